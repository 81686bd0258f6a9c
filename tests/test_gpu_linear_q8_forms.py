"""Every form that a product of codes (qw_op_linear_q8) can take, under every epilogue: a shape for each way of cutting the work
(tests/test_linear_q8_plan.py checks that these shapes reach them all).

STORE and RESID are compared for equality: the sum is a whole number, and its rounding to fp32, its products with the two scales,
the bias or residual and the rounding to bf16 are each the one of real arithmetic.  SWIGLU within the bound of
test_gpu_linear_q8.py, without an absolute term."""
import pytest

from common_b200 import native
from tests.test_gpu_linear_q8 import RESID, STORE, SWIGLU, Case

pytestmark = pytest.mark.gpu

# (tokens, features, codes): small and ragged ones, one to a form; then ordinary ones
SHAPES = [(2, 64, 20), (2, 8480, 1797), (2, 4768, 1549), (2, 64, 1537), (2, 64, 2049), (2, 64, 3841), (129, 64, 20),
          (17, 9056, 2307), (17, 4800, 2055), (129, 64, 1295), (130, 64, 2050), (129, 64, 3865), (257, 64, 20),
          (33, 6368, 2576), (259, 800, 1666), (257, 64, 1673), (257, 64, 2070), (260, 64, 3842), (513, 64, 20),
          (517, 1056, 2615), (897, 288, 2065), (514, 64, 1800), (4635, 800, 21), (1026, 64, 20), (2822, 288, 2597),
          (3882, 64, 2062), (1030, 64, 1795),
          (64, 6144, 4096), (64, 4096, 12288), (128, 4096, 12288), (256, 4096, 12288), (384, 4096, 12288), (512, 4096, 12288),
          (40, 1024, 8192), (1024, 6144, 4096)]


def expected(c):
    """What STORE and RESID write, rounding by rounding."""
    import torch
    s = c.x[:, : c.k].double() @ c.w[:, : c.k].double().T  # whole numbers below 2^53
    y = s.float() * c.ws * c.xs[:, None]
    if c.resid is not None:
        y = c.resid[:, : c.cols] + y
    elif c.bias is not None:
        y = y + c.bias
    return y.to(torch.bfloat16) if c.bf16 else y


def check(c):
    import torch
    torch.cuda.synchronize()
    assert c.err.item() == 0
    assert torch.equal(c.out[: c.t, : c.cols], expected(c))
    assert bool((c.out[c.t] == 7).all()) and bool((c.out[:, c.cols :] == 7).all())


@pytest.mark.parametrize("t,n_out,k", SHAPES)
@pytest.mark.parametrize("gap", [0, 3])
def test_store(t, n_out, k, gap):
    for bf16 in (False, True):
        for bias in (False, True):
            c = Case(t, n_out, k, bf16=bf16, bias=bias, seed=t + k, gap=gap, pad=gap * 16, lowest=-128)
            c.run()
            check(c)


@pytest.mark.parametrize("t,n_out,k", SHAPES)
@pytest.mark.parametrize("gap", [0, 3])
def test_resid(t, n_out, k, gap):
    import torch
    c = Case(t, n_out, k, epi=RESID, seed=t + k + 1, gap=gap)
    c.run()
    check(c)
    want, around = expected(c), c.resid[:, n_out:].clone()
    c.run(out=c.resid)
    torch.cuda.synchronize()
    assert torch.equal(c.resid[:, :n_out], want) and torch.equal(c.resid[:, n_out:], around)


@pytest.mark.parametrize("t,n_out,k", SHAPES)
@pytest.mark.parametrize("gap", [0, 3])
def test_swiglu(t, n_out, k, gap):
    import torch
    c = Case(t, n_out, k, epi=SWIGLU, bf16=True, seed=t + k + 2, gap=gap)
    c.run()
    c.check()
    y = (c.x[:, :k].double() @ c.w[:, :k].double().T) * c.ws.double() * c.xs.double()[:, None]
    gate, up = (part.reshape(t, -1) for part in y.view(t, -1, 2, 16).unbind(2))
    want = up * gate / (1 + torch.exp(-gate))
    e = 2.0 ** -22
    bound = e * want.abs() + 1.1 * e * (up * gate).abs() + (gate.abs() + 8) * e * want.abs()
    off = (c.out[:t, : c.cols].double() - want).abs() - bound * (1 + 2.0 ** -8) - 2.0 ** -8 * want.abs()
    assert bool((off <= 0).all()), off.max().item()


@pytest.mark.parametrize("t,n_out,k", SHAPES)
def test_marked_rows_of_codes(t, n_out, k):
    """A token whose scale is NaN gives NaN, and no other token does; one whose scale is zero gives its residual."""
    import torch
    c = Case(t, n_out, k, epi=RESID, seed=t, gap=4)
    c.xs[t - 1], c.xs[t // 2 - 1] = float("nan"), 0.0
    c.run()
    torch.cuda.synchronize()
    assert bool(torch.isnan(c.out[t - 1, :n_out]).all()) and torch.equal(c.out[t // 2 - 1, :n_out], c.resid[t // 2 - 1, :n_out])
    assert torch.equal(c.out[: t - 1, :n_out], expected(c)[: t - 1])


@pytest.mark.parametrize("t,n_out,k", [(40, 512, 700), (64, 4096, 12288), (300, 1056, 2615), (1500, 4096, 256)])
@pytest.mark.parametrize("out_off,resid_off", [(1, 0), (0, 1), (1, 1)])
def test_results_and_residuals_off_16_bytes(t, n_out, k, out_off, resid_off):
    """Pointers that lie on their elements only, in rows whose strides are whole pieces."""
    import torch
    c = Case(t, n_out, k, epi=RESID, seed=t, gap=4)
    whole = torch.full((t + 1, n_out + 4), 7.0, device="cuda")
    c.out, c.resid = whole[:, out_off:], c.resid[:, resid_off:]
    c.run()
    check(c)
    assert bool((whole[:, :out_off] == 7).all())
    for bf16 in (False, True):
        c = Case(t, n_out, k, bf16=bf16, bias=True, seed=t, gap=8)
        whole = torch.full((t + 1, n_out + 8), 7.0, dtype=c.out.dtype, device="cuda")
        c.out = whole[:, out_off:]
        c.run()
        check(c)
        assert bool((whole[:, :out_off] == 7).all())
