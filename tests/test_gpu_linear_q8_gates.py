"""SwiGLU products (qw_op_linear_q8) of gates far below zero, where e^-gate comes to the end of fp32.

gate = s w_scale x_scale is within 3 * 2^-24 of its value, relative; silu' there is about silu, so that up silu(gate) moves by
3 * 2^-24 |gate| of itself, and by 3 * 2^-24 for up.  The exponential of the gate: its argument (two roundings) brings 2^-23 |gate|, its
approximation 2^-22; sum, division and products 2^-21.  Together below (|gate| + 4) 2^-21 of the result, and 2^-8 of it in bf16.
Below gates of -92 silu(gate) is no normal number of fp32 (-91.7 gives 2^-126): there the result is anything from 0 to its value."""
import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu


# few tokens, a tile per pair, pairs that stay; a cut stride leaves the 16-byte stores
@pytest.mark.parametrize("t,n_out,gap", [(1, 512, 0), (40, 512, 0), (40, 512, 1), (300, 512, 0), (1500, 8192, 0), (1500, 8192, 1)])
@pytest.mark.parametrize("k", [16, 640])
def test_low_gates(t, n_out, gap, k):
    import torch
    g = torch.Generator(device="cuda").manual_seed(t)
    w = torch.zeros((n_out, k), dtype=torch.int8, device="cuda")
    x = torch.zeros((t, k), dtype=torch.int8, device="cuda")
    w[:, 3], x[:, 3] = 127, 127
    f = torch.arange(n_out, device="cuda")
    is_gate = f % 32 < 16
    # gates -84 .. -101, most of them where the exponential leaves fp32's normal numbers; ups that bring the products back
    values = torch.where(is_gate, -84 - 17 * torch.rand(n_out, device="cuda", generator=g).square(), 1e30 * (1 + torch.rand(n_out, device="cuda", generator=g)))
    values[:2] = torch.tensor([-87.5, -88.6], device="cuda")
    ws = values / 127 ** 2
    xs = torch.ones(t, device="cuda")
    out = torch.full((t, n_out // 2 + gap), 7.0, dtype=torch.bfloat16, device="cuda")
    native.LinearQ8(w.data_ptr(), ws.data_ptr(), n_out, k, epi=native.LINEAR_SWIGLU, out_dtype=native.DTYPE_BF16)(
        x.data_ptr(), xs.data_ptr(), t, out.data_ptr(), ld_out=n_out // 2 + gap)
    torch.cuda.synchronize()
    y = 127.0 ** 2 * ws.double()
    gate, up = y[is_gate], y[~is_gate]
    want = up * gate / (1 + torch.exp(-gate))
    bound = (gate.abs() + 4) * 2.0 ** -21 * want.abs()
    bound = torch.where(gate < -92, want.abs(), bound * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs())
    off = (out[:, : n_out // 2].double() - want).abs() - bound
    assert bool((off <= 0).all()), (off.max().item(), out[0, :2], want[:2])
    assert bool((out[:, : n_out // 2] <= 0).all())
    assert bool((out[:, n_out // 2 :] == 7).all())


@pytest.mark.parametrize("t,n_out", [(3, 64), (300, 512), (1500, 8192)])
def test_ends_of_the_gates(t, n_out):
    """Gates beyond every exponential, zero of either sign, and infinite ones."""
    import math
    import torch
    ends = [-1e4, -1e30, 0.0, -0.0, 90.0, 1e4, 1e30, math.inf, math.nan, -3e38, 3e38]
    w = torch.zeros((n_out, 16), dtype=torch.int8, device="cuda")
    x = torch.zeros((t, 16), dtype=torch.int8, device="cuda")
    w[:, 0] = x[:, 0] = 1
    f = torch.arange(n_out, device="cuda")
    gates = torch.tensor([ends[i % len(ends)] for i in range(n_out // 2)], device="cuda")
    ws = torch.full((n_out,), 0.75, device="cuda")
    ws[f % 32 < 16] = gates
    xs = torch.ones(t, device="cuda")
    out = torch.empty((t, n_out // 2), dtype=torch.bfloat16, device="cuda")
    native.LinearQ8(w.data_ptr(), ws.data_ptr(), n_out, 16, epi=native.LINEAR_SWIGLU, out_dtype=native.DTYPE_BF16)(
        x.data_ptr(), xs.data_ptr(), t, out.data_ptr())
    torch.cuda.synchronize()
    want = (0.75 * torch.where(gates < -200, 0.0, gates.double() / (1 + torch.exp(-gates.double())))).expand(t, -1)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    ok = torch.isfinite(want)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * 1.001 * want.abs())[ok].all())
    assert torch.equal(out[~ok & ~torch.isnan(want)].double(), want[~ok & ~torch.isnan(want)])


@pytest.mark.parametrize("t,n_out", [(3, 64), (300, 512), (1500, 8192)])
def test_small_gates(t, n_out):
    """Gates down to the smallest normal number: silu is half of them.  The gate is rounded at 2^-142 (2^-16 of the smallest one), the
    rest as above."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n_out)
    w = torch.zeros((n_out, 16), dtype=torch.int8, device="cuda")
    x = torch.zeros((t, 16), dtype=torch.int8, device="cuda")
    w[:, 0] = x[:, 0] = 1
    is_gate = torch.arange(n_out, device="cuda") % 32 < 16
    power = torch.randint(-126, -20, (n_out,), device="cuda", generator=g)
    gates = torch.ldexp(1 + torch.rand(n_out, device="cuda", generator=g), power) * (1 - 2 * (power % 2))
    ws = torch.where(is_gate, gates, 1e30 * (1 + torch.rand(n_out, device="cuda", generator=g)))
    xs = torch.ones(t, device="cuda")
    out = torch.empty((t, n_out // 2), dtype=torch.bfloat16, device="cuda")
    native.LinearQ8(w.data_ptr(), ws.data_ptr(), n_out, 16, epi=native.LINEAR_SWIGLU, out_dtype=native.DTYPE_BF16)(
        x.data_ptr(), xs.data_ptr(), t, out.data_ptr())
    torch.cuda.synchronize()
    gate, up = ws.double()[is_gate], ws.double()[~is_gate]
    want = up * gate / (1 + torch.exp(-gate))
    bound = 4 * 2.0 ** -21 * want.abs() + up.abs() * 2.0 ** -142
    bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    off = (out.double() - want).abs() - bound
    assert bool((off <= 0).all()), off.max().item()
