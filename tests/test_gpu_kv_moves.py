"""Compaction of positions that move up, far, or not at all.  A turned key is computed in fp32 from two products (relative
error below 2^-22 of the pair's length) and rounded once: |error| <= u |k'| + 2^-21 |pair|, u = 2^-8 in bf16 and 2^-23 in
fp32; the table's entries are themselves rounded to fp32, which the reference takes as they are."""
import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu


def _check(fp32, heads, ps, d, keeps, base, rope_len, layers=2, seed=5):
    """Compacts sequences of 20 pages each; a row that moves by rope_len or more has to be left out."""
    import torch
    dt = torch.float32 if fp32 else torch.bfloat16
    B, mp = len(keeps), 20
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = 2 * B * mp
    k = torch.randn((layers, pages, heads, ps, d), device="cuda", generator=g).to(dt)
    v = torch.randn((layers, pages, heads, ps, d), device="cuda", generator=g).to(dt)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    src, dst = order[: B * mp].view(B, mp).contiguous(), order[B * mp :].view(B, mp).contiguous()
    angle = torch.arange(rope_len, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
    rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    keep, bs = ints([p for x in keeps for p in x]), ints(base)
    start = ints([sum(len(x) for x in keeps[:b]) for b in range(B + 1)])
    pool = native.KvPool(k.data_ptr(), v.data_ptr(), layers, pages, heads, ps, d,
                         native.DTYPE_F32 if fp32 else native.DTYPE_BF16)
    wk, wv, tol = k.double(), v.double(), torch.zeros_like(k, dtype=torch.float64)
    u = 2.0 ** -23 if fp32 else 2.0 ** -8
    for b in range(B):
        for i, p in enumerate(keeps[b]):
            t = base[b] + i
            if abs(p - t) >= rope_len:
                continue
            sp, dp = int(src[b, p // ps]), int(dst[b, t // ps])
            x = k[:, sp, :, p % ps].double()
            z = torch.complex(x[..., : d // 2], x[..., d // 2 :])
            a = torch.view_as_complex(rope.double())[abs(p - t)]
            y = z * (a.conj() if p > t else a)
            wk[:, dp, :, t % ps] = torch.cat([y.real, y.imag], -1)
            wv[:, dp, :, t % ps] = v[:, sp, :, p % ps].double()
            if p != t:
                tol[:, dp, :, t % ps] = u * wk[:, dp, :, t % ps].abs() + 2.0 ** -21 * torch.cat([z.abs(), z.abs()], -1)
    native.op_kv_compact(pool, src.data_ptr(), dst.data_ptr(), mp, keep.data_ptr(), start.data_ptr(), B,
                         int(keep.numel()), rope=rope.data_ptr(), rope_len=rope_len, dst_base=bs.data_ptr())
    torch.cuda.synchronize()
    assert bool(((k.double() - wk).abs() <= tol).all())
    assert torch.equal(v.double(), wv)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("heads,ps,d", [(8, 64, 128), (3, 16, 64), (2, 32, 80)])
def test_keys_that_move_up_turn_forward(fp32, heads, ps, d):
    """Kept positions appended behind a longer base, and a sequence whose rows move up, not at all and down."""
    n = 20 * ps
    _check(fp32, heads, ps, d, [list(range(0, 100)), [5, 6, 7, 20, 23, 24, 200], [3]], [n - 110, 18, 3], n)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("heads,ps,d", [(8, 64, 128), (3, 16, 64), (2, 32, 80)])
def test_rows_that_move_beyond_the_table_are_left_out(fp32, heads, ps, d):
    _check(fp32, heads, ps, d, [[0, 1, 40, 41, 42, 43, 99], list(range(50, 60))], [0, 10], 40)
    _check(fp32, heads, ps, d, [[0, 1, 2], [100]], [40, 99], 1)
    _check(fp32, heads, ps, d, [[0, 1, 2], [39]], [40, 0], 40)
