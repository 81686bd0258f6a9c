"""Copying pages and compacting sequences of the paged cache, every layer, against plain indexing in 64 bits.

Copies are bit-exact.  A turned key is computed in fp32 from two products (relative error below 2^-22 of the pair's
length) and rounded once: |error| <= u |k'| + 2^-21 |pair|, u = 2^-8 in bf16 and 2^-23 in fp32."""
import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu


def _pool(layers, pages, heads, ps, d, fp32, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.float32 if fp32 else torch.bfloat16
    k = torch.randn((layers, pages, heads, ps, d), device="cuda", generator=g).to(dt)
    v = torch.randn((layers, pages, heads, ps, d), device="cuda", generator=g).to(dt)
    return k, v, native.KvPool(k.data_ptr(), v.data_ptr(), layers, pages, heads, ps, d,
                               native.DTYPE_F32 if fp32 else native.DTYPE_BF16)


def _ints(*v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("layers,heads,ps,d,fp32,rows", [
    (3, 8, 64, 128, False, [37, 64, 0, 1]), (1, 1, 16, 64, False, [5, 16, 3, 2]), (2, 3, 256, 128, True, [255, 256, 9, 100]),
    (28, 2, 32, 64, True, [31, 32, 1, 17]), (2, 5, 64, 80, False, [13, 64, 2, 7]), (1, 2, 1, 16, False, [1, 0, 1, 1]),
])
def test_copies_the_asked_rows_and_nothing_else(layers, heads, ps, d, fp32, rows):
    import torch
    k, v, pool = _pool(layers, 9, heads, ps, d, fp32, 1)
    k[0, 2, 0, 0, :3] = torch.tensor([float("nan"), float("inf"), -0.0])
    src, dst = [2, 2, 5, 7], [0, 8, 1, 4]
    wk, wv = k.clone(), v.clone()
    for a, b, n in zip(src, dst, rows):
        wk[:, b, :, :n] = k[:, a, :, :n]
        wv[:, b, :, :n] = v[:, a, :, :n]
    s, t, r = _ints(*src), _ints(*dst), _ints(*rows)
    native.op_kv_copy_pages(pool, s.data_ptr(), t.data_ptr(), r.data_ptr(), 4)
    torch.cuda.synchronize()
    it = torch.int32 if fp32 else torch.int16
    assert torch.equal(k.view(it), wk.view(it)) and torch.equal(v.view(it), wv.view(it))


def test_copies_whole_pages_without_row_counts_and_skips_numbers_outside_the_pool():
    import torch
    k, v, pool = _pool(2, 6, 2, 16, 64, False, 2)
    wk, wv = k.clone(), v.clone()
    wk[:, 4] = k[:, 1]
    wv[:, 4] = v[:, 1]
    s, t = _ints(1, -1, 6, 3, 5), _ints(4, 0, 0, 6, 5)
    native.op_kv_copy_pages(pool, s.data_ptr(), t.data_ptr(), 0, 5)
    native.op_kv_copy_pages(pool, s.data_ptr(), t.data_ptr(), 0, 0)
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_copies_past_32_bit_offsets():
    """A pool of more than 2^32 bytes (and 2^31 elements) per tensor: the last page of the last layer."""
    import torch
    layers, pages, heads, ps, d = 5, 1700, 4, 256, 256
    k = torch.zeros((layers, pages, heads, ps, d), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    k[:, 0] = torch.arange(layers, device="cuda").view(-1, 1, 1, 1).to(torch.bfloat16) + 1
    v[:, pages - 1, :, 7] = 3
    pool = native.KvPool(k.data_ptr(), v.data_ptr(), layers, pages, heads, ps, d, native.DTYPE_BF16)
    s, t = _ints(0, pages - 1), _ints(pages - 2, 5)
    native.op_kv_copy_pages(pool, s.data_ptr(), t.data_ptr(), 0, 2)
    torch.cuda.synchronize()
    assert torch.equal(k[:, pages - 2], k[:, 0]) and float(k[layers - 1, pages - 2, 3, 255, 255]) == layers
    assert torch.equal(v[:, 5], v[:, pages - 1]) and float(v[layers - 1, 5].float().sum()) == 3 * heads * d


def _compact(fp32, layers, heads, ps, d, ctx, keeps, base, rope_len=400, turn=True, seed=3):
    import torch
    mp = max(-(-(c + 1) // ps) for c in ctx)
    B = len(ctx)
    k, v, pool = _pool(layers, 2 * B * mp + 1, heads, ps, d, fp32, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    order = torch.randperm(2 * B * mp + 1, device="cuda", generator=g).to(torch.int32)
    src, dst = order[: B * mp].view(B, mp).contiguous(), order[B * mp : 2 * B * mp].view(B, mp).contiguous()
    angle = torch.arange(rope_len, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
    rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    keep = _ints(*[p for x in keeps for p in x])
    start = _ints(*[sum(len(x) for x in keeps[:b]) for b in range(B + 1)])
    bs = _ints(*base) if base else None
    k0, v0 = k.clone(), v.clone()
    native.op_kv_compact(pool, src.data_ptr(), dst.data_ptr(), mp, keep.data_ptr(), start.data_ptr(), B,
                         sum(len(x) for x in keeps), rope=rope.data_ptr() if turn else 0, rope_len=rope_len,
                         dst_base=bs.data_ptr() if base else 0)
    torch.cuda.synchronize()
    wk, wv, tol = k0.double(), v0.double(), torch.zeros_like(k0, dtype=torch.float64)
    u = 2.0 ** -23 if fp32 else 2.0 ** -8
    for b in range(B):
        for i, p in enumerate(keeps[b]):
            t = i + (base[b] if base else 0)
            sp, dp = int(src[b, p // ps]), int(dst[b, t // ps])
            x = k0[:, sp, :, p % ps].double()
            wv[:, dp, :, t % ps] = v0[:, sp, :, p % ps].double()
            if turn and p != t:
                z = torch.complex(x[..., : d // 2], x[..., d // 2 :])
                y = z * torch.view_as_complex(rope.double())[p - t].conj()
                x = torch.cat([y.real, y.imag], -1)
                pair = torch.cat([z.abs(), z.abs()], -1)
                tol[:, dp, :, t % ps] = u * x.abs() + 2.0 ** -21 * pair
            wk[:, dp, :, t % ps] = x
    assert bool(((k.double() - wk).abs() <= tol).all())
    assert torch.equal(v.double(), wv)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("layers,heads,ps,d", [(2, 8, 64, 128), (3, 1, 16, 64), (1, 3, 256, 128), (2, 2, 32, 80)])
def test_compacts_ragged_sequences_and_turns_their_keys(fp32, layers, heads, ps, d):
    ctx = [150, 1, 77, 300]
    keeps = [[p for p in range(150) if not 20 <= p < 90],   # a gap in the middle
             [0],                                           # a single position, which stays
             [p for p in range(77) if p % 3 == 1],          # scattered
             []]                                            # nothing kept
    _compact(fp32, layers, heads, ps, d, ctx, keeps, None)


def test_compacts_behind_an_untouched_prefix():
    _compact(False, 2, 2, 16, 64, [100, 64], [list(range(40, 100)), list(range(50, 64))], [32, 48])


def test_copies_keys_as_they_are_without_a_table():
    _compact(False, 2, 2, 16, 64, [100], [list(range(7, 100, 2))], None, turn=False)


def test_compaction_skips_positions_without_a_page():
    import torch
    k, v, pool = _pool(1, 4, 1, 16, 64, False, 9)
    k0 = k.clone()
    src, dst = _ints(0, -1).view(1, 2), _ints(3, 9).view(1, 2)
    keep = _ints(3, 20, 31, 40, -2)  # no page, no page, beyond the table, before the first position
    start = _ints(0, 5)
    native.op_kv_compact(pool, src.data_ptr(), dst.data_ptr(), 2, keep.data_ptr(), start.data_ptr(), 1, 5)
    torch.cuda.synchronize()
    want = k0.clone()
    want[:, 3, :, 0] = k0[:, 0, :, 3]
    assert torch.equal(k, want)
