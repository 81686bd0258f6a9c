"""What malformed lengths and page numbers may do to qw_op_chunk_attn: they are clamped to the call's rows, the slot's
positions and the pool's pages, nothing outside the call's rows is written, and the rest of the batch comes out right.
References and tolerances are those of test_gpu_chunk_attn.py."""
import pytest

from tests.test_gpu_chunk_attn import Case

pytestmark = pytest.mark.gpu

GUARD = 128  # rows before and after the results


def _guarded(c):
    """Puts c's results between guard rows; returns the buffers that hold both."""
    import torch
    H, d = c.H, c.d
    out = torch.full((c.rows + 2 * GUARD, H * d), -7.0, device="cuda", dtype=c.dt)
    lse = torch.full((c.rows + 2 * GUARD, H), -7.0, device="cuda")
    c.obuf, c.lse = out[GUARD : GUARD + c.rows], lse[GUARD : GUARD + c.rows]
    return out, lse


def _check(c, bufs):
    import torch
    c.check()
    for b in bufs:
        assert bool((b[:GUARD] == -7.0).all()) and bool((b[GUARD + c.rows :] == -7.0).all())
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new,lengths", [
    ([3, 37, 20], [-5, 3, 40, 1000]),                  # fp32: tiles of rows
    ([3, 37, 20], [-2 ** 31, 3, 40, 2 ** 31 - 1]),
    ([1, 1, 1], [-1, 1, 2, 99]),                       # fp32: single rows
])
def test_row_starts_outside_the_rows_are_clamped(dtype, new, lengths):
    import torch
    c = Case(new, [90, 400, 33], 16, 8, 128, 64, dtype=dtype, seed=31)
    bufs = _guarded(c)
    c.row_start = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    c.run()
    _check(c, bufs)


def _reference(c, kv):
    """(out, A, lse) in 64 bits with the lengths `kv` (within the table), where a page that is none reads as zeros."""
    import torch
    G, d, r = c.H // c.Hkv, c.d, 0
    out = torch.zeros((c.rows, c.H, d), dtype=torch.float64, device="cuda")
    A, lse = torch.zeros_like(out), torch.zeros((c.rows, c.H), dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(c.new, kv)):
        p = torch.arange(m, device="cuda")
        pg = c.table[len(c.new) - b].long()[p // c.page]
        there = ((pg >= 0) & (pg < c.num_pages))[:, None, None]
        pg = torch.where(there[:, 0, 0], pg, 0)
        k = torch.where(there, c.k[pg, :, p % c.page].double(), 0.0)
        v = torch.where(there, c.v[pg, :, p % c.page].double(), 0.0)
        q = c.q[r : r + n].double().view(n, c.Hkv, G, d)
        x = torch.einsum("nhgd,lhd->hgnl", q, k) / d ** 0.5
        x = x.masked_fill(p[None] > torch.arange(m - n, m, device="cuda")[:, None], -float("inf"))
        w = torch.softmax(x, -1)
        out[r : r + n] = torch.einsum("hgnl,lhd->nhgd", w, v).reshape(n, c.H, d)
        A[r : r + n] = torch.einsum("hgnl,lhd->nhgd", w, v.abs()).reshape(n, c.H, d)
        lse[r : r + n] = torch.logsumexp(x, -1).permute(2, 0, 1).reshape(n, c.H)
        r += n
    return out, A, lse


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new,kv", [([3, 2, 7], [100, 60, 500]), ([1, 1, 1], [100, 60, 500]), ([40, 90, 1], [100, 130, 9000])])
def test_lengths_beyond_the_table_are_clamped_and_pages_that_are_none_read_as_zeros(dtype, new, kv):
    """Sequence 0 is said to be longer than its slot, sequence 1's first page and sequence 2's second one have numbers outside
    the pool; the third is itself in order beyond that."""
    import torch
    c = Case(new, kv, 16, 8, 128, 64, dtype=dtype, seed=10)
    g = torch.Generator(device="cuda").manual_seed(32)
    c.k = torch.randn(c.k.shape, device="cuda", generator=g).to(c.dt)  # all of the pool: the clamped length reaches further
    c.v = torch.randn(c.v.shape, device="cuda", generator=g).to(c.dt)
    c.kv_len[0] = 1 << 30
    c.table[2, 0] = 1 << 30
    c.table[1, 1] = -(1 << 31)
    bufs = _guarded(c)
    c.run()
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0
    out, A, lse = _reference(c, [c.max_pages * 64] + kv[1:])
    got = c.obuf.view(c.rows, c.H, c.d).double()
    tol = 2.0 ** -8 * (A + out.abs()) + 2.0 ** -12 * A if dtype == "bf16" else 2e-5 * A
    assert bool(((got - out).abs() <= tol).all())
    assert (c.lse.double() - lse).abs().max().item() < (1e-4 if dtype == "bf16" else 2e-5)
    for b in bufs:
        assert bool((b[:GUARD] == -7.0).all()) and bool((b[GUARD + c.rows :] == -7.0).all())


def test_more_rows_that_see_nothing_than_32_bits_count_vectors_of():
    """2^21 rows of 64 heads of 128 are 2^31 vectors of 16 bytes (34 GB): a sequence with nothing cached."""
    import torch
    from common_b200 import native
    rows, H, d = 2 ** 21 + 1000, 64, 128
    out = torch.full((rows, H * d), -7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((rows, H), -7.0, device="cuda")
    cache = torch.zeros((1, 8, 64, d), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    start = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    kv_len = torch.zeros(1, dtype=torch.int32, device="cuda")
    n = native.chunk_attn_workspace(H, 8, d)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    attn = native.ChunkAttention(H, 8, d, 64, 1, 1, ws.data_ptr(), n)
    attn(out.data_ptr(), cache.data_ptr(), cache.data_ptr(), table.data_ptr(), start.data_ptr(), kv_len.data_ptr(), 1, rows,
         out.data_ptr(), lse=lse.data_ptr())
    torch.cuda.synchronize()
    for part in out.split(2 ** 18):
        assert not bool(part.any())
    assert bool((lse == -float("inf")).all())


def test_overlapping_sequences_of_more_work_than_32_bits_number_do_nothing():
    """512 sequences that all name the same 2^20 rows over 2^22 positions: 2^40 units of work; some are empty."""
    import torch
    from common_b200 import native
    rows, H, d, B = 2 ** 20, 8, 64, 1024
    out = torch.full((rows, H * d), -7.0, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros((1, H, 256, d), dtype=torch.bfloat16, device="cuda")
    table = torch.full((B, 2 ** 14), -1, dtype=torch.int32, device="cuda")
    start = torch.tensor([0, rows] * (B // 2) + [0], dtype=torch.int32, device="cuda")
    kv_len = torch.full((B,), 2 ** 22, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    n = native.chunk_attn_workspace(H, H, d)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    attn = native.ChunkAttention(H, H, d, 256, 1, 2 ** 14, ws.data_ptr(), n)

    def call(batch, rows):
        attn(out.data_ptr(), cache.data_ptr(), cache.data_ptr(), table.data_ptr(), start.data_ptr(), kv_len.data_ptr(), batch,
             rows, out.data_ptr(), err=err.data_ptr())
        torch.cuda.synchronize()

    call(B, rows)
    assert int(err.item()) != 0 and bool((out == -7.0).all())
    err.zero_()
    start[: 2] = torch.tensor([0, 1], dtype=torch.int32)
    call(1, 1)                                # the workspace is as it was: one row over pages that are not there
    assert int(err.item()) == 0 and not bool(out[0].any()) and bool((out[1:] == -7.0).all())
