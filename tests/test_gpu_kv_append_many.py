"""The append (qw_op_kv_append) of more than 1024 rows, which a CTA takes four at a time: what test_gpu_kv_append.py asks of fewer,
with its definition and tolerances."""
import math

import pytest

from common_b200 import native
from tests.test_gpu_kv_append import GEOMETRIES, HEAD, NONE, VECTOR, Case

pytestmark = pytest.mark.gpu

# sequences that begin and end inside a group of four rows: chunks, single tokens, none; 1029 rows in all
NEW = [411, 1, 0, 350, 1, 1, 2, 3, 200, 60]
KV = [411, 300, 77, 400, 1, 700, 2, 90, 333, 61]


def lengths(rows):
    """NEW with a last chunk that makes it `rows` rows."""
    return NEW + [rows - sum(NEW)], KV + [rows - sum(NEW) + 13]


@pytest.mark.parametrize("mode", [NONE, VECTOR, HEAD])
@pytest.mark.parametrize("heads,kv_heads,d", GEOMETRIES)
def test_geometries(heads, kv_heads, d, mode):
    c = Case(NEW, KV, heads, kv_heads, d, 16, mode, seed=heads + d)
    c.run()
    c.check()


@pytest.mark.parametrize("in_kind,kind", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("mode", [NONE, HEAD])
def test_types_and_strides(in_kind, kind, fused, rope, mode):
    for heads, kv_heads, d in ((16, 4, 64), (14, 2, 64), (28, 4, 128)):
        c = Case(NEW, KV, heads, kv_heads, d, 32, mode, in_kind, kind, fused, rope, seed=3, slots=fused)
        c.run()
        c.check()


@pytest.mark.parametrize("rows", [1030, 1031, 1032, 1033, 2050, 4099])
@pytest.mark.parametrize("spare", [0, 1, 2, 3])
def test_row_counts(rows, spare):
    """Buffers and sequences that end one to four rows into a group."""
    new, kv = lengths(rows)
    c = Case(new, kv, 14, 2, 64, 16, HEAD, "bf16", seed=rows, spare=spare)
    c.run()
    c.check()


@pytest.mark.parametrize("page", [1, 2, 16, 64, 256])
@pytest.mark.parametrize("mode", [NONE, HEAD])
def test_pages_and_lengths(page, mode):
    """Chunks that end inside pages, single tokens, sequences without rows, unused places, rows before position 0."""
    new = [1, 0, 130, 1, 517, 1, 64, 300, 1, 2, 90]
    kv = [1, 40, 130, 0, 600, 257, 64, 200, -5, 1, 90]
    c = Case(new, kv, 16, 8, 128, page, mode, seed=page)
    c.run()
    c.check()


@pytest.mark.parametrize("heads,kv_heads,d", [(32, 8, 128), (14, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("mode", [NONE, HEAD])
def test_single_tokens_of_the_largest_batch(heads, kv_heads, d, mode):
    B = 1024
    c = Case([1] * B, [(37 * b) % 90 for b in range(B)], heads, kv_heads, d, 16, mode, seed=B, spare=6)
    c.run()
    c.check()


def test_positions_beyond_the_table_of_angles_and_without_pages():
    c = Case([630, 440], [700, 450], 4, 2, 64, 16, HEAD, seed=1, rope_len=580)
    c.table[2, 9] = -1       # sequence 0 stands in row 2: positions 144..159 have no page
    c.table[1, 1] = 1 << 20  # sequence 1: positions 16..31 name a page that is none
    c.run()
    c.check()


def test_lengths_beyond_the_slot_are_limited():
    c = Case([1040], [1056], 4, 2, 64, 16, HEAD, seed=1, rope_len=1200)
    c.table[1, 66] = int(next(i for i in range(c.num_pages) if i not in c.table[1].tolist()))
    c.kv = [c.max_pages * c.page + 1000]
    c.kv_len.fill_(c.kv[0])
    c.run()
    c.check()


def test_wild_row_starts_stay_inside():
    """Row starts that do not ascend or pass the buffers: nothing is written outside rows, pages and slots."""
    import torch
    c = Case([400, 400, 400], [408, 408, 408], 4, 2, 64, 16, HEAD, seed=2)
    used = torch.zeros(c.num_pages, dtype=torch.bool, device="cuda")
    used[c.table[c.table >= 0].long()] = True
    for wild in ([500, 200, 900, 300], [-7, 400, 4000, 1 << 30], [0, 0, 0, 0], [-(1 << 31), (1 << 31) - 1, -1, 500]):
        c.row_start.copy_(torch.tensor(wild, dtype=torch.int32))
        c.run()
        torch.cuda.synchronize()
    assert torch.equal(c.qo[:, c.H * c.d :], c.before[2][:, c.H * c.d :])
    assert torch.equal(c.kc[~used], c.before[0][~used]) and torch.equal(c.vc[~used], c.before[1][~used])


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 4, 64), (14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("mode", [NONE, VECTOR, HEAD])
def test_queries_in_place(heads, kv_heads, d, kind, mode):
    import torch
    a = Case(NEW, KV, heads, kv_heads, d, 32, mode, kind, kind, seed=3, spare=0)
    b = Case(NEW, KV, heads, kv_heads, d, 32, mode, kind, kind, seed=3, spare=0)
    a.run()
    b.run(q_out=b.q)
    torch.cuda.synchronize()
    assert torch.equal(a.qo[:, : heads * d], b.q) and torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    a.check()


@pytest.mark.parametrize("mode", [NONE, HEAD])
def test_no_queries_wanted(mode):
    import torch
    c, d = (Case(NEW, KV, 14, 2, 64, 32, mode, seed=3) for _ in range(2))
    c.run(q_out=False)
    d.run()
    torch.cuda.synchronize()
    assert torch.equal(c.kc, d.kc) and torch.equal(c.vc, d.vc) and torch.equal(c.qo, c.before[2])
    d.check()


@pytest.mark.parametrize("mode", [NONE, HEAD])
def test_nan_rows_stay_by_themselves(mode):
    import torch
    c, d = (Case(NEW, KV, 14, 2, 64, 16, mode, seed=4) for _ in range(2))
    bad = [1, 410, 411, 1000]  # inside a chunk, its last, a single token, the last chunk
    c.q[bad], c.k[bad] = math.nan, math.inf
    c.run()
    d.run()
    torch.cuda.synchronize()
    keep = [r for r in range(c.rows) if r not in bad]
    assert torch.equal(c.qo[keep], d.qo[keep]) and bool(torch.isnan(c.qo[bad, : 14 * 64]).all())
    same = torch.isfinite(c.kc)
    # an infinite key is NaN behind a norm or a rotation with a sine of either sign, infinite at the least
    assert int((~same).sum()) == len(bad) * 2 * 64 and torch.equal(c.kc[same], d.kc[same]) and torch.equal(c.vc, d.vc)


def test_rows_agree_with_fewer():
    """Rows by fours have the bits of rows by one: the same sequences in calls of less than 1024 rows."""
    import torch
    a = Case(NEW, KV, 28, 4, 128, 16, HEAD, "bf16", seed=7, spare=0)
    b = Case(NEW, KV, 28, 4, 128, 16, HEAD, "bf16", seed=7, spare=0)
    a.run()
    for s in range(len(NEW)):
        r0, n = sum(NEW[:s]), NEW[s]
        if n == 0:
            continue
        start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        b.append(b.q[r0].data_ptr(), b.k[r0].data_ptr(), b.v[r0].data_ptr(), b.qo[r0].data_ptr(), b.kc.data_ptr(), b.vc.data_ptr(),
                 b.table.data_ptr(), start.data_ptr(), b.kv_len[s:].data_ptr(), 1, n, slots=b.slots[s:].data_ptr(),
                 ld_q=b.q.stride(0), ld_k=b.k.stride(0), ld_v=b.v.stride(0), ld_q_out=b.qo.stride(0))
        torch.cuda.synchronize()
    assert torch.equal(a.qo, b.qo) and torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
