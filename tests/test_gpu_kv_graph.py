"""Page copies and compaction on a stream of their own and in a captured graph that follows new lists, against plain
indexing, bit for bit (copies, and keys that move without a table)."""
import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu


def _pool(layers, pages, heads, ps, d, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn((layers, pages, heads, ps, d), device="cuda", generator=g).to(torch.bfloat16)
    v = torch.randn((layers, pages, heads, ps, d), device="cuda", generator=g).to(torch.bfloat16)
    return k, v, native.KvPool(k.data_ptr(), v.data_ptr(), layers, pages, heads, ps, d, native.DTYPE_BF16)


def _ints(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _behind_work(call, set_lists, first, second, check):
    """`call(stream)` behind work on a stream of its own that brings its lists, then captured and replayed on others."""
    import torch
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        x = torch.randn((4096, 4096), device="cuda")
        for _ in range(10):
            x = x @ x * 1e-2
        set_lists(first)
        call(st.cuda_stream)
    st.synchronize()
    check(first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        call(torch.cuda.current_stream().cuda_stream)
    for lists in (second, first):
        set_lists(lists)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(lists)


def test_copies_follow_their_lists():
    import torch
    k, v, pool = _pool(3, 12, 2, 16, 64, 61)
    state = [k.clone(), v.clone()]
    src, dst, rows = _ints([0] * 3), _ints([0] * 3), _ints([0] * 3)

    def set_lists(x):
        for t, y in zip((src, dst, rows), x):
            t.copy_(_ints(y))

    def check(x):
        for w, t in zip(state, (k, v)):
            for a, b, n in zip(*x):
                w[:, b, :, :n] = w[:, a, :, :n]
            assert torch.equal(w, t)

    _behind_work(lambda st: native.op_kv_copy_pages(pool, src.data_ptr(), dst.data_ptr(), rows.data_ptr(), 3, st), set_lists,
                 ([0, 0, 5], [1, 2, 3], [16, 7, 1]), ([1, 6, 6], [4, 7, 8], [9, 16, 0]), check)


@pytest.mark.parametrize("d", [64, 128, 80])
def test_compaction_follows_its_lists(d):
    import torch
    k, v, pool = _pool(2, 16, 3, 16, d, 62)
    state = [k.clone(), v.clone()]
    tables = _ints([[0, 1, 2, 3], [4, 5, 6, 7]]), _ints([[8, 9, 10, 11], [12, 13, 14, 15]])
    keep, start, base = _ints([0] * 40), _ints([0] * 3), _ints([0, 0])

    def set_lists(x):
        keep.copy_(_ints(x[0] + x[1] + [0] * (40 - len(x[0]) - len(x[1]))))
        start.copy_(_ints([0, len(x[0]), len(x[0]) + len(x[1])]))
        base.copy_(_ints(x[2]))

    def check(x):
        for w, t in zip(state, (k, v)):
            for b in range(2):
                for i, p in enumerate(x[b]):
                    to = x[2][b] + i
                    w[:, tables[1][b, to // 16], :, to % 16] = w[:, tables[0][b, p // 16], :, p % 16]
            assert torch.equal(w, t)

    # rows is the most that the lists hold: what start does not name is left alone
    _behind_work(lambda st: native.op_kv_compact(pool, tables[0].data_ptr(), tables[1].data_ptr(), 4, keep.data_ptr(),
                                                 start.data_ptr(), 2, 40, dst_base=base.data_ptr(), stream=st), set_lists,
                 (list(range(3, 60, 3)), [1, 2, 50], [0, 16]), ([9], list(range(20, 55)), [5, 0]), check)
