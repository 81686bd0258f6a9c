"""Attention of ragged chunks over the paged cache (qw_op_chunk_attn) against the definition in 64 bits: lengths from
none and one to long ones, every group size, page sizes below, at and above a key block, windows, rows that see
nothing, and non-finite values wherever no row of the sequence looks.

Tolerances, per element, with A = sum_j p_j |v_j| / sum_j p_j (the value sum without cancellation).  bf16: the
probabilities and the result are each rounded once to 8 significant bits, so |error| <= 2^-8 (A + |out|); exponentials
and fp32 sums add at most 2^-12 A.  fp32: 2^-24 sqrt(128) of a score sum of |q||k| scale <~ 10 moves each score by
<~ 7e-6, a probability by as much relative to itself: 2e-5 A.  lse: the same score error plus that of the exponentials:
1e-4 in bf16 and 2e-5 in fp32, absolute."""
import math

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


class Case:
    """A cache in which pages lie in random order and everything unwritten is NaN, and a batch of rows over it."""

    def __init__(self, new, kv, heads, kv_heads, d, page, window=0, dtype="bf16", seed=0, fused=0, gap=0, spread=1.0):
        torch = _torch()
        self.new, self.kv, self.H, self.Hkv, self.d, self.page, self.window = new, kv, heads, kv_heads, d, page, window
        self.dt = torch.bfloat16 if dtype == "bf16" else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [max(0, -(-k // page)) for k in kv]
        self.num_pages, self.max_pages = sum(need) + 3, max(need + [1]) + 1
        order = torch.randperm(self.num_pages, device="cuda", generator=g).to(torch.int32)
        B = len(new)
        # slots in reverse order, one table row of nobody in between
        self.slots = torch.arange(B, 0, -1, dtype=torch.int32, device="cuda")
        self.table = torch.full((B + 1, self.max_pages), -1, dtype=torch.int32, device="cuda")
        shape = (self.num_pages, kv_heads, page, d)
        self.k = torch.full(shape, float("nan"), device="cuda", dtype=self.dt)
        self.v = torch.full(shape, float("inf"), device="cuda", dtype=self.dt)
        at = 0
        for b in range(B):
            s = B - b
            self.table[s, : need[b]] = order[at : at + need[b]]
            at += need[b]
            lo = max(0, kv[b] - new[b] - window + 1) if window else 0
            if kv[b] > lo:
                p = torch.arange(lo, kv[b], device="cuda")
                pg = self.table[s].long()[p // page]
                n = kv[b] - lo
                self.k[pg, :, p % page] = torch.randn((n, kv_heads, d), device="cuda", generator=g).mul_(spread).to(self.dt)
                self.v[pg, :, p % page] = torch.randn((n, kv_heads, d), device="cuda", generator=g).to(self.dt)
            self.table[s, : lo // page] = -1
        self.rows = sum(new)
        wide = heads * d + fused
        self.qbuf = torch.randn((max(self.rows, 1), wide), device="cuda", generator=g).to(self.dt)
        self.q = self.qbuf[: self.rows, : heads * d].view(self.rows, heads, d)
        self.obuf = torch.full((max(self.rows, 1), heads * d + gap), -7.0, device="cuda", dtype=self.dt)
        self.lse = torch.full((max(self.rows, 1), heads), -7.0, device="cuda")
        self.row_start = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        n = native.chunk_attn_workspace(heads, kv_heads, d)
        self.ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
        self.attn = native.ChunkAttention(heads, kv_heads, d, page, self.num_pages, self.max_pages, self.ws.data_ptr(),
                                          n, window=window,
                                          dtype=native.DTYPE_BF16 if dtype == "bf16" else native.DTYPE_F32)

    def run(self, stream=0, lse=True):
        self.attn(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(),
                  self.row_start.data_ptr(), self.kv_len.data_ptr(), len(self.new), self.rows, self.obuf.data_ptr(),
                  lse=self.lse.data_ptr() if lse else 0, slots=self.slots.data_ptr(), ld_q=self.qbuf.stride(0),
                  ld_out=self.obuf.stride(0), err=self.err.data_ptr(), stream=stream)

    def reference(self):
        """(out, A, lse) in 64 bits."""
        torch = _torch()
        G, d = self.H // self.Hkv, self.d
        out = torch.zeros((self.rows, self.H, d), dtype=torch.float64, device="cuda")
        A = torch.zeros_like(out)
        lse = torch.full((self.rows, self.H), -math.inf, dtype=torch.float64, device="cuda")
        r = 0
        for b, (n, kv) in enumerate(zip(self.new, self.kv)):
            lo = max(0, kv - n - self.window + 1) if self.window else 0
            skip = max(0, n - kv)
            if kv > lo and n > skip:
                p = torch.arange(lo, kv, device="cuda")
                pg = self.table[len(self.new) - b].long()[p // self.page]
                k, v = self.k[pg, :, p % self.page].double(), self.v[pg, :, p % self.page].double()  # (L, Hkv, d)
                q = self.q[r + skip : r + n].double().view(n - skip, self.Hkv, G, d)
                x = torch.einsum("nhgd,lhd->hgnl", q, k) / math.sqrt(d)
                pos = torch.arange(kv - n + skip, kv, device="cuda")[:, None]
                hide = p[None] > pos
                if self.window:
                    hide |= p[None] <= pos - self.window
                x = x.masked_fill(hide, -math.inf)
                w = torch.softmax(x, -1)
                lse[r + skip : r + n] = torch.logsumexp(x, -1).permute(2, 0, 1).reshape(n - skip, self.H)
                out[r + skip : r + n] = torch.einsum("hgnl,lhd->nhgd", w, v).reshape(n - skip, self.H, d)
                A[r + skip : r + n] = torch.einsum("hgnl,lhd->nhgd", w, v.abs()).reshape(n - skip, self.H, d)
            r += n
        return out, A, lse

    def check(self):
        torch = _torch()
        torch.cuda.synchronize()
        assert int(self.err.item()) == 0
        out, A, lse = self.reference()
        bf16 = self.dt == torch.bfloat16
        got = self.obuf[: self.rows, : self.H * self.d].view(self.rows, self.H, self.d).double()
        tol = 2.0 ** -8 * (A + out.abs()) + 2.0 ** -12 * A if bf16 else 2e-5 * A
        assert bool(torch.isfinite(got).all())
        over = ((got - out).abs() - tol).max().item() if self.rows else 0.0
        assert over <= 1e-30, (over, (got - out).abs().max().item())
        gl = self.lse[: self.rows].double()
        empty = lse == -math.inf
        assert bool((gl[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
        if bool((~empty).any()):
            assert (gl - lse)[~empty].abs().max().item() < (1e-4 if bf16 else 2e-5)
        assert bool((self.obuf[:, self.H * self.d :] == -7.0).all())  # nothing between the rows is written


SHAPES = [
    # new rows, cached positions (with them), heads, KV heads, head_dim, page, window
    ([1], [1], 16, 8, 128, 64, 0),                                  # the first token of a sequence
    ([1], [128], 16, 8, 128, 64, 0),                                # a context of exactly one block
    ([1], [129], 16, 8, 128, 64, 0),
    ([1, 1, 1, 1], [300, 17, 64, 1025], 32, 8, 128, 64, 0),         # one token each: ragged decode
    ([5, 1, 37, 2], [5, 700, 250, 130], 32, 8, 128, 16, 0),         # chunks and single tokens together
    ([130, 64, 65], [130, 64, 400], 8, 8, 128, 32, 0),              # no grouping: 128 positions a tile
    ([129, 33], [1000, 33], 16, 8, 128, 128, 0),                    # group 2
    ([64, 100], [64, 357], 24, 8, 128, 256, 0),                     # group 3: tiles of 42 positions
    ([50, 19], [555, 19], 12, 2, 128, 64, 0),                       # group 6
    ([70, 1], [333, 900], 28, 4, 128, 64, 0),                       # group 7
    ([40, 3], [40, 500], 64, 8, 128, 64, 0),                        # group 8
    ([20, 1], [290, 77], 16, 1, 128, 64, 0),                        # group 16
    ([90, 1], [400, 211], 14, 2, 64, 16, 0),                        # head_dim 64
    ([300, 2], [300, 130], 8, 8, 64, 64, 0),
    ([10, 30], [4, 0], 16, 8, 128, 64, 0),                          # rows before the first position see nothing
    ([1, 1, 3], [0, 9, 0], 16, 8, 128, 64, 0),                      # unused places of a batch
    ([0, 7, 0, 1, 0], [50, 7, 0, 20, 9], 16, 8, 128, 64, 0),        # sequences without new rows
    ([100, 1, 1], [700, 800, 90], 32, 8, 128, 64, 100),             # a window, released pages before it
    ([300], [300], 16, 8, 128, 16, 1),                              # a window of one: every row copies its value
    ([40, 200], [5000, 260], 14, 2, 64, 32, 129),
    ([1], [9001], 32, 8, 128, 64, 0),                               # one row, a long context: split over the GPU
    ([3, 1], [20000, 15000], 8, 1, 64, 256, 0),
    ([600], [2900], 32, 8, 128, 64, 0),
]


@pytest.mark.parametrize("new,kv,heads,kv_heads,d,page,window", SHAPES)
def test_matches_the_definition_bf16(new, kv, heads, kv_heads, d, page, window):
    c = Case(new, kv, heads, kv_heads, d, page, window, seed=hash((sum(kv), heads, page)) & 0xFFFF)
    c.run()
    c.check()


@pytest.mark.parametrize("new,kv,heads,kv_heads,d,page,window", [SHAPES[i] for i in (0, 3, 4, 9, 12, 14, 16, 17, 20)])
def test_matches_the_definition_fp32(new, kv, heads, kv_heads, d, page, window):
    c = Case(new, kv, heads, kv_heads, d, page, window, dtype="fp32", seed=7)
    c.run()
    c.check()


def test_rows_inside_wider_buffers():
    c = Case([33, 1, 9], [60, 300, 1000], 16, 8, 128, 64, fused=16 * 128, gap=64, seed=3)
    c.run()
    c.check()


@pytest.mark.parametrize("d,window", [(128, 0), (64, 0), (128, 70)])
def test_rows_aligned_to_16_bytes_and_no_more(d, window):
    """Rows of q and out that begin on odd multiples of 16 bytes, in whole items, cut ones and single tokens."""
    c = Case([300, 1, 9, 130, 1], [2500, 300, 1000, 130, 4000], 16, 4, d, 64, window=window, fused=8, gap=8, seed=13)
    c.run()
    c.check()


def test_large_scores_and_a_late_maximum():
    """Scores over a wide range in which every later block holds a larger one: the running maximum is raised."""
    torch = _torch()
    c = Case([60], [1500], 16, 8, 128, 64, seed=4)
    ramp = torch.linspace(0.1, 4.0, 1500, device="cuda")
    p = torch.arange(1500, device="cuda")
    pg = c.table[1].long()[p // 64]
    c.k[pg, :, p % 64] = (c.q.view(60, 8, 2, 128)[:, :, 0].float().mean(0)[None] * 8 * ramp[:, None, None]).to(c.dt)
    c.run()
    c.check()


def test_repeats_bit_for_bit_and_leaves_the_workspace_usable():
    torch = _torch()
    c = Case([3, 1, 260], [4000, 9000, 700], 32, 8, 128, 64, seed=5)
    c.run()
    torch.cuda.synchronize()
    a, l = c.obuf.clone(), c.lse.clone()
    for _ in range(3):
        c.obuf.fill_(-7.0)
        c.run()
    torch.cuda.synchronize()
    assert torch.equal(a, c.obuf) and torch.equal(l, c.lse)
    c.check()


def test_one_workspace_serves_batches_of_different_shapes():
    torch = _torch()
    cases = [Case([1], [9001], 32, 8, 128, 64, seed=1), Case([300, 1], [900, 4000], 32, 8, 128, 64, seed=2),
             Case([1] * 40, list(range(1, 4001, 100)), 32, 8, 128, 64, seed=3)]
    for c in cases:
        c.attn.args.workspace = cases[0].ws.data_ptr()
    for _ in range(2):
        for c in cases:
            c.run()
    torch.cuda.synchronize()
    for c in cases:
        c.check()


def test_runs_on_its_own_stream_and_in_a_graph_that_follows_new_lengths():
    torch = _torch()
    c = Case([1, 1], [700, 90], 32, 8, 128, 64, seed=6)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        c.run(stream=st.cuda_stream)
    st.synchronize()
    c.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        c.run(stream=torch.cuda.current_stream().cuda_stream)
    c.kv = [333, 17]
    c.kv_len.copy_(torch.tensor(c.kv, dtype=torch.int32))
    c.obuf.fill_(-7.0)
    g.replay()
    c.check()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_window_longer_than_any_sequence_cuts_nothing_off(dtype):
    """The longest window there is, on rows before the first position, in the first pages and far beyond them."""
    c = Case([40, 130, 300, 3], [25, 130, 1500, 0], 8, 2, 64, 16, window=2 ** 31 - 1, dtype=dtype, seed=12)
    c.run()
    c.check()


def test_long_chunks_of_every_group_size():
    """The place of every item of many-item sequences: group sizes whose tiles are no power of two among them."""
    for G, window in ((1, 0), (3, 0), (5, 200), (6, 1), (7, 333), (11, 0), (13, 90), (16, 2000)):
        c = Case([700, 1, 451, 90], [2111, 300, 451, 60], 2 * G, 2, 64, 16, window=window, seed=G)
        c.run()
        c.check()


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(seed):
    """Batches of random shapes: items left whole, cut once and cut often, empty rows and sequences, every group size."""
    import random
    rng = random.Random(seed)
    for _ in range(6):
        G, kv_heads, d = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        B, longest = rng.choice([(1, 9000), (2, 6000), (3, 3000), (7, 2000), (30, 900)])
        single = rng.random() < 0.4
        new = [1 if single else rng.choice([0, 1, 2, rng.randint(1, 40), rng.randint(1, 300)]) for _ in range(B)]
        kv = [max(0, n + rng.choice([0, -1, -5, rng.randint(0, longest), rng.randint(0, longest)])) for n in new]
        c = Case(new, kv, G * kv_heads, kv_heads, d, rng.choice([16, 64, 256]), window=rng.choice([0, 0, 1, 130, 1500]),
                 seed=seed, fused=rng.choice([0, 64]), gap=rng.choice([0, 8]))
        c.run()
        c.run()
        c.check()


def test_without_lse():
    c = Case([40, 1], [400, 1200], 16, 8, 128, 64, seed=8)
    c.run(lse=False)
    torch = _torch()
    torch.cuda.synchronize()
    assert bool((c.lse == -7.0).all())
    c.run()
    c.check()


def test_a_cache_past_32_bit_offsets():
    """More than 2^32 bytes of keys (and of values): sequences in the pool's first and last pages."""
    torch = _torch()
    c = Case([1, 40], [200, 300], 32, 8, 128, 64, seed=9)
    pages = 36000
    k = torch.zeros((pages, 8, 64, 128), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() * 2 > 2 ** 32
    used = sorted({int(x) for x in c.table.flatten().tolist() if x >= 0})
    where = {p: (i if i % 2 else pages - 1 - i) for i, p in enumerate(used)}
    for p, to in where.items():
        k[to], v[to] = c.k[p], c.v[p]
    table = c.table.tolist()
    c.table = torch.tensor([[where.get(x, -1) for x in r] for r in table], dtype=torch.int32, device="cuda")
    c.k, c.v = k, v
    c.attn.args.num_pages = pages
    c.run()
    c.check()


def test_lengths_beyond_the_table_and_wild_page_numbers_stay_in_bounds():
    torch = _torch()
    c = Case([3, 2], [100, 60], 16, 8, 128, 64, seed=10)
    c.kv_len[0] = 1 << 30                       # clamped to what the table can name
    c.table[1, 0] = 1 << 30                     # slot of sequence 1: not a page, read as zeros
    c.run()
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0 and bool((c.obuf[5:] == -7.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_many_sequences(dtype):
    """More sequences than CTAs and than one warp's lanes, some without rows."""
    new = [i % 3 for i in range(300)]
    kv = [n and n + (37 * i) % 500 for i, n in enumerate(new)]
    c = Case(new, kv, 16, 8, 128, 64, dtype=dtype, seed=11)
    c.run()
    c.check()
