"""New rows on their way into the paged cache (qw_op_kv_append) against the definition in 64 bits.

Tolerances: a norm's sum of squares is a tree over at most 16 * 32 terms in a thread and 2^10 threads, so that 1 / rms is within
2^-18 of its value; rotation and the weights take four roundings: |error| <= 2^-17 (|x| + |y|), x and y being the
normalised pair, and 2^-8 of the result in bf16.  Values are rounded once and compared for equality; so are queries and keys
where there is neither norm nor rotation."""
import math

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu
NONE, VECTOR, HEAD = native.QKNORM_NONE, native.QKNORM_VECTOR, native.QKNORM_HEAD
TYPES = {"f32": native.DTYPE_F32, "bf16": native.DTYPE_BF16}


def rope_table(n, d, theta=1e6):
    import torch
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * \
        theta ** (-torch.arange(d // 2, dtype=torch.float64, device="cuda") * 2 / d)
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


class Case:
    def __init__(self, new, kv, heads, kv_heads, d, page, mode=NONE, in_kind="f32", kind="bf16", fused=True, rope=True,
                 seed=0, spare=2, rope_len=0, slots=True):
        import torch
        self.new, self.kv, self.H, self.Hkv, self.d, self.page, self.mode = new, kv, heads, kv_heads, d, page, mode
        tin, self.dt = ({"f32": torch.float32, "bf16": torch.bfloat16}[t] for t in (in_kind, kind))
        g = torch.Generator(device="cuda").manual_seed(seed)
        B = len(new)
        need = [max(0, -(-k // page)) for k in kv]
        self.num_pages, self.max_pages = sum(need) + 3, max(need + [1]) + 1
        order = torch.randperm(self.num_pages, device="cuda", generator=g).to(torch.int32)
        self.slots = torch.arange(B, 0, -1, dtype=torch.int32, device="cuda") if slots else None
        self.table = torch.full((B + 1, self.max_pages), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b in range(B):
            s = B - b if slots else b
            self.table[s, : need[b]] = order[at : at + need[b]]
            at += need[b]
        shape = (self.num_pages, kv_heads, page, d)
        self.kc = torch.randn(shape, device="cuda", generator=g).to(self.dt)
        self.vc = torch.randn(shape, device="cuda", generator=g).to(self.dt)
        self.n = sum(new)
        self.rows = self.n + spare
        widths = [heads * d, kv_heads * d, kv_heads * d]
        if fused:
            buf = torch.randn((self.rows, sum(widths) + 16), device="cuda", generator=g).mul_(2).to(tin)
            self.q, self.k, self.v, _ = buf.split(widths + [16], 1)
        else:
            self.q, self.k, self.v = (torch.randn((self.rows, w), device="cuda", generator=g).mul_(2).to(tin) for w in widths)
        self.qn = self.kn = None
        if mode != NONE:
            self.qn = 1 + 0.3 * torch.randn(heads * d if mode == VECTOR else d, device="cuda", generator=g)
            self.kn = 1 + 0.3 * torch.randn(kv_heads * d if mode == VECTOR else d, device="cuda", generator=g)
        self.rope_len = rope_len or max(kv + [1])
        self.rope = rope_table(self.rope_len, d) if rope else None
        self.qo = torch.full((self.rows, heads * d + 8), 7.0, dtype=self.dt, device="cuda")
        self.row_start = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device="cuda")
        p = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
        self.append = native.KvAppend(heads, kv_heads, d, page, self.num_pages, self.max_pages, rope=p(self.rope),
                                      rope_len=self.rope_len if rope else 0, qk_norm=mode, q_norm=p(self.qn), k_norm=p(self.kn),
                                      in_dtype=TYPES[in_kind], dtype=TYPES[kind])
        self.before = self.kc.clone(), self.vc.clone(), self.qo.clone()

    def run(self, stream=0, q_out=None):
        qo = self.qo if q_out is None else q_out
        self.append(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), qo.data_ptr() if qo is not False else 0,
                    self.kc.data_ptr(), self.vc.data_ptr(), self.table.data_ptr(), self.row_start.data_ptr(),
                    self.kv_len.data_ptr(), len(self.new), self.rows,
                    slots=self.slots.data_ptr() if self.slots is not None else 0, ld_q=self.q.stride(0),
                    ld_k=self.k.stride(0), ld_v=self.v.stride(0), ld_q_out=qo.stride(0) if qo is not False else 0, stream=stream)

    def normed(self, x, heads, w):
        """Rows r of x, (n, heads, d), normalised, in 64 bits."""
        import torch
        x = x.double().reshape(-1, heads, self.d)
        if self.mode != NONE:
            axes = (1, 2) if self.mode == VECTOR else (2,)
            x = x / torch.sqrt(x.square().mean(axes, keepdim=True) + 1e-6)
            x = x * w.double().reshape((heads, self.d) if self.mode == VECTOR else (1, self.d))
        return x

    def turned(self, x, pos):
        """(values, bound) of normalised rows at positions pos."""
        import torch
        half = self.d // 2
        lo, hi = x[..., :half], x[..., half:]
        size = torch.cat([lo.abs() + hi.abs()] * 2, -1)
        if self.rope is not None:
            c, s = self.rope[pos].double()[:, None].unbind(-1)
            x = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
        elif self.mode == NONE:
            return x, torch.zeros_like(size) + (2.0 ** -8 * x.abs() if self.dt == torch.bfloat16 else 0)
        bound = 2.0 ** -17 * size
        return x, bound * (1 + 2.0 ** -8) + 2.0 ** -8 * x.abs() if self.dt == torch.bfloat16 else bound

    def check(self):
        import torch
        torch.cuda.synchronize()
        kc, vc, qo = self.before
        kb = torch.zeros_like(kc, dtype=torch.float64)
        want_k, want_v = kc.double(), vc.clone()
        W = self.H * self.d
        assert torch.equal(self.qo[self.n :], qo[self.n :]) and torch.equal(self.qo[:, W:], qo[:, W:])
        at = 0
        for b, (n, m) in enumerate(zip(self.new, self.kv)):
            m = min(max(m, 0), self.max_pages * self.page)
            for_i = torch.arange(n, device="cuda")
            pos = m - n + for_i
            live = (pos >= 0) & (pos < self.rope_len if self.rope is not None else True)
            rows = slice(at, at + n)
            got = self.qo[rows, :W].double().view(n, self.H, self.d)
            if n:
                assert bool((got[~live] == 0).all())
            if bool(live.any()):
                p = pos[live]
                q, qb = self.turned(self.normed(self.q[rows][live], self.H, self.qn), p)
                assert bool(((got[live] - q).abs() <= qb).all()), (b, ((got[live] - q).abs() - qb).max().item())
                k, kbound = self.turned(self.normed(self.k[rows][live], self.Hkv, self.kn), p)
                v = self.v[rows][live].float().to(self.dt).reshape(-1, self.Hkv, self.d)
                s = int(self.slots[b]) if self.slots is not None else b
                pg = self.table[s].long()[p // self.page]
                held = (pg >= 0) & (pg < self.num_pages)
                pg, row = pg[held], p[held] % self.page
                want_k[pg, :, row] = k[held]
                kb[pg, :, row] = kbound[held]
                want_v[pg, :, row] = v[held]
            at += n
        off = (self.kc.double() - want_k).abs() - kb
        assert bool((off <= 0).all()), off.max().item()
        assert torch.equal(self.vc, want_v)


GEOMETRIES = [(16, 8, 128), (32, 8, 128), (64, 8, 128), (14, 2, 64), (28, 4, 128), (8, 1, 64), (3, 1, 16), (4, 4, 32),
              (6, 2, 256), (1, 1, 128), (2, 5, 64), (240, 8, 256)]


@pytest.mark.parametrize("mode", [NONE, VECTOR, HEAD])
@pytest.mark.parametrize("heads,kv_heads,d", GEOMETRIES)
def test_geometries(heads, kv_heads, d, mode):
    c = Case([3, 1, 0, 7], [10, 1, 5, 90], heads, kv_heads, d, 16, mode, seed=heads + d)
    c.run()
    c.check()


@pytest.mark.parametrize("in_kind,kind", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("mode", [NONE, VECTOR, HEAD])
def test_types_and_strides(in_kind, kind, fused, rope, mode):
    c = Case([5, 1, 20], [5, 300, 33], 16, 4, 64, 32, mode, in_kind, kind, fused, rope, seed=3, slots=fused)
    c.run()
    c.check()


@pytest.mark.parametrize("page", [1, 2, 16, 64, 256])
@pytest.mark.parametrize("mode", [VECTOR, HEAD])
def test_pages_and_lengths(page, mode):
    """Chunks that end inside pages, single tokens, sequences without rows, unused places, rows before position 0."""
    new = [1, 0, 130, 1, 17, 1, 64, 300, 1, 2]
    kv = [1, 40, 130, 0, 500, 257, 64, 200, -5, 1]
    c = Case(new, kv, 16, 8, 128, page, mode, seed=page)
    c.run()
    c.check()


def test_single_tokens_of_many_sequences():
    for B in (1, 64, 300, 1024):
        c = Case([1] * B, [1 + (37 * b) % 150 for b in range(B)], 8, 2, 64, 16, HEAD, seed=B, spare=B % 3)
        c.run()
        c.check()


def test_positions_beyond_the_table_of_angles_and_without_pages():
    c = Case([30, 40], [100, 50], 4, 2, 64, 16, HEAD, seed=1, rope_len=80)
    c.table[2, 5] = -1       # sequence 0 stands in row 2: positions 80..95 have no page
    c.table[1, 1] = 1 << 20  # sequence 1: positions 16..31 name a page that is none
    c.run()
    c.check()


def test_lengths_beyond_the_slot_are_limited():
    c = Case([10], [32], 4, 2, 64, 16, HEAD, seed=1, rope_len=200)
    c.table[1, 2] = int(next(i for i in range(c.num_pages) if i not in c.table[1].tolist()))
    c.kv = [c.max_pages * c.page + 1000]
    c.kv_len.fill_(c.kv[0])
    c.run()
    c.check()


def test_wild_row_starts_stay_inside():
    """Row starts that do not ascend or pass the buffers: nothing is written outside rows, pages and slots."""
    import torch
    c = Case([4, 4, 4], [8, 8, 8], 4, 2, 64, 16, HEAD, seed=2)
    for wild in ([5, 2, 9, 3], [-7, 4, 4000, 1 << 30], [0, 0, 0, 0], [-(1 << 31), (1 << 31) - 1, -1, 5]):
        c.row_start.copy_(torch.tensor(wild, dtype=torch.int32))
        c.run()
        torch.cuda.synchronize()
    assert torch.equal(c.qo[:, c.H * c.d :], c.before[2][:, c.H * c.d :])


@pytest.mark.parametrize("mode", [NONE, VECTOR, HEAD])
def test_queries_in_place(mode):
    import torch
    a = Case([5, 1, 20], [5, 300, 33], 16, 4, 64, 32, mode, "bf16", seed=3, spare=0)
    b = Case([5, 1, 20], [5, 300, 33], 16, 4, 64, 32, mode, "bf16", seed=3, spare=0)
    a.run()
    b.run(q_out=b.q)
    torch.cuda.synchronize()
    assert torch.equal(a.qo[:, : 16 * 64], b.q) and torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)


def test_no_queries_wanted():
    import torch
    c = Case([5, 1, 20], [5, 300, 33], 16, 4, 64, 32, HEAD, seed=3)
    d = Case([5, 1, 20], [5, 300, 33], 16, 4, 64, 32, HEAD, seed=3)
    c.run(q_out=False)
    d.run()
    torch.cuda.synchronize()
    assert torch.equal(c.kc, d.kc) and torch.equal(c.vc, d.vc) and torch.equal(c.qo, c.before[2])


def test_nan_rows_stay_by_themselves():
    import torch
    c = Case([3, 3], [3, 3], 4, 2, 64, 16, VECTOR, seed=4)
    d = Case([3, 3], [3, 3], 4, 2, 64, 16, VECTOR, seed=4)
    c.q[1], c.k[1] = math.nan, math.inf
    c.run()
    d.run()
    torch.cuda.synchronize()
    keep = [r for r in range(c.rows) if r != 1]
    assert torch.equal(c.qo[keep], d.qo[keep]) and torch.isnan(c.qo[1, : 4 * 64]).all()
    assert torch.isnan(c.kc).sum().item() == 2 * 64


def test_cache_past_32_bit_offsets():
    import torch
    H, Hkv, d, page, pages = 4, 8, 128, 256, 10000  # 2.6e9 elements
    kc = torch.zeros((pages, Hkv, page, d), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    q, k, v = (torch.randn((2, h * d), device="cuda") for h in (H, Hkv, Hkv))
    table = torch.tensor([[3, pages - 1]], dtype=torch.int32, device="cuda")
    qo = torch.empty((2, H * d), dtype=torch.bfloat16, device="cuda")
    rs, kl = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.tensor([512], dtype=torch.int32, device="cuda")
    native.KvAppend(H, Hkv, d, page, pages, 2)(q.data_ptr(), k.data_ptr(), v.data_ptr(), qo.data_ptr(), kc.data_ptr(),
                                               vc.data_ptr(), table.data_ptr(), rs.data_ptr(), kl.data_ptr(), 1, 2)
    torch.cuda.synchronize()
    for x, c in ((k, kc), (v, vc)):
        assert torch.equal(c[pages - 1, :, 254:].transpose(0, 1).reshape(2, -1), x.to(torch.bfloat16))
        assert int(torch.count_nonzero(c[: pages - 1])) == 0 and int(torch.count_nonzero(c[pages - 1, :, : 254])) == 0
