"""A decoder layer in 8 bits as a program runs it: norm_q8 -> linear_q8 (q, k, v) -> kv_append -> chunk_attn -> quant_q8 ->
linear_q8 (o, residual) -> norm_q8 -> linear_q8 (gate and up, SWIGLU) -> quant_q8 -> linear_q8 (down, residual), queued on one
stream without a pause, then each step checked against the definition in 64 bits on what the step before it left.

Tolerances are those of the operators' own tests; for the whole layer: codes are off by half a step of 1 / 127 of a row's
largest number each, so that a product's error is about (1 / 254) max / rms of a row / sqrt(3) of its size, twice (both
operands); with rows of normal numbers (max / rms about 4) 1.3 %, four products deep below 4 %."""
import math

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu
PAGE, THETA = 32, 1e6


class Layer:
    """Weights in 8 bits, a paged cache and buffers for `rows` rows; run() queues one pass."""

    def __init__(self, dim, hidden, heads, kv_heads, d, new, kv, seed=0, qk_norm=native.QKNORM_HEAD):
        import torch
        self.dim, self.hidden, self.H, self.Hkv, self.d = dim, hidden, heads, kv_heads, d
        self.new, self.kv, self.batch, self.rows = new, kv, len(new), sum(new)
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        wide = (heads + 2 * kv_heads) * d
        self.wide = wide
        rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
        self.plain = {"qkv": rand(wide, dim) / math.sqrt(dim), "o": rand(dim, heads * d) / math.sqrt(heads * d),
                      "gu": rand(2 * hidden, dim) / math.sqrt(dim), "down": rand(dim, hidden) / math.sqrt(hidden)}
        self.q8 = {}
        for name, w in self.plain.items():
            codes = torch.zeros(w.shape, dtype=torch.int8, device="cuda")
            scale = torch.zeros(w.shape[0], device="cuda")
            native.op_quant_q8(w.data_ptr(), native.DTYPE_F32, w.shape[0], w.shape[1], codes.data_ptr(), scale.data_ptr())
            self.q8[name] = codes, scale
        self.n1, self.n2 = 1 + 0.1 * rand(dim), 1 + 0.1 * rand(dim)
        self.qn, self.kn = 1 + 0.1 * rand(d), 1 + 0.1 * rand(d)
        need = [-(-k // PAGE) for k in kv]
        self.pages, self.max_pages = sum(need) + 2, max(need)
        order = torch.randperm(self.pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((self.batch, self.max_pages), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at : at + n]
            at += n
        shape = (self.pages, kv_heads, PAGE, d)
        self.kc, self.vc = rand(*shape).to(torch.bfloat16), rand(*shape).to(torch.bfloat16)
        self.row_start = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device="cuda")
        n = max(kv)
        ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * \
            THETA ** (-torch.arange(d // 2, dtype=torch.float64, device="cuda") * 2 / d)
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        R = self.rows
        self.x, self.delta = rand(R, dim), rand(R, dim).to(torch.bfloat16)
        e = lambda *s, t=torch.float32: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        self.h, self.h2, self.y = e(R, dim), e(R, dim), e(R, dim)
        self.c1, self.s1 = e(R, dim, t=torch.int8), e(R)
        self.qkv = e(R, wide)
        self.q, self.att = e(R, heads * d, t=torch.bfloat16), e(R, heads * d, t=torch.bfloat16)
        self.c2, self.s2 = e(R, heads * d, t=torch.int8), e(R)
        self.c3, self.s3 = e(R, dim, t=torch.int8), e(R)
        self.act = e(R, hidden, t=torch.bfloat16)
        self.c4, self.s4 = e(R, hidden, t=torch.int8), e(R)
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        ws = native.chunk_attn_workspace(heads, kv_heads, d)
        self.ws = torch.zeros(ws, dtype=torch.uint8, device="cuda")
        lin = lambda k, epi, dt: native.LinearQ8(self.q8[k][0].data_ptr(), self.q8[k][1].data_ptr(), *self.q8[k][0].shape,  # noqa: E731
                                                 epi=epi, out_dtype=dt)
        f32, bf16 = native.DTYPE_F32, native.DTYPE_BF16
        self.norm1 = native.NormQ8(dim, self.n1.data_ptr(), 1e-6, f32, bf16)
        self.norm2 = native.NormQ8(dim, self.n2.data_ptr(), 1e-6, f32)
        self.l_qkv = lin("qkv", native.LINEAR_STORE, f32)
        self.l_o, self.l_down = lin("o", native.LINEAR_RESID, f32), lin("down", native.LINEAR_RESID, f32)
        self.l_gu = lin("gu", native.LINEAR_SWIGLU, bf16)
        self.append = native.KvAppend(heads, kv_heads, d, PAGE, self.pages, self.max_pages, rope=self.rope.data_ptr(),
                                      rope_len=n, qk_norm=qk_norm, q_norm=self.qn.data_ptr(), k_norm=self.kn.data_ptr())
        self.attn = native.ChunkAttention(heads, kv_heads, d, PAGE, self.pages, self.max_pages, self.ws.data_ptr(), ws)

    def run(self, stream=0):
        R, H, Hkv, d, wide = self.rows, self.H, self.Hkv, self.d, self.wide
        p, err = lambda t: t.data_ptr(), self.err.data_ptr()  # noqa: E731
        self.norm1(p(self.x), p(self.c1), p(self.s1), R, delta=p(self.delta), sum_out=p(self.h), stream=stream)
        self.l_qkv(p(self.c1), p(self.s1), R, p(self.qkv), err=err, stream=stream)
        q, k, v = (self.qkv[:, a:] for a in (0, H * d, (H + Hkv) * d))
        self.append(p(q), p(k), p(v), p(self.q), p(self.kc), p(self.vc), p(self.table), p(self.row_start), p(self.kv_len),
                    self.batch, R, ld_q=wide, ld_k=wide, ld_v=wide, stream=stream)
        self.attn(p(self.q), p(self.kc), p(self.vc), p(self.table), p(self.row_start), p(self.kv_len), self.batch, R,
                  p(self.att), err=err, stream=stream)
        native.op_quant_q8(p(self.att), native.DTYPE_BF16, R, H * d, p(self.c2), p(self.s2), stream=stream)
        self.l_o(p(self.c2), p(self.s2), R, p(self.h2), resid=p(self.h), err=err, stream=stream)
        self.norm2(p(self.h2), p(self.c3), p(self.s3), R, stream=stream)
        self.l_gu(p(self.c3), p(self.s3), R, p(self.act), err=err, stream=stream)
        native.op_quant_q8(p(self.act), native.DTYPE_BF16, R, self.hidden, p(self.c4), p(self.s4), stream=stream)
        self.l_down(p(self.c4), p(self.s4), R, p(self.y), resid=p(self.h2), err=err, stream=stream)

    # ---- the definitions, in 64 bits ----
    def product(self, codes, scale, name):
        w, ws = self.q8[name]
        return codes.double() @ w.double().T * ws.double() * scale.double()[:, None]

    @staticmethod
    def coded(g):
        import torch
        g = g.double()
        top = g.abs().amax(1, keepdim=True)
        return torch.round(127 * g / top).to(torch.int8), top.squeeze(1) / 127

    def rotated(self, x, heads, w):
        import torch
        x = x.double().reshape(-1, heads, self.d)
        x = x / torch.sqrt(x.square().mean(2, keepdim=True) + 1e-6) * w.double()
        lo, hi = x.chunk(2, -1)
        c, s = self.rope[self.positions()].double()[:, None].unbind(-1)
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)

    def positions(self):
        import torch
        return torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(self.new, self.kv)])

    def cached(self, b, n):
        import torch
        p = torch.arange(n, device="cuda")
        pg = self.table[b].long()[p // PAGE]
        return self.kc[pg, :, p % PAGE].double(), self.vc[pg, :, p % PAGE].double()

    def attention(self, q, bf16=True):
        import torch
        out = torch.zeros((self.rows, self.H, self.d), dtype=torch.float64, device="cuda")
        at = 0
        for b, (n, m) in enumerate(zip(self.new, self.kv)):
            k, v = self.cached(b, m)
            k, v = (t.repeat_interleave(self.H // self.Hkv, 1) for t in (k, v))
            s = torch.einsum("nhd,mhd->hnm", q[at : at + n].double(), k) / math.sqrt(self.d)
            hidden = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None]
            s[:, hidden] = -math.inf
            out[at : at + n] = torch.einsum("hnm,mhd->nhd", torch.softmax(s, -1), v)
            at += n
        return out.reshape(self.rows, -1)

    def check_steps(self):
        import torch
        torch.cuda.synchronize()
        assert self.err.item() == 0
        near = lambda a, b, r: (a.double() - b).norm().item() <= r * b.norm().item()  # noqa: E731
        h = self.x + self.delta.float()
        assert torch.equal(self.h, h)
        codes, top = self.coded(h * self.n1)
        assert torch.equal(self.c1, codes)
        assert near(self.s1, top / torch.sqrt(h.double().square().mean(1) + 1e-6), 2.0 ** -22)
        assert near(self.qkv, self.product(self.c1, self.s1, "qkv"), 2.0 ** -22)
        H, Hkv, d = self.H, self.Hkv, self.d
        assert near(self.q.view(-1, H, d), self.rotated(self.qkv[:, : H * d], H, self.qn), 2.0 ** -8)
        k = torch.cat([self.cached(b, m)[0][m - n :] for b, (n, m) in enumerate(zip(self.new, self.kv))])
        v = torch.cat([self.cached(b, m)[1][m - n :] for b, (n, m) in enumerate(zip(self.new, self.kv))])
        assert near(k, self.rotated(self.qkv[:, H * d : (H + Hkv) * d], Hkv, self.kn), 2.0 ** -8)
        assert torch.equal(v.reshape(self.rows, -1).bfloat16(), self.qkv[:, (H + Hkv) * d :].bfloat16())
        assert near(self.att, self.attention(self.q.view(-1, H, d)), 2.0 ** -7)
        codes, top = self.coded(self.att.float())
        assert torch.equal(self.c2, codes) and near(self.s2, top, 2.0 ** -24)
        assert near(self.h2, self.h.double() + self.product(self.c2, self.s2, "o"), 2.0 ** -22)
        codes, top = self.coded(self.h2 * self.n2)
        assert torch.equal(self.c3, codes)
        y = self.product(self.c3, self.s3, "gu").view(self.rows, -1, 2, 16)
        gate, up = y[:, :, 0].reshape(self.rows, -1), y[:, :, 1].reshape(self.rows, -1)
        assert near(self.act, up * gate * torch.sigmoid(gate), 2.0 ** -8)
        codes, _ = self.coded(self.act.float())
        assert torch.equal(self.c4, codes)
        assert near(self.y, self.h2.double() + self.product(self.c4, self.s4, "down"), 2.0 ** -22)

    def uncoded(self):
        """The layer in 64 bits with the weights and activations as they were before they were coded."""
        import torch
        P = {k: w.double() for k, w in self.plain.items()}
        norm = lambda x, w: x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-6) * w.double()  # noqa: E731
        h = self.x.double() + self.delta.double()
        qkv = norm(h, self.n1) @ P["qkv"].T
        H, Hkv, d = self.H, self.Hkv, self.d
        q = self.rotated(qkv[:, : H * d], H, self.qn)
        k = self.rotated(qkv[:, H * d : (H + Hkv) * d], Hkv, self.kn)
        keep = self.kc.clone(), self.vc.clone()
        pos = self.positions()
        b = torch.repeat_interleave(torch.arange(self.batch, device="cuda"), torch.tensor(self.new, device="cuda"))
        pg = self.table[b, pos // PAGE].long()
        self.kc, self.vc = self.kc.double(), self.vc.double()
        self.kc[pg, :, pos % PAGE] = k
        self.vc[pg, :, pos % PAGE] = qkv[:, (H + Hkv) * d :].reshape(-1, Hkv, d)
        att = self.attention(q)
        self.kc, self.vc = keep
        h2 = h + att @ P["o"].T
        y = (norm(h2, self.n2) @ P["gu"].T).view(self.rows, -1, 2, 16)
        gate, up = y[:, :, 0].reshape(self.rows, -1), y[:, :, 1].reshape(self.rows, -1)
        return h2 + (up * gate * torch.sigmoid(gate)) @ P["down"].T


SHAPES = [(512, 1024, 4, 2, 128, [1, 40, 7], [60, 40, 33]),                # turns
          (896, 1216, 14, 2, 64, [1] * 16, [5 + 7 * i for i in range(16)]),  # decoding
          (1024, 2048, 8, 8, 128, [300, 200], [300, 260])]                 # prompts


@pytest.mark.parametrize("shape", SHAPES)
def test_layer_step_by_step(shape):
    layer = Layer(*shape)
    layer.run()
    layer.check_steps()


@pytest.mark.parametrize("shape", SHAPES)
def test_layer_against_itself_without_codes(shape):
    import torch
    layer = Layer(*shape, seed=3)
    layer.run()
    torch.cuda.synchronize()
    want = layer.uncoded()
    off = ((layer.y.double() - want).norm() / want.norm()).item()
    assert off < 0.04, off


def test_layer_in_a_graph_follows_new_inputs():
    """A captured pass, replayed on other rows, lengths and pages, gives what the eager calls give, bit for bit."""
    import torch
    layer = Layer(*SHAPES[0], seed=1)
    layer.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.run(stream=torch.cuda.current_stream().cuda_stream)
    for seed in (5, 6):
        other = Layer(*SHAPES[0], seed=seed)
        for name in ("x", "delta", "kc", "vc", "table", "row_start", "kv_len"):
            getattr(layer, name).copy_(getattr(other, name))
        if seed == 6:  # the sequences' rows dealt out otherwise
            layer.new, layer.kv = [8, 30, 10], [32, 40, 33]
            layer.row_start.copy_(torch.tensor([0, 8, 38, 48], dtype=torch.int32))
            layer.kv_len.copy_(torch.tensor(layer.kv, dtype=torch.int32))
        keep = layer.kc.clone(), layer.vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        layer.check_steps()
        got = [t.clone() for t in (layer.y, layer.kc, layer.vc, layer.c4, layer.s4)]
        layer.kc.copy_(keep[0])
        layer.vc.copy_(keep[1])
        layer.run()
        torch.cuda.synchronize()
        for a, b in zip(got, (layer.y, layer.kc, layer.vc, layer.c4, layer.s4)):
            assert torch.equal(a, b)


def test_layers_on_two_streams_at_once():
    import torch
    layers = [Layer(*SHAPES[i], seed=7) for i in (0, 1, 2)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(4):
        for layer, s in zip(layers, streams):
            layer.run(stream=s.cuda_stream)
    for layer in layers:
        layer.check_steps()


def test_two_graphs_of_the_operators_at_once():
    """Nothing is shared between calls: two captured passes over the same weights run together."""
    import torch
    a, b = Layer(*SHAPES[2], seed=8), Layer(*SHAPES[2], seed=8)
    for name in ("q8", "l_qkv", "l_o", "l_gu", "l_down"):
        setattr(b, name, getattr(a, name))
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for layer, s in zip((a, b), streams):
        layer.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            layer.run(stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    a.check_steps()
    b.check_steps()
    assert torch.equal(a.y, b.y)


def test_codes_that_the_kernel_before_writes():
    """Weights coded right in front of the product that reads them, on one stream: nothing is read early."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(0)
    n, k, t = 4096, 4096, 64
    x = torch.randn((t, k), device="cuda", generator=g)
    cx, sx = torch.zeros((t, k), dtype=torch.int8, device="cuda"), torch.zeros(t, device="cuda")
    cw, sw = torch.zeros((n, k), dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    out = torch.zeros((t, n), device="cuda")
    lin = native.LinearQ8(cw.data_ptr(), sw.data_ptr(), n, k)
    for i in range(6):
        w = torch.randn((n, k), device="cuda", generator=g)
        torch.cuda.synchronize()
        native.op_quant_q8(x.data_ptr(), native.DTYPE_F32, t, k, cx.data_ptr(), sx.data_ptr())
        native.op_quant_q8(w.data_ptr(), native.DTYPE_F32, n, k, cw.data_ptr(), sw.data_ptr())
        lin(cx.data_ptr(), sx.data_ptr(), t, out.data_ptr())
        torch.cuda.synchronize()
        want = cx.double() @ cw.double().T * sw.double() * sx.double()[:, None]
        assert torch.equal(cw, Layer.coded(w)[0])
        assert bool(((out.double() - want).abs() <= 2.0 ** -22 * want.abs()).all())


FIRST = """
import torch
from tests.test_gpu_layer_q8 import Layer, SHAPES
torch.cuda.set_device(0)
layer = Layer(*SHAPES[0], seed=1)  # codes its weights: the only call before the capture
torch.cuda.synchronize()
side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    layer.run(stream=torch.cuda.current_stream().cuda_stream)
graph.replay()
layer.check_steps()
print("captured first")
"""


def test_first_calls_may_be_captured_ones():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_graphs_with_copies_and_joined_streams():
    """Captured behind copies, fills and another stream's kernels, each operator waits for all of them."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    n, k, t = 2048, 2048, 100
    src = torch.randn((4, t, k), device="cuda", generator=g)
    x, x2 = torch.zeros((t, k), device="cuda"), torch.zeros((t, k), device="cuda")
    w = torch.randn((n, k), device="cuda", generator=g)
    cw, sw = torch.zeros((n, k), dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    cx, sx = torch.zeros((t, k), dtype=torch.int8, device="cuda"), torch.zeros(t, device="cuda")
    w2, out, resid = torch.zeros_like(w), torch.zeros((t, n), device="cuda"), torch.zeros((t, n), device="cuda")
    lin = native.LinearQ8(cw.data_ptr(), sw.data_ptr(), n, k, epi=native.LINEAR_RESID)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        here = torch.cuda.current_stream()
        st = here.cuda_stream
        x.copy_(src[0])                                      # a copy in front
        other.wait_stream(here)
        with torch.cuda.stream(other):                       # weights coded on another stream meanwhile
            w2.copy_(w).mul_(2.0)
            native.op_quant_q8(w2.data_ptr(), native.DTYPE_F32, n, k, cw.data_ptr(), sw.data_ptr(), stream=other.cuda_stream)
        x2.copy_(x)
        native.op_quant_q8(x2.data_ptr(), native.DTYPE_F32, t, k, cx.data_ptr(), sx.data_ptr(), stream=st)
        resid.zero_()
        resid.add_(1.0)
        here.wait_stream(other)                              # two kernels and a fill in front of the product
        lin(cx.data_ptr(), sx.data_ptr(), t, out.data_ptr(), resid=resid.data_ptr(), stream=st)
        out.mul_(0.5)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        body()
    for i in range(1, 4):
        src[0].copy_(src[i])
        w.copy_(torch.randn((n, k), device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cx, Layer.coded(src[i])[0]) and torch.equal(cw, Layer.coded(2 * w)[0])
        y = cx.double() @ cw.double().T * sw.double() * sx.double()[:, None]
        assert bool(((2 * out.double() - 1 - y).abs() <= 2.0 ** -22 * y.abs() + 2.0 ** -24 * (1 + y).abs()).all())
        got = out.clone()
        with torch.cuda.stream(side):
            body()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
