"""Products of 8-bit codes (qw_op_linear_q8) against the definition in 64 bits.

The integer sums are exact, y = (s w_scale) x_scale takes three roundings to 24 bits (s itself the first): |error| <= 3 * 2^-24
|y| < 2^-22 |y|; a bias or residual adds one of the result, 2^-24 |out|.  bf16 results are rounded once more, 2^-8 |out|.
SWIGLU: with e = 2^-22 the relative errors of gate and up, up silu(gate) moves by e |up silu| and 1.1 e |up gate| (silu' <= 1.1),
and the exponential of gate, whose argument is rounded, brings (|gate| + 8) 2^-22 of it."""
import math

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu
STORE, RESID, SWIGLU = native.LINEAR_STORE, native.LINEAR_RESID, native.LINEAR_SWIGLU


class Case:
    def __init__(self, t, n_out, k, epi=STORE, bf16=False, bias=False, seed=0, pad=0, gap=0, lowest=-127):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.t, self.n, self.k, self.epi, self.bf16 = t, n_out, k, epi, bf16
        self.ld = (k + 15) // 16 * 16 + pad
        self.w = torch.randint(lowest, 128, (n_out, self.ld), dtype=torch.int8, device="cuda", generator=g)
        self.x = torch.randint(lowest, 128, (t, self.ld), dtype=torch.int8, device="cuda", generator=g)
        self.ws = (torch.rand(n_out, device="cuda", generator=g) + 0.5) / (40 * math.sqrt(k))
        self.xs = (torch.rand(t, device="cuda", generator=g) + 0.5) / 60
        self.bias = torch.randn(n_out, device="cuda", generator=g) if bias else None
        self.cols = n_out // 2 if epi == SWIGLU else n_out
        self.resid = torch.randn((t, self.cols + gap), device="cuda", generator=g) if epi == RESID else None
        dt = torch.bfloat16 if bf16 else torch.float32
        self.out = torch.full((t + 1, self.cols + gap), 7.0, dtype=dt, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(self, stream=0, out=None):
        lin = native.LinearQ8(self.w.data_ptr(), self.ws.data_ptr(), self.n, self.k, ld_w=self.ld, epi=self.epi,
                              bias=self.bias.data_ptr() if self.bias is not None else 0,
                              out_dtype=native.DTYPE_BF16 if self.bf16 else native.DTYPE_F32)
        out = self.out if out is None else out
        lin(self.x.data_ptr(), self.xs.data_ptr(), self.t, out.data_ptr(),
            resid=self.resid.data_ptr() if self.resid is not None else 0, ld_x=self.ld, ld_out=out.stride(0),
            ld_resid=self.resid.stride(0) if self.resid is not None else 0, err=self.err.data_ptr(), stream=stream)

    def check(self):
        import torch
        torch.cuda.synchronize()
        assert self.err.item() == 0
        s = self.x[:, : self.k].double() @ self.w[:, : self.k].double().T
        y = s * self.ws.double() * self.xs.double()[:, None]
        got = self.out[: self.t, : self.cols].double()
        if self.epi == SWIGLU:
            gate, up = y.view(self.t, -1, 2, 16).unbind(2)
            gate, up = gate.reshape(self.t, -1), up.reshape(self.t, -1)
            want = up * gate / (1 + torch.exp(-gate))
            e = 2.0 ** -22
            bound = e * want.abs() + 1.1 * e * (up * gate).abs() + (gate.abs() + 8) * e * want.abs()
        else:
            want = y
            if self.bias is not None:
                want = want + self.bias.double()
            if self.resid is not None:
                want = want + self.resid[:, : self.cols].double()
            bound = 2.0 ** -22 * y.abs() + 2.0 ** -24 * want.abs()
        if self.bf16:
            bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
        off = (got - want).abs() - bound
        assert bool((off <= 1e-30).all()), (off.max().item(), int((off > 1e-30).sum()))
        assert bool((self.out[self.t] == 7).all()) and bool((self.out[:, self.cols :] == 7).all())


# tokens below, at and above every tile; features and codes that end inside one
@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 127, 128, 129, 200, 256, 257, 300])
@pytest.mark.parametrize("n_out,k", [(1, 1), (31, 17), (32, 16), (100, 127), (128, 128), (130, 129), (257, 136), (384, 896)])
def test_store(t, n_out, k):
    c = Case(t, n_out, k, seed=t + k, bias=t % 2 == 0, gap=t % 3, pad=16 * (t % 2))
    c.run()
    c.check()


@pytest.mark.parametrize("t,n_out,k", [(1, 6144, 4096), (3, 4096, 12288), (8, 24576, 896), (16, 1152, 896), (64, 4096, 12288),
                                       (40, 10240, 2048), (128, 6144, 4096), (333, 1152, 896), (512, 2048, 6144),
                                       (700, 5120, 1000), (1024, 6144, 1024), (1500, 8192, 512), (2500, 4100, 300),
                                       (4100, 4096, 640), (77, 151936, 64)])
@pytest.mark.parametrize("bf16", [False, True])
def test_store_larger(t, n_out, k, bf16):
    c = Case(t, n_out, k, bf16=bf16, bias=True, seed=1, gap=5)
    c.run()
    c.check()


@pytest.mark.parametrize("t", [1, 7, 16, 40, 64, 100, 128, 200, 256, 513, 1030, 2048])
@pytest.mark.parametrize("n_out,k", [(32, 64), (96, 100), (512, 256), (4864 * 2, 896), (2048, 2050)])
def test_swiglu(t, n_out, k):
    c = Case(t, n_out, k, epi=SWIGLU, bf16=True, seed=t, gap=3 * (t % 2))
    c.run()
    c.check()


@pytest.mark.parametrize("t,n_out,k", [(1, 4096, 512), (5, 33, 70), (64, 896, 4864), (100, 2048, 300), (300, 4096, 4096),
                                       (2100, 4096, 1024)])
@pytest.mark.parametrize("in_place", [False, True])
def test_resid(t, n_out, k, in_place):
    import torch
    c = Case(t, n_out, k, epi=RESID, seed=2, gap=4)
    if in_place:
        want = c.resid.clone()
        c.run(out=c.resid)
        torch.cuda.synchronize()
        c.out[:t] = c.resid
        c.out[:t, n_out:] = 7
        assert torch.equal(c.resid[:, n_out:], want[:, n_out:])
        c.resid = want
    else:
        c.run()
    c.check()


@pytest.mark.parametrize("t", [1, 64, 300])
def test_largest_sums(t):
    """The longest rows of the largest codes: sums of 2^31 - 16384."""
    import torch
    k = 131071
    c = Case(t, 192, k, seed=0)
    c.w[: 64].fill_(-128)
    c.x[: t // 2 + 1].fill_(-128)
    c.w[64:128].fill_(127)
    c.run()
    c.check()
    assert torch.isfinite(c.out).all()


@pytest.mark.parametrize("epi,bf16", [(STORE, False), (STORE, True), (RESID, False), (SWIGLU, True)])
@pytest.mark.parametrize("t", [1, 40, 64, 128, 300, 1500])
def test_same_bits_every_time(t, epi, bf16):
    """Integer sums: nothing depends on the order in which parts are joined."""
    import torch
    c = Case(t, 4096, 2100, epi=epi, bf16=bf16, seed=5)
    first = None
    for _ in range(4):
        c.run()
        torch.cuda.synchronize()
        first = c.out.clone() if first is None else first
        assert torch.equal(first, c.out)


@pytest.mark.parametrize("epi,bf16,bias", [(STORE, False, False), (STORE, True, False), (STORE, False, True), (STORE, True, True),
                                           (RESID, False, False), (SWIGLU, True, False)])
@pytest.mark.parametrize("n_out,k,gap", [(1024, 2304, 0), (1024, 300, 3), (4096, 4096, 0)])
def test_rows_do_not_depend_on_their_batch(epi, bf16, bias, n_out, k, gap):
    """A token's results are the same bits in every batch, whatever kernel and split it takes."""
    import torch
    big = Case(5000, n_out, k, epi=epi, bf16=bf16, bias=bias, seed=6, gap=gap)
    big.run()
    torch.cuda.synchronize()
    for t in (1, 16, 33, 64, 128, 257, 700, 1500):
        c = Case(t, n_out, k, epi=epi, bf16=bf16, gap=gap)
        c.w, c.ws, c.x, c.xs, c.bias = big.w, big.ws, big.x[:t], big.xs[:t], big.bias
        c.resid = big.resid[:t] if epi == RESID else None
        c.run()
        torch.cuda.synchronize()
        assert torch.equal(c.out[:t], big.out[:t]), t


def test_scales_that_are_none():
    """Scales of zero and NaN: marked rows of codes give NaN, rows of zeros zero (and the residual as it was)."""
    import torch
    for t, epi, bf16 in ((5, STORE, False), (5, SWIGLU, True), (300, RESID, False), (2000, SWIGLU, True)):
        c = Case(t, 4096, 256, epi=epi, bf16=bf16, seed=9)
        c.xs[2], c.xs[3] = math.nan, 0.0
        c.x[2] = 0
        c.run()
        torch.cuda.synchronize()
        assert torch.isnan(c.out[2, : c.cols]).all() and torch.isfinite(c.out[: 2]).all()
        want = c.resid[3, : c.cols] if epi == RESID else torch.zeros_like(c.out[3, : c.cols])
        assert torch.equal(c.out[3, : c.cols], want)


def test_gates_far_from_zero():
    import torch
    c = Case(64, 512, 64, epi=SWIGLU, bf16=True, seed=3)
    c.ws *= 400  # gates up to several thousand: exponentials beyond fp32
    c.run()
    c.check()
    assert torch.isfinite(c.out).all()


def test_weights_past_32_bit_offsets():
    """Weight rows whose offsets pass 2^31 codes."""
    import torch
    n, k, ld = 300, 512, 1 << 23
    buf = torch.zeros((n, ld), dtype=torch.int8, device="cuda")
    c = Case(20, n, k, seed=4)
    buf[:, :k] = c.w[:, :k]
    lin = native.LinearQ8(buf.data_ptr(), c.ws.data_ptr(), n, k, ld_w=ld)
    lin(c.x.data_ptr(), c.xs.data_ptr(), c.t, c.out.data_ptr(), ld_x=c.ld, ld_out=c.out.stride(0))
    c.check()


@pytest.mark.parametrize("t,n_out,k,epi,bf16,ld", [(20, 300, 600, STORE, True, 1 << 27), (20, 256, 2048, RESID, False, 1 << 27),
                                                   (300, 19456, 256, SWIGLU, True, 1 << 23), (300, 19456, 256, STORE, True, 1 << 23)])
def test_results_past_32_bit_offsets(t, n_out, k, epi, bf16, ld):
    """Result (and residual) rows whose offsets pass 2^31 elements, by joined tiles and by pairs."""
    import torch
    c = Case(t, n_out, k, epi=epi, bf16=bf16, seed=8)
    out = torch.zeros(((t - 1) * ld + n_out,), dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    rows = out.as_strided((t, c.cols), (ld, 1))
    if epi == RESID:
        rows.copy_(c.resid)
        want, c.resid = c.resid, rows
    c.run(out=rows)
    torch.cuda.synchronize()
    c.out[:t] = rows
    if epi == RESID:
        c.resid = want
    c.check()
    rows.zero_()
    assert int(torch.count_nonzero(out)) == 0


def test_other_streams_at_once():
    import torch
    cases = [Case(t, 4096, 1024, seed=t, epi=e, bf16=b) for t, e, b in
             ((1, STORE, False), (64, RESID, False), (200, STORE, True), (1200, SWIGLU, True))]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cases, streams):
            c.run(stream=s.cuda_stream)
    torch.cuda.synchronize()
    for c in cases:
        c.check()
