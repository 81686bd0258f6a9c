"""Rows to 8-bit codes (qw_op_quant_q8) and the residual's addition with the root-mean-square norm in front of them
(qw_op_norm_q8) against the definition in 64 bits.

Codes are compared for equality: (127 g) / t in 64 bits is exact where it is a half (254 |g| and t are whole numbers of at most
32 and 24 bits times powers of two), and a quotient that is none keeps 2^-25 of distance from one, so that rounding it to
whole numbers gives the codes of real arithmetic.  h = x + delta and h w are fp32 numbers by definition, so they are compared
for equality too (bf16 sums as the rounded h).  scale: the root of the mean, its product with t and the division by 127 are
rounded once each to 24 bits: 3 * 2^-24 < 2^-22, relative; without a norm one rounding, 2^-24."""
import math

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu
TINY = 127 * 2.0 ** -126
TYPES = {"f32": native.DTYPE_F32, "bf16": native.DTYPE_BF16}


def torch_type(t):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16}[t]


def placed(values, ld, lead=0):
    """`values` in rows of ld elements that begin `lead` elements behind an aligned address; NaN around them."""
    import torch
    rows, dim = values.shape
    buf = torch.full((lead + rows * ld + 8,), math.nan, dtype=values.dtype, device="cuda")
    view = buf[lead : lead + rows * ld].view(rows, ld)[:, :dim]
    view.copy_(values)
    return buf, view


def codes_of(g):
    """(codes, scale without a norm) of rows of fp32 numbers, in 64 bits."""
    import torch
    g = g.double()
    top = g.abs().amax(1)
    bad = ~torch.isfinite(g).all(1)
    top = torch.where(bad | (top < TINY), torch.zeros_like(top), top)
    codes = torch.where((top > 0)[:, None], torch.round(127 * g / top[:, None]), torch.zeros_like(g))
    scale = torch.where(bad, torch.full_like(top, math.nan), top / 127)
    return codes.to(torch.int8), scale


def rows_of(rows, dim, seed, kind="f32"):
    """Rows that try the codes: ordinary ones, outliers, halves of a code, one value, zeros, tiny and huge numbers."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, dim), device="cuda", generator=g)
    for r in range(rows):
        k = r % 8
        if k == 1:
            x[r] *= torch.exp(torch.randn(dim, device="cuda", generator=g))
        elif k == 2:  # quarter steps of a code: every second one a half
            x[r] = torch.randint(-508, 509, (dim,), device="cuda", generator=g) / 4.0
            x[r, 0] = 127.0
        elif k == 3:
            x[r] = 0.0
            x[r, r % dim] = -3.5
        elif k == 4:
            x[r] = 0.0
        elif k == 5:
            x[r] *= 1e-38  # the largest is near the border below which rows count as zeros
        elif k == 6:
            x[r] *= 1e37
        elif k == 7:  # halves of a code for a largest value with many bits
            x[r] = (torch.randint(-127, 127, (dim,), device="cuda", generator=g) + 0.5) * (1.7320508 / 127)
            x[r, dim // 2] = 1.7320508
    return x.to(torch_type(kind))


def check_codes(q, scale, g, factor, bound):
    import torch
    codes, plain = codes_of(g)
    assert torch.equal(q, codes)
    want = plain * factor
    assert torch.equal(torch.isnan(scale), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert bool(((scale.double() - want).abs()[ok] <= bound * want[ok]).all())


# widths below, at and above a thread's, a warp's and a CTA's share; odd ones; rows that lie apart and off alignment
ROWS = [(1, 1, 0, 0), (3, 5, 1, 0), (9, 31, 0, 0), (16, 32, 0, 0), (40, 100, 4, 0), (40, 128, 0, 0), (17, 255, 1, 3),
        (33, 256, 0, 0), (24, 896, 0, 0), (24, 1000, 24, 0), (24, 1001, 0, 0), (24, 1023, 1, 0), (16, 1024, 0, 1),
        (16, 2048, 16, 0), (16, 4095, 1, 0), (16, 4096, 0, 0), (300, 4096, 0, 0), (16, 4097, 15, 0), (8, 6478, 2, 0),
        (8, 8192, 0, 0), (8, 9000, 0, 0), (8, 12288, 0, 0), (8, 16384, 0, 0), (8, 20000, 0, 0), (8, 32768, 0, 0),
        (8, 32772, 0, 0), (8, 40001, 7, 1)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,gap,lead", ROWS)
def test_quant(rows, dim, gap, lead, kind):
    import torch
    x = rows_of(rows, dim, dim, kind)
    buf, view = placed(x, dim + gap, lead)
    q = torch.full((rows + 1, dim + gap), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((rows + 1,), -5.0, device="cuda")
    native.op_quant_q8(view.data_ptr(), TYPES[kind], rows, dim, q.data_ptr(), scale.data_ptr(), ld_x=dim + gap,
                       ld_q=dim + gap)
    torch.cuda.synchronize()
    check_codes(q[:rows, :dim], scale[:rows], x.float(), 1.0, 2.0 ** -24)
    assert bool((q[rows] == 99).all()) and bool((q[:, dim:] == 99).all()) and scale[rows].item() == -5.0


@pytest.mark.parametrize("x_kind,d_kind", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32"),
                                           ("f32", None), ("bf16", None)])
@pytest.mark.parametrize("rows,dim,gap,lead", ROWS)
def test_norm(rows, dim, gap, lead, x_kind, d_kind):
    import torch
    x = rows_of(rows, dim, dim + 1, x_kind)
    x = torch.where(x.abs() > 1e30, torch.ones_like(x), x)  # squares are summed in 64 bits, products with w must stay in fp32
    g = torch.Generator(device="cuda").manual_seed(3)
    delta = None
    if d_kind:
        delta = torch.randn((rows, dim), device="cuda", generator=g).to(torch_type(d_kind))
        delta[torch.arange(rows) % 8 >= 2] = 0  # those rows stay what they are
    w = 1 + 0.3 * torch.randn(dim, device="cuda", generator=g)
    w[torch.rand(dim, device="cuda", generator=g) < 0.5] = 1.0
    _, xv = placed(x, dim + gap, lead)
    if d_kind:
        _, dv = placed(delta, dim + gap, lead)
    out = torch.full((rows + 1, dim + gap), 7.0, dtype=x.dtype, device="cuda")
    q = torch.full((rows + 1, dim + gap), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((rows + 1,), -5.0, device="cuda")
    norm = native.NormQ8(dim, w.data_ptr(), 1e-6, TYPES[x_kind], TYPES[d_kind or "f32"])
    norm(xv.data_ptr(), q.data_ptr(), scale.data_ptr(), rows, delta=dv.data_ptr() if d_kind else 0,
         sum_out=out.data_ptr(), ld_x=dim + gap, ld_delta=dim + gap, ld_sum=dim + gap, ld_q=dim + gap)
    torch.cuda.synchronize()
    h = x.float() + delta.float() if d_kind else x.float()
    assert torch.equal(out[:rows, :dim], h.to(x.dtype))
    rms = 1 / torch.sqrt(h.double().square().mean(1) + 1e-6)
    check_codes(q[:rows, :dim], scale[:rows], h * w, rms, 2.0 ** -22)
    assert bool((q[rows] == 99).all()) and bool((q[:, dim:] == 99).all()) and scale[rows].item() == -5.0
    assert bool((out[rows] == 7).all()) and bool((out[:, dim:] == 7).all())


@pytest.mark.parametrize("power", [0, 100, -100])
def test_every_pair_of_bf16_significands(power):
    """A row for every significand of its largest number, holding every significand at every exponent that has a code, and
    numbers without a full significand: halves are told from what is next to them, whatever the two numbers."""
    import torch
    a = torch.arange(128, 256, dtype=torch.float64, device="cuda")
    halvings = torch.tensor([2.0 ** -j for j in range(12)], dtype=torch.float64, device="cuda")
    g = (a[:, None] * halvings).reshape(-1)
    x = torch.stack([torch.cat([b[None], torch.where(g <= b, g, torch.zeros_like(g)), -torch.where(g <= b, g, torch.zeros_like(g))])
                     for b in a]) * 2.0 ** power
    rows, dim = x.shape
    for ld in (dim, (dim + 7) // 8 * 8):  # by every number, by whole pieces
        buf = torch.zeros((rows, ld), dtype=torch.bfloat16, device="cuda")
        buf[:, :dim] = x
        assert torch.equal(buf[:, :dim].double(), x)
        q, scale = torch.zeros((rows, ld), dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
        native.op_quant_q8(buf.data_ptr(), native.DTYPE_BF16, rows, dim, q.data_ptr(), scale.data_ptr(), ld_x=ld, ld_q=ld)
        torch.cuda.synchronize()
        check_codes(q[:, :dim], scale, x.float(), 1.0, 2.0 ** -24)


@pytest.mark.parametrize("dim", [40, 4096, 40001])
def test_rows_with_nan_or_infinity_are_marked(dim):
    import torch
    x = torch.randn((6, dim), device="cuda")
    x[0, dim - 1] = math.nan
    x[2, 0] = math.inf
    x[3, dim // 2] = -math.inf
    x[4, 0], x[4, 1] = math.nan, math.inf
    w = torch.ones(dim, device="cuda")
    for norm in (False, True):
        q = torch.full((6, dim), 99, dtype=torch.int8, device="cuda")
        scale = torch.zeros(6, device="cuda")
        if norm:
            native.NormQ8(dim, w.data_ptr())(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 6)
        else:
            native.op_quant_q8(x.data_ptr(), native.DTYPE_F32, 6, dim, q.data_ptr(), scale.data_ptr())
        torch.cuda.synchronize()
        assert torch.isnan(scale).tolist() == [True, False, True, True, True, False]
        assert bool((q[torch.isnan(scale)] == 0).all())
        assert torch.equal(q[1], codes_of(x)[0][1]) and torch.equal(q[5], codes_of(x)[0][5])


def test_norm_products_that_leave_fp32_mark_their_row():
    import torch
    x = torch.full((2, 64), 1e30, device="cuda")
    x[1] = 1.0
    w = torch.ones(64, device="cuda")
    w[3] = 1e20
    q, scale = torch.zeros((2, 64), dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda")
    native.NormQ8(64, w.data_ptr())(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 2)
    torch.cuda.synchronize()
    assert math.isnan(scale[0].item()) and q[1, 3].item() == 127 and abs(scale[1].item() * 127 / 1e20 - 1) < 1e-6


def test_norm_of_numbers_whose_squares_leave_fp32():
    import torch
    x = torch.randn((4, 4096), device="cuda") * torch.tensor([[1e25], [1e-25], [1e36], [1.0]], device="cuda")
    w = torch.ones(4096, device="cuda")
    q, scale = torch.zeros((4, 4096), dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    native.NormQ8(4096, w.data_ptr(), 0.0)(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 4)
    torch.cuda.synchronize()
    check_codes(q, scale, x, 1 / torch.sqrt(x.double().square().mean(1)), 2.0 ** -22)


@pytest.mark.parametrize("dim", [64, 4096, 40001])
def test_norm_of_zeros_without_eps(dim):
    import torch
    x = torch.zeros((3, dim), device="cuda")
    x[1] = 2.0
    w = torch.ones(dim, device="cuda")
    q, scale = torch.full((3, dim), 9, dtype=torch.int8, device="cuda"), torch.full((3,), 9.0, device="cuda")
    native.NormQ8(dim, w.data_ptr(), 0.0)(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 3)
    torch.cuda.synchronize()
    assert scale[0].item() == 0 and scale[2].item() == 0 and abs(scale[1].item() * 127 - 1) < 2.0 ** -21
    assert bool((q[0] == 0).all()) and bool((q[1] == 127).all()) and bool((q[2] == 0).all())


@pytest.mark.parametrize("dim", [100, 4096, 40001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_norm_in_place(dim, kind):
    """The sum may take the stream's place or the delta's."""
    import torch
    x0, d0 = (torch.randn((30, dim), device="cuda").to(torch_type(kind)) for _ in range(2))
    w = torch.randn(dim, device="cuda")
    norm = native.NormQ8(dim, w.data_ptr(), 1e-6, TYPES[kind], TYPES[kind])
    got = []
    for where in range(3):
        x, d, s = x0.clone(), d0.clone(), torch.empty_like(x0)
        to = (s, x, d)[where]
        q, scale = torch.zeros((30, dim), dtype=torch.int8, device="cuda"), torch.zeros(30, device="cuda")
        norm(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 30, delta=d.data_ptr(), sum_out=to.data_ptr())
        torch.cuda.synchronize()
        got.append((to, q, scale))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_scale_of_codes_gives_back_the_rows():
    """code * scale is within half a step of the row: what a product with them stands for."""
    import torch
    x = torch.randn((64, 4096), device="cuda")
    q, scale = torch.zeros((64, 4096), dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda")
    native.op_quant_q8(x.data_ptr(), native.DTYPE_F32, 64, 4096, q.data_ptr(), scale.data_ptr())
    torch.cuda.synchronize()
    off = (q.double() * scale.double()[:, None] - x.double()).abs()
    # half a step, and 127 steps of a scale that is rounded once
    assert bool((off <= scale.double()[:, None] * (0.5 + 127 * 2.0 ** -24)).all())


def test_long_rows_past_32_bit_offsets():
    """Row strides whose offsets pass 2^31 elements."""
    import torch
    ld = 1 << 30
    buf = torch.zeros(2 * ld + 4096, dtype=torch.bfloat16, device="cuda")
    rows = torch.randn((3, 4096), device="cuda").to(torch.bfloat16)
    for r in range(3):
        buf[r * ld : r * ld + 4096] = rows[r]
    q, scale = torch.zeros((3, 4096), dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
    native.op_quant_q8(buf.data_ptr(), native.DTYPE_BF16, 3, 4096, q.data_ptr(), scale.data_ptr(), ld_x=ld)
    torch.cuda.synchronize()
    check_codes(q, scale, rows.float(), 1.0, 2.0 ** -24)
