"""Rows to 8-bit codes, with and without the norm, for more than 296 rows, where a lane holds many numbers and a CTA several rows: what
test_gpu_q8_rows.py asks of fewer, with its definition and tolerances."""
import pytest

from tests import test_gpu_q8_rows as few

pytestmark = pytest.mark.gpu

# (rows, dim, gap, lead): a warp, two, four, eight and sixteen of them a row; widths that end inside a piece, a lane's share, a warp's;
# numbers of rows that leave a CTA part empty; rows off alignment
MANY = [(1001, 1, 7, 0), (997, 5, 3, 0), (513, 31, 1, 0), (511, 64, 0, 0), (403, 100, 4, 0), (401, 250, 6, 0), (299, 257, 7, 0),
        (301, 500, 4, 0), (297, 520, 0, 0), (299, 896, 0, 0), (301, 1000, 0, 0), (298, 1025, 7, 0), (300, 1536, 0, 0), (299, 2040, 8, 0),
        (298, 2048, 0, 0), (301, 2056, 0, 0), (299, 3584, 0, 0), (298, 4095, 1, 0), (299, 4095, 0, 0), (301, 4100, 4, 1), (299, 5120, 0, 0),
        (298, 6144, 0, 0), (301, 8184, 0, 0), (299, 8200, 0, 0), (298, 9728, 0, 0), (297, 12288, 0, 0), (299, 16380, 4, 0), (298, 16384, 0, 0),
        (297, 16392, 0, 0), (299, 25600, 0, 0), (297, 32767, 1, 0)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,gap,lead", MANY)
def test_quant(rows, dim, gap, lead, kind):
    few.test_quant(rows, dim, gap, lead, kind)


@pytest.mark.parametrize("x_kind,d_kind", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", None), ("bf16", None)])
@pytest.mark.parametrize("rows,dim,gap,lead", MANY)
def test_norm(rows, dim, gap, lead, x_kind, d_kind):
    few.test_norm(rows, dim, gap, lead, x_kind, d_kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 896, 4096, 12288])
def test_norm_in_place(dim, kind):
    """The sum in the stream's place or the delta's, for 600 rows."""
    import torch
    from common_b200 import native
    x0, d0 = (torch.randn((600, dim), device="cuda").to(few.torch_type(kind)) for _ in range(2))
    w = torch.randn(dim, device="cuda")
    norm = native.NormQ8(dim, w.data_ptr(), 1e-6, few.TYPES[kind], few.TYPES[kind])
    got = []
    for where in range(3):
        x, d, s = x0.clone(), d0.clone(), torch.empty_like(x0)
        to = (s, x, d)[where]
        q, scale = torch.zeros((600, dim), dtype=torch.int8, device="cuda"), torch.zeros(600, device="cuda")
        norm(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 600, delta=d.data_ptr(), sum_out=to.data_ptr())
        torch.cuda.synchronize()
        got.append((to, q, scale))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    h = x0.float() + d0.float()
    assert torch.equal(got[0][0], h.to(x0.dtype)) and torch.equal(got[0][1], few.codes_of(h * w)[0])


def test_rows_do_not_depend_on_their_batch():
    """A row's codes, scale and sum are the same bits among few rows and many, but for the order of the sum of squares in 64 bits."""
    import torch
    from common_b200 import native
    for dim in (896, 4096, 12288):
        x, d = torch.randn((700, dim), device="cuda"), torch.randn((700, dim), device="cuda").to(torch.bfloat16)
        w = 1 + 0.2 * torch.randn(dim, device="cuda")
        norm = native.NormQ8(dim, w.data_ptr(), 1e-6, native.DTYPE_F32, native.DTYPE_BF16)
        got = []
        for n in (1, 64, 700):
            q, s, h = torch.zeros((n, dim), dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros((n, dim), device="cuda")
            norm(x.data_ptr(), q.data_ptr(), s.data_ptr(), n, delta=d.data_ptr(), sum_out=h.data_ptr())
            torch.cuda.synchronize()
            got.append((q, s, h))
        for q, s, h in got[:2]:
            n = len(s)
            assert torch.equal(q, got[2][0][:n]) and torch.equal(h, got[2][2][:n])
            assert bool(((s - got[2][1][:n]).abs() <= 2.0 ** -23 * s).all())
