"""Scales of the normalised rows' codes (qw_op_norm_q8) where 1 / rms, or its product with the row's largest number, is outside
fp32's normal range and the scale is not.  A scale is computed in 64 bits and rounded once: 2^-24 of it, and below the normal
range half of 2^-149; sums of up to 40001 squares in 64 bits add less than 2^-36."""
import math

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu


def scales(x, w, eps=0.0):
    import torch
    rows, dim = x.shape
    q, scale = torch.zeros((rows, dim), dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    native.NormQ8(dim, w.data_ptr(), eps)(x.data_ptr(), q.data_ptr(), scale.data_ptr(), rows)
    torch.cuda.synchronize()
    g = (x * w).double()
    top = g.abs().amax(1)
    assert torch.equal(q, torch.round(127 * g / top[:, None]).to(torch.int8))
    want = top / 127 / torch.sqrt(x.double().square().mean(1) + eps)
    assert bool((want > 0).all()) and bool((want < 3.4e38).all())
    off = (scale.double() - want).abs()
    assert bool((off <= 2.0 ** -24 * (1 + 2.0 ** -12) * want + 2.0 ** -150).all()), (scale, want)


def normal(rows, dim, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((rows, dim), device="cuda", generator=g).clamp_(-3, 3)


@pytest.mark.parametrize("dim", [64, 100, 4096, 40001])
def test_rows_below_the_normal_range(dim):
    """1 / rms is beyond fp32; the weights bring the products back."""
    scales(normal(9, dim, 1) * 1e-39, 1e5 + normal(1, dim, 2)[0])


@pytest.mark.parametrize("dim", [64, 100, 4096, 40001])
def test_rows_near_the_largest_number(dim):
    """1 / rms is below fp32's normal range."""
    scales(normal(9, dim, 3) * 1.1e38, 1 + 0.01 * normal(1, dim, 4)[0])


@pytest.mark.parametrize("dim", [64, 100, 4096, 40001])
def test_largest_number_times_a_factor_beyond_fp32(dim):
    """A row of a single number, whose factor is the root of its width, under large weights."""
    import torch
    x = torch.zeros((5, dim), device="cuda")
    x[torch.arange(5), torch.arange(5) * 7] = torch.tensor([1.0, -2.0, 1e-3, 5.0, 0.1], device="cuda")
    scales(x, torch.full((dim,), 1e38, device="cuda") / torch.tensor([1.0, 3.0], device="cuda").repeat(dim // 2 + 1)[:dim])


def test_scales_below_the_normal_range():
    """Small weights under large rows: what is left of the scale is rounded once."""
    scales(normal(9, 4096, 5) * 1e30, 1e-37 * (2 + 0.1 * normal(1, 4096, 6)[0]))


@pytest.mark.parametrize("dim", [64, 4096, 40001])
def test_ordinary_rows(dim):
    scales(normal(300, dim, 7), 1 + 0.2 * normal(1, dim, 8)[0], 1e-6)


def test_marks_are_kept():
    import torch
    x = normal(4, 4096, 9)
    x[0] = 0
    x[1, 5] = math.nan
    x[2, 4095] = math.inf
    w = torch.ones(4096, device="cuda")
    for eps in (0.0, 1e-6):
        q, scale = torch.full((4, 4096), 9, dtype=torch.int8, device="cuda"), torch.full((4,), 9.0, device="cuda")
        native.NormQ8(4096, w.data_ptr(), eps)(x.data_ptr(), q.data_ptr(), scale.data_ptr(), 4)
        torch.cuda.synchronize()
        assert scale[0].item() == 0 and torch.isnan(scale).tolist() == [False, True, True, False]
        assert int(q[:3].count_nonzero()) == 0
