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
