"""A query row of NaN gives NaN, not the zeros of a row that sees nothing, however the row's keys are split and joined;
the other rows stay right.  References and tolerances are those of test_gpu_chunk_attn.py."""
import pytest

from tests.test_gpu_chunk_attn import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new,kv,heads,kv_heads,window,bad", [
    ([1, 1], [300, 90], 16, 8, 0, 0),              # keys in one CTA
    ([1], [9001], 32, 8, 0, 0),                    # one token over the whole GPU
    ([3, 1], [20000, 15000], 8, 1, 0, 2),
    ([16], [4000], 8, 2, 0, 7),                    # fp32: a tile whose keys are split
    ([60], [2900], 32, 8, 0, 59),                  # a chunk in several shares
    ([600], [2900], 32, 8, 0, 333),
    ([5, 200], [700, 260], 16, 8, 130, 100),
    ([1] * 200, [500] * 200, 16, 8, 0, 150),       # fp32: rows that fill the GPU
])
def test_a_row_of_nan_gives_nan(dtype, new, kv, heads, kv_heads, window, bad):
    import torch
    c = Case(new, kv, heads, kv_heads, 128, 64, window=window, dtype=dtype, seed=41)
    clean = c.q[bad].clone()
    c.q[bad] = float("nan")
    c.run()
    torch.cuda.synchronize()
    assert bool(c.obuf[bad].isnan().all()) and bool(c.lse[bad].isnan().all())
    got, lse = c.obuf.clone(), c.lse.clone()
    c.q[bad] = clean
    c.run()
    c.check()                                      # the workspace is as it was
    others = [r for r in range(c.rows) if r != bad]
    assert torch.equal(got[others], c.obuf[others]) and torch.equal(lse[others], c.lse[others])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new,kv", [([1], [9001]), ([16], [4000])])
def test_keys_of_nan_reach_the_rows_that_see_them(dtype, new, kv):
    """A stretch of keys of NaN that is a whole part of a split row's keys."""
    import torch
    c = Case(new, kv, 8, 2, 128, 64, dtype=dtype, seed=42)
    c.k[c.table[1, 10:30].long()] = float("nan")
    c.run()
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0 and bool(c.obuf.isnan().all()) and bool(c.lse.isnan().all())
