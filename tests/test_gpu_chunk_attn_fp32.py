"""The fp32 kernels of qw_op_chunk_attn: tiles and single rows, keys split over the GPU and not, windows, every group
size, lengths out of range.  References and tolerances are those of test_gpu_chunk_attn.py."""
import pytest

from tests.test_gpu_chunk_attn import Case

pytestmark = pytest.mark.gpu


def _repeats(c, times):
    """`times` calls give the same out and lse, bit for bit."""
    import torch
    c.run()
    c.check()
    out, lse = c.obuf.clone(), c.lse.clone()
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(times):
        c.obuf.fill_(-7.0)
        c.lse.fill_(-7.0)
        c.run()
        differ += (c.obuf != out).sum() + (c.lse != lse).sum()
    assert int(differ.item()) == 0


@pytest.mark.parametrize("new,kv,heads,kv_heads,d", [([16], [4000], 8, 2, 128), ([9, 16], [3000, 2500], 4, 1, 64),
                                                     ([60], [6000], 2, 2, 128)])
def test_tiles_whose_keys_are_split_repeat_bit_for_bit(new, kv, heads, kv_heads, d):
    """Many rows a sequence and few tiles: the last CTA of a tile joins its ranges of keys."""
    _repeats(Case(new, kv, heads, kv_heads, d, 64, dtype="fp32", seed=21), 300)


@pytest.mark.parametrize("batch,heads,kv_heads,d", [(200, 16, 8, 128), (320, 6, 2, 64), (8, 8, 2, 128)])
def test_single_rows_repeat_bit_for_bit(batch, heads, kv_heads, d):
    """One row a sequence: rows enough to fill the GPU, whose keys one CTA takes, and few, whose keys are split."""
    _repeats(Case([1] * batch, [1 + 37 * i % 700 for i in range(batch)], heads, kv_heads, d, 64, dtype="fp32", seed=22), 100)
