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


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 7, 8, 16])
@pytest.mark.parametrize("window", [0, 1, 100, 129, 5000])
def test_single_rows_under_windows(d, G, window):
    """Every group size's kernel, keys split (few rows) and not (many), rows that see nothing and places without rows."""
    c = Case([1, 1, 0, 1, 2], [700, 9000, 40, 0, 64], 2 * G, 2, d, 64, window=window, dtype="fp32", seed=23)
    c.run()
    c.check()
    c = Case([1] * 300, [1 + 31 * i % 400 for i in range(300)], 2 * G, 2, d, 16, window=window, dtype="fp32", seed=24)
    c.run()
    c.check()


@pytest.mark.parametrize("seed", range(12))
def test_random_batches_fp32(seed):
    """Batches of random shapes: tiles and single rows, split and whole, empty rows and sequences, every group size."""
    import random
    rng = random.Random(100 + seed)
    for _ in range(6):
        G, kv_heads, d = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16]), rng.choice([1, 2, 4]), rng.choice([64, 128])
        B, longest = rng.choice([(1, 6000), (2, 3000), (3, 2000), (7, 900), (30, 400)])
        single = rng.random() < 0.4
        new = [1 if single else rng.choice([0, 1, 2, rng.randint(1, 40), rng.randint(1, 150)]) for _ in range(B)]
        kv = [max(0, n + rng.choice([0, -1, -5, rng.randint(0, longest), rng.randint(0, longest)])) for n in new]
        c = Case(new, kv, G * kv_heads, kv_heads, d, rng.choice([16, 64, 256]), window=rng.choice([0, 0, 1, 130, 1500]),
                 dtype="fp32", seed=seed, fused=rng.choice([0, 64]), gap=rng.choice([0, 8]))
        c.run()
        c.run()
        c.check()
