"""qw_extend, qw_fork, qw_truncate and qw_compact on models: ragged turns against the oracle fed token by token (bf16
within 2e-2 relative L2 of the oracle holding the same bf16-rounded weights, fp32 within 1e-3), forks that share pages,
copies before writes to shared pages, and page accounts that add up."""
import numpy as np
import pytest

from common_b200 import native
from tests.helpers import cfg_dict, native_model, oracle_model, rel_l2, state_dict

pytestmark = pytest.mark.gpu

TOL = {"bf16": 2e-2, "fp32": 1e-3}


def _same(a, b, precision):
    """The same tokens on the same history twice: bit for bit in fp32; in bf16 the projections' split sums are added in any
    order, before roundings, so the two only agree as closely as both agree with the oracle."""
    return np.array_equal(a, b) if precision == "fp32" else rel_l2(a, b) < TOL["bf16"]


def _tokens(rng, c, n):
    return rng.integers(0, c["vocab"], n).astype(np.int32)


def _oracle_logits(o, toks):
    o.reset()
    for p, t in enumerate(toks):
        want = o.forward_token(int(t), p)
    return want


@pytest.mark.parametrize("precision,heads,kv_heads,head_dim,page,max_tokens,bias", [
    ("bf16", 8, 2, 128, 64, 0, 0),
    ("bf16", 7, 1, 64, 16, 0, 1),      # seven query heads per KV head, biases
    ("bf16", 12, 2, 128, 32, 90, 0),   # passes of 90 rows: a sequence is cut between passes
    ("bf16", 4, 4, 64, 256, 0, 0),
    ("fp32", 4, 2, 64, 64, 0, 0),      # token by token
])
def test_ragged_turns_match_the_oracle(precision, heads, kv_heads, head_dim, page, max_tokens, bias):
    c = cfg_dict(dim=512, hidden_dim=1024, heads=heads, kv_heads=kv_heads, head_dim=head_dim, seq_len=320,
                 has_qkv_bias=bias, qk_norm=0 if bias else 1)
    sd = state_dict(c, seed=70, std=0.05, norm_noise=0.1)
    rng = np.random.default_rng(71)
    m = native_model(c, sd, precision=precision, max_batch=5, max_tokens=max_tokens or 400, page_size=page)
    turns = [[_tokens(rng, c, n) for n in t] for t in ([37, 1, 130, 5], [1, 64, 3, 90], [17, 1, 1, 1])]
    slots = [4, 0, 2, 1]
    have = [np.zeros(0, np.int32)] * 4
    for turn in turns:
        lg, am = m.extend(turn, [h.size for h in have], slots)
        have = [np.concatenate([h, t]) for h, t in zip(have, turn)]
        for b in range(4):
            assert am[b] == int(np.argmax(lg[b]))
    # then one decode step on top of the extended cache
    nxt = [int(a) for a in am]
    dl, _ = m.decode_step(nxt, [h.size for h in have], slots)
    m.synchronize()
    o = oracle_model(c, sd, bf16_weights=precision == "bf16")
    for b in range(4):
        assert rel_l2(lg[b], _oracle_logits(o, have[b])) < TOL[precision], b
        assert rel_l2(dl[b], o.forward_token(nxt[b], have[b].size)) < TOL[precision], b
    o.close()
    m.close()


def test_extend_from_nothing_equals_prefill():
    c = cfg_dict(dim=512, hidden_dim=1024, heads=8, kv_heads=2, head_dim=128, seq_len=256)
    m = native_model(c, None, precision="bf16", synthetic_seed=3, max_batch=6, max_tokens=6 * 200)
    p = np.random.default_rng(5).integers(0, c["vocab"], (6, 200)).astype(np.int32)
    a, _ = m.prefill(p)
    m.reset()
    b, _ = m.extend(list(p), [0] * 6)
    m.synchronize()
    for i in range(6):  # two attention kernels with different roundings of the probabilities
        assert rel_l2(a[i], b[i]) < 1.5e-2
    m.close()


def _small(layers=2, precision="bf16", num_pages=0, page=16, max_batch=5):
    c = cfg_dict(dim=512, hidden_dim=1024, layers=layers, heads=8, kv_heads=2, head_dim=128, seq_len=256)
    sd = state_dict(c, seed=80, std=0.05)
    return c, sd, native_model(c, sd, precision=precision, max_batch=max_batch, max_tokens=256, page_size=page,
                               num_pages=num_pages)


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
@pytest.mark.parametrize("prefix", [48, 53, 7])
def test_forks_share_pages_and_go_their_own_ways(prefix, precision):
    c, sd, m = _small(precision=precision)
    rng = np.random.default_rng(81)
    total = m.free_pages
    base, x, y = _tokens(rng, c, prefix), _tokens(rng, c, 40), _tokens(rng, c, 40)
    m.extend([base], [0], [0])
    pages = -(-prefix // 16)
    assert m.free_pages == total - pages
    m.fork(0, [1, 3], prefix)
    assert m.free_pages == total - pages - (2 if prefix % 16 else 0)
    l0, _ = m.extend([x], [prefix], [0])
    l1, _ = m.extend([x], [prefix], [1])
    assert _same(l0, l1, precision)
    l3, _ = m.extend([y], [prefix], [3])
    m.synchronize()
    o = oracle_model(c, sd, bf16_weights=precision == "bf16")
    assert rel_l2(l3[0], _oracle_logits(o, np.concatenate([base, y]))) < TOL[precision]
    assert rel_l2(l1[0], _oracle_logits(o, np.concatenate([base, x]))) < TOL[precision]
    o.close()
    m.reset(0)                               # the children keep the shared pages
    d1, _ = m.decode_step([5], [prefix + 40], [1])
    m.fork(1, [0], prefix + 41)
    l0, _ = m.extend([y], [prefix + 41], [0])
    l1, _ = m.extend([y], [prefix + 41], [1])
    assert _same(l0, l1, precision)
    m.reset()
    assert m.free_pages == total
    m.close()


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_writes_to_shared_pages_copy_them_first(precision):
    c, sd, m = _small(precision=precision)
    rng = np.random.default_rng(82)
    total = m.free_pages
    base = _tokens(rng, c, 64)
    m.extend([base], [0], [0])
    m.fork(0, [1, 2], 64)
    assert m.free_pages == total - 4         # four whole pages, held three times
    before, _ = m.decode_step([9], [64], [0])
    m.truncate(0, 64)
    other = _tokens(rng, c, 30)
    m.extend([other], [10], [1])             # rewinds the child into shared pages 0..2
    m.decode_step([3], [50], [2])
    assert m.free_pages == total - 4 - 3 - 1
    m.prefill(_tokens(rng, c, 20)[None], [2])
    after, _ = m.decode_step([9], [64], [0])
    assert _same(before, after, precision)
    m.reset()
    assert m.free_pages == total
    m.close()


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_compaction_is_as_if_the_dropped_tokens_had_not_been(precision):
    """One layer: keys and values depend on their own token only, so the compacted cache is that of the kept tokens."""
    c, sd, m = _small(layers=1, precision=precision)
    rng = np.random.default_rng(83)
    total = m.free_pages
    toks = _tokens(rng, c, 150)
    for t in range(0, 150, 50):
        m.extend([toks[t : t + 50]], [t], [2])
    m.fork(2, [0], 150)
    o = oracle_model(c, sd, bf16_weights=precision == "bf16")
    for keep in ([p for p in range(150) if not 37 <= p < 90], [p for p in range(97) if p % 3 != 1], list(range(20))):
        m.compact(2, keep)
        toks = toks[keep]
        lg, _ = m.extend([[11, 12, 13]], [len(keep)], [2])
        want = _oracle_logits(o, np.concatenate([toks, [11, 12, 13]]))
        assert rel_l2(lg[0], want) < TOL[precision], len(keep)
        m.truncate(2, len(keep))
    o.close()
    assert m.free_pages == total - 2 - 10    # 20 positions, and the fork's 150 of which nothing is shared any more
    m.compact(2, [])
    m.reset(0)
    assert m.free_pages == total
    m.close()


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_compaction_leaves_the_other_holders_alone(precision):
    c, sd, m = _small(precision=precision)
    rng = np.random.default_rng(84)
    base = _tokens(rng, c, 100)
    m.extend([base], [0], [0])
    m.fork(0, [1], 100)
    before, _ = m.decode_step([9], [100], [1])
    m.compact(0, [p for p in range(100) if not 20 <= p < 50])
    m.extend([_tokens(rng, c, 60)], [70], [0])
    after, _ = m.decode_step([9], [100], [1])
    assert _same(before, after, precision)
    m.close()


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_refusals_and_exhaustion_change_nothing(precision):
    c, sd, m = _small(num_pages=9, precision=precision)
    rng = np.random.default_rng(85)
    m.extend([_tokens(rng, c, 100)], [0], [0])   # 7 of 9 pages
    before, _ = m.decode_step([9], [100], [0])
    for status, call in [
        (3, lambda: m.fork(0, [1, 2, 3], 99)),                        # three copies, two pages
        (3, lambda: m.compact(0, list(range(1, 100)))),               # seven new pages
        (3, lambda: m.extend([_tokens(rng, c, 60)], [0], [1])),
        (1, lambda: m.fork(0, [0], 10)), (1, lambda: m.fork(0, [1, 1], 10)), (1, lambda: m.fork(0, [7], 10)),
        (1, lambda: m.fork(-1, [1], 0)), (2, lambda: m.fork(0, [1], 113)),
        (1, lambda: m.compact(0, [3, 3])), (1, lambda: m.compact(0, [5, 4])), (1, lambda: m.compact(0, [-1])),
        (1, lambda: m.compact(0, [112])), (1, lambda: m.compact(9, [])), (1, lambda: m.truncate(9, 0)),
        (1, lambda: m.truncate(0, -1)),
        (2, lambda: m.extend([[]], [0], [1])), (2, lambda: m.extend([[1] * 10], [250], [0])),
        (2, lambda: m.extend([[1]], [-1], [0])), (1, lambda: m.extend([[1], [2]], [0, 0], [1, 1])),
        (1, lambda: m.extend([[c["vocab"]]], [0], [1])), (1, lambda: m.extend([[1]], [0], [8])),
        (2, lambda: m.extend([[1]] * 6, [0] * 6)), (2, lambda: m.extend([], [])), (2, lambda: m.extend([[1]], [0, 1])),
    ]:
        with pytest.raises(native.QwenError) as e:
            call()
        assert e.value.status == status, (status, str(e.value))
    assert m.free_pages >= 1
    m.truncate(0, 101)
    after, _ = m.decode_step([9], [100], [0])
    assert _same(before, after, precision)
    m.close()
