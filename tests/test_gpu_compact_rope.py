"""qw_compact with a RoPE table of the checkpoint's own: tables whose angles grow evenly with the position move keys (one
layer: as if the dropped tokens had not been, within 1e-3 of the oracle in fp32), others are refused and nothing changes."""
import numpy as np
import pytest

from common_b200 import native
from tests.helpers import cfg_dict, native_model, oracle_model, rel_l2, state_dict

pytestmark = pytest.mark.gpu

SEQ, HEAD = 512, 64


def _angles(pos, theta=1e4):
    return np.outer(pos, theta ** (-np.arange(0, HEAD, 2) / HEAD))


def _table(ang, scale=1.0):
    return (scale * np.stack([np.cos(ang), np.sin(ang)], -1)).astype(np.float32)


def _bf16(x):
    u = x.view(np.uint32)
    return ((u + 0x7FFF + (u >> 16 & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def _fp32_angles():
    inv = (1e4 ** (-np.arange(0, HEAD, 2, dtype=np.float32) / HEAD)).astype(np.float32)
    return np.outer(np.arange(SEQ, dtype=np.float32), inv)


def _model(table):
    c = cfg_dict(dim=256, hidden_dim=512, layers=1, heads=4, kv_heads=2, head_dim=HEAD, seq_len=SEQ, rope_theta=1e4)
    sd = state_dict(c, seed=90, std=0.05)
    if table is not None:
        sd["rope.freq_cis"] = table
    return c, sd, native_model(c, sd, precision="fp32", max_batch=2, page_size=16)


P = np.arange(SEQ)


@pytest.mark.parametrize("table,tol", [
    (None, 1e-3), (_table(_fp32_angles()), 1e-3),
    (_table(_angles(P / 4.0, 5e5)), 1e-3),          # positions interpolated by four
    (_bf16(_table(_angles(P))), 3e-2),              # a table stored in bf16: its own entries are off by 2^-9
], ids=["computed", "float", "interpolated", "bf16"])
def test_even_tables_move_keys(table, tol):
    c, sd, m = _model(table)
    rng = np.random.default_rng(91)
    toks = rng.integers(0, c["vocab"], 120).astype(np.int32)
    m.extend([toks], [0], [1])
    keep = [p for p in range(120) if not 30 <= p < 75]
    m.compact(1, keep)
    lg, _ = m.extend([[11, 12, 13]], [len(keep)], [1])
    m.synchronize()
    o = oracle_model(c, sd)
    for p, t in enumerate([*toks[keep], 11, 12, 13]):
        want = o.forward_token(int(t), p)
    assert rel_l2(lg[0], want) < tol
    o.close()
    m.close()


@pytest.mark.parametrize("table", [
    _table(_angles(P), 1.1),                                   # off the unit circle
    _table(_angles(P ** 0.97)), _table(_angles(P + 1)),        # not even; row 0 is no angle of no distance
    _table(np.where(P[:, None] < 300, _angles(P), _angles(300 + (P - 300) * 0.25))),   # bent at 300
    np.where(np.arange(SEQ)[:, None, None] == 400, np.float32("nan"), _table(_angles(P))),
], ids=["scaled", "power", "shifted", "bent", "nan"])
def test_other_tables_are_refused(table):
    c, sd, m = _model(table)
    toks = np.random.default_rng(92).integers(0, c["vocab"], 120).astype(np.int32)
    m.extend([toks], [0], [1])
    before, _ = m.decode_step([9], [120], [1])
    free = m.free_pages
    with pytest.raises(native.QwenError) as e:
        m.compact(1, list(range(1, 120)))
    assert e.value.status == 8 and "rope.freq_cis" in str(e.value)
    assert m.free_pages == free
    after, _ = m.decode_step([9], [120], [1])
    assert np.array_equal(before, after)
    m.compact(1, list(range(40)))                              # the first positions stay where they are
    assert m.free_pages == free + 5
    m.load_tensor("rope.freq_cis", _table(_angles(P)))         # another table
    m.finalize()
    m.compact(1, list(range(3, 40)))
    m.close()
