"""Page-table writes keep their place among the kernels that read the table: a slot that grows, shrinks, is cleared or is
filled anew while a compaction, a fork or device steps are still queued gives the same logits, bit for bit (fp32), as
the same calls with a wait between them."""
import numpy as np
import pytest

from tests.helpers import cfg_dict, native_model

pytestmark = pytest.mark.gpu

CTX, KEPT, PAGE = 2100, 1470, 64  # 33 pages, 23 after the compaction


def _calls(m, rng, script, wait):
    """The logits of `script` on a slot 0 that holds slot 2's history, behind queued device steps on slot 1."""
    import torch
    V = m.cfg.vocab
    toks = lambda n: rng.integers(0, V, n).astype(np.int32)  # noqa: E731
    pause = m.synchronize if wait else (lambda: None)
    for s in (0, 1, 3):
        m.reset(s)
    m.fork(2, [0], CTX)
    m.reserve(1, 200)
    tok = torch.tensor([5], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0], dtype=torch.int32, device="cuda")
    slot = torch.tensor([1], dtype=torch.int32, device="cuda")
    out = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    m.synchronize()
    for _ in range(60):  # keeps the stream busy while the host goes on
        m.decode_step_device(tok.data_ptr(), slot.data_ptr(), pos.data_ptr(), 1, 0, out.data_ptr(), 1)
    keep = [p for p in range(CTX) if not 300 <= p < 300 + CTX - KEPT]
    got = []
    if script == "grow":            # into pages past those that the compaction left
        m.compact(0, keep)
        pause()
        got.append(m.extend([toks(60)], [KEPT], [0])[0])
        end = KEPT + 60
    elif script == "grow-by-step":  # 22 whole pages: the next position needs a new one
        end = KEPT - KEPT % PAGE
        m.compact(0, keep[:end])
        pause()
        got.append(m.decode_step([7], [end], [0])[0])
        end += 1
    elif script == "shrink-and-grow":
        m.compact(0, keep)
        pause()
        m.truncate(0, 640)
        pause()
        m.reserve(3, 600)           # another slot takes pages that the compaction had filled
        pause()
        got.append(m.extend([toks(30), toks(40)], [640, 0], [0, 3])[0])
        end = 670
    elif script == "clear-and-refill":
        m.compact(0, keep)
        pause()
        m.reset(0)
        pause()
        m.reserve(3, KEPT)          # the freed pages go to another slot
        pause()
        got.append(m.extend([toks(70), toks(70)], [0, 0], [0, 3])[0])
        end = 70
    else:                           # "fork-and-refill"
        m.fork(2, [3], CTX - 30)
        pause()
        m.reset(3)
        pause()
        m.reserve(0, CTX + 100)
        pause()
        got.append(m.extend([toks(70), toks(20)], [0, CTX], [3, 0])[0])
        end = CTX + 20
    got.append(m.decode_step([9], [end], [0])[0])
    m.synchronize()
    return got


@pytest.fixture(scope="module")
def model():
    c = cfg_dict(dim=256, hidden_dim=512, layers=16, heads=4, kv_heads=4, head_dim=128, vocab=500, seq_len=2304)
    m = native_model(c, None, precision="fp32", synthetic_seed=11, max_batch=4, max_tokens=64, page_size=PAGE)
    m.extend([np.random.default_rng(1).integers(0, 500, CTX).astype(np.int32)], [0], [2], want_logits=False)
    yield m
    m.close()


@pytest.mark.parametrize("script", ["grow", "grow-by-step", "shrink-and-grow", "clear-and-refill", "fork-and-refill"])
def test_table_writes_wait_for_the_kernels_that_read_the_table(model, script):
    want = _calls(model, np.random.default_rng(2), script, True)
    for _ in range(3):
        got = _calls(model, np.random.default_rng(2), script, False)
        for a, b in zip(got, want):
            assert np.array_equal(a, b)
