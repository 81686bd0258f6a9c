"""Several answers from one prompt over a shared paged cache: a system prompt is read once and forked into conversations
that share its pages, their turns of different lengths go through the model together, one conversation drops its oldest
turn, and pages go back as conversations end.

    python examples/shared_prefix.py            # a small random model on cuda:0

Uses the model calls qw_extend, qw_fork, qw_compact, qw_truncate and qw_decode_step (see include/qwen3_b200.h)."""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from common_b200 import native  # noqa: E402

PAGE = 64


def make_model(slots: int, seq_len: int) -> native.NativeModel:
    cfg = native.make_config(dim=1024, hidden_dim=2816, layers=4, heads=16, kv_heads=8, head_dim=128, vocab=32000,
                             seq_len=seq_len, max_batch=slots, max_tokens=1024, page_size=PAGE)
    m = native.NativeModel(cfg)
    m.init_synthetic(0, 0.02)
    m.finalize()
    return m


def main() -> dict:
    rng = np.random.default_rng(0)
    m = make_model(slots=5, seq_len=1024)
    pages = {"at the start": m.free_pages}

    # the system prompt, once
    system = rng.integers(0, 32000, 300)
    m.extend([system], start=[0], slots=[0], want_logits=False)
    pages["after the prompt"] = m.free_pages

    # four conversations on it: whole pages shared, the partly filled one copied
    users = [1, 2, 3, 4]
    m.fork(0, users, len(system))
    pages["after the forks"] = m.free_pages
    length = {u: len(system) for u in users}

    # their first turns, of different lengths, in one call; then eight tokens each
    def turn(lengths):
        toks = [rng.integers(0, 32000, n) for n in lengths]
        _, nxt = m.extend(toks, [length[u] for u in users], users, want_logits=False)
        for u, t in zip(users, toks):
            length[u] += len(t)
        said = [list() for _ in users]
        for _ in range(8):
            for s, t in zip(said, nxt):
                s.append(int(t))
            _, nxt = m.decode_step(nxt, [length[u] for u in users], users, want_logits=False)
            for u in users:
                length[u] += 1
        return said

    first = {u: length[u] for u in users}
    turn([17, 120, 64, 1])
    turn([5, 33, 1, 80])
    pages["after two turns"] = m.free_pages

    # conversation 2 drops its first turn: what stays moves down, keys turned to their new positions
    gone = range(first[2], first[2] + 128)
    m.compact(2, [p for p in range(length[2]) if p not in gone])
    length[2] -= len(gone)
    # conversation 4 takes its last answer back
    length[4] -= 8
    m.truncate(4, length[4])
    answers = turn([9, 10, 11, 12])
    pages["after compacting and a third turn"] = m.free_pages

    for u in users:
        m.reset(u)
    pages["with only the prompt held"] = m.free_pages
    m.reset()
    pages["at the end"] = m.free_pages
    m.synchronize()
    m.close()
    return {"pages": pages, "answers": answers, "lengths": length}


if __name__ == "__main__":
    r = main()
    for k, v in r["pages"].items():
        print(f"{v:4d} free pages {k}")
    for u, a in enumerate(r["answers"], 1):
        print(f"conversation {u} ({r['lengths'][u]} positions): {a}")
