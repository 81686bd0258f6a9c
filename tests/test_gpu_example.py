"""examples/shared_prefix.py runs, and its page account adds up."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_shared_prefix_example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "shared_prefix.py")
    spec = importlib.util.spec_from_file_location("shared_prefix", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main()
    p = r["pages"]
    assert p["after the prompt"] == p["at the start"] - 5          # 300 positions in pages of 64
    assert p["after the forks"] == p["after the prompt"] - 4       # one copied page each
    assert p["with only the prompt held"] == p["after the prompt"] and p["at the end"] == p["at the start"]
    assert all(len(a) == 8 for a in r["answers"])
