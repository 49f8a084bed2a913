"""The example that serves a small decoder from an 8-bit cache and parks the cache."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parked_cache_gives_the_same_tokens(gpu, capsys):
    spec = importlib.util.spec_from_file_location("park_cache", os.path.join(ROOT, "examples", "park_cache.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main(["--tokens", "6", "--layers", "2"]) == 0
    out = capsys.readouterr().out
    print(out)
    assert "bit for bit" in out and "the same" in out
