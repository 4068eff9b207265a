"""The long-context example runs: prompt, rounds with rollbacks, evictions, rounds in the smaller cache."""
import importlib.util
import pathlib

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = pathlib.Path(__file__).resolve().parents[1] / "examples" / "long_context.py"


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_example(la, cuda, fmt):
    import torch

    spec = importlib.util.spec_from_file_location("long_context", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(prompt=1000, rounds=30, limit=520, budget=300, fmt=fmt, chunk=300)
    cache = got["cache"]
    assert got["evictions"] >= 1 and 300 <= cache.length <= 520 + 8
    assert got["position"] > 1000 + 30
    assert torch.isfinite(got["out"].float()).all()
    w = got["weights"][:, :cache.length]
    assert torch.isfinite(w).all() and (w >= 0).all() and (w.sum(dim=1) > 1).all()
