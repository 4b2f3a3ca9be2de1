"""The dense retrieval example: quantised scores, distributions and a training loop together.

8 bits leave each product off by about 0.001 of vectors of length 1, so the exact nearest row stays among
the ten best unless ten others lie within that of it; the contrastive loss falls when its gradient is right.
"""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "quiver-ae_amd" / "examples" / "dense_retrieval.py"


def test_example():
    from quiver import _lib

    if _lib.device_count() == 0:
        pytest.skip("no GPU")
    print("[gpu] dense retrieval example", flush=True)
    spec = importlib.util.spec_from_file_location("dense_retrieval", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(rows=20_000, queries=256, steps=15)
    assert r["recall"] > 0.98
    assert 0 <= r["entropy"] < 9.91  # ln 20,000
    assert r["losses"][-1] < 0.7 * r["losses"][0]
    torch.cuda.empty_cache()
