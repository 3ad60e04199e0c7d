"""The example that trains an encoder and searches with it (needs an MI355X)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "cuda-vector-search_amd" / "examples" / "train_encoder.py"


def test_example_learns_to_find_documents(eng):
    spec = importlib.util.spec_from_file_location("train_encoder", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    before, after = mod.main(["--steps", "200"])
    # ten of 1024 by chance is 0.01; a trained encoder finds most
    assert after > before + 0.2 and after > 0.5
