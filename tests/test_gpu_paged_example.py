"""examples/paged_decoding.py: the operators of a paged cache as a program uses them."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["NN_CACHE_PLAIN", "NN_CACHE_MXFP4"])
def test_serving_agrees_with_plain_attention(nn, L, kind):
    """fp32 sums of up to 100 terms of values up to about 5, in another order."""
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_decoding.py"
    spec = importlib.util.spec_from_file_location("paged_decoding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.serve(nn, L, getattr(nn, kind)) <= 100 * 5 * 2.0**-24
