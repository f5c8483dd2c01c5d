"""examples/attention_block.py: the attention operators as a program uses them."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "attention_block.py"
    spec = importlib.util.spec_from_file_location("attention_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_training_lowers_the_loss(nn, L, example):
    losses = example.train(nn, L, 20)
    assert all(b < a for a, b in zip(losses, losses[1:])) and losses[-1] < 0.9 * losses[0], losses


def test_decoding_agrees_with_the_whole(nn, L, example):
    """fp32 sums of up to 100 terms of values up to about 5, in another order."""
    assert example.decode(nn, L) <= 100 * 5 * 2.0**-24
