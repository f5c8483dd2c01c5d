"""Attention at the ends of its arguments' ranges: ids of documents, caps, positions, sizes of values."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_attention import TYPES, Call, case, run

pytestmark = pytest.mark.gpu


def _negative(rng, shape):
    return rng.choice([-1, -2, -3, -(2**31)], shape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["none", "causal"])
@pytest.mark.parametrize("batch, n, heads", [(2, 300, 2), (32, 130, 8)])
def test_negative_documents_of_any_number(nn, L, rng, dtype, mask, batch, n, heads):
    """Padding labelled with other numbers than -1, in blocks that also hold real documents: it is
    neither seen nor sees, whatever it holds."""
    doc = np.sort(rng.integers(0, 3, (batch, n)), axis=1)
    doc[0, n - 40:] = -2  # queries and keys of the same negative document
    pad = rng.random((batch - 1, n)) < 0.2
    doc[1:][pad] = _negative(rng, int(pad.sum()))
    other = np.where(doc < 0, _negative(rng, doc.shape), doc)
    run(nn, L, rng, case(dtype, batch, n, n, heads, heads, 16, mask, doc_q=doc, doc_k=doc), "packed")
    run(nn, L, rng, case(dtype, batch, n, n, heads, heads, 16, mask, doc_q=doc, doc_k=other), "packed")


@pytest.mark.parametrize("dtype", TYPES)
def test_negative_documents_of_few_queries(nn, L, rng, dtype):
    dk = np.sort(rng.integers(0, 3, (3, 900)), axis=1)
    pad = rng.random(dk.shape) < 0.2
    dk[pad] = _negative(rng, int(pad.sum()))
    dk[2, 100:] = -2
    dq = np.array([[2, -2], [-2, -(2**31)], [-2, 0]])
    c = case(dtype, 3, 2, 900, 8, 2, 40, "none", doc_q=dq, doc_k=dk)
    print(f"[case] few queries {c}", flush=True)
    call = Call(nn, L, rng, c, "cache", backward=False)
    call.forward()
    L.sync()
    call.compare()
