"""A workspace that serves attention over tensors and over a paged cache in turn."""
from __future__ import annotations

import numpy as np
import pytest

import test_gpu_attention as plain
import test_gpu_cache_attention as paged
from test_gpu_attention import case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["plain", "mxfp4"])
def test_both_operators_in_turn(nn, L, rng, kind, dtype):
    """Few queries over tensors in parts, documents, and paged requests of more units than tickets have lines, each
    after every other one: all hold against the formulas, and the paged calls give what they give with a workspace
    of their own."""
    docs = np.sort(rng.integers(0, 5, (2, 700)), 1)
    tensors = [plain.Call(nn, L, rng, c, backward=False) for c in (
        case(dtype, 3, 2, 4000, 8, 2, 64, "causal"),
        case(dtype, 2, 700, 700, 2, 2, 32, "causal", doc_q=docs, doc_k=docs))]
    pages = [paged.Call(nn, L, rng, case(dtype, b, 1, 900, 8, 4, 32, "causal", k_len=[900 - 7 * i for i in range(b)]), kind, 64)
             for b in (40, 3)]
    size = max(x.ws.n for x in tensors + pages)
    assert min(x.ws.n for x in tensors + pages) > 1
    shared = L.to_device(np.zeros(size, np.float32))
    own = []
    for x in pages:
        x.launch()
        L.sync()
        own.append(x.compare())
    for x in tensors:
        x.ws = shared
    for t in (0, 1, 0):
        for n in (0, 1):
            print(f"[case] workspace of {size} floats: tensors {t}, pages {n}, {kind} {dtype}", flush=True)
            tensors[t].forward()
            pages[n].out.dev.fill_bytes(0xFF)
            pages[n].launch(ws=shared)
            L.sync()
            tensors[t].compare()
            got = pages[n].compare()
            assert all(np.array_equal(got[name], own[n][name]) for name in got)
