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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("long, short", [
    (dict(len_q=3008, len_k=3008, heads=1, kv_heads=1, batch=1), dict(len_q=2944, len_k=2944)),
    (dict(len_q=1, len_k=8193, heads=8, kv_heads=8, batch=1), dict(len_k=8192)),
    (dict(len_q=900, len_k=2000, heads=8, kv_heads=2, batch=3), dict(len_q=1, len_k=1999, batch=1)),
    (dict(len_q=900, len_k=2000, heads=8, kv_heads=2, batch=3), dict(len_q=700, len_k=300, batch=1)),
])
def test_workspaces_of_longer_calls(nn, L, rng, dtype, long, short):
    """A program's workspaces have the sizes of its longest call; shorter ones write nothing past them."""
    guard = 4096
    big = case(dtype, long["batch"], long["len_q"], long["len_k"], long["heads"], long["kv_heads"], 16)
    c = case(dtype, **{**long, **short}, dim=16, mask="causal")
    print(f"[case] workspace of {big} for {c}", flush=True)
    a = nn.NnAttention(dtype=nn.NN_BF16 if dtype == "bf16" else nn.NN_F32, scale=1.0, head_dim=16,
                       **{n: long[n] for n in ("batch", "len_q", "len_k", "heads", "kv_heads")})
    call = Call(nn, L, rng, c)
    sizes = {"ws": L.nnhip_attention_forward_workspace(a), "bws": L.nnhip_attention_backward_workspace(a)}
    for name, n in sizes.items():
        assert n >= getattr(call, name).n or getattr(call, name).n == 1
        host = np.zeros(n + guard, np.float32)
        host[n:] = 7.0
        setattr(call, name, L.to_device(host))
    for _ in range(2):
        call.forward()
        call.grad()
    L.sync()
    for name, n in sizes.items():
        assert (getattr(call, name).download()[n:] == 7.0).all(), name
    call.compare()
