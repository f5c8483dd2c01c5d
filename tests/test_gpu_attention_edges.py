"""Attention at the ends of its arguments' ranges: ids of documents, caps, positions, sizes of values."""
from __future__ import annotations

import numpy as np
import pytest

from attention_ref import Tensor, check, ints
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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch, heads", [(1, 1), (64, 8)])
@pytest.mark.parametrize("scale, cap", [(1.0, 5e-5), (1.0, 1e-3), (100.0, 0.01), (1e-3, 50.0), (1e-4, 50.0), (1e-5, 30.0),
                                        (1e-6, 1.0), (0.125, 5e3), (0.1, 1e4), (0.125, 30.0), (1.0, 50.0)])
def test_caps_of_any_size(nn, L, dtype, batch, heads, scale, cap):
    """One key of 128 has a score of y caps before the tanh, the others 0, the same for all queries of a call, so
    that each of the forms of the cap is met by itself; workgroups of 64 rows and of 128.

    The capped score x is off by up to 20 u of itself (c1 2 u, the product 1, tanh 10, c2 2, its product 1, the
    reference 2), a log-sum by that and 12 u of its own; a probability by twice that and 32 u, a gradient by two
    of them and its slope, whose exponential's argument is up to 30."""
    u, n, dim = 2.0**-24, 128, 8
    scale, cap = float(np.float32(scale)), float(np.float32(cap))
    t = nn.NN_BF16 if dtype == "bf16" else nn.NN_F32
    for y in (0.0, 1e-6, 1e-3, 0.1, 0.139, 0.141, 0.3, 0.37, 0.374, 0.376, 0.5, 1.0, 3.0, 10.0, -1e-3, -0.1, -0.139, -0.3,
              -0.37, -0.376, -1.0, -10.0):
        print(f"[case] cap {dtype} {batch} {heads} {scale} {cap} {y}", flush=True)
        shape = (batch, n, heads, dim)
        q, k, v = np.zeros(shape, np.float32), np.zeros(shape, np.float32), np.zeros(shape, np.float32)
        q[..., 0] = y * cap / scale
        k[:, 100, :, 0] = 1.0
        v[:, 100] = 1.0
        x = {m: Tensor(L, shape, dtype, values=val) for m, val in
             (("q", q), ("k", k), ("v", v), ("dout", np.ones(shape)), ("out", 0), ("dq", 0), ("dk", 0), ("dv", 0))}
        lse = L.alloc(batch * heads * n)
        strides = x["q"].strides[:3]
        a = nn.NnAttention(dtype=t, batch=batch, len_q=n, len_k=n, heads=heads, kv_heads=heads, head_dim=dim, scale=scale,
                           softcap=cap, q_stride=strides, k_stride=strides, v_stride=strides, out_stride=strides)
        ws = L.to_device(np.zeros(max(1, L.nnhip_attention_forward_workspace(a)), np.float32))
        bws = L.alloc(max(1, L.nnhip_attention_backward_workspace(a)))
        L.launch_attention_forward(x["out"].p, lse.p, x["q"].p, x["k"].p, x["v"].p, a, ws.p, None)
        L.launch_attention_backward(x["dq"].p, x["dk"].p, x["dv"].p, None, x["dout"].p, x["q"].p, x["k"].p, x["v"].p,
                                    x["out"].p, lse.p, a, bws.p, None)
        L.sync()
        raw = x["q"].values()[0, 0, 0, 0]
        tanh = np.tanh(raw * scale / cap)
        score = tanh * cap
        own = np.logaddexp(np.log(n - 1), score)
        p = np.exp(score - own)
        grad = scale / np.cosh(raw * scale / cap) ** 2 * p * np.exp(np.log(n - 1) - own) * dim
        want = {"out": (p, 32 * abs(score) + 32), "dq": (grad, 64 * abs(score) + 128), "dv": (n * p, 32 * abs(score) + 64)}
        got = lse.download().astype(np.float64)
        assert (abs(got - own) <= 32 * u * (abs(score) + abs(own) + 1)).all(), (y, "lse", abs(got - own).max())
        for m, (ref, bound) in want.items():
            got = x[m].result()
            got = got[..., 0] if m == "dq" else got[:, 100] if m == "dv" else got
            assert np.isfinite(got).all(), (y, m)
            if score > 0 and m == "dq":
                continue  # 1 - p cancels: the size of dq is that of its terms, not its own
            # bf16: the probability or score gradient, and the result
            off = abs(got - ref)
            limit = (bound * u + (2 * 2.0**-8 if dtype == "bf16" else 0)) * abs(ref) + 2.0**-120
            assert (off <= limit).all(), (y, m, float((off / limit).max()))
        assert np.isfinite(x["dk"].result()).all(), y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale, cap", [(1.0, 5e-5), (1e-5, 30.0), (0.125, 30.0)])
@pytest.mark.parametrize("part", [0.1, 0.3, 1.0])
def test_caps_of_any_size_with_a_bias(nn, L, rng, dtype, scale, cap, part):
    """Scores of about `part` of the cap, a seventh of the queries with scores of exactly 0."""
    c = case(dtype, 2, 130, 130, 2, 2, 16, cap=cap, scale=scale, buckets=4, max_distance=9)
    print(f"[case] capped {part} {c}", flush=True)
    call = Call(nn, L, rng, c, spoil=False)
    q = call.t["q"]
    view = q.view(q.host)
    view *= part * cap / scale / c["dim"] ** 0.5
    view[:, ::7] = 0
    q.upload()
    call.forward()
    call.grad()
    L.sync()
    call.compare(scores=max(10.0, min(1.0, 4 * part) * cap))


def test_positions_past_2_to_the_29(nn, L):
    """A query past the end of a cache of 2^29 + 100 keys (one row, at strides of 0): every key lies more than
    max_distance before it, none in the buckets of the near ones."""
    n, m = (1 << 29) + 100, 300
    print("[case] positions past 2^29", flush=True)
    ones = L.to_device(np.ones(8, np.float32))
    out, lse = L.alloc(8), L.alloc(2)
    bias, bucket = L.to_device(np.array([[0.0], [60.0]], np.float32)), ints(L, np.arange(2 * m + 1) > 0)
    start = ints(L, [(1 << 29) + 500])
    a = nn.NnAttention(dtype=nn.NN_F32, batch=1, len_q=1, len_k=n, heads=1, kv_heads=1, head_dim=8, scale=0.125,
                       mask=nn.NN_MASK_CAUSAL, buckets=2, max_distance=m, q_stride=(8, 8, 8), k_stride=(0, 0, 0),
                       v_stride=(0, 0, 0), out_stride=(8, 8, 8), q_start=start.p, bucket=bucket.p, bias=bias.p)
    ws = L.to_device(np.zeros(max(1, L.nnhip_attention_forward_workspace(a)), np.float32))
    L.launch_attention_forward(out.p, lse.p, ones.p, ones.p, ones.p, a, ws.p, None)
    L.sync()
    # 2^29 equal terms in fp32 sums of up to 2^19 each: 2^-5 at worst, far from the bias of 60
    assert abs(lse.download()[0] - (1.0 + np.log(n))) < 0.05
    assert np.allclose(out.download(), 1.0, rtol=0.05)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("len_q", [3, 150])
def test_starts_at_the_ends_of_the_type(nn, L, rng, dtype, mask, len_q):
    """Queries far before the keys see none of them unless a prefix or no mask shows them; far behind, all."""
    starts = [-(2**31), -(2**30) - 7, -len_q - 40, 2**29 + 1, 2**30, 2**31 - 1 - len_q, 233, 260]
    run(nn, L, rng, case(dtype, len(starts), len_q, 230, 2, 2, 16, mask, buckets=7, max_distance=30, q_start=starts,
                         prefix=[100] * len(starts)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2.0**100, 2.0**-100])
@pytest.mark.parametrize("len_q, batch, heads", [(100, 1, 2), (130, 32, 8), (3, 1, 2)])
@pytest.mark.parametrize("low, high", [(-200.0, 200.0), (-15.0, 15.0), (-200.0, -200.0), (15.0, -15.0)])
def test_values_of_any_size_under_a_cap(nn, L, rng, dtype, size, len_q, batch, heads, low, high):
    """Values near the ends of the type: probabilities that are formed from a fixed reference may not
    carry their products past them.  The first 64 keys' scores are about `low`, the later ones' `high`."""
    c = case(dtype, batch, len_q, 200, heads, heads, 16, cap=50.0, scale=1.0)
    print(f"[case] values of {size} {low} {high} {c}", flush=True)
    call = Call(nn, L, rng, c, backward=False, spoil=False)
    for n in "qkv":
        x = call.t[n]
        view = x.view(x.host)
        if n == "q":
            view[...] = 1.0
        if n == "k":
            view *= 0.01
            view[:, :64] += low / 16
            view[:, 64:] += high / 16
        if n == "v":
            view *= size
        x.upload()
    call.forward()
    L.sync()
    got, (ref, mag) = call.results(), call.expected()
    check("out", got["out"] / size, ref["out"] / size, mag["out"] / size, dtype, scores=50.0)
    check("lse", got["lse"], ref["lse"], mag["lse"], "f32", scores=50.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, distance", [(8, 1, 500), (4, 1, 1023), (8, 2, 1023), (4, 1, 511), (4, 1, 512), (1, 1, 1023)])
def test_bias_of_few_queries_by_any_distance(nn, L, rng, dtype, heads, kv, distance):
    """Tables of the bias that fit in LDS (16 KB: 4 heads of 511 distances) and that do not; keys within
    max_distance, past it, and after the query."""
    c = case(dtype, 2, 2, 3001, heads, kv, 40, "prefix", buckets=32, max_distance=distance, prefix=[3001, 100],
             q_start=[1500, 2999], k_len=[3001, 2990])
    print(f"[case] few queries {c}", flush=True)
    call = Call(nn, L, rng, c, "cache", backward=False)
    call.forward()
    L.sync()
    call.compare()
