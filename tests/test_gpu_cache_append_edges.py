"""Appends to a paged cache at the ends of what their inputs may hold."""
from __future__ import annotations

import numpy as np
import pytest

from cache_ref import Cache
from test_gpu_cache import Append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["plain", "mxfp4"])
@pytest.mark.parametrize("dim, rot, inter", [(64, 32, False), (64, 32, True), (64, 36, False), (72, 16, False), (64, 0, False)])
def test_infinite_features_that_are_not_turned(nn, L, rng, kind, dtype, dim, rot, inter):
    """Behind rot_dim, without the norm, a feature stays what it is: in q_out and in plain pages, by pairs that lie
    whole chunks apart (32 and 16 of them) or otherwise.  In 4 bits its 32 become NaN and no others."""
    print(f"[case] infinities {kind} {dtype} {dim} {rot} {inter}", flush=True)
    t, heads, kv = 20, 3, 2
    values = {n: 1.3 * rng.standard_normal((t, h, dim)) for n, h in (("q", heads), ("k", kv), ("v", kv))}
    at = (np.arange(t) + 37) % (dim - rot) + rot  # one of a row's features
    infinite = np.where(np.arange(t) % 3 == 0, -np.inf, np.inf)
    for x in values.values():
        x[np.arange(t), :, at] = infinite[:, None]
    finite = {n: np.where(np.isfinite(x), x, 0) for n, x in values.items()}
    got = {}
    for name, v in (("infinite", values), ("finite", finite)):
        cache = Cache(nn, L, np.random.default_rng(3), kind, dtype, kv, dim, 16, [2])
        a = Append(nn, L, np.random.default_rng(4), cache, np.zeros(t, int), np.arange(t), heads, rot, interleaved=inter,
                   norm=False, values={n: x.copy() for n, x in v.items()})
        a.launch()
        L.sync()
        pool = {n: cache.download(n) for n in ("k", "v")}
        got[name] = {"q": a.t["q_out"].result()}
        for n in pool:
            got[name][n] = np.stack([cache.get(n, cache.where(0, i), pool[n]) for i in range(t)])
    for n in ("q", "k", "v"):
        want = got["finite"][n].copy()
        if kind == "mxfp4" and n != "q":
            for i in range(t):
                want[i, :, at[i] // 32 * 32:at[i] // 32 * 32 + 32] = np.nan
        else:
            want[np.arange(t), :, at] = infinite[:, None]
        assert np.array_equal(got["infinite"][n], want, equal_nan=True), n


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim, rot", [(64, 32), (64, 36), (40, 0)])
def test_signs_of_zeros_that_are_not_turned(nn, L, rng, dtype, dim, rot):
    """Every bit of a feature behind rot_dim, without the norm, is what it was."""
    x = rng.standard_normal((6, 1, dim))
    x[:, :, rot:] = np.where(rng.integers(0, 2, x[:, :, rot:].shape), -0.0, 0.0)
    cache = Cache(nn, L, rng, "plain", dtype, 1, dim, 16, [1])
    a = Append(nn, L, rng, cache, np.zeros(6, int), np.arange(6), 1, rot, norm=False, values={n: x.copy() for n in "qkv"})
    a.launch()
    L.sync()
    pool = cache.download("k")
    k = np.stack([cache.get("k", cache.where(0, i), pool) for i in range(6)])
    for got in (a.t["q_out"].result(), k):
        assert np.array_equal(np.signbit(got[:, :, rot:]), np.signbit(x[:, :, rot:])) and not got[:, :, rot:].any()
