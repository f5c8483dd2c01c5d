"""Attention over a paged cache by the form for many queries (csrc/attn_fwd.h over csrc/attn_paged.h), against the 64-bit
formulas.  Every case is one that the library's choice sends there: both widths of its workgroups, every kind of pages that
it has, entries that are no page, caps, biases, more keys than are looked up at once, pools past 32 bits."""
from __future__ import annotations

import numpy as np
import pytest

from cache_ref import Cache, Tensor, ints
from test_cache_forms import is_few
from test_gpu_attention import case
from test_gpu_cache import Append
from test_gpu_cache_attention import Call

pytestmark = pytest.mark.gpu

KINDS = [("plain", "bf16"), ("plain", "f32"), ("mxfp4", "bf16")]  # fp32 queries over 4 bits take the other form always
# requests, queries, heads that share nothing: 64 queries a workgroup, and 128
NARROW, WIDE = (16, 140, 4), (64, 100, 8)


def many(kind, dtype, shape, len_k, dim, mask="causal", cap=0.0, kv=None, **more):
    batch, len_q, heads = shape
    return case(dtype, batch, len_q, len_k, heads, kv or heads, dim, mask, cap, **more)


def check_form(nn, c, kind):
    assert not is_few(nn, c["dtype"], kind, c["batch"], c["len_q"], c["len_k"], c["heads"], c["kv_heads"], c["dim"]), "the other form"
    groups = -(-c["len_q"] // 128) * c["heads"] * c["batch"]
    return "128 queries a workgroup" if groups >= 512 else "64 queries a workgroup"


def run(nn, L, rng, c, kind, page, layout="plain", scores=10.0, holes=()):
    print(f"[case] cache attention, many queries ({check_form(nn, c, kind)}), {kind} pages of {page} {layout} holes {holes} {c}", flush=True)
    call = Call(nn, L, rng, c, kind, page, layout, holes)
    call.launch()
    L.sync()
    return call.compare(scores)


def lengths(c, rng):
    """Uneven ones from a quarter of len_k on, the first whole, and every request's last queries behind them."""
    n = rng.integers(c["len_k"] // 4, c["len_k"] + 1, c["batch"])
    n[0] = c["len_k"]
    return dict(c, k_len=list(n), q_start=list(n - c["len_q"]))


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("shape", [NARROW, WIDE])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_entries_that_are_no_page(nn, L, rng, kind, dtype, shape, page, mask):
    """Quarters of a block without a page, whole blocks, the first and the last, and a request without any."""
    len_k = 320 if shape == NARROW else 192
    c = lengths(many(kind, dtype, shape, len_k, 32, mask), rng)
    c["k_len"][1:4] = [len_k, len_k - 21, 64]
    last = (len_k - 1) // page
    holes = [(0, 0), (0, last), (1, 1), (2, 0), (2, last - 1)] + [(3, p) for p in range(64 // page)]
    holes += [(int(r), int(p)) for r, p in zip(rng.integers(4, shape[0], 40), rng.integers(0, last + 1, 40))]
    got = run(nn, L, rng, c, kind, page, holes=holes)
    assert not got["out"][3].any() and np.isneginf(got["lse"][3]).all()


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("shape", [NARROW, WIDE])
@pytest.mark.parametrize("cap, buckets, scale", [(20.0, 0, 0.2), (50.0, 0, 4.0), (100.0, 0, 0.2), (0.0, 16, 0.2), (8.0, 8, 0.5)])
def test_caps_and_biases(nn, L, rng, kind, dtype, shape, cap, buckets, scale):
    """Caps with a fixed reference (up to 55) and with a running one, scores far below a cap and at it, biases with and without."""
    more = dict(buckets=buckets, max_distance=40) if buckets else {}
    c = lengths(many(kind, dtype, shape, 320 if shape == NARROW else 160, 32, "causal", cap, scale=scale, **more), rng)
    run(nn, L, rng, c, kind, 32, scores=max(10.0, cap))


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_values_that_a_fixed_reference_cannot_hold(nn, L, rng, kind, dtype):
    """First keys of score 0, later ones near a cap of 50: shares of up to 2^72 of values near 2^60 leave fp32, and the
    workgroup goes over its pages again."""
    c = many(kind, dtype, NARROW, 320, 32, "causal", 50.0, scale=4.0)
    check_form(nn, c, kind)
    call = Call(nn, L, rng, c, kind, 16)
    cache = call.cache
    for r in range(c["batch"]):
        for i, page in enumerate(cache.table[r]):
            x = {n: cache._page(n, page) for n in ("k", "v")}
            if i < 4:
                x["k"] *= 0
            cache._put_page("k", page, x["k"])
            cache._put_page("v", page, x["v"] * 2.0**60)
    cache.upload()
    call.launch()
    L.sync()
    call.compare(50.0)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("len_k, page", [(1100, 16), (1024, 64), (1025, 32), (2300, 4096)])
def test_more_keys_than_are_looked_up_at_once(nn, L, rng, kind, dtype, len_k, page):
    """1024 keys' entries are read together; a page of 4096 has more blocks than that."""
    c = lengths(many(kind, dtype, (40 if len_k < 2000 else 60, 66, 4), len_k, 16), rng)
    run(nn, L, rng, c, kind, page)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("dim, layout", [(1, "odd"), (8, "plain"), (33, "odd"), (64, "plain"), (72, "heads"), (72, "odd"),
                                         (96, "plain"), (128, "plain"), (128, "odd")])
def test_features_and_strides(nn, L, rng, kind, dtype, dim, layout):
    c = lengths(many(kind, dtype, NARROW, 200, dim), rng)
    run(nn, L, rng, c, kind, 16, layout)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("shape, kv", [((16, 140, 8), 4), ((12, 200, 12), 3), ((16, 260, 8), 1)])
def test_shared_heads(nn, L, rng, kind, dtype, shape, kv):
    c = lengths(many(kind, dtype, shape, 300, 24, kv=kv), rng)
    run(nn, L, rng, c, kind, 128)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
def test_masks(nn, L, rng, kind, dtype, mask):
    """Positions before the cache, behind it and inside; empty caches; queries that see nothing."""
    b, len_q, _ = NARROW
    c = many(kind, dtype, NARROW, 180, 48, mask, k_len=[180, 0, 1, 100, 180, 999, -3, 63] * 2,
             q_start=[40, 3, -2, 400, -500, 20, 5, -77] * 2, prefix=[0, 5, 180, 17, 0, 1000, 9, 40] * 2)
    got = run(nn, L, rng, c, kind, 16)
    for r in (1, 6):
        assert not got["out"][r].any() and np.isneginf(got["lse"][r]).all()


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_large_scores(nn, L, rng, kind, dtype):
    """Scores of a deviation of some 40: the running maximum moves, shares vanish."""
    run(nn, L, rng, lengths(many(kind, dtype, NARROW, 320, 32, scale=7.0), rng), kind, 32, scores=200.0)


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_pools_past_32_bits(nn, L, rng, kind, dtype):
    """Requests that share three pages, whose offsets need 33 bits: against the formulas, and to the bit what the same pages
    close together give."""
    heads, dim, tokens = WIDE[2], 32, 4096
    c = lengths(many(kind, dtype, WIDE, 150, dim), rng)
    check_form(nn, c, kind)
    cache = Cache(nn, L, rng, kind, dtype, heads, dim, tokens, [1, 1, 1], spare=0)
    cache.fill(rng, [150] * 3, spoil=False)
    cache.table = np.tile(cache.table, (-(-c["batch"] // 3), 1))[:c["batch"]]
    cache.table_dev = ints(L, cache.table)
    cache.args.table, cache.args.requests = cache.table_dev.p, c["batch"]
    call = Call(nn, L, rng, c, kind, tokens, cache=cache)
    call.launch()
    L.sync()
    near = call.compare()
    size = cache.block * heads
    pages = (1 << 32) // size + 3
    far = [pages - 1, pages // 2, pages - 2]
    pool = {n: L.alloc(pages * size // 4) for n in ("k", "v")}
    for n in pool:
        for i, at in enumerate(far):
            raw = np.ascontiguousarray(cache.bytes[n][i]).ravel()
            assert L.dll.nnhip_memcpy_htod(pool[n].ptr + at * size, raw.ctypes.data, raw.nbytes) == 0
    table = ints(L, np.array(far)[cache.table])
    call.cache.args = nn.NnCache(kind=cache.args.kind, page_tokens=tokens, pages=pages, requests=c["batch"], table_pages=1,
                                 table=table.p, k=pool["k"].p, v=pool["v"].p)
    call.out.dev.fill_bytes(0xFF)
    call.launch()
    L.sync()
    got = call.results()
    assert np.array_equal(got["out"], near["out"]) and np.array_equal(got["lse"], near["lse"])


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_capture(nn, L, rng, kind, dtype):
    """A chunk's append and attention in a graph, replayed with new lengths and table between eager calls."""
    b, len_q, heads = 16, 140, 4
    cache = Cache(nn, L, rng, kind, dtype, heads, 32, 16, [20] * b)
    held = rng.integers(0, 150, b)
    cache.fill(rng, held, spoil=False)
    request = np.repeat(np.arange(b), len_q)
    a = Append(nn, L, rng, cache, request, (held[:, None] + np.arange(len_q)).ravel(), heads, 32)
    c = many(kind, dtype, (b, len_q, heads), 320, 32, k_len=list(held + len_q), q_start=list(held))
    check_form(nn, c, kind)
    call = Call(nn, L, rng, c, kind, 16, cache=cache)
    stream = L.nnhip_stream_create()
    L.nnhip_graph_capture_begin(stream)
    a.launch(stream)
    call.launch(stream)
    graph = L.nnhip_graph_capture_end(stream)
    assert graph
    for step in range(3):
        now = np.minimum(held + 11 * step, 320 - len_q)
        a.place = (now[:, None] + np.arange(len_q)).ravel()
        for dev, x in ((a.keep[3], a.place), (call.keep["k_len"], now + len_q), (call.keep["q_start"], now)):
            dev.upload(np.append(x.astype(np.int32), np.int32(0)).view(np.float32))
        call.c = dict(c, k_len=list(now + len_q), q_start=list(now))
        assert L.nnhip_graph_launch(graph, stream) == 0
        assert L.nnhip_stream_synchronize(stream) == 0
        a.compare()
        replayed = call.compare()
        call.launch()
        L.sync()
        eager = call.results()
        assert np.array_equal(eager["out"], replayed["out"]) and np.array_equal(eager["lse"], replayed["lse"])
    L.nnhip_graph_destroy(graph)
    L.nnhip_stream_destroy(stream)


def test_more_requests_than_ordinary(nn, L, rng):
    """600 requests of a few keys, 128 queries a workgroup, results of their own."""
    c = many("plain", "bf16", (600, 33, 2), 40, 16, "none", k_len=list(rng.integers(0, 41, 600)))
    run(nn, L, rng, c, "plain", 16)
