"""Attention over a paged cache through the C-ABI against the 64-bit formulas: types, kinds of pages, head layouts,
lengths, masks, strides, tables with entries that are no page, and what slots that nothing sees may hold."""
from __future__ import annotations

import numpy as np
import pytest

from attention_ref import attention, check
from cache_ref import Cache, Tensor, ints
from test_gpu_attention import bias_of, case
from test_gpu_cache import KINDS, Append

pytestmark = pytest.mark.gpu


class Call:
    """A case's cache, queries and launches, and its 64-bit results."""

    def __init__(self, nn, L, rng, c, kind, page, layout="plain", holes=(), cache=None, most=None):
        self.nn, self.L, self.c = nn, L, c
        b, lq, lk, h, kv, d, t = (c[n] for n in ("batch", "len_q", "len_k", "heads", "kv_heads", "dim", "dtype"))
        lengths = np.clip(c.get("k_len", [lk] * b), 0, lk)
        if cache is None:
            cache = Cache(nn, L, rng, kind, t, kv, d, page, [-(-int(n) // page) for n in lengths] or [0], width=max(1, -(-lk // page)))
            cache.fill(rng, lengths)
            for r, p in holes:
                cache.table[r, p] = rng.choice([-1, -9, cache.pages, 2**31 - 1])
            if holes:
                cache.table_dev = ints(L, cache.table)
                cache.args.table = cache.table_dev.p
        self.cache = cache
        stride, offset = {"plain": (None, 0), "odd": ((lq * (h * (d + 1) + 1) + 3, h * (d + 1) + 1, d + 1, 1), 1),
                          "heads": ((lq * h * d, d, lq * d, 1), 0)}[layout]
        self.q = Tensor(L, (b, lq, h, d), t, stride, offset, values=rng.standard_normal((b, lq, h, d)).astype(np.float32))
        self.out = Tensor(L, (b, lq, h, d), t, stride, offset)
        self.lse = L.alloc(max(1, b * h * lq))
        self.lse.fill_bytes(0xFF)
        self.bias, self.bucket = bias_of(c, rng)
        self.keep = {n: ints(L, c[n]) for n in ("q_start", "k_len", "prefix") if n in c}
        if self.bias is not None:
            self.keep["bias"], self.keep["bucket"] = L.to_device(self.bias), ints(L, self.bucket)
        self.args = nn.NnAttention(
            dtype=nn.NN_BF16 if t == "bf16" else nn.NN_F32, batch=b, len_q=lq, len_k=lk, heads=h, kv_heads=kv,
            head_dim=d, scale=c["scale"], softcap=c["cap"],
            mask={"none": nn.NN_MASK_NONE, "causal": nn.NN_MASK_CAUSAL, "prefix": nn.NN_MASK_PREFIX}[c["mask"]],
            buckets=c.get("buckets", 0), max_distance=c.get("max_distance", 0), q_stride=self.q.strides[:3],
            out_stride=self.out.strides[:3], **{n: x.p for n, x in self.keep.items()})
        self.ws = L.to_device(np.zeros(max(1, L.nnhip_cache_attention_workspace(self.args, cache.args)), np.float32))

    def launch(self, stream=None, ws=None):
        self.L.launch_cache_attention_forward(self.out.p, self.lse.p, self.q.p, self.args, self.cache.args,
                                              (ws or self.ws).p, stream)

    def results(self):
        c = self.c
        shape = (c["batch"], c["heads"], c["len_q"])
        return {"out": self.out.result(), "lse": self.lse.download(int(np.prod(shape)), shape).astype(np.float64)}

    def expected(self):
        c = dict(self.c)
        b, lk = c["batch"], c["len_k"]
        x = {n: np.zeros((b, lk, c["kv_heads"], c["dim"])) for n in ("k", "v")}
        c["doc_q"], c["doc_k"] = np.zeros((b, c["len_q"]), int), np.full((b, lk), -1)
        for r in range(b):
            n = int(np.clip(c.get("k_len", [lk] * b)[r], 0, lk))
            for name in x:
                x[name][r, :n], held = self.cache.rows(name, r, n)
            c["doc_k"][r, :n][held] = 0  # a key of no page is in no document
        return attention(c, self.q.values(), x["k"], x["v"], bias=None if self.bias is None else self.bias.astype(np.float64),
                         bucket=self.bucket)

    def compare(self, scores=10.0):
        got, (ref, mag) = self.results(), self.expected()
        for n in ("out", "lse"):
            check(n, got[n], ref[n], mag[n], "f32" if n == "lse" else self.c["dtype"], scores)
        return got


def run(nn, L, rng, c, kind, page, layout="plain", scores=10.0, holes=()):
    print(f"[case] cache attention {kind} pages of {page} {layout} holes {holes} {c}", flush=True)
    call = Call(nn, L, rng, c, kind, page, layout, holes)
    call.launch()
    L.sync()
    return call.compare(scores)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (4, 4, 64), (3, 1, 72), (32, 2, 32), (5, 5, 1), (6, 3, 33), (2, 2, 96),
                                            (7, 1, 100), (64, 1, 40), (16, 1, 8)])
def test_heads(nn, L, rng, kind, dtype, heads, kv, dim):
    """A decoding step of two requests, every head layout."""
    c = case(dtype, 2, 1, 203, heads, kv, dim, "causal", k_len=[203, 77], q_start=[202, 76])
    run(nn, L, rng, c, kind, 16)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("len_q, len_k", [(1, 1), (1, 15), (1, 16), (1, 17), (1, 64), (1, 1025), (2, 2), (3, 33), (5, 129),
                                          (16, 40), (17, 17), (33, 300), (64, 64), (65, 200), (130, 131), (200, 100), (257, 512)])
def test_lengths(nn, L, rng, kind, dtype, len_q, len_k):
    c = case(dtype, 2, len_q, len_k, 4, 2, 64, "causal", k_len=[len_k, max(1, len_k // 2)])
    run(nn, L, rng, c, kind, 32)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("len_q", [1, 6, 150])
def test_masks(nn, L, rng, kind, dtype, mask, len_q):
    """Positions before the cache, behind it and inside; empty caches; queries that see nothing."""
    b = 6
    c = case(dtype, b, len_q, 180, 6, 3, 48, mask, k_len=[180, 0, 1, 100, 180, 999], q_start=[180 - len_q, 3, -2, 400, -500, 20],
             prefix=[0, 5, 180, 17, 0, 1000])
    got = run(nn, L, rng, c, kind, 16)
    assert not got["out"][1].any() and np.isneginf(got["lse"][1]).all()  # an empty cache


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("len_q, cap, buckets", [(1, 20.0, 0), (1, 0.0, 16), (4, 5.0, 16), (90, 30.0, 0), (90, 0.0, 8), (40, 8.0, 8)])
def test_caps_and_biases(nn, L, rng, kind, dtype, len_q, cap, buckets):
    c = case(dtype, 2, len_q, 333, 4, 2, 64, "causal", cap, k_len=[333, 150], q_start=[333 - len_q, 150 - len_q],
             **(dict(buckets=buckets, max_distance=40) if buckets else {}))
    run(nn, L, rng, c, kind, 64)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("page", [16, 32, 128, 4096])
@pytest.mark.parametrize("len_q", [1, 20, 100])
def test_pages(nn, L, rng, kind, dtype, page, len_q):
    c = case(dtype, 3, len_q, 700, 4, 1, 80, "causal", k_len=[700, 513, 100], q_start=[700 - len_q, 513 - len_q, 100 - len_q])
    run(nn, L, rng, c, kind, page)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("layout", ["odd", "heads"])
@pytest.mark.parametrize("len_q", [1, 7, 129])
def test_strides(nn, L, rng, kind, dtype, layout, len_q):
    c = case(dtype, 2, len_q, 260, 6, 2, 72, "causal", k_len=[260, 131], q_start=[260 - len_q, 131 - len_q])
    run(nn, L, rng, c, kind, 16, layout)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("len_q", [1, 9, 140])
def test_entries_that_are_no_page(nn, L, rng, kind, dtype, page, len_q):
    """Their keys are not seen, first, last, between others, and all of a request."""
    c = case(dtype, 4, len_q, 320, 4, 2, 64, "none", k_len=[320, 200, 290, 64])
    last = 319 // page
    holes = [(0, 0), (0, 2), (0, last), (1, 1), (2, 3)] + [(3, p) for p in range(-(-64 // page))]
    got = run(nn, L, rng, c, kind, page, holes=holes)
    assert not got["out"][3].any() and np.isneginf(got["lse"][3]).all()


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_large_scores(nn, L, rng, kind, dtype):
    """Scores of a deviation of some 60: the running maximum moves, shares vanish."""
    c = case(dtype, 1, 3, 600, 2, 1, 64, "causal", scale=7.0)
    run(nn, L, rng, c, kind, 32, scores=200.0)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("batch, len_q, len_k", [(1, 1, 9000), (3, 1, 5000), (1, 8, 20000), (1, 300, 5000)])
def test_long(nn, L, rng, kind, dtype, batch, len_q, len_k):
    """Keys divided over workgroups."""
    c = case(dtype, batch, len_q, len_k, 2, 1, 32, "causal", k_len=[len_k - 700 * b for b in range(batch)],
             q_start=[len_k - 700 * b - len_q for b in range(batch)])
    run(nn, L, rng, c, kind, 64)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("batch, heads, kv", [(65, 4, 2), (150, 2, 1), (300, 8, 8)])
def test_many_requests(nn, L, rng, kind, dtype, batch, heads, kv):
    """Lengths from none to several pages, more requests than a wave has lanes, and (300 x 8) a unit a workgroup."""
    k_len = rng.integers(0, 400, batch)
    k_len[rng.integers(0, batch, 5)] = 0
    c = case(dtype, batch, 1, 400, heads, kv, 32, "causal", k_len=list(k_len), q_start=list(k_len - 1))
    run(nn, L, rng, c, kind, 64)


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_prompt_chunk_and_steps(nn, L, rng, kind, dtype):
    """A prompt, a chunk and single tokens appended and attended to, as a program serves a request: each agrees with
    the 64-bit attention over what the cache then holds."""
    heads, kv, dim = 4, 2, 64
    cache = Cache(nn, L, rng, kind, dtype, kv, dim, 16, [14, 9])
    held = np.zeros(2, int)
    for new in (100, 37, 1, 1, 1):
        place = np.concatenate([h + np.arange(new) for h in held])
        request = np.repeat([0, 1], new)
        a = Append(nn, L, rng, cache, request, place, heads, dim, far=4096)
        a.launch()
        a.L.sync()
        a.compare()  # and the host image follows
        held += new
        c = case(dtype, 2, new, int(held.max()), heads, kv, dim, "causal", k_len=list(held), q_start=list(held - new))
        call = Call(nn, L, rng, c, kind, 16, cache=cache)
        call.launch()
        L.sync()
        call.compare()


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_capture(nn, L, rng, kind, dtype):
    """An append and the attention that reads it in a graph, replayed with new rows and lengths between eager calls."""
    heads, kv, dim = 4, 2, 64
    cache = Cache(nn, L, rng, kind, dtype, kv, dim, 32, [20, 20])
    cache.fill(rng, [500, 300], spoil=False)
    c = case(dtype, 2, 1, 640, heads, kv, dim, "causal", k_len=[501, 301], q_start=[500, 300])
    call = Call(nn, L, rng, c, kind, 32, cache=cache)
    a = Append(nn, L, rng, cache, np.arange(2), np.array([500, 300]), heads, dim)
    stream = L.nnhip_stream_create()
    L.nnhip_graph_capture_begin(stream)
    a.launch(stream)
    call.launch(stream)
    graph = L.nnhip_graph_capture_end(stream)
    assert graph
    for step in range(4):
        held = np.array([500, 300]) + step
        for dev, x in ((a.keep[3], held), (call.keep["k_len"], held + 1), (call.keep["q_start"], held)):
            dev.upload(np.append(x.astype(np.int32), np.int32(0)).view(np.float32))
        a.place = held
        call.c = dict(c, k_len=list(held + 1), q_start=list(held))
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


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_one_workspace_serves_smaller_calls(nn, L, rng, kind, dtype):
    """The workspace of the largest call, used by others in turn, gives each the results of its own."""
    big = Call(nn, L, rng, case(dtype, 4, 8, 3000, 4, 2, 64, "causal", k_len=[3000, 2000, 1, 555]), kind, 64)
    for batch, len_q, len_k in [(1, 1, 3000), (4, 8, 3000), (2, 3, 100), (1, 8, 2999), (3, 1, 1500), (4, 8, 3000)]:
        c = case(dtype, batch, len_q, len_k, 4, 2, 64, "causal")
        small = Call(nn, L, rng, c, kind, 64)
        assert small.ws.n <= big.ws.n
        small.launch(ws=big.ws)
        L.sync()
        got = small.compare()
        small.launch()
        L.sync()
        own = small.results()
        assert np.array_equal(own["out"], got["out"]) and np.array_equal(own["lse"], got["lse"])


@pytest.mark.parametrize("kind", ["mxfp4", "plain"])
def test_two_streams(nn, L, rng, kind):
    """Two calls at once, a workspace each."""
    calls = [Call(nn, L, rng, case("bf16", 2, 1, 4000, 8, 2, 128, "causal", k_len=[4000, 3000 - i]), kind, 64) for i in range(2)]
    streams = [L.nnhip_stream_create() for _ in calls]
    for _ in range(5):
        for call, stream in zip(calls, streams):
            call.launch(stream)
    for call, stream in zip(calls, streams):
        assert L.nnhip_stream_synchronize(stream) == 0
        call.compare()
        L.nnhip_stream_destroy(stream)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("table_pages, pages", [(0, 0), (0, 3), (2, 0)])
@pytest.mark.parametrize("len_q", [1, 200])
def test_empty_tables_and_pools(nn, L, kind, dtype, table_pages, pages, len_q):
    """No entries, or no pages, and no pointers where there is nothing: every query sees nothing."""
    heads, kv, dim = 2, 1, 32
    table = ints(L, np.zeros(max(1, 2 * table_pages)))
    pool = {n: L.alloc(max(1, pages) * 16 * 512) for n in ("k", "v")}
    cache = nn.NnCache(kind=nn.NN_CACHE_MXFP4 if kind == "mxfp4" else nn.NN_CACHE_PLAIN, page_tokens=16, pages=pages,
                       requests=2, table_pages=table_pages, table=table.p if table_pages else None,
                       k=pool["k"].p if pages else None, v=pool["v"].p if pages else None)
    q = Tensor(L, (2, len_q, heads, dim), dtype, values=np.ones((2, len_q, heads, dim)))
    out, lse = Tensor(L, (2, len_q, heads, dim), dtype, fill=7.0), L.alloc(2 * heads * len_q)
    a = nn.NnAttention(dtype=nn.NN_BF16 if dtype == "bf16" else nn.NN_F32, batch=2, len_q=len_q, len_k=16 * table_pages,
                       heads=heads, kv_heads=kv, head_dim=dim, scale=1.0, mask=nn.NN_MASK_NONE, q_stride=q.strides[:3],
                       out_stride=out.strides[:3])
    assert L.nnhip_cache_attention_workspace(a, cache) == 0
    L.launch_cache_attention_forward(out.p, lse.p, q.p, a, cache, None, None)
    L.sync()
    assert not out.result().any() and np.isneginf(lse.download(2 * heads * len_q)).all()


@pytest.mark.parametrize("batch, heads, kv, len_k", [(300, 8, 8, 9000), (64, 16, 8, 16384)])
def test_requests_that_share_pages(nn, L, rng, batch, heads, kv, len_k):
    """All requests read the same pages with the same queries, in a workgroup's long row of keys (9000) and
    in long shares of them (16384), both of more blocks than are looked up at once."""
    dim, page = 32, 64
    cache = Cache(nn, L, rng, "mxfp4", "bf16", kv, dim, page, [-(-len_k // page)])
    cache.fill(rng, [len_k])
    one = Call(nn, L, rng, case("bf16", 1, 1, len_k, heads, kv, dim, "causal"), "mxfp4", page, cache=cache)
    one.launch()
    L.sync()
    one.compare()
    ref, mag = one.expected()
    table = ints(L, np.repeat(cache.table, batch, 0))
    shared = nn.NnCache(kind=nn.NN_CACHE_MXFP4, page_tokens=page, pages=cache.pages, requests=batch,
                        table_pages=cache.table.shape[1], table=table.p, k=cache.dev["k"].p, v=cache.dev["v"].p)
    q = Tensor(L, (batch, 1, heads, dim), "bf16", values=np.repeat(one.q.values(), batch, 0))
    out, lse = Tensor(L, (batch, 1, heads, dim), "bf16"), L.alloc(batch * heads)
    a = nn.NnAttention(dtype=nn.NN_BF16, batch=batch, len_q=1, len_k=len_k, heads=heads, kv_heads=kv, head_dim=dim,
                       scale=dim**-0.5, mask=nn.NN_MASK_CAUSAL, q_stride=q.strides[:3], out_stride=out.strides[:3])
    ws = L.to_device(np.zeros(max(1, L.nnhip_cache_attention_workspace(a, shared)), np.float32))
    L.launch_cache_attention_forward(out.p, lse.p, q.p, a, shared, ws.p, None)
    L.sync()
    # Against the formulas and not against the one request's results: there the keys are divided otherwise, so
    # shares are rounded relative to another reference, each by up to 2^-8 of itself on either side.
    check("out", out.result(), np.repeat(ref["out"], batch, 0), np.repeat(mag["out"], batch, 0), "bf16")
    got = lse.download(shape=(batch, heads, 1)).astype(np.float64)
    check("lse", got, np.repeat(ref["lse"], batch, 0), np.repeat(mag["lse"], batch, 0), "f32")


@pytest.mark.parametrize("len_q", [1, 300])
def test_pools_past_32_bits(nn, L, rng, len_q):
    """Pages whose offsets need more than 32 bits, read by both forms."""
    heads, kv, dim, tokens, length = 8, 8, 128, 4096, 8192 + 700
    size = tokens * 68 * kv
    pages = (1 << 32) // size + 3
    pool = {n: L.alloc(pages * size // 4) for n in ("k", "v")}
    order = [pages - 1, 0, pages - 2]
    table = ints(L, [order])
    far = nn.NnCache(kind=nn.NN_CACHE_MXFP4, page_tokens=tokens, pages=pages, requests=1, table_pages=3, table=table.p,
                     k=pool["k"].p, v=pool["v"].p)
    cache = Cache(nn, L, rng, "mxfp4", "bf16", kv, dim, tokens, [3])
    cache.fill(rng, [length])
    for n in pool:  # the same pages, far apart
        for i, at in enumerate(order):
            raw = np.ascontiguousarray(cache.bytes[n][cache.table[0, i]]).ravel().view(np.float32)
            assert L.dll.nnhip_memcpy_htod(pool[n].ptr + at * size, raw.ctypes.data, raw.nbytes) == 0
    c = case("bf16", 1, len_q, length, heads, kv, dim, "causal")
    call = Call(nn, L, rng, c, "mxfp4", tokens, cache=cache)
    call.launch()
    L.sync()
    near = call.results()
    call.cache.args = far
    call.out.dev.fill_bytes(0xFF)
    call.launch()
    L.sync()
    got = call.results()
    assert np.array_equal(got["out"], near["out"]) and np.array_equal(got["lse"], near["lse"])
    if len_q == 1:
        call.compare()


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_append_attend_and_read(nn, L, rng, kind, dtype):
    """What is read out of the cache is what attention over it used: attention over tensors of it agrees."""
    heads, kv, dim, tokens = 4, 2, 64, 150
    cache = Cache(nn, L, rng, kind, dtype, kv, dim, 32, [5])
    a = Append(nn, L, rng, cache, np.zeros(tokens, int), np.arange(tokens), heads, dim)
    a.launch()
    c = case(dtype, 1, tokens, tokens, heads, kv, dim, "causal")
    rows = {n: Tensor(L, (tokens, kv, dim), dtype) for n in ("k", "v")}
    L.launch_cache_read(rows["k"].p, rows["v"].p, nn.NnCacheRead(
        dtype=cache.nn_dtype(), tokens=tokens, kv_heads=kv, head_dim=dim, k_stride=rows["k"].strides[:2],
        v_stride=rows["v"].strides[:2], request=a.keep[2].p, place=a.keep[3].p), cache.args, None)
    out = {n: Tensor(L, (1, tokens, heads, dim), dtype) for n in ("paged", "plain")}
    lse = {n: L.alloc(heads * tokens) for n in out}
    q = a.t["q_out"]
    args = nn.NnAttention(dtype=cache.nn_dtype(), batch=1, len_q=tokens, len_k=tokens, heads=heads, kv_heads=kv, head_dim=dim,
                          scale=c["scale"], mask=nn.NN_MASK_CAUSAL, q_stride=(0, heads * dim, dim),
                          k_stride=(0, kv * dim, dim), v_stride=(0, kv * dim, dim), out_stride=(tokens * heads * dim, heads * dim, dim))
    ws = L.to_device(np.zeros(max(1, L.nnhip_cache_attention_workspace(args, cache.args),
                                  L.nnhip_attention_forward_workspace(args)), np.float32))
    L.launch_cache_attention_forward(out["paged"].p, lse["paged"].p, q.p, args, cache.args, ws.p, None)
    L.launch_attention_forward(out["plain"].p, lse["plain"].p, q.p, rows["k"].p, rows["v"].p, args, ws.p, None)
    L.sync()
    ref, mag = attention(c, q.result()[None], rows["k"].result()[None], rows["v"].result()[None])
    for n in out:
        check(n, out[n].result(), ref["out"], mag["out"], dtype)
        check(n, lse[n].download(shape=(1, heads, tokens)).astype(np.float64), ref["lse"], mag["lse"], "f32")
