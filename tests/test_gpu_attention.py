"""Attention through the C-ABI against the 64-bit formulas: types, head layouts, lengths,
masks, biases, strides, and what masked places may hold."""
from __future__ import annotations

import numpy as np
import pytest

from attention_ref import Tensor, attention, check, from_bf16, ints, rounded, sees_of

pytestmark = pytest.mark.gpu


def case(dtype, batch, len_q, len_k, heads, kv_heads, dim, mask="none", cap=0.0, **more):
    return dict(dtype=dtype, batch=batch, len_q=len_q, len_k=len_k, heads=heads, kv_heads=kv_heads, dim=dim, mask=mask,
                cap=cap, scale=more.pop("scale", dim**-0.5), **more)


def bias_of(c, rng):
    if not c.get("buckets"):
        return None, None
    m = c["max_distance"]
    bucket = np.sort(rng.integers(0, c["buckets"], 2 * m + 1)).astype(np.int32)
    return rng.standard_normal((c["buckets"], c["heads"])).astype(np.float32), bucket


class Call:
    """A case's tensors on the device, its launches and its 64-bit results."""

    def __init__(self, nn, L, rng, c, layout="plain", backward=True, spoil=True):
        self.nn, self.L, self.c, self.backward = nn, L, c, backward
        b, lq, lk, h, kv, d = (c[n] for n in ("batch", "len_q", "len_k", "heads", "kv_heads", "dim"))
        t = c["dtype"]
        shapes = {"q": (b, lq, h, d), "k": (b, lk, kv, d), "v": (b, lk, kv, d), "out": (b, lq, h, d)}
        values = {n: rng.standard_normal(shapes[n]).astype(np.float32) for n in ("q", "k", "v")}
        dout = rng.standard_normal(shapes["out"]).astype(np.float32)
        strides = {n: None for n in shapes}
        offset = {n: 0 for n in shapes}
        if layout == "packed":  # one projection's rows; queries, keys and values of a token together
            row = (h + 2 * kv) * d
            for n, at in (("q", 0), ("k", h * d), ("v", (h + kv) * d)):
                strides[n] = (shapes[n][1] * row, row, d, 1)
                offset[n] = at
        elif layout == "cache":  # a head's tokens together
            for n in ("k", "v"):
                strides[n] = (kv * lk * d, d, lk * d, 1)
        elif layout == "odd":  # nothing on 16 bytes
            for n in shapes:
                heads, length = shapes[n][2], shapes[n][1]
                strides[n] = (length * (heads * (d + 1) + 1) + 3, heads * (d + 1) + 1, d + 1, 1)
                offset[n] = 1
        self.sees, _ = sees_of(c)
        dead_q, dead_k = ~self.sees.any(2) if lk else np.ones((b, lq), bool), ~self.sees.any(1) if lq else np.ones((b, lk), bool)
        self.dead_q, self.dead_k = dead_q, dead_k
        # keys that no one can see by their length or document, and queries that see nothing, hold anything
        gone = np.arange(lk)[None] >= np.asarray(c.get("k_len", [lk] * b))[:, None]
        if "doc_k" in c:
            gone |= np.asarray(c["doc_k"]) < 0
        if spoil:
            for n in ("k", "v"):
                values[n][gone] = rng.choice([np.nan, np.inf, -np.inf, 3e38], values[n][gone].shape)
            values["q"][dead_q] = np.nan
            dout[dead_q] = np.inf
        make = lambda n, v=None, like=None: Tensor(L, shapes[like or n], t, strides[like or n], offset[like or n], values=v)  # noqa: E731
        self.t = {n: make(n, values[n]) for n in ("q", "k", "v")}
        self.t["out"] = make("out")
        self.lse = L.alloc(max(1, b * h * lq))
        self.lse.fill_bytes(0xFF)
        self.bias, self.bucket = bias_of(c, rng)
        self.keep = {}
        for n in ("q_start", "k_len", "prefix", "doc_q", "doc_k"):
            if n in c:
                self.keep[n] = ints(L, c[n])
        if self.bias is not None:
            self.keep["bias"], self.keep["bucket"] = L.to_device(self.bias), ints(L, self.bucket)
        self.args = nn.NnAttention(
            dtype=nn.NN_BF16 if t == "bf16" else nn.NN_F32, batch=b, len_q=lq, len_k=lk, heads=h, kv_heads=kv,
            head_dim=d, scale=c["scale"], softcap=c["cap"],
            mask={"none": nn.NN_MASK_NONE, "causal": nn.NN_MASK_CAUSAL, "prefix": nn.NN_MASK_PREFIX}[c["mask"]],
            buckets=c.get("buckets", 0), max_distance=c.get("max_distance", 0),
            **{f"{n}_stride": self.t[n].strides[:3] for n in ("q", "k", "v", "out")},
            **{n: d_.p for n, d_ in self.keep.items()})
        self.ws = L.to_device(np.zeros(max(1, L.nnhip_attention_forward_workspace(self.args)), np.float32))
        if backward:
            self.t["dout"] = make("dout", dout, "out")
            for n in ("q", "k", "v"):
                self.t["d" + n] = make("d" + n, None, n)
            self.dbias = L.alloc(self.bias.size) if self.bias is not None else None
            self.bws = L.alloc(max(1, L.nnhip_attention_backward_workspace(self.args)))
            self.bws.fill_bytes(0xFF)

    def forward(self, stream=None):
        t = self.t
        self.L.launch_attention_forward(t["out"].p, self.lse.p, t["q"].p, t["k"].p, t["v"].p, self.args, self.ws.p, stream)

    def grad(self, stream=None):
        t = self.t
        self.L.launch_attention_backward(t["dq"].p, t["dk"].p, t["dv"].p, self.dbias.p if self.dbias else None,
                                         t["dout"].p, t["q"].p, t["k"].p, t["v"].p, t["out"].p, self.lse.p, self.args,
                                         self.bws.p, stream)

    def results(self):
        c = self.c
        got = {"out": self.t["out"].result(),
               "lse": self.lse.download(c["batch"] * c["heads"] * c["len_q"], (c["batch"], c["heads"], c["len_q"])).astype(np.float64)}
        if self.backward:
            got.update({n: self.t[n].result() for n in ("dq", "dk", "dv")})
            if self.dbias:
                got["dbias"] = self.dbias.download(shape=self.bias.shape).astype(np.float64)
        return got

    def expected(self):
        x = {n: self.t[n].values() for n in ("q", "k", "v")}
        return attention(self.c, **x, bias=None if self.bias is None else self.bias.astype(np.float64),
                         bucket=self.bucket, dout=self.t["dout"].values() if self.backward else None)

    def compare(self, scores=10.0):
        got, (ref, mag) = self.results(), self.expected()
        assert set(got) == set(ref)
        for n in ref:
            check(n, got[n], ref[n], mag[n], "f32" if n in ("lse", "dbias") else self.c["dtype"], scores)
        assert not got["out"][self.dead_q].any() and np.isneginf(got["lse"].transpose(0, 2, 1)[self.dead_q]).all()
        if self.backward:
            assert not got["dq"][self.dead_q].any()
            assert not got["dk"][self.dead_k].any() and not got["dv"][self.dead_k].any()
            alone = self.sees.sum(2) == 1
            if alone[self.sees.any(2)].all():  # every query sees one key at most: its share is 1 whatever the score
                assert not got["dq"].any() and not got["dk"].any()
                assert self.dbias is None or not got["dbias"].any()
        return got


def run(nn, L, rng, c, layout="plain", scores=10.0):
    print(f"[case] attention {layout} {c}", flush=True)
    call = Call(nn, L, rng, c, layout)
    call.forward()
    call.grad()
    L.sync()
    return call.compare(scores)


TYPES = ("f32", "bf16")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 8, 33, 40, 64, 72, 100, 128])
def test_head_dims(nn, L, rng, dtype, dim):
    run(nn, L, rng, case(dtype, 2, 70, 93, 2, 2, dim))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("len_q, len_k", [(1, 1), (1, 65), (65, 1), (64, 64), (130, 257), (257, 130), (3, 400)])
def test_lengths_and_masks(nn, L, rng, dtype, mask, len_q, len_k):
    run(nn, L, rng, case(dtype, 2, len_q, len_k, 2, 1, 24, mask, prefix=[len_k // 3, 0]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (3, 3), (6, 2), (8, 1)])
def test_shared_key_heads(nn, L, rng, dtype, heads, kv_heads):
    run(nn, L, rng, case(dtype, 2, 97, 97, heads, kv_heads, 48, "causal"), "packed")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["plain", "packed", "cache", "odd"])
def test_layouts(nn, L, rng, dtype, layout):
    run(nn, L, rng, case(dtype, 2, 140, 140, 4, 2, 40, "causal", cap=20.0), layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.05, 1.0, 5.0, 50.0, 1e4])
def test_capped_scores(nn, L, rng, dtype, cap):
    run(nn, L, rng, case(dtype, 1, 100, 130, 2, 2, 64, cap=cap, scale=0.4))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("buckets, distance", [(1, 0), (2, 1), (7, 20), (32, 128), (5, 1023)])
@pytest.mark.parametrize("mask, cap, heads, kv", [("none", 0.0, 2, 2), ("causal", 3.0, 4, 2)])
def test_distance_bias(nn, L, rng, dtype, buckets, distance, mask, cap, heads, kv):
    run(nn, L, rng, case(dtype, 2, 150, 310, heads, kv, 32, mask, cap, buckets=buckets, max_distance=distance))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_everything_at_once(nn, L, rng, dtype, dim):
    doc = np.sort(rng.integers(-1, 3, (2, 200)), axis=1)
    run(nn, L, rng, case(dtype, 2, 200, 200, 4, 2, dim, "prefix", 4.0, prefix=[150, 20], buckets=16, max_distance=60,
                         doc_q=doc, doc_k=doc, k_len=[200, 170]), "packed")


def _docs(kind, rng, n):
    if kind == "runs":
        return np.repeat(np.arange(n), 37)[:n]
    if kind == "single":  # a document a token: each query sees one key
        return np.arange(n)
    if kind == "shuffled":
        return rng.integers(-1, 5, n)
    if kind == "blocks":  # documents that end on the kernels' blocks
        return np.arange(n) // 64
    return np.full(n, -1)  # none


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["runs", "single", "shuffled", "blocks", "padding"])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_documents(nn, L, rng, dtype, kind, mask):
    n = 50 if kind == "single" else 300
    doc = np.stack([_docs(kind, rng, n), _docs(kind, rng, n)[::-1]])
    run(nn, L, rng, case(dtype, 2, n, n, 2, 2, 16, mask, doc_q=doc, doc_k=doc))


@pytest.mark.parametrize("dtype", TYPES)
def test_documents_of_other_keys(nn, L, rng, dtype):
    dq, dk = rng.integers(-1, 4, (2, 90)), rng.integers(-1, 4, (2, 210))
    run(nn, L, rng, case(dtype, 2, 90, 210, 2, 2, 16, doc_q=dq, doc_k=dk))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
def test_lengths_of_requests(nn, L, rng, dtype, mask):
    """Lengths of zero, of one, inside a block and past the tensor's; queries before key 0 see nothing."""
    run(nn, L, rng, case(dtype, 5, 6, 200, 4, 1, 64, mask, k_len=[0, 1, 100, 200, 999], q_start=[-3, 0, 94, 194, 500],
                         prefix=[0, 0, 50, 300, -4]), "cache")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("len_q, len_k", [(0, 5), (5, 0)])
def test_empty_sides(nn, L, rng, dtype, len_q, len_k):
    doc_q, doc_k = np.zeros((2, len_q), int), np.zeros((2, len_k), int)
    run(nn, L, rng, case(dtype, 2, len_q, len_k, 2, 2, 8, buckets=3, max_distance=2, doc_q=doc_q, doc_k=doc_k))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("len_q", [1, 2, 5, 17, 40])
@pytest.mark.parametrize("heads, kv_heads", [(2, 2), (8, 2), (24, 3)])
@pytest.mark.parametrize("len_k", [63, 777, 3001])
def test_few_queries(nn, L, rng, dtype, len_q, heads, kv_heads, len_k):
    """The form for few queries over a cache: lengths that end anywhere, one request of a single key."""
    k_len = [len_k, max(len_q, len_k // 3), 1]
    c = case(dtype, 3, len_q, len_k, heads, kv_heads, 72 if len_k == 777 else 64, "causal", 30.0 if heads == 8 else 0.0,
             k_len=k_len, q_start=[n - len_q for n in k_len])
    print(f"[case] few queries {c}", flush=True)
    call = Call(nn, L, rng, c, "cache", backward=False)
    call.forward()
    first = call.results()
    call.forward()  # the workspace is as before
    L.sync()
    got = call.compare()
    for n in got:
        assert np.array_equal(got[n], first[n]), f"{n}: another result on the second call"


@pytest.mark.parametrize("dtype", TYPES)
def test_few_queries_with_bias_and_documents(nn, L, rng, dtype):
    dq, dk = np.array([[2, 1], [0, -1]]), np.sort(rng.integers(-1, 3, (2, 900)), axis=1)
    c = case(dtype, 2, 2, 900, 8, 2, 40, "prefix", 5.0, prefix=[900, 300], buckets=9, max_distance=100, doc_q=dq, doc_k=dk)
    print(f"[case] few queries {c}", flush=True)
    call = Call(nn, L, rng, c, "odd", backward=False)
    call.forward()
    L.sync()
    call.compare()


def test_workspace_of_a_larger_call(nn, L, rng):
    """One workspace for calls of several shapes in turn."""
    big = Call(nn, L, rng, case("bf16", 4, 1, 4000, 8, 2, 64, "causal", k_len=[4000, 9, 2500, 64], q_start=[3999, 8, 2499, 63]), "cache", backward=False)
    small = Call(nn, L, rng, case("bf16", 1, 2, 1900, 4, 4, 64, "causal"), "cache", backward=False)
    docs = Call(nn, L, rng, case("f32", 1, 40, 40, 2, 2, 8, doc_q=np.arange(40)[None] // 9, doc_k=np.arange(40)[None] // 9), backward=False)
    shared = L.to_device(np.zeros(max(big.ws.n, small.ws.n, docs.ws.n), np.float32))
    big.ws = small.ws = docs.ws = shared
    for call in (big, small, docs, big, docs, small):
        print(f"[case] shared workspace {call.c}", flush=True)
        call.forward()
        L.sync()
        call.compare()


def test_results_repeat_bit_for_bit(nn, L, rng):
    doc = np.sort(rng.integers(0, 3, (1, 500)), axis=1)
    c = case("bf16", 1, 500, 500, 8, 2, 64, "causal", 10.0, buckets=8, max_distance=30, doc_q=doc, doc_k=doc)
    print(f"[case] repeated {c}", flush=True)
    call = Call(nn, L, rng, c, "packed")
    got = []
    for _ in range(3):
        call.forward()
        call.grad()
        L.sync()
        got.append(call.results())
    for n in got[0]:
        assert np.array_equal(got[0][n], got[1][n]) and np.array_equal(got[0][n], got[2][n]), n


@pytest.mark.parametrize("few", [False, True])
def test_captured_and_replayed(nn, L, rng, few):
    """Forward and backward captured on a stream; every replay on new inputs agrees with an
    eager call, eager work and other graphs in between."""
    c = (case("bf16", 2, 1, 2500, 8, 2, 64, "causal", k_len=[2500, 1200], q_start=[2499, 1199]) if few else
         case("bf16", 2, 150, 150, 4, 2, 64, "causal", 8.0, buckets=8, max_distance=20))
    print(f"[case] graph {c}", flush=True)
    call = Call(nn, L, rng, c, "cache" if few else "packed", backward=not few, spoil=False)
    s = L.nnhip_stream_create()
    call.forward(s)
    if not few:
        call.grad(s)
    L.nnhip_stream_synchronize(s)
    assert L.nnhip_graph_capture_begin(s) == 0
    call.forward(s)
    if not few:
        call.grad(s)
    g = L.nnhip_graph_capture_end(s)
    assert g
    for _ in range(4):
        for n in ("q", "k", "v") + (() if few else ("dout",)):
            call.t[n].view(call.t[n].host)[...] = rng.standard_normal(call.t[n].shape)
            call.t[n].upload()
        assert L.nnhip_graph_launch(g, s) == 0
        L.nnhip_stream_synchronize(s)
        replayed = call.compare()
        call.forward()
        if not few:
            call.grad()
        L.sync()
        eager = call.results()
        for n in eager:
            assert np.array_equal(eager[n], replayed[n]), n
    L.nnhip_graph_destroy(g)
    L.nnhip_stream_destroy(s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("len_q", [1, 70])
def test_offsets_past_32_bits(nn, L, rng, dtype, len_q):
    """A cache whose tokens lie 2^26 elements apart: element offsets pass 2^32."""
    n, dim, step = 90, 16, 1 << 26
    c = case(dtype, 1, len_q, n, 2, 1, dim, "causal")
    print(f"[case] far rows {c}", flush=True)
    small = Call(nn, L, rng, c, backward=False)
    size = small.t["k"].size
    far = {m: L.alloc(((n - 1) * step + dim) * size // 4 + 4) for m in ("k", "v")}
    for m in far:
        rows = small.t[m].dev.download().view(np.uint8)
        for j in range(n):
            row = np.ascontiguousarray(rows[j * dim * size:(j + 1) * dim * size])
            assert L.nnhip_memcpy_htod(far[m].p + j * step * size, row.ctypes.data, row.nbytes) == 0
    small.args.k_stride = small.args.v_stride = (n * step, step, dim)
    t = small.t
    L.launch_attention_forward(t["out"].p, small.lse.p, t["q"].p, far["k"].p, far["v"].p, small.args, small.ws.p, None)
    L.sync()
    small.compare()
    for m in far:
        far[m].close()


@pytest.mark.parametrize("dtype, len_q", [("bf16", 1), ("bf16", 130), ("f32", 3)])
def test_long_cache_of_aligned_rows(nn, L, rng, dtype, len_q):
    """Tokens 2^20 bytes apart: a block's offsets fit in 32 bits, a block's address does not."""
    n, dim, size = 4500, 64, 2 if dtype == "bf16" else 4
    step = (1 << 20) // size
    c = case(dtype, 1, len_q, n, 1, 1, dim, "causal")
    print(f"[case] long cache {c}", flush=True)
    small = Call(nn, L, rng, c, backward=False)
    far = {m: L.alloc(((n - 1) * step + dim) * size // 4 + 4) for m in ("k", "v")}
    for m in far:
        rows = small.t[m].dev.download().view(np.uint8)
        for j in range(n):
            row = np.ascontiguousarray(rows[j * dim * size:(j + 1) * dim * size])
            assert L.nnhip_memcpy_htod(far[m].p + j * step * size, row.ctypes.data, row.nbytes) == 0
    small.args.k_stride = small.args.v_stride = (n * step, step, dim)
    t = small.t
    L.launch_attention_forward(t["out"].p, small.lse.p, t["q"].p, far["k"].p, far["v"].p, small.args, small.ws.p, None)
    L.sync()
    small.compare()
    for m in far:
        far[m].close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask, cap, buckets", [("none", 0.0, 0), ("causal", 30.0, 0), ("prefix", 0.0, 8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_enough_workgroups_for_whole_tiles(nn, L, rng, dtype, mask, cap, buckets, dim):
    """Sizes at which a workgroup keeps 128 rows (fewer tiles are split), with documents that end anywhere."""
    doc = np.sort(rng.integers(-1, 4, (32, 130)), axis=1)
    run(nn, L, rng, case(dtype, 32, 130, 130, 8, 4 if mask == "causal" else 8, dim, mask, cap, prefix=[60] * 32,
                         buckets=buckets, max_distance=40, **({"doc_q": doc, "doc_k": doc} if mask != "none" else {})))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
def test_tiles_dealt_out_by_their_work(nn, L, rng, dtype, mask):
    """Documents and as many workgroups as make an order of the tiles worth it, heads that do not divide over XCDs."""
    doc = np.sort(rng.integers(-1, 6, (60, 130)), axis=1)
    doc[7], doc[8] = -1, rng.integers(0, 3, 130)
    run(nn, L, rng, case(dtype, 60, 130, 130, 3, 3, 16, mask, prefix=[40] * 60, doc_q=doc, doc_k=doc,
                         k_len=[0] + [130] * 58 + [77]), "packed")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("len_q, len_k, heads, kv, dim, mask, cap, buckets, docs, layout", [
    (900, 1100, 1, 1, 72, "prefix", 20.0, 0, False, "plain"),
    (1030, 1030, 2, 1, 33, "causal", 0.0, 0, False, "odd"),
    (777, 777, 3, 3, 128, "none", 0.0, 12, True, "packed"),
    (70, 2500, 2, 2, 64, "causal", 3.0, 40, False, "cache"),
    (2500, 70, 4, 2, 24, "none", 0.0, 0, False, "plain"),
    (1200, 1200, 2, 2, 40, "causal", 0.0, 0, True, "plain"),
])
def test_long_axes_in_parts(nn, L, rng, dtype, len_q, len_k, heads, kv, dim, mask, cap, buckets, docs, layout):
    """Few heads and long sequences: the other axis is divided over workgroups, some of which have nothing."""
    more = {}
    if docs:
        doc = np.sort(rng.integers(-1, 5, (1, len_q)), axis=1)
        more = {"doc_q": doc, "doc_k": doc}
    run(nn, L, rng, case(dtype, 1, len_q, len_k, heads, kv, dim, mask, cap, prefix=[len_k // 3], buckets=buckets,
                         max_distance=50, **more), layout)


def test_large_scores_and_infinite_bias(nn, L, rng):
    """Scores of hundreds (one key takes all), and a bias of -inf, which hides its bucket."""
    c = case("f32", 1, 80, 80, 2, 2, 16, scale=40.0)
    run(nn, L, rng, c, scores=40.0 * 16)
    c = case("f32", 1, 70, 70, 1, 1, 8, buckets=2, max_distance=1)
    call = Call(nn, L, rng, c)
    call.bias[...] = [[0.5], [-np.inf]]
    call.bucket[...] = [0, 0, 1]  # keys past the query's own are hidden
    call.keep["bias"].upload(call.bias)
    call.keep["bucket"].upload(call.bucket.view(np.float32))
    call.forward()
    call.grad()
    L.sync()
    got = call.results()
    call.c = dict(c, mask="causal", buckets=1)
    call.bias, call.bucket = call.bias[:1], np.zeros(3, np.int32)
    ref, mag = call.expected()
    for n in ("out", "lse", "dq", "dk", "dv"):
        check(n, got[n], ref[n], mag[n], "f32")
    assert got["dbias"][1] == 0


def test_bf16_probabilities_are_not_all_that_is_kept(nn, L, rng):
    """The log-sum and the bias gradient of bf16 calls are fp32 values, not bf16 ones."""
    c = case("bf16", 2, 300, 300, 2, 2, 64, buckets=8, max_distance=40)
    got = run(nn, L, rng, c)
    for n in ("lse", "dbias"):
        assert (rounded(got[n], "bf16") != got[n]).mean() > 0.9
    assert from_bf16(np.uint16(0x3F80)) == 1.0
