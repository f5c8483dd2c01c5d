"""The paged cache through the C-ABI: appends and reads against the 64-bit formulas, in the tensors' type and in 4
bits, for types, head layouts, strides, padded batches and tables with entries that are no page."""
from __future__ import annotations

import numpy as np
import pytest

from attention_ref import check, norm_rope
from cache_ref import Cache, Tensor, ints, rounded

pytestmark = pytest.mark.gpu


def turned(x, w, eps, norm, pos, freq, rot, axes, interleaved):
    """x [tokens, heads, dim] as the append has it: norm_rope, or its turn alone."""
    if norm:
        return norm_rope(x, w, eps, pos, freq, rot, axes, interleaved)
    size = np.sqrt((x * x).mean(-1, keepdims=True))
    return norm_rope(np.where(size == 0, 1, x / np.where(size == 0, 1, size)), 1.0, 0.0, pos, freq, rot, axes, interleaved) * size


class Append:
    def __init__(self, nn, L, rng, cache, request, place, heads, rot, axes=1, interleaved=False, norm=True, layout="packed",
                 far=1 << 20, values=None, given_request=True):
        self.nn, self.L, self.cache, self.request, self.place, self.norm = nn, L, cache, request, place, norm
        t, kv, dim = len(place), cache.kv, cache.dim
        self.shape = dict(rot=rot, axes=axes, interleaved=interleaved)
        if layout == "packed":
            row = (heads + 2 * kv) * dim
            spec = {"q": ((row, dim, 1), 0), "k": ((row, dim, 1), heads * dim), "v": ((row, dim, 1), (heads + kv) * dim)}
        else:  # nothing on 16 bytes
            spec = {n: ((h * (dim + 1) + 3, dim + 1, 1), 1) for n, h in (("q", heads), ("k", kv), ("v", kv))}
        dead = np.asarray(place) < 0
        self.t = {}
        for n, h in (("q", heads), ("k", kv), ("v", kv)):
            x = values[n] if values else 1.3 * rng.standard_normal((t, h, dim))
            x[dead] = np.nan
            self.t[n] = Tensor(L, (t, h, dim), cache.dtype, spec[n][0], spec[n][1], values=x)
        self.t["q_out"] = Tensor(L, (t, heads, dim), cache.dtype, None if layout == "packed" else spec["q"][0],
                                 0 if layout == "packed" else 1, fill=7.0)
        self.pos = rng.integers(0, far, (t, axes)).astype(np.int32)
        per = max(1, rot // 2 // axes)
        self.freq = 500000.0 ** (-(np.arange(rot // 2) % per) / per)
        self.w = {n: (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for n in ("q", "k")} if norm else {}
        self.eps = 1e-6
        self.keep = [ints(L, self.pos), L.to_device(self.freq.view(np.float32)), ints(L, request), ints(L, place)]
        self.keep_w = {n: L.to_device(w) for n, w in self.w.items()}
        self.args = nn.NnCacheAppend(
            rope=nn.NnQkNormRope(
                dtype=cache.nn_dtype(), tokens=t, heads=heads, kv_heads=kv, head_dim=dim, rot_dim=rot, axes=axes,
                interleaved=int(interleaved), eps=self.eps, q_stride=self.t["q"].strides[:2], k_stride=self.t["k"].strides[:2],
                q_out_stride=self.t["q_out"].strides[:2], pos=self.keep[0].p, freq=self.keep[1].p,
                **{f"{n}_weight": d.p for n, d in self.keep_w.items()}),
            norm=int(norm), v_stride=self.t["v"].strides[:2], request=self.keep[2].p if given_request else None,
            place=self.keep[3].p)

    def launch(self, stream=None):
        t = self.t
        self.L.launch_cache_append(t["q_out"].p, t["q"].p, t["k"].p, t["v"].p, self.args, self.cache.args, stream)

    def rows(self, name):
        x = np.nan_to_num(self.t[name].values())
        return turned(x, self.w[name].astype(np.float64) if self.norm else 1.0, self.eps, self.norm, self.pos, self.freq,
                      self.shape["rot"], self.shape["axes"], self.shape["interleaved"])

    def compare(self):
        """q_out, and every byte of both pools."""
        c, live = self.cache, np.asarray(self.place) >= 0
        if self.t["q"].shape[1]:
            q = self.t["q_out"].result()
            assert (q[~live] == 7.0).all(), "a row that is no token was written"
            ref = self.rows("q")[live]
            check("q_out", q[live], ref, np.broadcast_to(np.abs(ref).max(-1, keepdims=True), ref.shape), c.dtype)
        k, v = self.rows("k"), np.nan_to_num(self.t["v"].values())
        slots = {}
        for t in np.flatnonzero(live):
            at = c.where(int(self.request[t]), int(self.place[t]))
            if at is not None:
                slots[at] = t
        near = {t: c.put("k", at, k[t]) for at, t in slots.items()}
        for at, t in slots.items():
            c.put("v", at, v[t])
        got = {n: c.download(n) for n in ("k", "v")}
        assert np.array_equal(got["v"], c.bytes["v"])
        if c.groups:
            if not np.array_equal(got["k"], c.bytes["k"]):
                for at, t in slots.items():
                    assert near[t] < 1e-8 or np.array_equal(c.get("k", at, got["k"]), c.get("k", at)), (at, t, near[t])
                    if near[t] < 1e-8:  # either way: then the same elsewhere
                        c.bytes["k"][at[0]] = got["k"][at[0]]
            assert np.array_equal(got["k"], c.bytes["k"])
        else:
            rows = np.stack([c.get("k", at, got["k"]) for at in slots]) if slots else np.zeros((0, c.kv, c.dim))
            ref = np.stack([k[t] for t in slots.values()]) if slots else rows
            check("k", rows, ref, np.broadcast_to(np.abs(ref).max(-1, keepdims=True), ref.shape), c.dtype)
            for at in slots:  # and nothing else, apart from the row's own values
                size = c.dim * (2 if c.dtype == "bf16" else 4)
                c.bytes["k"][at[0]][:, at[1] * c.row:at[1] * c.row + size] = got["k"][at[0]][:, at[1] * c.row:at[1] * c.row + size]
            assert np.array_equal(got["k"], c.bytes["k"])


KINDS = [("mxfp4", "bf16"), ("mxfp4", "f32"), ("plain", "bf16"), ("plain", "f32")]


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("heads, kv, dim, rot, axes, inter, norm, layout", [
    (8, 2, 128, 128, 1, False, True, "packed"),
    (4, 4, 64, 64, 2, True, True, "packed"),
    (3, 1, 72, 48, 2, True, False, "packed"),
    (2, 2, 33, 16, 1, False, True, "odd"),
    (5, 5, 1, 0, 1, False, False, "odd"),
    (0, 3, 96, 96, 3, False, True, "packed"),
    (2, 1, 40, 34, 1, False, False, "odd"),
    (6, 2, 128, 0, 1, False, False, "packed"),
    (2, 2, 8, 8, 1, False, True, "packed"),
])
def test_append(nn, L, rng, kind, dtype, heads, kv, dim, rot, axes, inter, norm, layout):
    """Two requests that hold something already, one of them over a page's end, and rows that are no tokens."""
    print(f"[case] append {kind} {dtype} {heads} {kv} {dim} {rot} {axes} {inter} {norm} {layout}", flush=True)
    cache = Cache(nn, L, rng, kind, dtype, kv, dim, 16, [3, 1, 2])
    place = np.array(list(range(10, 40)) + [0, 1, 2, -1, -5] + [31, -1])
    request = np.array([0] * 30 + [2] * 5 + [2, 1])
    order = rng.permutation(len(place))  # any order of rows
    a = Append(nn, L, rng, cache, request[order], place[order], heads, rot, axes, inter, norm, layout)
    a.launch()
    L.sync()
    a.compare()


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("tokens, page", [(1, 16), (2, 4096), (1023, 32), (1024, 16), (2500, 64)])
def test_append_lengths(nn, L, rng, kind, dtype, tokens, page):
    print(f"[case] append {kind} {dtype} {tokens} tokens, pages of {page}", flush=True)
    first = 5
    cache = Cache(nn, L, rng, kind, dtype, 2, 64, page, [-(-(first + tokens) // page)])
    a = Append(nn, L, rng, cache, np.zeros(tokens, int), first + np.arange(tokens), 3, 64)
    a.launch()
    L.sync()
    a.compare()


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_append_without_requests(nn, L, rng, kind, dtype):
    """A decoding step: row t is of request t."""
    cache = Cache(nn, L, rng, kind, dtype, 1, 32, 16, [2] * 9)
    a = Append(nn, L, rng, cache, np.arange(9), np.array([0, 1, 15, 16, 31, 7, -1, 20, 3]), 4, 32, given_request=False)
    a.launch()
    L.sync()
    a.compare()


@pytest.mark.parametrize("kind, dtype", KINDS)
def test_append_to_what_is_no_page(nn, L, rng, kind, dtype):
    """Entries outside of the pool, places past the table and requests that are none: queries alone are written."""
    cache = Cache(nn, L, rng, kind, dtype, 2, 48, 16, [2, 2, 2], width=3)
    cache.table[0, 0], cache.table[1, 1], cache.table[2] = -7, cache.pages, [2**31 - 1, -(2**31), cache.table[2, 0]]
    cache.table_dev = ints(L, cache.table)
    cache.args.table = cache.table_dev.p
    place = np.array([0, 17, 5, 20, 3, 18, 33, 48, 2**31 - 1, 1, 1, 1])
    request = np.array([0, 0, 1, 1, 2, 2, 2, 2, 0, 3, -1, 2**31 - 1])
    a = Append(nn, L, rng, cache, request, place, 4, 32)
    a.launch()
    L.sync()
    a.compare()


def test_four_bits_at_their_borders(nn, L, rng):
    """Values on borders go to the even code, sizes near the ends of the range are kept or end as they should."""
    cache = Cache(nn, L, rng, "mxfp4", "f32", 1, 32, 16, [2])
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    rows = np.zeros((12, 1, 32))
    rows[0, 0, :8] = borders
    rows[1, 0, :8] = -borders
    rows[2, 0, :8] = np.nextafter(borders.astype(np.float32), np.float32(0)).astype(np.float64)
    rows[3, 0, :7] = np.nextafter(borders[:7].astype(np.float32), np.float32(9)).astype(np.float64)
    rows[3, 0, 7] = 7
    rows[4, 0, 0] = np.nextafter(np.float32(7), np.float32(8))
    rows[5, 0, :3] = [3.4e38, -3.3e38, 2.0**125]
    rows[6, 0, :3] = [1e-45, -1e-38, 0]
    rows[7, 0, :4] = 2.0**-120 * np.array([0.5, 1, -3, 7])
    rows[8] = 0
    rows[9, 0, :2] = [np.inf, 1]
    rows[10, 0, :2] = [1, np.nan]
    rows[11, 0] = rng.standard_normal(32) * 2.0**100
    values = {"q": np.zeros((12, 0, 32)), "k": rows.copy(), "v": rows.copy()}
    a = Append(nn, L, rng, cache, np.zeros(12, int), np.arange(12), 0, 0, norm=False, values=values)
    a.launch()
    L.sync()
    rows = rows.astype(np.float32).astype(np.float64)
    for name in ("k", "v"):
        got = cache.download(name)
        for t in range(12):
            cache.put(name, cache.where(0, t), rows[t])
            have, want = cache.get(name, cache.where(0, t), got), cache.get(name, cache.where(0, t))
            assert np.array_equal(have, want, equal_nan=True), (name, t, have, want)


@pytest.mark.parametrize("kind, dtype", KINDS)
@pytest.mark.parametrize("kv, dim, odd", [(2, 128, False), (1, 33, True), (3, 72, False), (1, 1, True), (2, 20, False)])
def test_read(nn, L, rng, kind, dtype, kv, dim, odd):
    """Every value exactly, in any order and twice; rows that are no tokens stay, entries that are no page give zeros."""
    cache = Cache(nn, L, rng, kind, dtype, kv, dim, 16, [2, 3], width=3)
    cache.fill(rng, [21, 48], spoil=False)
    place = np.array([20, 0, 5, 5, -1, 47, 16, 33, 0, 15, 40, 1])
    request = np.array([0, 0, 0, 0, 1, 1, 1, 0, 1, 1, 2, -1])
    stride = (kv * (dim + 1) + 2, dim + 1, 1) if odd else None
    out = {n: Tensor(L, (len(place), kv, dim), dtype, stride, int(odd), fill=7.0) for n in ("k", "v")}
    keep = [ints(L, request), ints(L, place)]
    a = nn.NnCacheRead(dtype=cache.nn_dtype(), tokens=len(place), kv_heads=kv, head_dim=dim, k_stride=out["k"].strides[:2],
                       v_stride=out["v"].strides[:2], request=keep[0].p, place=keep[1].p)
    L.launch_cache_read(out["k"].p, out["v"].p, a, cache.args, None)
    L.sync()
    for n in ("k", "v"):
        got = out[n].result()
        for t in range(len(place)):
            at = cache.where(int(request[t]), int(place[t]))
            want = np.full((kv, dim), 7.0) if place[t] < 0 else np.zeros((kv, dim)) if at is None else cache.get(n, at)
            assert np.array_equal(got[t], rounded(want, dtype).astype(np.float64)), (n, t)


def test_append_in_place(nn, L, rng):
    """q_out may be q."""
    cache = Cache(nn, L, rng, "mxfp4", "bf16", 2, 64, 16, [4])
    a = Append(nn, L, rng, cache, np.zeros(40, int), np.arange(40), 6, 64)
    ref = a.rows("q")
    a.args.rope.q_out_stride = a.args.rope.q_stride
    L.launch_cache_append(a.t["q"].p, a.t["q"].p, a.t["k"].p, a.t["v"].p, a.args, cache.args, None)
    L.sync()
    got = a.t["q"].view(a.t["q"].flat()).astype(np.float64)
    check("q", got, ref, np.broadcast_to(np.abs(ref).max(-1, keepdims=True), ref.shape), "bf16")


def test_pools_past_32_bits(nn, L, rng):
    """Pages whose offsets need more than 32 bits: pools of 4.3 GB each, three of their pages in use."""
    tokens, kv, dim = 4096, 8, 128
    size = tokens * 68 * kv
    pages = (1 << 32) // size + 3
    pool = {n: L.alloc(pages * size // 4) for n in ("k", "v")}
    table = ints(L, [[pages - 1, 0, pages // 2]])
    args = nn.NnCache(kind=nn.NN_CACHE_MXFP4, page_tokens=tokens, pages=pages, requests=1, table_pages=3, table=table.p,
                      k=pool["k"].p, v=pool["v"].p)
    place = np.array([5, 4095, 4096, 8191, 8192, 12287])
    t = len(place)
    x = {n: rounded(rng.standard_normal((t, kv, dim)), "bf16") for n in ("k", "v")}
    src = {n: Tensor(L, (t, kv, dim), "bf16", values=x[n]) for n in x}
    out = {n: Tensor(L, (t, kv, dim), "bf16") for n in x}
    zeros, keep = ints(L, np.zeros(t)), ints(L, place)
    rope = nn.NnQkNormRope(dtype=nn.NN_BF16, tokens=t, kv_heads=kv, head_dim=dim, axes=1, k_stride=(kv * dim, dim))
    a = nn.NnCacheAppend(rope=rope, v_stride=(kv * dim, dim), request=zeros.p, place=keep.p)
    r = nn.NnCacheRead(dtype=nn.NN_BF16, tokens=t, kv_heads=kv, head_dim=dim, k_stride=(kv * dim, dim),
                       v_stride=(kv * dim, dim), request=zeros.p, place=keep.p)
    L.launch_cache_append(None, None, src["k"].p, src["v"].p, a, args, None)
    L.launch_cache_read(out["k"].p, out["v"].p, r, args, None)
    L.sync()
    from cache_ref import codes, unpacked

    for n in x:
        code, e, _ = codes(x[n].astype(np.float64))
        assert np.array_equal(out[n].result(), unpacked(code, e, dim)), n
