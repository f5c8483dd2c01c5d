"""A layer that serves requests out of a paged cache: prompts of different lengths, then tokens one by one.

Two requests share a pool of pages. Their prompts come as one padded batch: the projection's rows
are normalised, turned by their positions and appended (launch_cache_append), and attention reads
the pages (launch_cache_attention_forward). Then every step appends one token of each request; a
request takes a page from the pool when its last one is full. At the end what the pages hold is
read back (launch_cache_read), and the last step is formed again by attention over plain tensors
of it: both agree.

    python examples/paged_decoding.py [steps]
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

from __graft_entry__ import load_package  # noqa: E402

HEADS, KV, DIM, PAGE, PAGES, MOST = 8, 2, 64, 16, 24, 12  # MOST: pages of a request
ROW = (HEADS + 2 * KV) * DIM


def ints(L, x):
    return L.to_device(np.ascontiguousarray(x, np.int32).view(np.float32))


class Layer:
    def __init__(self, nn, L, kind, rng):
        self.nn, self.L, self.kind = nn, L, kind
        self.free = list(rng.permutation(PAGES))
        self.table = np.full((2, MOST), -1, np.int32)
        self.held = np.zeros(2, np.int32)
        self.table_dev = ints(L, self.table)
        self.weights = [L.to_device((1 + 0.1 * rng.standard_normal(DIM)).astype(np.float32)) for _ in range(2)]
        self.freq = L.to_device((10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))).view(np.float32))
        self.cache = nn.NnCache(kind=kind, page_tokens=PAGE, pages=PAGES, requests=2, table_pages=MOST, table=self.table_dev.p)
        page = L.nnhip_cache_page_bytes(self.cache, nn.NN_F32, KV, DIM)
        self.pools = [L.alloc(PAGES * page // 4) for _ in range(2)]
        self.cache.k, self.cache.v = (p.p for p in self.pools)
        largest = self.attention(2, 1, MOST * PAGE)  # its workspace serves every smaller call
        self.workspace = L.to_device(np.zeros(max(1, *(L.nnhip_cache_attention_workspace(a, self.cache)
                                                       for a in (largest, self.attention(2, 64, MOST * PAGE)))), np.float32))

    def attention(self, batch, length, keys, **more):
        return self.nn.NnAttention(
            dtype=self.nn.NN_F32, batch=batch, len_q=length, len_k=keys, heads=HEADS, kv_heads=KV, head_dim=DIM,
            scale=DIM**-0.5, mask=self.nn.NN_MASK_CAUSAL, q_stride=(length * HEADS * DIM, HEADS * DIM, DIM),
            out_stride=(length * HEADS * DIM, HEADS * DIM, DIM), **more)

    def step(self, rows, lengths):
        """Appends lengths[r] tokens to request r, whose rows are the first of rows[r], and gives their outputs."""
        nn, L, n = self.nn, self.L, rows.shape[1]
        place = np.full((2, n), -1, np.int32)  # rows behind a request's tokens are none
        for r in range(2):
            place[r, :lengths[r]] = self.held[r] + np.arange(lengths[r])
            while (self.table[r] >= 0).sum() * PAGE < self.held[r] + lengths[r]:
                self.table[r, (self.table[r] >= 0).sum()] = self.free.pop()
        start, self.held = self.held.copy(), self.held + np.asarray(lengths, np.int32)
        self.table_dev.upload(self.table.view(np.float32))
        x, q, out, lse = L.to_device(rows.astype(np.float32)), L.alloc(2 * n * HEADS * DIM), L.alloc(2 * n * HEADS * DIM), L.alloc(2 * n * HEADS)
        request, place_dev, first, held = ints(L, np.repeat([0, 1], n)), ints(L, place), ints(L, start), ints(L, self.held)
        pos = ints(L, np.maximum(place, 0))
        rope = nn.NnQkNormRope(
            dtype=nn.NN_F32, tokens=2 * n, heads=HEADS, kv_heads=KV, head_dim=DIM, rot_dim=DIM, axes=1, eps=1e-6,
            q_stride=(ROW, DIM), k_stride=(ROW, DIM), q_out_stride=(HEADS * DIM, DIM), q_weight=self.weights[0].p,
            k_weight=self.weights[1].p, pos=pos.p, freq=self.freq.p)
        append = nn.NnCacheAppend(rope=rope, norm=1, v_stride=(ROW, DIM), request=request.p, place=place_dev.p)
        L.launch_cache_append(q.p, x.p, x.offset(HEADS * DIM), x.offset((HEADS + KV) * DIM), append, self.cache, None)
        a = self.attention(2, n, int(self.held.max()), q_start=first.p, k_len=held.p)
        L.launch_cache_attention_forward(out.p, lse.p, q.p, a, self.cache, self.workspace.p, None)
        L.sync()
        return q.download(shape=(2, n, HEADS, DIM)), out.download(shape=(2, n, HEADS, DIM))

    def rows(self, r):
        """Keys and values of request r, [tokens, KV, DIM]."""
        nn, L, n = self.nn, self.L, int(self.held[r])
        request, place = ints(L, np.full(n, r)), ints(L, np.arange(n))
        out = [L.alloc(n * KV * DIM) for _ in range(2)]
        read = nn.NnCacheRead(dtype=nn.NN_F32, tokens=n, kv_heads=KV, head_dim=DIM, k_stride=(KV * DIM, DIM),
                              v_stride=(KV * DIM, DIM), request=request.p, place=place.p)
        L.launch_cache_read(out[0].p, out[1].p, read, self.cache, None)
        L.sync()
        return out


def serve(nn, L, kind, steps=20, seed=0):
    """Largest difference of the last step's outputs from attention over plain tensors of what the pages hold."""
    rng = np.random.default_rng(seed)
    layer = Layer(nn, L, kind, rng)
    layer.step(rng.standard_normal((2, 61, ROW)), [61, 23])
    for _ in range(steps):
        q, got = layer.step(rng.standard_normal((2, 1, ROW)), [1, 1])
    off = 0.0
    for r in range(2):
        k, v = layer.rows(r)
        a = layer.attention(1, 1, int(layer.held[r]), k_stride=(0, KV * DIM, DIM), v_stride=(0, KV * DIM, DIM))
        out, lse, mine = L.alloc(HEADS * DIM), L.alloc(HEADS), L.to_device(q[r])
        ws = L.to_device(np.zeros(max(1, L.nnhip_attention_forward_workspace(a)), np.float32))
        L.launch_attention_forward(out.p, lse.p, mine.p, k.p, v.p, a, ws.p, None)
        L.sync()
        off = max(off, float(np.abs(out.download(shape=(1, HEADS, DIM)) - got[r]).max()))
    return off


def main():
    nn = load_package()
    L = nn.lib()
    steps = int(sys.argv[1]) if len(sys.argv) > 1 else 20
    for name, kind in (("fp32", nn.NN_CACHE_PLAIN), ("4-bit", nn.NN_CACHE_MXFP4)):
        print(f"{name} pages: off by {serve(nn, L, kind, steps):.2e} at most")


if __name__ == "__main__":
    main()
