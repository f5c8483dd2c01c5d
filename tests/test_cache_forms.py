"""Which form of attention over a paged cache a call takes (csrc/k_cache_few.hip, nnk_cache_is_few)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_ref import Cache, Tensor, ints
from attention_ref import check


def is_few(nn, dtype, kind, batch, len_q, len_k, heads, kv_heads, head_dim):
    f = nn.lib().dll.nnk_cache_is_few
    f.argtypes, f.restype = [ctypes.POINTER(nn.NnAttention), ctypes.c_int], ctypes.c_int
    a = nn.NnAttention(dtype=nn.NN_BF16 if dtype == "bf16" else nn.NN_F32, batch=batch, len_q=len_q, len_k=len_k, heads=heads,
                       kv_heads=kv_heads, head_dim=head_dim)
    return bool(f(a, kind == "mxfp4"))


# microseconds on an MI355X of the form for few queries and of the one for many, where one is 9 % longer at least
MEASURED = [
    # one token of requests whose heads share no keys
    ("bf16", "plain", 16, 1, 32768, 32, 32, 128, 1241, 1377), ("bf16", "plain", 32, 1, 4096, 32, 32, 128, 317, 351),
    ("bf16", "plain", 64, 1, 32768, 32, 32, 128, 5000, 5551), ("bf16", "plain", 48, 1, 32768, 8, 8, 128, 642, 847),
    ("bf16", "plain", 43, 1, 4096, 8, 8, 128, 83, 110), ("bf16", "plain", 300, 1, 9000, 8, 8, 32, 301, 364),
    ("f32", "plain", 16, 1, 4096, 32, 32, 128, 460, 1156), ("f32", "plain", 64, 1, 32768, 32, 32, 128, 11520, 36165),
    ("f32", "plain", 256, 1, 512, 16, 16, 64, 173, 491), ("f32", "plain", 2000, 1, 128, 12, 12, 64, 442, 1122),
    ("f32", "plain", 64, 1, 64, 16, 16, 128, 40, 58), ("bf16", "mxfp4", 48, 1, 32768, 8, 8, 128, 197, 602),
    # few keys
    ("bf16", "plain", 1, 1, 200, 8, 2, 128, 10.0, 11.2), ("bf16", "plain", 1, 6, 200, 8, 2, 128, 13.6, 11.9),
    ("f32", "plain", 1, 1, 130, 8, 2, 128, 13.6, 23.3), ("f32", "plain", 4, 6, 280, 8, 2, 128, 24.9, 34.8),
    ("bf16", "mxfp4", 4, 1, 200, 32, 8, 128, 9.6, 11.5), ("bf16", "mxfp4", 4, 6, 130, 32, 8, 128, 13.4, 10.4),
    # one token, shared key heads
    ("bf16", "plain", 32, 1, 4096, 32, 8, 128, 70, 187), ("f32", "plain", 64, 1, 4096, 64, 32, 128, 1066, 5765),
    ("bf16", "mxfp4", 64, 1, 2048, 32, 16, 128, 47, 165),
    # several tokens of many requests
    ("bf16", "plain", 64, 16, 300, 8, 8, 128, 36, 20), ("f32", "plain", 64, 16, 300, 8, 8, 128, 53, 106),
    ("bf16", "mxfp4", 64, 16, 300, 8, 8, 128, 31, 16), ("f32", "plain", 64, 32, 2048, 8, 8, 128, 319, 594),
    ("bf16", "mxfp4", 64, 32, 300, 8, 8, 128, 38, 16), ("bf16", "plain", 64, 40, 2048, 16, 16, 128, 251, 145),
    ("bf16", "mxfp4", 16, 64, 1024, 16, 4, 128, 48, 28), ("bf16", "mxfp4", 32, 20, 4096, 32, 16, 128, 110, 178),
    # prompts and chunks
    ("bf16", "plain", 1, 2048, 16384, 16, 4, 128, 881, 443), ("f32", "plain", 1, 2048, 16384, 16, 4, 128, 3953, 2555),
    ("bf16", "mxfp4", 1, 2048, 16384, 16, 4, 128, 369, 402), ("bf16", "mxfp4", 8, 128, 2048, 16, 4, 128, 60, 48),
    ("bf16", "mxfp4", 2, 256, 8192, 16, 4, 128, 68, 161), ("bf16", "plain", 3, 150, 3000, 6, 2, 96, 34, 61),
    ("f32", "plain", 4, 300, 300, 8, 8, 64, 33, 22),
]


@pytest.mark.parametrize("case", MEASURED, ids=lambda c: "-".join(map(str, c[:8])))
def test_the_quicker_form_is_taken(nn, case):
    few, many = case[8:]
    assert is_few(nn, *case[:8]) == (few < many)


def test_fp32_queries_over_four_bits(nn):
    assert is_few(nn, "f32", "mxfp4", 1, 2048, 16384, 16, 4, 128)


DUMMY, FAR = 16, 1 << 40  # never dereferenced
# more (request, head) pairs than a launch has workgroups, fewer units: 128 heads of one key head are four of these
MANY, HEADS = 131100, 128


def _cache(nn, kind, requests, table_pages):
    return nn.NnCache(kind=nn.NN_CACHE_MXFP4 if kind == "mxfp4" else nn.NN_CACHE_PLAIN, page_tokens=16, pages=1,
                      requests=requests, table_pages=table_pages, table=DUMMY, k=DUMMY, v=FAR)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["plain", "mxfp4"])
def test_sizes_are_those_of_the_form_taken(nn, dtype, kind):
    """What a launch of the form for few queries has room for is not refused for the other form's workgroups."""
    L = nn.lib()
    L.last_error()
    t = nn.NN_BF16 if dtype == "bf16" else nn.NN_F32
    a = nn.NnAttention(dtype=t, batch=MANY, len_q=1, len_k=200, heads=HEADS, kv_heads=1, head_dim=8)
    assert is_few(nn, dtype, kind, MANY, 1, 200, HEADS, 1, 8)
    assert L.nnhip_cache_attention_workspace(a, _cache(nn, kind, MANY, 13)) > 0
    a.batch = 1 << 22  # units past a launch
    with pytest.raises(nn.NnHipError, match="nnhip_cache_attention_workspace: error 1: .*too many rows"):
        L.nnhip_cache_attention_workspace(a, _cache(nn, kind, a.batch, 13))
    assert L.last_error()[0] == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["plain", "mxfp4"])
@pytest.mark.parametrize("len_q", [1 << 17, (1 << 17) + 32, (1 << 18) - 128])
def test_tiles_past_32_bits(nn, dtype, kind, len_q):
    """2^20 heads of one key head: 2^32 tiles of queries and more, which are too many, not the few that 32 bits hold of them."""
    L = nn.lib()
    L.last_error()
    t = nn.NN_BF16 if dtype == "bf16" else nn.NN_F32
    a = nn.NnAttention(dtype=t, batch=1, len_q=len_q, len_k=200, heads=1 << 20, kv_heads=1, head_dim=8, scale=1.0,
                       q_stride=(0, 0, 8), out_stride=(0, 8 << 20, 8))
    c = _cache(nn, kind, 1, 13)
    with pytest.raises(nn.NnHipError, match="nnhip_cache_attention_workspace: error 1: .*too many rows"):
        L.nnhip_cache_attention_workspace(a, c)
    with pytest.raises(nn.NnHipError, match="launch_cache_attention_forward: error 1: .*too many rows"):
        L.launch_cache_attention_forward(DUMMY, DUMMY, DUMMY, a, c, DUMMY, None)
    assert L.last_error()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "mxfp4"])
def test_more_heads_than_a_launch_has_workgroups(nn, L, rng, kind):
    """Every request has the same page and the same queries (strides of 0), and a result of its own."""
    from test_gpu_attention import case
    from test_gpu_cache_attention import Call

    dim, len_k = 8, 13
    cache = Cache(nn, L, rng, kind, "bf16", 1, dim, 16, [1])
    cache.fill(rng, [len_k])
    one = Call(nn, L, rng, case("bf16", 1, 1, len_k, HEADS, 1, dim), kind, 16, cache=cache)
    one.launch()
    L.sync()
    one.compare()
    ref, mag = one.expected()
    table = ints(L, np.repeat(cache.table, MANY, 0))
    many = nn.NnCache(kind=cache.args.kind, page_tokens=16, pages=cache.pages, requests=MANY, table_pages=1, table=table.p,
                      k=cache.dev["k"].p, v=cache.dev["v"].p)
    out, lse = Tensor(L, (MANY, 1, HEADS, dim), "bf16"), L.alloc(MANY * HEADS)
    a = nn.NnAttention(dtype=nn.NN_BF16, batch=MANY, len_q=1, len_k=len_k, heads=HEADS, kv_heads=1, head_dim=dim,
                       scale=dim**-0.5, mask=nn.NN_MASK_NONE, q_stride=(0, 0, dim), out_stride=out.strides[:3])
    assert L.nnhip_cache_attention_workspace(a, many) == 0
    L.launch_cache_attention_forward(out.p, lse.p, one.q.p, a, many, None, None)
    L.sync()
    got, sums = out.result(), lse.download(shape=(MANY, HEADS, 1))
    assert (got == got[:1]).all() and (sums == sums[:1]).all()
    check("out", got[:1], ref["out"], mag["out"], "bf16")
    check("lse", sums[:1].astype(np.float64), ref["lse"], mag["lse"], "f32")
