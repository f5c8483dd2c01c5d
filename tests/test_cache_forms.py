"""Which form of attention over a paged cache a call takes (csrc/k_cache_few.hip, nnk_cache_is_few)."""
from __future__ import annotations

import ctypes

import pytest


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
