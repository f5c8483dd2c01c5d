"""Attention to many queries by workgroups whose waves share a block's keys: what their parts add up to."""
from __future__ import annotations

import numpy as np
import pytest

import test_gpu_attention as plain
import test_gpu_cache_attention as paged
from attention_ref import Tensor
from test_cache_forms import is_few
from test_gpu_attention import case

pytestmark = pytest.mark.gpu

CAP, KEY = 50.0, 64.0
SHARE = CAP * np.log2(np.e) * np.tanh(KEY / CAP)  # units of log2: of a key of this score, where the first ones' is 0
VALUE = 2.0 ** np.floor(127.9 - SHARE)            # with it past 2^127, and two of them past fp32's range


def rows(b, len_k, heads, dim):
    """Keys of score 0 and values of 0, but for one key in each half of the second block of 64."""
    k, v = np.zeros((b, len_k, heads, dim)), np.zeros((b, len_k, heads, dim))
    k[:, [70, 100], :, 0] = KEY
    v[:, [70, 100]] = VALUE
    return k, v


def test_the_sums_are_near_the_end_of_the_type():
    assert 2.0**127 < 2.0**SHARE * VALUE < 2.0**128


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tensors(nn, L, rng, dtype):
    """Each half's sum fits in fp32, both do not, and the mean is an ordinary value."""
    c = case(dtype, 2, 70, 192, 3, 3, 8, "none", CAP, scale=1.0)
    call = plain.Call(nn, L, rng, c, backward=False, spoil=False)
    k, v = rows(2, 192, 3, 8)
    q = np.zeros((2, 70, 3, 8))
    q[..., 0] = 1
    call.t.update(q=Tensor(L, q.shape, dtype, values=q), k=Tensor(L, k.shape, dtype, values=k), v=Tensor(L, v.shape, dtype, values=v))
    call.forward()
    L.sync()
    call.compare(CAP)


@pytest.mark.parametrize("kind, dtype", [("plain", "bf16"), ("plain", "f32"), ("mxfp4", "bf16")])
def test_pages(nn, L, rng, kind, dtype):
    """The same out of a paged cache."""
    b, len_q, heads, dim = 16, 140, 4, 32
    c = case(dtype, b, len_q, 192, heads, heads, dim, "none", CAP, scale=1.0)
    assert not is_few(nn, dtype, kind, b, len_q, 192, heads, heads, dim)
    call = paged.Call(nn, L, rng, c, kind, 64)
    k, v = rows(1, 192, heads, dim)
    for table in call.cache.table:
        for i, page in enumerate(table):
            for name, x in (("k", k), ("v", v)):
                call.cache._put_page(name, page, x[0, 64 * i:64 * i + 64])
    call.cache.upload()
    q = np.zeros((b, len_q, heads, dim))
    q[..., 0] = 1
    call.q = Tensor(L, q.shape, dtype, values=q)
    call.launch()
    L.sync()
    call.compare(CAP)
