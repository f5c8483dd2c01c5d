"""Pages of 4 bits that a program filled itself: every scale that the layout has, those among them that no append writes."""
from __future__ import annotations

import numpy as np
import pytest

from cache_ref import SIZES, Cache, Tensor, ints
from test_cache_forms import is_few
from test_gpu_attention import case
from test_gpu_cache_attention import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [32, 40])
def test_read_every_scale_and_code(nn, L, rng, dtype, dim):
    """Code c under scale s is size(c) 2^(s - 127), from 2^-128 to past the type's end (infinite); 255 makes NaN."""
    groups, tokens = -(-dim // 32), 256
    cache = Cache(nn, L, rng, "mxfp4", dtype, 1, dim, 256, [1])
    page = cache.table[0, 0]
    code = np.tile(np.arange(16, dtype=np.uint8), (tokens, 2 * groups))
    to = cache.bytes["k"][page, 0]
    to[:tokens * cache.row] = (code[:, 0::2] | code[:, 1::2] << 4).ravel()
    to[tokens * cache.row:] = np.repeat(np.arange(256), groups)
    cache.bytes["v"][page] = cache.bytes["k"][page]
    cache.upload()
    out = {n: Tensor(L, (tokens, 1, dim), dtype, fill=7.0) for n in "kv"}
    zeros, place = ints(L, np.zeros(tokens)), ints(L, np.arange(tokens))
    L.launch_cache_read(out["k"].p, out["v"].p, nn.NnCacheRead(
        dtype=cache.nn_dtype(), tokens=tokens, kv_heads=1, head_dim=dim, k_stride=(dim, dim), v_stride=(dim, dim),
        request=zeros.p, place=place.p), cache.args, None)
    L.sync()
    sign = np.where(code & 8, -1.0, 1.0)
    with np.errstate(over="ignore"):
        want = (SIZES[code & 7] * sign * 2.0 ** (np.arange(256) - 127.0)[:, None]).astype(np.float32)
    want[255] = np.nan
    want = want[:, None, :dim]
    for n in "kv":
        got = out[n].result()
        off = ~((got == want) | (np.isnan(got) & np.isnan(want)))
        assert not off.any(), (n, sorted(set(np.nonzero(off)[0])), got[off][:8], want[off][:8])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 3, 400, 4, 2), (16, 140, 192, 4, 4)])
@pytest.mark.parametrize("k_power, v_power", [(60, 60), (-60, -60), (100, -40)])
def test_attention_with_far_scales(nn, L, rng, dtype, shape, k_power, v_power):
    """Keys and values far from 1, queries as far the other way, by the form for few queries and, in bf16, the one for many."""
    b, len_q, len_k, heads, kv = shape
    c = case(dtype, b, len_q, len_k, heads, kv, 64, "causal")
    assert is_few(nn, dtype, "mxfp4", b, len_q, len_k, heads, kv, 64) == (dtype == "f32" or len_q == 3)
    call = Call(nn, L, rng, c, "mxfp4", 16)
    for n, power in (("k", k_power), ("v", v_power)):
        scales = call.cache.bytes[n][:, :, call.cache.tokens * call.cache.row:]
        scales[...] = np.where(scales < 255, np.clip(scales.astype(int) + power, 0, 254), 255)
    call.cache.upload()
    call.q = Tensor(L, call.q.shape, dtype, values=call.q.values() * 2.0**-k_power)
    call.launch()
    L.sync()
    call.compare()
