"""The paged cache's host side: refusals, sizes, calls with nothing to do, and the tests' own 4 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_ref import SIZES, codes, exponents, unpacked

DUMMY = 16  # never dereferenced: every check of the host comes before a launch
FAR = 1 << 40


def _cache(nn, **more):
    a = dict(kind=nn.NN_CACHE_MXFP4, page_tokens=16, pages=4, requests=2, table_pages=2, table=DUMMY, k=DUMMY, v=FAR)
    a.update(more)
    return nn.NnCache(**a)


def _append(nn, **more):
    rope = dict(dtype=nn.NN_F32, tokens=4, heads=2, kv_heads=1, head_dim=8, rot_dim=8, axes=1, interleaved=0, eps=1e-6,
                q_stride=(16, 8), k_stride=(8, 8), q_out_stride=(16, 8), pos=DUMMY, freq=DUMMY)
    own = dict(norm=1, v_stride=(8, 8), place=DUMMY)
    for k, v in more.items():
        (own if k in own or k == "request" else rope)[k] = v
    return nn.NnCacheAppend(rope=nn.NnQkNormRope(**rope), **own)


def _read(nn, **more):
    a = dict(dtype=nn.NN_F32, tokens=4, kv_heads=1, head_dim=8, k_stride=(8, 8), v_stride=(8, 8), place=DUMMY)
    a.update(more)
    return nn.NnCacheRead(**a)


def _attn(nn, **more):
    a = dict(dtype=nn.NN_F32, batch=1, len_q=4, len_k=32, heads=2, kv_heads=1, head_dim=8, scale=0.3, softcap=0.0,
             mask=nn.NN_MASK_CAUSAL, q_stride=(64, 16, 8), out_stride=(64, 16, 8))
    a.update(more)
    return nn.NnAttention(**a)


def _calls(nn, cache):
    """Every call on a cache, as (name, function)."""
    L = nn.lib()
    return [
        ("launch_cache_append", lambda: L.launch_cache_append(DUMMY, DUMMY, DUMMY, DUMMY, _append(nn), cache, None)),
        ("launch_cache_read", lambda: L.launch_cache_read(DUMMY, DUMMY, _read(nn), cache, None)),
        ("launch_cache_attention_forward",
         lambda: L.launch_cache_attention_forward(DUMMY, DUMMY, DUMMY, _attn(nn), cache, DUMMY, None)),
    ]


BAD_CACHE = [
    (dict(kind=2), "unknown kind of cache 2"),
    (dict(page_tokens=8), "page_tokens=8"),
    (dict(page_tokens=48), "page_tokens=48"),
    (dict(page_tokens=0), "page_tokens=0"),
    (dict(page_tokens=-16), "page_tokens=-16"),
    (dict(page_tokens=8192), "page_tokens=8192"),
    (dict(pages=-1), "pages=-1"),
    (dict(requests=-1), "requests=-1"),
    (dict(table_pages=-1), "table_pages=-1"),
    (dict(table_pages=1 << 26), "are too many"),
    (dict(table=None), "null table"),
    (dict(k=None), "null pool"),
    (dict(v=None), "null pool"),
    (dict(k=24), "not aligned"),
    (dict(v=FAR + 4), "not aligned"),
    (dict(v=DUMMY), "overlap"),
    (dict(v=DUMMY + 4 * 16 * 17 - 16), "overlap"),
]


@pytest.mark.parametrize("more, text", BAD_CACHE, ids=[f"{n}-{t}" for n, (_, t) in enumerate(BAD_CACHE)])
def test_cache_refusals(nn, more, text):
    L = nn.lib()
    L.last_error()
    for name, call in _calls(nn, _cache(nn, **more)):
        with pytest.raises(nn.NnHipError, match=f"{name}: error 1: .*{text}"):
            call()
    assert L.last_error()[0] == 0


def test_null_descriptions(nn):
    L = nn.lib()
    L.last_error()
    for _, call in _calls(nn, None):
        with pytest.raises(nn.NnHipError, match="null cache"):
            call()
    c = _cache(nn)
    with pytest.raises(nn.NnHipError, match="null description"):
        L.launch_cache_append(DUMMY, DUMMY, DUMMY, DUMMY, None, c, None)
    with pytest.raises(nn.NnHipError, match="null description"):
        L.launch_cache_read(DUMMY, DUMMY, None, c, None)
    with pytest.raises(nn.NnHipError, match="null description"):
        L.launch_cache_attention_forward(DUMMY, DUMMY, DUMMY, None, c, DUMMY, None)
    with pytest.raises(nn.NnHipError, match="null description"):
        L.nnhip_cache_attention_workspace(None, c)


BAD_APPEND = [
    (dict(dtype=3), "unknown dtype 3"),
    (dict(tokens=-1), "tokens=-1"),
    (dict(heads=-1), "heads=-1"),
    (dict(kv_heads=0), "kv_heads=0"),
    (dict(head_dim=129, rot_dim=0), "head_dim=129"),
    (dict(head_dim=0, rot_dim=0), "head_dim=0"),
    (dict(rot_dim=10), "rot_dim=10"),
    (dict(rot_dim=3), "rot_dim=3"),
    (dict(axes=3), "axes=3"),
    (dict(axes=0), "axes=0"),
    (dict(eps=-1.0), "eps=-1"),
    (dict(eps=float("nan")), "eps=nan"),
    (dict(pos=None), "null pos or freq"),
    (dict(freq=None), "null pos or freq"),
    (dict(place=None), "null place"),
    (dict(tokens=1 << 28), "too many rows"),
    (dict(q_out_stride=(8, 8)), "rows of q_out overlap"),
    (dict(q_out_stride=(16, 4)), "rows of q_out overlap"),
]


@pytest.mark.parametrize("more, text", BAD_APPEND, ids=[f"{n}-{t}" for n, (_, t) in enumerate(BAD_APPEND)])
def test_append_refusals(nn, more, text):
    L = nn.lib()
    L.last_error()
    with pytest.raises(nn.NnHipError, match=f"launch_cache_append: error 1: .*{text}"):
        L.launch_cache_append(DUMMY, DUMMY, DUMMY, DUMMY, _append(nn, **more), _cache(nn), None)
    assert L.last_error()[0] == 0


BAD_READ = [
    (dict(dtype=3), "unknown dtype 3"),
    (dict(tokens=-1), "tokens=-1"),
    (dict(kv_heads=0), "kv_heads=0"),
    (dict(head_dim=129), "head_dim=129"),
    (dict(place=None), "null place"),
    (dict(k_stride=(0, 8)), "rows of k overlap"),
    (dict(v_stride=(4, 8)), "rows of v overlap"),
    (dict(tokens=1 << 30), "too many rows"),
]


@pytest.mark.parametrize("more, text", BAD_READ, ids=[t for _, t in BAD_READ])
def test_read_refusals(nn, more, text):
    L = nn.lib()
    L.last_error()
    with pytest.raises(nn.NnHipError, match=f"launch_cache_read: error 1: .*{text}"):
        L.launch_cache_read(DUMMY, DUMMY, _read(nn, **more), _cache(nn), None)
    assert L.last_error()[0] == 0


BAD_ATTN = [
    (dict(dtype=7), "unknown dtype 7"),
    (dict(batch=-1), "bad shape"),
    (dict(batch=3), "batch=3 of a cache of 2 requests"),
    (dict(len_q=-2), "bad shape"),
    (dict(len_k=33), "len_k=33 does not fit"),
    (dict(heads=3, kv_heads=2), "not a multiple of kv_heads"),
    (dict(kv_heads=0), "kv_heads=0"),
    (dict(head_dim=129), "head_dim=129"),
    (dict(scale=0.0), "scale=0"),
    (dict(softcap=-1.0), "softcap=-1"),
    (dict(mask=9), "unknown mask 9"),
    (dict(mask=2), "null prefix"),
    (dict(doc_q=DUMMY, doc_k=DUMMY), "documents"),
    (dict(buckets=4, max_distance=4), "null bucket or bias"),
    (dict(buckets=4, max_distance=1024, bucket=DUMMY, bias=DUMMY), "max_distance=1024"),
    (dict(out_stride=(64, 8, 8)), "rows of out overlap"),
    (dict(len_q=1 << 30), "bad shape"),
]


@pytest.mark.parametrize("more, text", BAD_ATTN, ids=[f"{n}-{t}" for n, (_, t) in enumerate(BAD_ATTN)])
def test_attention_refusals(nn, more, text):
    L = nn.lib()
    L.last_error()
    with pytest.raises(nn.NnHipError, match=f"launch_cache_attention_forward: error 1: .*{text}"):
        L.launch_cache_attention_forward(DUMMY, DUMMY, DUMMY, _attn(nn, **more), _cache(nn), DUMMY, None)
    assert L.last_error()[0] == 0


BAD_SIZES = [
    (dict(dtype=7), "unknown dtype 7"),
    (dict(batch=-1), "bad shape"),
    (dict(batch=3), "batch=3 of a cache of 2 requests"),
    (dict(len_q=-2), "bad shape"),
    (dict(len_q=1 << 30), "bad shape"),
    (dict(len_k=-1), "bad shape"),
    (dict(len_k=1 << 20), "does not fit"),
    (dict(heads=3, kv_heads=2), "not a multiple of kv_heads"),
    (dict(heads=0), "not a multiple of kv_heads"),
    (dict(heads=-2), "not a multiple of kv_heads"),
    (dict(head_dim=0), "head_dim=0"),
    (dict(doc_q=DUMMY, doc_k=DUMMY), "documents"),
]


@pytest.mark.parametrize("more, text", BAD_SIZES, ids=[f"{n}-{t}" for n, (_, t) in enumerate(BAD_SIZES)])
def test_workspace_refusals(nn, more, text):
    """What the launch refuses by its sizes has no workspace either."""
    L = nn.lib()
    L.last_error()
    with pytest.raises(nn.NnHipError, match=f"nnhip_cache_attention_workspace: error 1: .*{text}"):
        L.nnhip_cache_attention_workspace(_attn(nn, **dict(dict(len_k=1000), **more)), _cache(nn, table_pages=64))
    assert L.last_error()[0] == 0


@pytest.mark.parametrize("kind", ["NN_CACHE_PLAIN", "NN_CACHE_MXFP4"])
@pytest.mark.parametrize("heads, kv", [(8, 8), (32, 1), (8, 1)])
def test_launches_past_32_bits(nn, kind, heads, kv):
    """Single queries of more requests than a launch has threads for, by either form: units or heads of 256."""
    L = nn.lib()
    L.last_error()
    batch = 1 << 24 if kv == 1 else 1 << 22
    a = _attn(nn, dtype=nn.NN_BF16, batch=batch, len_q=1, heads=heads, kv_heads=kv, out_stride=(8 * heads, 8 * heads, 8))
    c = _cache(nn, kind=getattr(nn, kind), requests=batch)
    with pytest.raises(nn.NnHipError, match="launch_cache_attention_forward: error 1: .*too many rows"):
        L.launch_cache_attention_forward(DUMMY, DUMMY, DUMMY, a, c, DUMMY, None)
    assert L.last_error()[0] == 0


def test_null_pointers(nn):
    L = nn.lib()
    L.last_error()
    c = _cache(nn)
    for hole in range(4):
        args = [None if i == hole else DUMMY for i in range(4)]
        with pytest.raises(nn.NnHipError, match="null pointer"):
            L.launch_cache_append(*args, _append(nn), c, None)
    for hole in range(2):
        with pytest.raises(nn.NnHipError, match="null pointer"):
            L.launch_cache_read(*[None if i == hole else DUMMY for i in range(2)], _read(nn), c, None)
    for hole in range(3):
        with pytest.raises(nn.NnHipError, match="null pointer"):
            L.launch_cache_attention_forward(*[None if i == hole else DUMMY for i in range(3)], _attn(nn), c, DUMMY, None)


def test_nothing_to_do(nn):
    """Calls without tokens, requests or queries end on the host."""
    L = nn.lib()
    L.last_error()
    L.launch_cache_append(None, None, None, None, _append(nn, tokens=0, pos=None, freq=None, place=None), _cache(nn), None)
    L.launch_cache_read(None, None, _read(nn, tokens=0, place=None), _cache(nn), None)
    for more in (dict(batch=0), dict(len_q=0)):
        L.launch_cache_attention_forward(None, None, None, _attn(nn, **more), _cache(nn), None, None)
    assert L.last_error()[0] == 0


@pytest.mark.parametrize("kind, dtype, dim, tokens, size", [
    ("mxfp4", "f32", 128, 64, 64 * 68), ("mxfp4", "bf16", 33, 16, 16 * 34), ("mxfp4", "bf16", 1, 16, 16 * 17),
    ("plain", "bf16", 72, 16, 16 * 144), ("plain", "bf16", 1, 32, 32 * 16), ("plain", "f32", 5, 16, 16 * 32),
])
def test_page_bytes(nn, kind, dtype, dim, tokens, size):
    L = nn.lib()
    c = _cache(nn, kind=nn.NN_CACHE_MXFP4 if kind == "mxfp4" else nn.NN_CACHE_PLAIN, page_tokens=tokens, table=None, k=None, v=None)
    assert L.nnhip_cache_page_bytes(c, nn.NN_BF16 if dtype == "bf16" else nn.NN_F32, 3, dim) == 3 * size
    with pytest.raises(nn.NnHipError, match="nnhip_cache_page_bytes: error 1: .*head_dim=200"):
        L.nnhip_cache_page_bytes(c, nn.NN_F32, 3, 200)


def test_structures_match_the_header(nn, tmp_path):
    """Sizes and offsets of the mirrors against the compiler's."""
    import subprocess

    structs = {"NnCache": nn.NnCache, "NnCacheAppend": nn.NnCacheAppend, "NnCacheRead": nn.NnCacheRead}
    lines = [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n, s in structs.items() for f, *_ in s._fields_]
    lines += [f'printf("{n} %zu\\n", sizeof({n}));' for n in structs]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "nn_cache.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", f"-I{nn.INCLUDE_DIR}", "-I/opt/rocm/include", str(src), "-o",
                    str(tmp_path / "sizes")], check=True)
    said = dict(line.rsplit(" ", 1) for line in
                subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.splitlines())
    for n, s in structs.items():
        assert int(said[n]) == ctypes.sizeof(s)
        for f, *_ in s._fields_:
            assert int(said[f"{n}.{f}"]) == getattr(s, f).offset, (n, f)


def test_sizes_are_the_nearest_and_off_by_half_a_step():
    """The tests' own 4 bits: every size is its own, and no value is off by more than half its step."""
    x = np.concatenate([SIZES, -SIZES, np.linspace(-7, 7, 1121)])
    for value in x:
        block = np.zeros((1, 32))
        block[0, :2] = [7, value]
        code, e, _ = codes(block)
        got = unpacked(code, e, 32)
        assert e[0, 0] == 0 and got[0, 0] == 6
        nearest = np.abs(np.concatenate([SIZES, -SIZES]) - value).min()
        assert abs(got[0, 1] - value) == nearest
        assert nearest <= (0.25 if abs(value) <= 2 else 0.5 if abs(value) <= 4 else 1)


def test_exponents():
    top = np.array([[0.0], [7.0], [np.nextafter(7, 8)], [3.5], [np.inf], [np.nan], [3.4e38], [1e-45], [6 * 2.0**-121]])
    assert exponents(top).tolist() == [-120, 0, 1, -1, 128, 128, 125, -120, -120]
    for value in np.exp2(np.linspace(-117, 126, 2000)):
        e = int(exponents(np.array([[value]]))[0])
        assert value <= 7 * 2.0**e and value > 7 * 2.0 ** (e - 1)
