"""The attention operators' host side: refusals, sizes of workspaces, calls with nothing
to do, and the tests' own gradient formulas against differences."""
from __future__ import annotations

import ctypes
import re

import numpy as np
import pytest

from attention_ref import attention, norm_rope

DUMMY = 16  # never dereferenced: every check of the host comes before a launch


def _attn(nn, **more):
    a = dict(dtype=nn.NN_F32, batch=1, len_q=4, len_k=4, heads=2, kv_heads=1, head_dim=8, scale=0.3, softcap=0.0,
             mask=nn.NN_MASK_NONE, q_stride=(64, 16, 8), k_stride=(32, 8, 8), v_stride=(32, 8, 8),
             out_stride=(64, 16, 8))
    a.update(more)
    return nn.NnAttention(**a)


def _rope(nn, **more):
    a = dict(dtype=nn.NN_F32, tokens=4, heads=2, kv_heads=1, head_dim=8, rot_dim=8, axes=1, interleaved=0, eps=1e-6,
             q_stride=(16, 8), k_stride=(8, 8), q_out_stride=(16, 8), k_out_stride=(8, 8), pos=DUMMY, freq=DUMMY)
    a.update(more)
    return nn.NnQkNormRope(**a)


BAD_ATTN = [
    (dict(dtype=7), "unknown dtype 7"),
    (dict(batch=-1), "bad shape"),
    (dict(len_q=-2), "bad shape"),
    (dict(heads=3, kv_heads=2), "not a multiple of kv_heads"),
    (dict(heads=0), "not a multiple of kv_heads|heads=0"),
    (dict(kv_heads=0), "kv_heads=0"),
    (dict(head_dim=0), "head_dim=0"),
    (dict(head_dim=129), "head_dim=129"),
    (dict(scale=0.0), "scale=0"),
    (dict(scale=float("nan")), "scale=nan"),
    (dict(softcap=-1.0), "softcap=-1"),
    (dict(scale=1e10, softcap=1e-35), "overflows"),
    (dict(mask=9), "unknown mask 9"),
    (dict(mask=2), "null prefix"),
    (dict(doc_q=DUMMY), "documents of queries or keys only"),
    (dict(buckets=4, max_distance=4), "null bucket or bias"),
    (dict(buckets=4, max_distance=1024, bucket=DUMMY, bias=DUMMY), "max_distance=1024"),
    (dict(buckets=-1), "buckets=-1"),
    (dict(batch=1 << 20, len_q=1 << 20), "too many rows"),
]


@pytest.mark.parametrize("more, text", BAD_ATTN, ids=[t for _, t in BAD_ATTN])
def test_attention_refusals(nn, more, text):
    L = nn.lib()
    L.last_error()
    a = _attn(nn, **more)
    with pytest.raises(nn.NnHipError, match=f"launch_attention_forward: error 1: .*({text})"):
        L.launch_attention_forward(DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, a, DUMMY, None)
    with pytest.raises(nn.NnHipError, match=f"launch_attention_backward: error 1: .*({text})"):
        L.launch_attention_backward(*[DUMMY] * 3, None, *[DUMMY] * 6, a, DUMMY, None)
    assert L.last_error()[0] == 0


def test_attention_null_pointers(nn):
    L = nn.lib()
    L.last_error()
    a = _attn(nn)
    for hole in range(5):
        args = [None if i == hole else DUMMY for i in range(5)]
        with pytest.raises(nn.NnHipError, match="null pointer"):
            L.launch_attention_forward(*args, a, None, None)
    for hole in (0, 1, 2, 4, 5, 6, 7, 8, 9):
        args = [None if i in (hole, 3) else DUMMY for i in range(10)]
        with pytest.raises(nn.NnHipError, match="null pointer"):
            L.launch_attention_backward(*args, a, DUMMY, None)
    with pytest.raises(nn.NnHipError, match="null description"):
        L.launch_attention_forward(*[DUMMY] * 5, None, None, None)
    with pytest.raises(nn.NnHipError, match="null workspace"):
        L.launch_attention_backward(*[DUMMY] * 3, None, *[DUMMY] * 6, a, None, None)
    with pytest.raises(nn.NnHipError, match="not aligned"):
        L.launch_attention_backward(*[DUMMY] * 3, None, *[DUMMY] * 6, a, 20, None)
    with pytest.raises(nn.NnHipError, match="bias gradient without a bias"):
        L.launch_attention_backward(*[DUMMY] * 10, a, DUMMY, None)


BAD_ROPE = [
    (dict(dtype=-1), "unknown dtype"),
    (dict(tokens=-1), "bad shape"),
    (dict(heads=-1), "bad shape"),
    (dict(head_dim=0, rot_dim=0), "head_dim=0"),
    (dict(head_dim=257), "head_dim=257"),
    (dict(rot_dim=10), "rot_dim=10"),
    (dict(rot_dim=3), "rot_dim=3"),
    (dict(axes=0), "axes=0"),
    (dict(axes=3), "axes=3"),
    (dict(eps=-1.0), "eps=-1"),
    (dict(pos=None), "null pos or freq"),
    (dict(freq=None), "null pos or freq"),
    (dict(tokens=1 << 30), "too many rows"),
]


@pytest.mark.parametrize("more, text", BAD_ROPE, ids=[t for _, t in BAD_ROPE])
def test_rope_refusals(nn, more, text):
    L = nn.lib()
    L.last_error()
    a = _rope(nn, **more)
    with pytest.raises(nn.NnHipError, match=f"launch_qk_norm_rope_forward: error 1: .*{text}"):
        L.launch_qk_norm_rope_forward(*[DUMMY] * 4, a, None)
    with pytest.raises(nn.NnHipError, match=f"launch_qk_norm_rope_backward: error 1: .*{text}"):
        L.launch_qk_norm_rope_backward(*[DUMMY] * 8, a, DUMMY, None)


def test_rope_null_pointers(nn):
    L = nn.lib()
    L.last_error()
    a = _rope(nn)
    for hole in range(4):
        with pytest.raises(nn.NnHipError, match="null pointer"):
            L.launch_qk_norm_rope_forward(*[None if i == hole else DUMMY for i in range(4)], a, None)
    with pytest.raises(nn.NnHipError, match="null workspace"):
        L.launch_qk_norm_rope_backward(*[DUMMY] * 8, a, None, None)


@pytest.mark.parametrize("len_q, len_k, heads, kv, buckets", [(1, 3000, 8, 2, 0), (1500, 1500, 1, 1, 0), (700, 700, 8, 2, 8),
                                                              (130, 4000, 2, 2, 4), (5, 5, 1, 1, 0)])
def test_workspaces_serve_smaller_batches(nn, len_q, len_k, heads, kv, buckets):
    """Fewer requests are divided into more parts; the reported sizes may not fall as the batch grows."""
    L = nn.lib()
    for size in (L.nnhip_attention_forward_workspace, L.nnhip_attention_backward_workspace):
        sizes = [size(_attn(nn, batch=b, len_q=len_q, len_k=len_k, heads=heads, kv_heads=kv, buckets=buckets,
                            max_distance=buckets, bucket=DUMMY, bias=DUMMY)) for b in list(range(1, 200)) + [1000, 3000]]
        assert sizes == sorted(sizes)


def test_nothing_to_do(nn):
    L = nn.lib()
    L.last_error()
    L.launch_attention_forward(*[None] * 5, _attn(nn, batch=0), None, None)
    L.launch_attention_forward(*[None] * 5, _attn(nn, len_q=0), None, None)
    L.launch_attention_backward(*[None] * 10, _attn(nn, batch=0), None, None)
    L.launch_qk_norm_rope_forward(*[None] * 4, _rope(nn, tokens=0), None)
    L.launch_qk_norm_rope_backward(*[None] * 8, _rope(nn, heads=0, kv_heads=0), None, None)
    assert L.last_error()[0] == 0


def test_structures_match_the_header(nn):
    """Field names and kinds of the ctypes mirrors, in the header's order."""
    text = (nn.INCLUDE_DIR / "nn_attention.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name in ("NnQkNormRope", "NnAttention"):
        body = re.search(r"typedef struct \{([^}]*)\} " + name, text).group(1)
        want = []
        for line in filter(None, (s.strip() for s in body.split(";"))):
            kind, names = re.match(r"((?:const )?(?:long long|\w+)\*?)\s*(.*)", line, flags=re.S).groups()
            for field in names.split(","):
                n = re.match(r"\s*(\w+)(?:\[(\d)\])?", field)
                base = {"int": ctypes.c_int, "float": ctypes.c_float, "long long": ctypes.c_longlong}.get(kind, ctypes.c_void_p)
                want.append((n.group(1), base * int(n.group(2)) if n.group(2) else base))
        assert getattr(nn, name)._fields_ == want


def test_reference_gradients_by_differences():
    """The formulas that the GPU tests compare with, against central differences in 64 bits."""
    rng = np.random.default_rng(3)
    c = dict(batch=2, len_q=5, len_k=6, heads=4, kv_heads=2, dim=3, scale=0.7, cap=2.0, mask="prefix", prefix=[3, 0],
             buckets=3, max_distance=2, doc_q=[[0, 0, 1, 1, -1], [0, 0, 0, 2, 2]],
             doc_k=[[0, 0, 0, 1, 1, -1], [0, 0, 0, 0, 2, 2]])
    x = {"q": rng.standard_normal((2, 5, 4, 3)), "k": rng.standard_normal((2, 6, 2, 3)),
         "v": rng.standard_normal((2, 6, 2, 3)), "bias": rng.standard_normal((3, 4))}
    bucket = np.array([0, 1, 1, 2, 2])
    dout = rng.standard_normal((2, 5, 4, 3))
    got, _ = attention(c, **x, bucket=bucket, dout=dout)
    for n in x:
        for _ in range(12):
            at = tuple(rng.integers(0, s) for s in x[n].shape)
            side = []
            for step in (1e-5, -1e-5):
                y = {m: z.copy() for m, z in x.items()}
                y[n][at] += step
                side.append((attention(c, **y, bucket=bucket)[0]["out"] * dout).sum())
            # truncation 1e-10 of the third derivative, cancellation 1e-16 / 1e-5
            assert abs((side[0] - side[1]) / 2e-5 - got["d" + n][at]) < 1e-7
    for interleaved in (False, True):
        x, w = rng.standard_normal((4, 2, 8)), rng.standard_normal(8)
        grad, pos, freq = rng.standard_normal((4, 2, 8)), rng.integers(0, 50, (4, 2)), rng.random(2)
        call = lambda x, w: (norm_rope(x, w, 1e-6, pos, freq, 4, 2, interleaved) * grad).sum()  # noqa: E731
        _, dx, dw, _ = norm_rope(x, w, 1e-6, pos, freq, 4, 2, interleaved, grad)
        for _ in range(12):
            at, d = tuple(rng.integers(0, s) for s in x.shape), rng.integers(0, 8)
            e = np.zeros_like(x)
            e[at] = 1e-5
            assert abs((call(x + e, w) - call(x - e, w)) / 2e-5 - dx[at]) < 1e-7
            f = np.zeros(8)
            f[d] = 1e-5
            assert abs((call(x, w + f) - call(x, w - f)) / 2e-5 - dw[d]) < 1e-7


@pytest.mark.parametrize("heads, kv, batch, docs", [(1, 1, 1, False), (8, 8, 1, True), (8, 2, 3, False), (32, 8, 16, False),
                                                    (3, 1, 200, True)])
@pytest.mark.parametrize("buckets", [0, 8])
def test_workspaces_serve_shorter_lengths(nn, heads, kv, batch, docs, buckets):
    """A program's workspaces have the sizes of its longest call: no shorter one may report more."""
    L = nn.lib()
    # where the division into parts changes: tiles of 32, 64 and 128, counts of workgroups, few queries
    lengths = sorted({*range(1, 200, 7), *(n + d for n in (64, 128, 512, 1024, 4096, 8192, 16384) for d in (-1, 0, 1)), 2944, 3008, 4160,
                      30000, 100000})
    for size in (L.nnhip_attention_forward_workspace, L.nnhip_attention_backward_workspace):
        got = np.array([[size(_attn(nn, batch=batch, len_q=q, len_k=k, heads=heads, kv_heads=kv, buckets=buckets,
                                    max_distance=buckets, doc_q=DUMMY if docs else None, doc_k=DUMMY if docs else None))
                         for k in lengths] for q in lengths], np.int64)
        assert (np.diff(got, axis=0) >= 0).all() and (np.diff(got, axis=1) >= 0).all()


@pytest.mark.parametrize("scale, cap", [(0.1, 1e38), (1e-38, 1e10), (1e-30, 1e9), (0.1, 1e-39)])
def test_caps_too_far_for_fp32_are_refused(nn, scale, cap):
    """scale / softcap, or the cap, below the normal fp32 values has lost its digits."""
    L = nn.lib()
    a = _attn(nn, scale=scale, softcap=cap)
    with pytest.raises(nn.NnHipError, match="underflows"):
        L.launch_attention_forward(*[DUMMY] * 5, a, DUMMY, None)
    with pytest.raises(nn.NnHipError, match="underflows"):
        L.launch_attention_backward(*[DUMMY] * 3, None, *[DUMMY] * 6, a, DUMMY, None)
    assert L.last_error()[0] == 0


@pytest.mark.parametrize("more", [dict(len_q=(1 << 30) - 4095), dict(len_k=(1 << 30) - 4095), dict(len_q=2**31 - 1)])
def test_lengths_whose_distances_pass_32_bits_are_refused(nn, more):
    L = nn.lib()
    with pytest.raises(nn.NnHipError, match="bad shape"):
        L.launch_attention_forward(*[DUMMY] * 5, _attn(nn, **more), DUMMY, None)
    assert L.nnhip_attention_forward_workspace(_attn(nn, len_k=(1 << 30) - 4096)) > 0
    assert L.last_error()[0] == 0


OVERLAPS = [
    (dict(batch=3, k_stride=(0, 8, 8)), "dk"),  # one request's keys for all
    (dict(batch=3, v_stride=(0, 8, 8)), "dv"),
    (dict(heads=4, kv_heads=2, k_stride=(64, 8, 0)), "dk"),  # one key head's keys for all
    (dict(k_stride=(64, 0, 8)), "dk"),
    (dict(v_stride=(64, 7, 8)), "dv"),
    (dict(q_stride=(64, 8, 8)), "dq"),  # tokens by the stride of heads
    (dict(batch=2, q_stride=(48, 16, 8)), "dq"),
    (dict(q_stride=(64, -8, 8)), "dq"),
    (dict(batch=2, q_stride=(1 << 62, 16, 0)), "dq"),
]


@pytest.mark.parametrize("more, name", OVERLAPS)
def test_gradients_that_would_overlap_are_refused(nn, more, name):
    """Rows repeated by their strides: workgroups would write one row's gradient over another's."""
    L = nn.lib()
    more = {"batch": 1, **more}
    a = _attn(nn, **{"q_stride": (128, 32, 8), "k_stride": (64, 16, 8), "v_stride": (64, 16, 8), **more})
    with pytest.raises(nn.NnHipError, match=f"rows of {name} overlap"):
        L.launch_attention_backward(*[DUMMY] * 3, None, *[DUMMY] * 6, a, DUMMY, None)
    assert L.last_error()[0] == 0


@pytest.mark.parametrize("stride", [(0, 16, 8), (64, 0, 8), (64, 16, 0), (64, 15, 8), (63, 16, 8), (64, 16, -4)])
def test_outputs_that_would_overlap_are_refused(nn, stride):
    L = nn.lib()
    with pytest.raises(nn.NnHipError, match="rows of out overlap"):
        L.launch_attention_forward(*[DUMMY] * 5, _attn(nn, batch=2, out_stride=stride), DUMMY, None)
    assert L.last_error()[0] == 0


def test_rotated_rows_that_would_overlap_are_refused(nn):
    L = nn.lib()
    for more, name in ((dict(q_out_stride=(0, 8)), "q_out"), (dict(k_out_stride=(7, 8)), "k_out"), (dict(q_out_stride=(16, 0)), "q_out")):
        with pytest.raises(nn.NnHipError, match=f"rows of {name} overlap"):
            L.launch_qk_norm_rope_forward(*[DUMMY] * 4, _rope(nn, **more), None)
    for more, name in ((dict(q_stride=(0, 8)), "dq"), (dict(k_stride=(0, 8)), "dk"), (dict(q_stride=(16, 4)), "dq")):
        with pytest.raises(nn.NnHipError, match=f"rows of {name} overlap"):
            L.launch_qk_norm_rope_backward(*[DUMMY] * 8, _rope(nn, **more), DUMMY, None)
    assert L.last_error()[0] == 0


WIDE = {n: (1 << 32, 1 << 20, 8) for n in ("q_stride", "k_stride", "v_stride", "out_stride")}


@pytest.mark.parametrize("more, forward", [
    (dict(batch=1 << 23, heads=2, kv_heads=2, len_q=1, len_k=1), True),
    (dict(batch=1 << 24, heads=1, len_q=1, len_k=1), True),
    (dict(batch=1 << 19, len_k=1, len_q=2049), True),
    (dict(batch=1 << 14, len_q=1, len_k=1 << 18, doc_q=DUMMY, doc_k=DUMMY), True),  # documents of its keys
    (dict(batch=1 << 19, len_k=2049, len_q=1), False),  # key gradients
    (dict(batch=1 << 19, heads=32, len_q=1, len_k=1), False),  # few queries; query gradients
])
def test_more_workgroups_than_a_launch_takes_are_refused(nn, more, forward):
    """2^32 threads and more: the first kernels of a call would run and a later one not."""
    L = nn.lib()
    a = _attn(nn, **WIDE, **more)
    calls = [lambda: L.launch_attention_backward(*[DUMMY] * 3, None, *[DUMMY] * 6, a, DUMMY, None),
             lambda: L.nnhip_attention_backward_workspace(a)]
    if forward:
        calls += [lambda: L.launch_attention_forward(*[DUMMY] * 5, a, DUMMY, None), lambda: L.nnhip_attention_forward_workspace(a)]
    else:
        L.nnhip_attention_forward_workspace(a)
    for call in calls:
        with pytest.raises(nn.NnHipError, match="too many rows"):
            call()
    assert L.last_error()[0] == 0


def test_heads_and_tokens_past_a_launch_are_refused(nn):
    L = nn.lib()
    with pytest.raises(nn.NnHipError, match="heads=1048577"):
        L.launch_attention_forward(*[DUMMY] * 5, _attn(nn, heads=(1 << 20) + 1), DUMMY, None)
    with pytest.raises(nn.NnHipError, match="too many rows"):
        L.launch_qk_norm_rope_forward(*[DUMMY] * 4, _rope(nn, tokens=1 << 28, heads=1, kv_heads=0, head_dim=256, rot_dim=256,
                                                          q_out_stride=(256, 256)), None)
    assert L.last_error()[0] == 0
    with pytest.raises(nn.NnHipError, match="too many rows"):
        L.launch_qk_norm_rope_backward(*[DUMMY] * 8, _rope(nn, tokens=(1 << 30) + 1, heads=1, kv_heads=0, q_stride=(8, 8)), DUMMY, None)
    assert L.last_error()[0] == 0
