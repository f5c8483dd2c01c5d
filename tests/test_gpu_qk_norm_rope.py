"""Per-head norms with the position rotation, through the C-ABI against the 64-bit formulas."""
from __future__ import annotations

import numpy as np
import pytest

from attention_ref import U, Tensor, norm_rope

pytestmark = pytest.mark.gpu

# An element is rounded once to its type (u of itself) from fp32 values: a product of five
# factors, each rounded, sines off by 2^-22 of 1, two terms: 32 u_32 of the terms' sizes.
# Weight gradients add up to `rows` such products: 64 u_32 of the sum of magnitudes.
U32 = U["f32"]


def _run(nn, L, rng, dtype, tokens, heads, kv, dim, rot, axes=1, interleaved=False, far=100, layout="packed",
         weights=True, in_place=False):
    print(f"[case] norm and rotation {dtype} {tokens} {heads} {kv} {dim} {rot} {axes} {interleaved} {far} {layout}", flush=True)
    row = (heads + 2 * kv) * dim + (3 if layout == "odd" else 0)
    place = {"q": ((tokens, heads, dim), (row, dim, 1), 1 if layout == "odd" else 0),
             "k": ((tokens, kv, dim), (row, dim, 1), heads * dim)}
    x = {n: Tensor(L, s, dtype, st, o, values=rng.standard_normal(s) * 1.5) for n, (s, st, o) in place.items()}
    outs = {n: Tensor(L, s, dtype, *((st, o) if in_place else (None, 0))) for n, (s, st, o) in place.items()}
    grads = {n: Tensor(L, s, dtype, outs[n].strides, outs[n].offset, values=rng.standard_normal(s)) for n, (s, _, _) in place.items()}
    dx = {n: Tensor(L, s, dtype, st, o) for n, (s, st, o) in place.items()}
    w = {n: (1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if weights else np.ones(dim, np.float32) for n in "qk"}
    wd = {n: L.to_device(w[n]) for n in "qk"}
    dw = {n: L.alloc(dim) for n in "qk"}
    pos = rng.integers(0, far, (tokens, axes)).astype(np.int32)
    freq = 10000.0 ** -rng.random(rot // 2)
    posd = L.to_device(np.append(pos.ravel(), np.int32(0)).view(np.float32))
    freqd = L.to_device(np.append(freq, 0.0).view(np.float32))
    a = nn.NnQkNormRope(dtype=nn.NN_BF16 if dtype == "bf16" else nn.NN_F32, tokens=tokens, heads=heads, kv_heads=kv,
                        head_dim=dim, rot_dim=rot, axes=axes, interleaved=int(interleaved), eps=1e-6,
                        q_stride=x["q"].strides[:2], k_stride=x["k"].strides[:2], q_out_stride=outs["q"].strides[:2],
                        k_out_stride=outs["k"].strides[:2], q_weight=wd["q"].p if weights else None,
                        k_weight=wd["k"].p if weights else None, pos=posd.p, freq=freqd.p)
    ws = L.alloc(max(1, L.nnhip_qk_norm_rope_workspace(a)))
    ws.fill_bytes(0xFF)
    L.launch_qk_norm_rope_backward(dx["q"].p, dx["k"].p, dw["q"].p, dw["k"].p, grads["q"].p, grads["k"].p, x["q"].p,
                                   x["k"].p, a, ws.p, None)
    if in_place:
        before = {n: x[n].values() for n in "qk"}
        outs = x
    L.launch_qk_norm_rope_forward(outs["q"].p, outs["k"].p, x["q"].p, x["k"].p, a, None)
    L.sync()
    eps = float(np.float32(1e-6))
    for n in "qk":
        if not x[n].shape[1]:
            continue
        xv = before[n] if in_place else x[n].values()
        gv = grads[n].values()
        out, dxr, dwr, mag = norm_rope(xv, w[n].astype(np.float64), eps, pos, freq, rot, axes, interleaved, gv)
        u = U[dtype]
        top = lambda y: abs(y).max(-1, keepdims=True)  # noqa: E731  # a row's terms are at most twice its largest value
        got = outs[n].result()
        assert (abs(got - out) <= u * abs(out) + 32 * U32 * 2 * top(out)).all(), n
        got = dx[n].result()
        rstd = 1 / np.sqrt((xv * xv).mean(-1, keepdims=True) + eps)
        terms = rstd * top(gv) * top(w[n]) * (2 + abs(xv * rstd))
        assert (abs(got - dxr) <= u * abs(dxr) + 32 * U32 * 2 * terms).all(), n
        got = dw[n].download().astype(np.float64)
        size = mag + 2 * U32 * np.sqrt(tokens) * abs(gv).max()
        assert (abs(got - dwr) <= U32 * abs(dwr) + 64 * U32 * size * 2).all(), (n, abs(got - dwr).max())


TYPES = ("f32", "bf16")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim, rot, axes", [(8, 8, 1), (16, 4, 2), (40, 40, 1), (64, 64, 2), (72, 48, 2), (72, 66, 3),
                                            (128, 128, 1), (128, 0, 1), (256, 256, 1), (33, 30, 1), (1, 0, 1), (96, 36, 3)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads(nn, L, rng, dtype, dim, rot, axes, interleaved):
    _run(nn, L, rng, dtype, 37, 4, 2, dim, rot, axes, interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 130, 2100])
@pytest.mark.parametrize("heads, kv", [(1, 1), (8, 1), (5, 5), (3, 0), (0, 3)])
def test_sizes(nn, L, rng, dtype, tokens, heads, kv):
    _run(nn, L, rng, dtype, tokens, heads, kv, 32, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_unaligned_rows(nn, L, rng, dtype, interleaved):
    _run(nn, L, rng, dtype, 50, 3, 1, 40, 24, 2, interleaved, layout="odd")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("far", [1 << 20, (1 << 31) - 1])
def test_far_positions(nn, L, rng, dtype, far):
    """fp32 angles would be off by whole turns here."""
    _run(nn, L, rng, dtype, 64, 2, 1, 64, 64, far=far)


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_and_without_weights(nn, L, rng, dtype):
    _run(nn, L, rng, dtype, 90, 4, 2, 64, 64, weights=False, in_place=True)


def test_many_tokens_and_rows_that_repeat(nn, L, rng):
    """More tokens than the backward pass has workgroups."""
    _run(nn, L, rng, "bf16", 9000, 2, 1, 16, 16)


def test_rows_of_zeros(nn, L):
    """eps keeps a row of zeros finite: its output is zero, its gradient the weight's over sqrt(eps)."""
    x, g = L.to_device(np.zeros(8, np.float32)), L.to_device(np.ones(8, np.float32))
    out, dx, dw, ws = L.alloc(8), L.alloc(8), L.alloc(8), L.alloc(64)
    a = nn.NnQkNormRope(dtype=nn.NN_F32, tokens=1, heads=1, kv_heads=0, head_dim=8, rot_dim=0, axes=1, eps=1e-4,
                        q_stride=(8, 8), q_out_stride=(8, 8))
    L.launch_qk_norm_rope_forward(out.p, None, x.p, None, a, None)
    L.launch_qk_norm_rope_backward(dx.p, None, dw.p, None, g.p, None, x.p, None, a, ws.p, None)
    L.sync()
    assert not out.download().any() and not dw.download().any()
    assert np.allclose(dx.download(), 100.0, rtol=1e-5)
