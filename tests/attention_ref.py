"""The attention operators in 64-bit numpy, and what their tests share.

Tolerances.  A result may be off by its own rounding, u of its value, and by what
the kernel rounds before: each probability or score gradient to the type that the
matrix cores take (u again, bf16 only), and fp32 arithmetic.  u is half the type's
step: 2^-8 for bf16, 2^-24 for fp32.

  * norm of the difference over the norm of the result: the roundings are independent,
    so u / sqrt(3) each at most, twice: under 1.25 u for bf16.  fp32: a score is a sum
    of up to 128 products (about sqrt(128) u of their size) of a size up to about 10, in
    an exponent, and sums over keys follow: 128 u.
  * every element: u of itself, and u_p (bf16: 2^-8) and the fp32 part, 1024 u_32, of the
    sum of the magnitudes that it adds up.
"""
from __future__ import annotations

import numpy as np

U = {"f32": 2.0**-24, "bf16": 2.0**-8}


def to_bf16(x):
    """Rounded to bf16 (ties to even), as its 16 bits."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    up = (b + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(np.asarray(x, np.float32)), 0x7FC0, up).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint32) << 16).view(np.float32)


def rounded(x, dtype):
    x = np.asarray(x, np.float32)
    return from_bf16(to_bf16(x)).reshape(x.shape) if dtype == "bf16" else x


class Tensor:
    """A device tensor of fp32 or bf16 values with the strides of a numpy view.

    `shape` lies in a buffer of `room` elements at element strides `strides` from
    `offset` on; the other elements are `fill` (NaN: reads of them show)."""

    def __init__(self, L, shape, dtype, strides=None, offset=0, room=None, values=None, fill=np.nan):
        self.L, self.shape, self.dtype, self.offset = L, tuple(shape), dtype, offset
        if strides is None:
            strides = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        self.strides = tuple(strides)
        need = offset + 1 + sum((n - 1) * s for n, s in zip(shape, strides)) if np.prod(shape) else offset + 1
        self.room = max(room or 0, need)
        self.host = np.full(self.room, fill, np.float32)
        if values is not None:
            self.view(self.host)[...] = values
        self.size = 2 if dtype == "bf16" else 4
        self.dev = L.alloc(-(-self.room * self.size // 4))
        self.upload()

    def view(self, flat):
        return np.lib.stride_tricks.as_strided(flat[self.offset:], self.shape, [s * flat.itemsize for s in self.strides])

    def upload(self):
        raw = to_bf16(self.host) if self.dtype == "bf16" else self.host
        if raw.size % 2 and self.dtype == "bf16":
            raw = np.append(raw, np.uint16(0))
        self.dev.upload(raw.view(np.float32))

    @property
    def p(self):
        return self.dev.p + self.offset * self.size

    def values(self):
        """What the inputs are, in 64 bits."""
        return self.view(rounded(self.host, self.dtype)).astype(np.float64)

    def flat(self):
        raw = self.dev.download()
        return from_bf16(raw.view(np.uint16)[:self.room]) if self.dtype == "bf16" else raw[:self.room]

    def result(self):
        """What is on the device now; the elements between the tensor's have to be as they were."""
        flat = self.flat()
        others = np.ones(self.room, bool)
        self.view(others)[...] = False
        assert np.array_equal(flat[others], rounded(self.host, self.dtype)[others], equal_nan=True), "written outside"
        return self.view(flat).astype(np.float64)


def ints(L, x):
    x = np.ascontiguousarray(x, np.int32)
    return L.to_device(np.append(x.ravel(), np.int32(0)).view(np.float32))


def sees_of(c):
    """[batch, len_q, len_k]: which keys each query sees; and positions [batch, len_q]."""
    b, lq, lk = c["batch"], c["len_q"], c["len_k"]
    start = np.asarray(c.get("q_start", [lk - lq] * b), np.int64)
    k_len = np.asarray(c.get("k_len", [lk] * b), np.int64)
    pos = start[:, None] + np.arange(lq)
    j = np.arange(lk)
    sees = np.broadcast_to(j < k_len[:, None, None], (b, lq, lk)).copy()
    if c["mask"] == "causal":
        sees &= j <= pos[:, :, None]
    elif c["mask"] == "prefix":
        sees &= (j <= pos[:, :, None]) | (j < np.asarray(c["prefix"])[:, None, None])
    if "doc_q" in c:
        dq, dk = np.asarray(c["doc_q"]), np.asarray(c["doc_k"])
        sees &= (dq[:, :, None] == dk[:, None, :]) & (dk[:, None, :] >= 0)
    return sees, pos


def attention(c, q, k, v, bias=None, bucket=None, dout=None):
    """Outputs, and gradients if dout; and per output the sum of magnitudes that it adds up."""
    sees, pos = sees_of(c)
    b, lq, lk, h, kv = c["batch"], c["len_q"], c["len_k"], c["heads"], c["kv_heads"]
    g, scale, cap = h // kv, c["scale"], c["cap"]
    dead_k = ~sees.any(1) if lq else np.ones((b, lk), bool)
    dead_q = ~sees.any(2) if lk else np.ones((b, lq), bool)
    k, v, q = k.copy(), v.copy(), q.copy()
    k[dead_k], v[dead_k], q[dead_q] = 0, 0, 0
    kk, vv = np.repeat(k, g, 2), np.repeat(v, g, 2)
    raw = np.einsum("bihd,bjhd->bhij", q, kk) * scale
    t = np.tanh(raw / cap) if cap else None
    x = t * cap if cap else raw
    if bias is not None:
        m = c["max_distance"]
        at = np.clip(np.arange(lk)[None, None] - pos[:, :, None], -m, m) + m
        x = x + np.moveaxis(bias[bucket[at]], 3, 1)
    x = np.where(sees[:, None], x, -np.inf)
    top = x.max(-1, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0)
    e = np.exp(x - top[..., None])
    total = e.sum(-1)
    with np.errstate(divide="ignore"):
        lse = np.log(total) + top
    p = e / np.where(total > 0, total, 1)[..., None]
    out = np.einsum("bhij,bjhd->bihd", p, vv)
    got = {"out": out, "lse": lse}
    # the log-sum adds up products of scores (those of the keys that count) and a logarithm
    dots = np.einsum("bihd,bjhd->bhij", abs(q), abs(kk)) * scale
    with np.errstate(divide="ignore"):
        mag = {"out": np.einsum("bhij,bjhd->bihd", p, abs(vv)), "lse": (p * dots).sum(-1) + abs(np.log(total)) + abs(lse)}
    if dout is None:
        return got, mag

    def heads_sum(y):
        return y.reshape(b, lk, kv, g, y.shape[-1]).sum(3)

    dout = dout.copy()
    dout[dead_q] = 0
    got["dv"] = heads_sum(np.einsum("bhij,bihd->bjhd", p, dout))
    mag["dv"] = heads_sum(np.einsum("bhij,bihd->bjhd", p, abs(dout)))
    dp = np.einsum("bihd,bjhd->bhij", dout, vv)
    delta = (dp * p).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    # what the terms of ds are made of: a rounded sum of products each, and delta
    size = p * (np.einsum("bihd,bjhd->bhij", abs(dout), abs(vv)) + abs(delta) +
                np.einsum("bihd,bihd->bhi", abs(dout), np.einsum("bhij,bjhd->bihd", p, abs(vv)))[..., None])
    if bias is not None:
        got["dbias"] = np.zeros_like(bias)
        mag["dbias"] = np.zeros_like(bias)
        for n in range(c["buckets"]):
            of = (bucket[at] == n)[:, None]
            got["dbias"][n] = (ds * of).sum((0, 2, 3))
            mag["dbias"][n] = (size * of).sum((0, 2, 3))
    if cap:
        ds, size = ds * (1 - t * t), size * (1 - t * t)
    got["dq"] = np.einsum("bhij,bjhd->bihd", ds, kk) * scale
    mag["dq"] = np.einsum("bhij,bjhd->bihd", size, abs(kk)) * scale
    got["dk"] = heads_sum(np.einsum("bhij,bihd->bjhd", ds, q)) * scale
    mag["dk"] = heads_sum(np.einsum("bhij,bihd->bjhd", size, abs(q))) * scale
    return got, mag


def norm_rope(x, w, eps, pos, freq, rot, axes, interleaved, grad=None):
    """x [tokens, heads, dim] normalised and turned; with grad the gradients too."""
    rstd = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    half = rot // 2
    axis = np.arange(half) // max(1, half // axes)
    angle = pos[:, axis].astype(np.float64) * freq
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(half), np.arange(half, rot))

    def turn(y, s):
        z = y.copy()
        z[..., a] = y[..., a] * cos - y[..., b] * s
        z[..., b] = y[..., a] * s + y[..., b] * cos
        return z

    out = turn(x * rstd * w, sin)
    if grad is None:
        return out
    g, xn = turn(grad, -sin), x * rstd
    return out, rstd * (g * w - xn * (g * w * xn).mean(-1, keepdims=True)), (g * xn).sum((0, 1)), (abs(g * xn)).sum((0, 1))


def check(name, got, ref, mag, dtype, scores=10.0):
    """`got` against `ref`; `dtype`: of the result; `mag`: the magnitudes that it adds up;
    `scores`: their size, in proportion to which an exponent's rounding grows."""
    u, u32 = U[dtype], U["f32"] * scores / 10.0
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    fine = np.isfinite(ref)
    assert np.array_equal(got[~fine], ref[~fine]), f"{name}: infinities differ"
    got, ref, mag = got[fine], ref[fine], np.broadcast_to(mag, fine.shape)[fine]
    assert np.isfinite(got).all(), f"{name}: {int((~np.isfinite(got)).sum())} values are not finite"
    part = (U["bf16"] if dtype == "bf16" else 0.0) + 1024 * u32
    bound = u * abs(ref) + part * mag + 1e-30
    worst = float((abs(got - ref) / bound).max()) if got.size else 0.0
    assert worst <= 1, f"{name}: an element is {worst:.3g} times its bound off"
    norm = float(np.linalg.norm(ref))
    off = float(np.linalg.norm(got - ref))
    limit = 1.25 * U["bf16"] if dtype == "bf16" else 128 * u32
    # what cancels in the result itself does not count as its size
    size = max(norm, float(np.linalg.norm(mag)) * 2.0**-6)
    assert off <= limit * size, f"{name}: {off / max(size, 1e-300):.3g} off, at most {limit:.3g}"
