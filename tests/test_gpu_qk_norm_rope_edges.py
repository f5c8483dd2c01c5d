"""Norms with the position rotation at angles where digits are easily lost."""
from __future__ import annotations

import numpy as np
import pytest

from attention_ref import U

pytestmark = pytest.mark.gpu

U32 = U["f32"]


@pytest.mark.parametrize("interleaved", [False, True])
def test_small_sines_and_cosines_keep_their_digits(nn, L, interleaved):
    """Angles near multiples of a quarter turn: the small one of sine and cosine is rounded as a value of
    its own, not as a part of 1.  x = (1, 0) and (0, 1): an output is one product of three fp32 factors."""
    rest = np.array([1e-6, -3e-6, 1e-5, -1e-4, 7e-4, -1e-3])
    angle = (np.arange(-9, 10)[:, None] * (np.pi / 2) + rest).ravel()
    pairs = 128
    angle = np.resize(angle, pairs)
    x = np.zeros((2, 1, 2 * pairs), np.float32)
    first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, pairs), slice(pairs, None))
    x[0, 0, first] = x[1, 0, second] = 1.0
    xd, out, pos = L.to_device(x), L.alloc(x.size), L.to_device(np.ones(2, np.int32).view(np.float32))
    freq = L.to_device(angle.view(np.float32))
    a = nn.NnQkNormRope(dtype=nn.NN_F32, tokens=2, heads=1, kv_heads=0, head_dim=2 * pairs, rot_dim=2 * pairs, axes=1,
                        interleaved=int(interleaved), eps=0.0, q_stride=(2 * pairs, 2 * pairs),
                        q_out_stride=(2 * pairs, 2 * pairs), pos=pos.p, freq=freq.p)
    L.launch_qk_norm_rope_forward(out.p, None, xd.p, None, a, None)
    L.sync()
    got = out.download(shape=x.shape).astype(np.float64)[:, 0]
    size = np.sqrt(2.0)  # 1 over the root of the mean square
    ref = np.empty((2, 2 * pairs))
    ref[0, first], ref[0, second] = size * np.cos(angle), size * np.sin(angle)
    ref[1, first], ref[1, second] = -size * np.sin(angle), size * np.cos(angle)
    # the root 2 u, the rounded angle 1 u of the small ones, sine or cosine 2 u, two products: 8 u; the
    # angle's 64-bit turns are off by some 2^-53 of up to 3 turns
    assert (abs(got - ref) <= 8 * U32 * abs(ref) + 2.0**-48).all()
