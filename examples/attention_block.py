"""The attention operators together: a training loop of one attention layer, then its decoding.

Training: queries, keys and values of a 28 x 28 image's tokens lie in one projection's rows.
Each step normalises and rotates queries and keys by their row and column
(launch_qk_norm_rope_*), mixes the values with capped scores and a learned bias by distance
(launch_attention_*), compares with a target, and goes back through both to the gradients
of the projection's rows, the norms' weights and the bias, which plain gradient steps lower.

Decoding: a causal layer over the same tokens, once for all of them and once token by token
over a cache that grows; both have to agree.

    python examples/attention_block.py [steps]
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

from __graft_entry__ import load_package  # noqa: E402

TOKENS, HEADS, KV, DIM, BUCKETS, DISTANCE = 28 * 28, 4, 2, 32, 16, 64
ROW = (HEADS + 2 * KV) * DIM


def ints(L, x):
    return L.to_device(np.ascontiguousarray(x, np.int32).view(np.float32))


class Layer:
    """One attention layer over the rows of a projection, [tokens, (heads + 2 kv heads) * dim] fp32."""

    def __init__(self, nn, L, rng):
        self.nn, self.L = nn, L
        self.rows = L.to_device(rng.standard_normal((TOKENS, ROW)).astype(np.float32))
        self.q_weight, self.k_weight = (L.to_device(np.ones(DIM, np.float32)) for _ in range(2))
        self.bias = L.to_device(np.zeros((BUCKETS, HEADS), np.float32))
        self.turned = L.alloc(TOKENS * (HEADS + KV) * DIM)  # queries and keys, normalised and rotated
        self.out, self.lse = L.alloc(TOKENS * HEADS * DIM), L.alloc(HEADS * TOKENS)
        yx = np.stack(np.divmod(np.arange(TOKENS), 28), 1)
        per = DIM // 4  # pairs of each axis
        freq = np.tile(100.0 ** (-np.arange(per) / per), 2)
        self.pos, self.freq = ints(L, yx), L.to_device(freq.view(np.float32))
        far = np.abs(np.arange(-DISTANCE, DISTANCE + 1))
        self.bucket = ints(L, np.minimum(BUCKETS - 1, (np.log2(far + 1) * 2.4).astype(int)))
        self.rope = nn.NnQkNormRope(
            dtype=nn.NN_F32, tokens=TOKENS, heads=HEADS, kv_heads=KV, head_dim=DIM, rot_dim=DIM, axes=2, eps=1e-6,
            q_stride=(ROW, DIM), k_stride=(ROW, DIM), q_out_stride=((HEADS + KV) * DIM, DIM),
            k_out_stride=((HEADS + KV) * DIM, DIM), q_weight=self.q_weight.p, k_weight=self.k_weight.p,
            pos=self.pos.p, freq=self.freq.p)
        turned = (TOKENS * (HEADS + KV) * DIM, (HEADS + KV) * DIM, DIM)
        self.attn = nn.NnAttention(
            dtype=nn.NN_F32, batch=1, len_q=TOKENS, len_k=TOKENS, heads=HEADS, kv_heads=KV, head_dim=DIM,
            scale=DIM**-0.5, softcap=20.0, mask=nn.NN_MASK_NONE, buckets=BUCKETS, max_distance=DISTANCE,
            q_stride=turned, k_stride=turned, v_stride=(TOKENS * ROW, ROW, DIM),
            out_stride=(TOKENS * HEADS * DIM, HEADS * DIM, DIM), bucket=self.bucket.p, bias=self.bias.p)
        zeros = lambda n: L.to_device(np.zeros(max(1, n), np.float32))  # noqa: E731
        self.forward_ws = zeros(L.nnhip_attention_forward_workspace(self.attn))
        self.backward_ws = zeros(L.nnhip_attention_backward_workspace(self.attn))
        self.rope_ws = zeros(L.nnhip_qk_norm_rope_workspace(self.rope))
        self.grads = {"rows": L.alloc(TOKENS * ROW), "q_weight": L.alloc(DIM), "k_weight": L.alloc(DIM),
                      "bias": L.alloc(BUCKETS * HEADS), "turned": L.alloc(TOKENS * (HEADS + KV) * DIM)}

    def forward(self, stream=None):
        L, k, v = self.L, HEADS * DIM, (HEADS + KV) * DIM
        L.launch_qk_norm_rope_forward(self.turned.p, self.turned.offset(k), self.rows.p, self.rows.offset(k), self.rope,
                                      stream)
        L.launch_attention_forward(self.out.p, self.lse.p, self.turned.p, self.turned.offset(k), self.rows.offset(v),
                                   self.attn, self.forward_ws.p, stream)

    def backward(self, dout, stream=None):
        L, g, k, v = self.L, self.grads, HEADS * DIM, (HEADS + KV) * DIM
        L.launch_attention_backward(g["turned"].p, g["turned"].offset(k), g["rows"].offset(v), g["bias"].p, dout.p,
                                    self.turned.p, self.turned.offset(k), self.rows.offset(v), self.out.p, self.lse.p,
                                    self.attn, self.backward_ws.p, stream)
        L.launch_qk_norm_rope_backward(g["rows"].p, g["rows"].offset(k), g["q_weight"].p, g["k_weight"].p,
                                       g["turned"].p, g["turned"].offset(k), self.rows.p, self.rows.offset(k),
                                       self.rope, self.rope_ws.p, stream)

    def step(self, rate, stream=None):
        for name in ("rows", "q_weight", "k_weight", "bias"):  # what all tokens share gets their sum: smaller steps
            mine = rate if name == "rows" else rate / TOKENS
            self.L.launch_sgd_step(getattr(self, name).p, self.grads[name].p, mine, getattr(self, name).n, stream)


def train(nn, L, steps=20, seed=0):
    """Losses of `steps` gradient steps."""
    rng = np.random.default_rng(seed)
    layer = Layer(nn, L, rng)
    target = L.to_device(0.3 * rng.standard_normal((TOKENS, HEADS * DIM)).astype(np.float32))
    dout, losses = L.alloc(TOKENS * HEADS * DIM), []
    for _ in range(steps):
        layer.forward()
        L.launch_weighted_sum(dout.p, layer.out.p, target.p, 1.0, -1.0, dout.n, None)  # of half the squared distance
        layer.backward(dout)
        layer.step(1.0)
        losses.append(0.5 * float(np.mean(dout.download().astype(np.float64) ** 2)))
    return losses


def decode(nn, L, tokens=100, seed=0):
    """Largest difference of the layer token by token over a cache from the layer at once."""
    rng = np.random.default_rng(seed)
    q = L.to_device(rng.standard_normal((tokens, HEADS, DIM)).astype(np.float32))
    # a cache of each key head's tokens together, with room for more
    room = tokens + 28
    k, v = (L.to_device(rng.standard_normal((KV, room, DIM)).astype(np.float32)) for _ in range(2))
    outs = []
    for at, length in [(0, tokens)] + [(i, 1) for i in range(tokens)]:
        start, held = ints(L, [at]), ints(L, [at + length])
        a = nn.NnAttention(dtype=nn.NN_F32, batch=1, len_q=length, len_k=room, heads=HEADS, kv_heads=KV, head_dim=DIM,
                           scale=DIM**-0.5, mask=nn.NN_MASK_CAUSAL, q_stride=(0, HEADS * DIM, DIM),
                           k_stride=(0, DIM, room * DIM), v_stride=(0, DIM, room * DIM),
                           out_stride=(0, HEADS * DIM, DIM), q_start=start.p, k_len=held.p)
        out, lse = L.alloc(length * HEADS * DIM), L.alloc(HEADS * length)
        ws = L.to_device(np.zeros(max(1, L.nnhip_attention_forward_workspace(a)), np.float32))
        L.launch_attention_forward(out.p, lse.p, q.offset(at * HEADS * DIM), k.p, v.p, a, ws.p, None)
        L.sync()
        outs.append(out.download(shape=(length, HEADS * DIM)))
    return float(np.abs(outs[0] - np.concatenate(outs[1:])).max())


def main():
    nn = load_package()
    L = nn.lib()
    losses = train(nn, L, int(sys.argv[1]) if len(sys.argv) > 1 else 20)
    print("loss", " ".join(f"{x:.5f}" for x in losses))
    print(f"decoding token by token differs by {decode(nn, L):.2e} at most")


if __name__ == "__main__":
    main()
