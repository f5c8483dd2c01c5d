"""The attention operators, as cases to measure: position-aware query/key norms, attention with capped scores, a
learned bias by distance buckets and document, prefix and length masks, its gradients, and its form for few queries.

A transformer block of a diffusion or token model runs them in this order: one projection makes queries, keys and
values; each head's query and key is normalised and rotated by its position; attention mixes the values.  listed()
holds sizes of this repository's images (28 x 28 and 64 x 64 tokens) and generic ones; draw() spreads over the
ranges that they stand for.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
DEV = "cuda"
own = False


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _rope(name, kind, dtype, tokens, heads, kv_heads, dim, rot, axes, interleaved, far):
    return {"name": name, "kind": kind, "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "axes": axes, "interleaved": interleaved, "far": far}


def _attn(name, kind, dtype, batch, len_q, len_k, heads, kv_heads, dim, mask="none", cap=0.0, buckets=0, distance=0,
          docs=0, ragged=False, packed=False):
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "len_q": len_q, "len_k": len_k,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "mask": mask, "cap": cap, "buckets": buckets,
            "distance": distance, "docs": docs, "ragged": ragged, "packed": packed}


def listed():
    return [
        # one decoding step's queries and keys, four requests far into their contexts: all launch and latency
        _rope("rope_4_tokens", "rope", "bf16", 4, 32, 8, 128, 128, 1, False, 1 << 20),
        # queries and keys of eight 64 x 64 images in fp32, rows and columns rotated by an axis each
        _rope("rope_64x64", "rope", "f32", 8 * 64 * 64, 16, 16, 64, 64, 2, True, 64),
        # a training step's forward and backward over a long packed batch, shared key heads
        _rope("rope_train_32k", "rope_train", "bf16", 32768, 32, 8, 128, 128, 1, False, 8192),
        # the same on ragged sizes: 785 tokens (28 x 28 and a class token), heads of 72 of which 48 are rotated
        _rope("rope_train_785", "rope_train", "f32", 3 * 785, 16, 16, 72, 48, 2, False, 28),
        # attention over a small image level's pixels in fp32, with a learned bias by distance
        _attn("attn_28x28_f32", "attn", "f32", 8, 784, 784, 4, 4, 32, buckets=32, distance=128, packed=True),
        # images of different sizes packed into one sequence, each attending to itself only; heads of 72
        _attn("attn_packed_8k", "attn", "bf16", 1, 8192, 8192, 16, 16, 72, docs=13, packed=True),
        # a long sequence whose first part is seen by all (a prompt), the rest by what follows; capped scores
        _attn("attn_prefix_16k", "attn", "bf16", 1, 16384, 16384, 16, 4, 128, mask="prefix", cap=50.0),
        # one new token of one request over a short cache
        _attn("decode_777", "attn", "bf16", 1, 1, 777, 8, 8, 64, mask="causal", ragged=True),
        # one new token of each of 16 requests, caches of up to 32768 tokens filled to different lengths
        _attn("decode_32k", "attn", "bf16", 16, 1, 32768, 32, 8, 128, mask="causal", cap=30.0, ragged=True),
        # a training step of an encoder's attention, the bias table's gradient with it
        _attn("train_1k_bias", "train", "bf16", 4, 1024, 1024, 16, 16, 64, buckets=32, distance=128, packed=True),
        # a training step over packed documents, causal, shared key heads, capped scores
        _attn("train_packed_8k", "train", "bf16", 1, 8192, 8192, 16, 4, 128, mask="causal", cap=50.0, docs=7),
        # a training step in fp32 on an odd length with a prefix, bias and all gradients
        _attn("train_1001_f32", "train", "f32", 2, 1001, 1001, 8, 8, 64, mask="prefix", buckets=32, distance=64),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_SCORES = {"attn": 16 * 16384 * 16384, "train": 16 * 8192 * 8192}
_MOST_CACHE = 16 * 32768 * 8 * 128
_MOST_ROWS = 32768 * 40 * 128


def draw(rng):
    kind = rng.choice(["rope", "rope_train", "attn", "attn", "train", "train", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    dim = rng.choice([8 * rng.randint(2, 16), 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4, 8])
    if kind.startswith("rope"):
        axes = rng.choice([1, 2, 3])
        rot = rng.choice([dim // (2 * axes) * (2 * axes), max(1, dim // (4 * axes)) * (2 * axes)])
        most = min(1 << 15, _MOST_ROWS // ((heads + kv) * dim))
        return {k: v for k, v in _rope("", kind, dtype, _log_int(rng, 1, most), heads, kv, dim, rot, axes,
                                       rng.random() < 0.5, rng.choice([32, 4096, 1 << 20])).items() if k != "name"}
    mask = rng.choice(["none", "causal", "prefix"])
    cap = rng.choice([0.0, 0.0, 15.0, 50.0])
    buckets, distance = rng.choice([(0, 0), (0, 0), (32, 128), (16, _log_int(rng, 20, 500))])
    while True:
        batch = _log_int(rng, 1, 16)
        if kind == "decode":
            len_k = _log_int(rng, 1, 32768)
            case = _attn("", "attn", dtype, batch, min(len_k, rng.choice([1, 1, 1, 2, 5])), len_k, heads, kv, dim,
                         mask if mask != "none" else "causal", cap, buckets, distance, 0, rng.random() < 0.8)
            fits = batch * len_k * kv * dim * (1 if dtype == "bf16" else 2) <= _MOST_CACHE
        else:
            len_q = _log_int(rng, 1, 8192)
            same = kind == "train" or rng.random() < 0.6
            len_k = len_q if same else _log_int(rng, 1, 8192)
            case = _attn("", kind, dtype, batch, len_q, len_k, heads, kv, dim, mask, cap, buckets, distance,
                         rng.choice([0, rng.randint(1, 20)]) if same else 0, False, same and rng.random() < 0.5)
            fits = batch * heads * len_q * len_k <= _MOST_SCORES[kind] // (1 if dtype == "bf16" else 4)
        if fits:
            return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------------------
# Masks: they follow from the case alone, so that its work does too
# ---------------------------------------------------------------------------
def _documents(c):
    """Document of each position: `docs` documents of uneven lengths, one after another, then 3 % of padding."""
    n = c["len_k"]
    sizes = [1.0 + (5 * i) % 7 for i in range(c["docs"])]
    ends, at = [], 0.0
    for size in sizes:
        at += size / sum(sizes) * 0.97 * n
        ends.append(round(at))
    doc, begin = [-1] * n, 0
    for d, end in enumerate(ends):
        doc[begin:end] = [d] * (end - begin)
        begin = end
    return doc


def _lengths(c):
    """Keys of each request that its cache holds so far."""
    n = c["len_k"]
    if not c["ragged"]:
        return [n] * c["batch"]
    return [max(c["len_q"], n - (b * 5 % 16) * n // 20 - b % 3) for b in range(c["batch"])]


def _prefixes(c):
    return [(c["len_k"] // 4 + 7 * b) % (c["len_k"] + 1) for b in range(c["batch"])]


def _visible(c):
    """Number of (query, key) pairs that the masks leave, over the batch."""
    total = 0
    for length, prefix in zip(_lengths(c), _prefixes(c)):
        start = length - c["len_q"] if c["ragged"] else c["len_k"] - c["len_q"]
        begin, bounds = 0, [(0, length)] * c["len_q"]
        if c["docs"]:
            doc, bounds = _documents(c), []
            while begin < len(doc):
                end = begin
                while end < len(doc) and doc[end] == doc[begin]:
                    end += 1
                bounds += [(begin, end) if doc[begin] >= 0 else (0, 0)] * (end - begin)
                begin = end
        for i, (lo, hi) in enumerate(bounds):
            limit = length
            if c["mask"] != "none":
                limit = min(length, max(start + i + 1, prefix if c["mask"] == "prefix" else 0))
            total += max(0, min(hi, limit) - lo)
    return total


def _bytes_of(c):
    return 2 if c["dtype"] == "bf16" else 4


def work(c):
    e = _bytes_of(c)
    if c["kind"].startswith("rope"):
        n = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        small = c["tokens"] * c["axes"] * 4 + 8 * c["dim"]
        if c["kind"] == "rope":
            return {"bytes": 2 * n * e + small, "flops": 8 * n}
        # forward: q, k in, rotated out; backward: their gradients in, the inputs' out (and the weights')
        return {"bytes": 4 * n * e + small + 8 * c["dim"], "flops": 24 * n}
    lengths = sum(_lengths(c)) if c["ragged"] else c["batch"] * c["len_k"]
    nq = c["batch"] * c["len_q"] * c["heads"] * c["dim"]
    nk = lengths * c["kv_heads"] * c["dim"]
    pairs = _visible(c) * c["heads"]
    lse = 4 * c["batch"] * c["len_q"] * c["heads"]
    if c["kind"] == "attn":
        return {"bytes": (2 * nq + 2 * nk) * e + lse, "flops": 4 * pairs * c["dim"]}
    # q, k, v and the output's gradient in; output, log-sum and three gradients out
    return {"bytes": (4 * nq + 4 * nk) * e + lse + 8 * c["buckets"] * c["heads"], "flops": 14 * pairs * c["dim"]}


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------
def _bucket_map(buckets, distance):
    """Bucket of each clamped distance -distance..distance: half of the buckets for either direction, the nearer
    half of those one distance each, the others spaced by the logarithm up to `distance`."""
    half, got = buckets // 2, []
    exact = half // 2
    for rel in range(-distance, distance + 1):
        d = abs(rel)
        if d >= exact:
            far = math.log(max(d, 1) / max(exact, 1)) / math.log(max(distance, exact + 1) / max(exact, 1))
            d = min(half - 1, exact + int(far * (half - exact) + 1e-9))
        got.append(d + (half if rel > 0 else 0))
    return got


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(to)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    s = {"case": c}
    h, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"].startswith("rope"):
        t = c["tokens"]
        qkv = normal(t, h + 2 * kv, dim, std=1.3)  # as the projection leaves it
        s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], eps=1e-6)
        s.update(q_weight=normal(dim, std=0.2, mean=1.0, to=torch.float32),
                 k_weight=normal(dim, std=0.2, mean=1.0, to=torch.float32))
        s["pos"] = torch.randint(0, c["far"], (t, c["axes"]), generator=g, device=DEV, dtype=torch.int32)
        per = max(1, c["rot"] // 2 // c["axes"])
        base = 10000.0 if c["far"] <= 8192 else 500000.0
        s["freq"] = base ** (-(torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64) % per) / per)
        if c["kind"] == "rope_train":
            s.update(dq_out=normal(t, h, dim), dk_out=normal(t, kv, dim))
        return s
    b, lq, lk = c["batch"], c["len_q"], c["len_k"]
    if c["packed"]:
        qkv = normal(b, lq, h + 2 * kv, dim)
        s.update(q=qkv[:, :, :h], k=qkv[:, :, h:h + kv], v=qkv[:, :, h + kv:])
    elif c["ragged"]:  # a cache: a head's tokens lie together
        s.update(q=normal(b, lq, h, dim), k=normal(b, kv, lk, dim).transpose(1, 2),
                 v=normal(b, kv, lk, dim).transpose(1, 2))
    else:
        s.update(q=normal(b, lq, h, dim), k=normal(b, lk, kv, dim), v=normal(b, lk, kv, dim))
    s["scale"] = dim ** -0.5
    if c["ragged"]:
        lengths = _lengths(c)
        s.update(k_len=ints(lengths), q_start=ints([n - lq for n in lengths]))
    if c["mask"] == "prefix":
        s["prefix"] = ints(_prefixes(c))
    if c["docs"]:
        s["doc"] = ints(_documents(c)).repeat(b, 1)
    if c["buckets"]:
        s["bias"] = normal(c["buckets"], h, to=torch.float32)
        s["bucket"] = ints(_bucket_map(c["buckets"], c["distance"]))
    if c["kind"] == "train":
        s["dout"] = normal(b, lq, h, dim)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _pairs(c, x):
    """The two members of each rotated pair and the features that are not rotated."""
    r = c["rot"]
    if c["interleaved"]:
        return x[..., 0:r:2], x[..., 1:r:2], x[..., r:]
    return x[..., :r // 2], x[..., r // 2:r], x[..., r:]


def _join(c, a, b, rest):
    turned = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1)


def _cos_sin(s):
    c = s["case"]
    pos = s["pos"].double().repeat_interleave(max(1, c["rot"] // 2 // c["axes"]), dim=1)[:, :c["rot"] // 2]
    angle = pos * s["freq"]  # far positions: 64 bits
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _norm_rope(s, x, weight, cos, sin):
    x = x.float()
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    a, b, rest = _pairs(s["case"], x * rstd * weight)
    return _join(s["case"], a * cos - b * sin, a * sin + b * cos, rest), rstd


def _norm_rope_grad(s, x, rstd, weight, grad, cos, sin):
    xn = x.float() * rstd
    a, b, rest = _pairs(s["case"], grad.float())
    g = _join(s["case"], a * cos + b * sin, b * cos - a * sin, rest)
    dweight = (g * xn).double().sum((0, 1)).float()
    gw = g * weight
    return rstd * (gw - xn * (gw * xn).mean(-1, keepdim=True)), dweight


def _plain_rope(s):
    cos, sin = _cos_sin(s)
    t = s["q"].dtype
    q_out, q_rstd = _norm_rope(s, s["q"], s["q_weight"], cos, sin)
    k_out, k_rstd = _norm_rope(s, s["k"], s["k_weight"], cos, sin)
    got = {"q_out": q_out.to(t), "k_out": k_out.to(t)}
    if s["case"]["kind"] == "rope_train":
        dq, dqw = _norm_rope_grad(s, s["q"], q_rstd, s["q_weight"], s["dq_out"], cos, sin)
        dk, dkw = _norm_rope_grad(s, s["k"], k_rstd, s["k_weight"], s["dk_out"], cos, sin)
        got.update(dq=dq.to(t), dk=dk.to(t), dq_weight=dqw, dk_weight=dkw)
    return got


def _mask_and_distance(s):
    """Which keys each query sees, [batch or 1, 1, len_q, len_k], and the map's entry of each pair."""
    c = s["case"]
    i = torch.arange(c["len_q"], device=DEV)[None, None, :, None]
    j = torch.arange(c["len_k"], device=DEV)[None, None, None, :]
    pos = i + (s["q_start"].view(-1, 1, 1, 1) if "q_start" in s else c["len_k"] - c["len_q"])
    seen = j < (s["k_len"].view(-1, 1, 1, 1) if "k_len" in s else c["len_k"])
    if c["mask"] == "causal":
        seen = seen & (j <= pos)
    elif c["mask"] == "prefix":
        seen = seen & ((j <= pos) | (j < s["prefix"].view(-1, 1, 1, 1)))
    if "doc" in s:
        seen = seen & (s["doc"][:, None, :, None] == s["doc"][:, None, None, :]) & (s["doc"][:, None, None, :] >= 0)
    at = None
    if c["buckets"]:
        at = (j - pos).clamp(-c["distance"], c["distance"]) + c["distance"]
    return seen, at


def _plain_attention(s):
    c = s["case"]
    b, lq, lk, h, kv, dim = (c[n] for n in ("batch", "len_q", "len_k", "heads", "kv_heads", "dim"))
    group, t = h // kv, s["q"].dtype

    def by_head(x, n):  # [batch, length, heads, dim] -> [batch, kv heads, group * length, dim]
        return x.float().transpose(1, 2).reshape(b, kv, group * n if x.shape[2] == h else n, dim)

    q, k, v = by_head(s["q"], lq), s["k"].float().transpose(1, 2).contiguous(), s["v"].float().transpose(1, 2).contiguous()
    seen, at = _mask_and_distance(s)
    x = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, h, lq, lk)
    if c["cap"]:
        capped = torch.tanh(x / c["cap"])
        x = capped * c["cap"]
    if at is not None:
        bucket = s["bucket"].long()[at]  # [batch or 1, 1, len_q, len_k]
        x = x + s["bias"][bucket[:, 0]].permute(0, 3, 1, 2)
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(x - top)
    del x
    total = p.sum(-1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(-1)  # -inf where a query sees nothing
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    pk = p.view(b, kv, group * lq, lk)

    def by_token(x):
        return x.reshape(b, h, lq, dim).transpose(1, 2)

    out = torch.matmul(pk, v)
    got = {"out": by_token(out).to(t), "lse": lse}
    if c["kind"] == "attn":
        return got
    dout = by_head(s["dout"], lq)
    got["dv"] = torch.matmul(pk.transpose(2, 3), dout).transpose(1, 2).to(t)
    dp = torch.matmul(dout, v.transpose(2, 3)).view(b, h, lq, lk)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True))
    del dp, p, pk
    if at is not None:
        # pairs of one distance lie on a diagonal: each row shifted by its number, the diagonals are columns
        skew = torch.nn.functional.pad(ds.sum(0).flip(1), (0, lq)).view(h, -1)[:, :-lq].view(h, lq, lq + lk - 1)
        rel = torch.arange(1 - lq, lk, device=DEV) - (lk - lq)
        of_rel = s["bucket"].long()[rel.clamp(-c["distance"], c["distance"]) + c["distance"]]
        which = torch.nn.functional.one_hot(of_rel, c["buckets"]).double()
        got["dbias"] = torch.matmul(skew.double().sum(1), which).t().float()
    if c["cap"]:
        ds = ds * (1 - capped * capped)
    ds = (ds * s["scale"]).view(b, kv, group * lq, lk)
    got["dq"] = by_token(torch.matmul(ds, k)).to(t)
    got["dk"] = torch.matmul(ds.transpose(2, 3), q).transpose(1, 2).to(t)
    return got


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _package():
    """The package; its folder's name is not an identifier, so it is loaded from its path."""
    name = "cuda_c_diffusion_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, ROOT / "cuda-c-diffusion_amd" / "__init__.py")
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _ptr(x):
    return None if x is None else x.data_ptr()


def _workspace(floats):
    return torch.zeros(max(1, floats), dtype=torch.float32, device=DEV)


def _rope_call(s):
    """What a program keeps beside its inputs: the description of the call, outputs and workspace."""
    nn, c = _package(), s["case"]
    L = nn.lib()
    q, k = s["q"], s["k"]
    r = {"L": L, "q_out": torch.empty(q.shape, dtype=q.dtype, device=DEV),
         "k_out": torch.empty(k.shape, dtype=k.dtype, device=DEV)}
    r["args"] = a = nn.NnQkNormRope(
        dtype=nn.NN_BF16 if c["dtype"] == "bf16" else nn.NN_F32, tokens=c["tokens"], heads=c["heads"],
        kv_heads=c["kv_heads"], head_dim=c["dim"], rot_dim=c["rot"], axes=c["axes"],
        interleaved=int(c["interleaved"]), eps=s["eps"], q_stride=q.stride()[:2], k_stride=k.stride()[:2],
        q_out_stride=r["q_out"].stride()[:2], k_out_stride=r["k_out"].stride()[:2], q_weight=_ptr(s["q_weight"]),
        k_weight=_ptr(s["k_weight"]), pos=_ptr(s["pos"]), freq=_ptr(s["freq"]))
    if c["kind"] == "rope_train":
        dqkv = torch.empty(c["tokens"], c["heads"] + 2 * c["kv_heads"], c["dim"], dtype=q.dtype, device=DEV)
        r.update(dq=dqkv[:, :c["heads"]], dk=dqkv[:, c["heads"]:c["heads"] + c["kv_heads"]],
                 dq_weight=torch.empty_like(s["q_weight"]), dk_weight=torch.empty_like(s["k_weight"]),
                 workspace=_workspace(L.nnhip_qk_norm_rope_workspace(a)))
    return r


def _own_rope(s):
    if "call" not in s:
        s["call"] = _rope_call(s)
    r = s["call"]
    L, a, stream = r["L"], r["args"], torch.cuda.current_stream().cuda_stream
    L.launch_qk_norm_rope_forward(_ptr(r["q_out"]), _ptr(r["k_out"]), _ptr(s["q"]), _ptr(s["k"]), a, stream)
    got = {"q_out": r["q_out"], "k_out": r["k_out"]}
    if s["case"]["kind"] == "rope_train":
        L.launch_qk_norm_rope_backward(_ptr(r["dq"]), _ptr(r["dk"]), _ptr(r["dq_weight"]), _ptr(r["dk_weight"]),
                                       _ptr(s["dq_out"]), _ptr(s["dk_out"]), _ptr(s["q"]), _ptr(s["k"]), a,
                                       _ptr(r["workspace"]), stream)
        got.update({n: r[n] for n in ("dq", "dk", "dq_weight", "dk_weight")})
    return got


def _attention_call(s):
    nn, c = _package(), s["case"]
    L = nn.lib()
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    r = {"L": L, "out": out, "lse": torch.empty(c["batch"], c["heads"], c["len_q"], device=DEV)}
    doc = s.get("doc")
    r["args"] = a = nn.NnAttention(
        dtype=nn.NN_BF16 if c["dtype"] == "bf16" else nn.NN_F32, batch=c["batch"], len_q=c["len_q"], len_k=c["len_k"],
        heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["dim"], scale=s["scale"], softcap=c["cap"],
        mask={"none": nn.NN_MASK_NONE, "causal": nn.NN_MASK_CAUSAL, "prefix": nn.NN_MASK_PREFIX}[c["mask"]],
        buckets=c["buckets"], max_distance=c["distance"], q_stride=q.stride()[:3], k_stride=k.stride()[:3],
        v_stride=v.stride()[:3], out_stride=out.stride()[:3], q_start=_ptr(s.get("q_start")),
        k_len=_ptr(s.get("k_len")), prefix=_ptr(s.get("prefix")), doc_q=_ptr(doc), doc_k=_ptr(doc),
        bucket=_ptr(s.get("bucket")), bias=_ptr(s.get("bias")))
    r["workspace"] = _workspace(L.nnhip_attention_forward_workspace(a))
    if c["kind"] == "train":
        if c["packed"]:
            h, kv = c["heads"], c["kv_heads"]
            grad = torch.empty(c["batch"], c["len_q"], h + 2 * kv, c["dim"], dtype=q.dtype, device=DEV)
            r.update(dq=grad[:, :, :h], dk=grad[:, :, h:h + kv], dv=grad[:, :, h + kv:])
        else:
            r.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
        if c["buckets"]:
            r["dbias"] = torch.empty_like(s["bias"])
        r["backward_workspace"] = _workspace(L.nnhip_attention_backward_workspace(a))
    return r


def _own_attention(s):
    if "call" not in s:
        s["call"] = _attention_call(s)
    r = s["call"]
    L, a, stream = r["L"], r["args"], torch.cuda.current_stream().cuda_stream
    q, k, v = _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"])
    L.launch_attention_forward(_ptr(r["out"]), _ptr(r["lse"]), q, k, v, a, _ptr(r["workspace"]), stream)
    got = {"out": r["out"], "lse": r["lse"]}
    if s["case"]["kind"] == "train":
        L.launch_attention_backward(_ptr(r["dq"]), _ptr(r["dk"]), _ptr(r["dv"]), _ptr(r.get("dbias")),
                                    _ptr(s["dout"]), q, k, v, _ptr(r["out"]), _ptr(r["lse"]), a,
                                    _ptr(r["backward_workspace"]), stream)
        got.update({n: r[n] for n in ("dq", "dk", "dv", "dbias") if n in r})
    return got


def run(s):
    if s["case"]["kind"].startswith("rope"):
        return _own_rope(s) if own else _plain_rope(s)
    return _own_attention(s) if own else _plain_attention(s)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rope_rows(s, x, weight, grad):
    """Rows [tokens, heads, dim] of one tensor: each pair as a complex number, turned by e^(i angle)."""
    c, r = s["case"], s["case"]["rot"]
    x, w = x.double(), weight.double()
    order = torch.arange(r, device=DEV)
    order = order.view(-1, 2) if c["interleaved"] else order.view(2, -1).t()
    first, second = order[:, 0], order[:, 1]
    axis = torch.arange(r // 2, device=DEV) // max(1, r // 2 // c["axes"])
    turn = torch.exp(1j * (s["pos"].double()[:, axis] * s["freq"]))[:, None, :]

    def turned(y, by):
        z, y = torch.complex(y[..., first], y[..., second]) * by, y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    size = (x.square().sum(-1, keepdim=True) / c["dim"] + s["eps"]).sqrt()
    unit = x / size
    out = turned(unit * w, turn)
    if grad is None:
        return out, None, None
    back = turned(grad.double(), turn.conj())
    dw = torch.einsum("thd,thd->d", back, unit)
    along = (back * w * unit).sum(-1, keepdim=True) / c["dim"]
    return out, (back * w - along * unit) / size, dw


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"].startswith("rope"):
        q_out, dq, dqw = _exact_rope_rows(s, s["q"], s["q_weight"], s.get("dq_out"))
        k_out, dk, dkw = _exact_rope_rows(s, s["k"], s["k_weight"], s.get("dk_out"))
        got = {"q_out": q_out, "k_out": k_out}
        if c["kind"] == "rope_train":
            got.update(dq=dq, dk=dk, dq_weight=dqw, dk_weight=dkw)
        return got
    b, lq, lk, h, kv = (c[n] for n in ("batch", "len_q", "len_k", "heads", "kv_heads"))
    train = c["kind"] == "train"
    f64 = {"dtype": torch.float64, "device": DEV}
    got = {"out": torch.zeros(s["q"].shape, **f64), "lse": torch.empty(b, h, lq, **f64)}
    if train:
        got.update(dq=torch.zeros(s["q"].shape, **f64), dk=torch.zeros(s["k"].shape, **f64),
                   dv=torch.zeros(s["v"].shape, **f64))
        if c["buckets"]:
            got["dbias"] = torch.zeros(c["buckets"], h, **f64)
    key = torch.arange(lk, device=DEV)
    for n in range(b):
        place = torch.arange(lq, device=DEV) + (int(s["q_start"][n]) if "q_start" in s else lk - lq)
        hidden = (key >= (int(s["k_len"][n]) if "k_len" in s else lk)).expand(lq, lk).clone()
        if c["mask"] != "none":
            late = key[None, :] > place[:, None]
            if c["mask"] == "prefix":
                late &= key[None, :] >= int(s["prefix"][n])
            hidden |= late
        if "doc" in s:
            d = s["doc"][n]
            hidden |= (d[:, None] != d[None, :]) | (d < 0)[None, :]
        empty = hidden.all(1)
        for m in range(h):
            q, k, v = s["q"][n, :, m].double(), s["k"][n, :, m * kv // h].double(), s["v"][n, :, m * kv // h].double()
            score = q @ k.t() * s["scale"]
            if c["cap"]:
                slope = 1 / torch.cosh(score / c["cap"]) ** 2
                score = torch.tanh(score / c["cap"]) * c["cap"]
            if c["buckets"]:
                far = (key[None, :] - place[:, None]).clamp(-c["distance"], c["distance"]) + c["distance"]
                which = s["bucket"].long()[far]
                score = score + s["bias"][:, m].double()[which]
            score[hidden] = -math.inf
            lse = torch.logsumexp(score, 1)
            p = torch.exp(score - lse[:, None])
            p[empty] = 0
            got["lse"][n, m] = lse
            out = p @ v
            got["out"][n, :, m] = out
            if train:
                dout = s["dout"][n, :, m].double()
                got["dv"][n, :, m * kv // h] += p.t() @ dout
                ds = p * (dout @ v.t() - (dout * out).sum(1, keepdim=True))
                if c["buckets"]:
                    got["dbias"][:, m] += torch.zeros(c["buckets"], **f64).index_add_(0, which.reshape(-1), ds.reshape(-1))
                if c["cap"]:
                    ds = ds * slope
                got["dq"][n, :, m] = ds @ k * s["scale"]
                got["dk"][n, :, m * kv // h] += ds.t() @ q * s["scale"]
    return got
