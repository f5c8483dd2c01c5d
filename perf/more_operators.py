"""The operators of a paged cache, as cases to measure: the append of a projection's rows (norm, rotation, the write into
pages, in the tensors' type or in 4 bits), attention that reads the pages, and the way back out of them.

A serving program runs them in this order for every layer: a projection makes queries, keys and values of the new
tokens; the append turns them and writes keys and values to the pages of their requests; attention reads the pages.
listed() holds prompts, decoding steps and small chunks; draw() spreads over the ranges that they stand for.
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
def _append(name, dtype, kind, requests, tokens, heads, kv_heads, dim, rot, axes, interleaved, norm, page, far, padded=0):
    """`tokens` new tokens of each of `requests` requests; `padded` rows of each are no tokens."""
    return {"name": name, "op": "append", "dtype": dtype, "kind": kind, "requests": requests, "tokens": tokens,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "axes": axes, "interleaved": interleaved,
            "norm": norm, "page": page, "far": far, "padded": padded}


def _attention(name, dtype, kind, batch, len_q, len_k, heads, kv_heads, dim, page, mask="causal", cap=0.0, buckets=0,
               distance=0, ragged=True):
    return {"name": name, "op": "attention", "dtype": dtype, "kind": kind, "batch": batch, "len_q": len_q, "len_k": len_k,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "mask": mask, "cap": cap, "buckets": buckets,
            "distance": distance, "ragged": ragged}


def _read(name, dtype, kind, requests, tokens, kv_heads, dim, page):
    return {"name": name, "op": "read", "dtype": dtype, "kind": kind, "requests": requests, "tokens": tokens,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def listed():
    return [
        # one decoding step's rows, four requests far into their contexts, pages of 4 bits: all launch and latency
        _append("append_4_mxfp4", "bf16", "mxfp4", 4, 1, 32, 8, 128, 128, 1, False, True, 64, 1 << 20),
        # a long prompt into pages of 4 bits, keys that are turned but not normalised
        _append("append_prompt_8k_mxfp4", "bf16", "mxfp4", 1, 8192, 32, 8, 128, 128, 1, False, False, 64, 8192),
        # three images of 28 x 28 tokens and a class token, a padded batch, fp32, heads of 72 of which 48 are turned
        _append("append_785_f32", "f32", "plain", 3, 785, 16, 16, 72, 48, 2, True, True, 16, 28, 13),
        # one new token of each of 16 requests, caches of up to 32768 tokens filled to different lengths, capped scores
        _attention("paged_32k", "bf16", "plain", 16, 1, 32768, 32, 8, 128, 64, cap=30.0),
        # a part of a long prompt over what came before it
        _attention("paged_prompt_16k", "bf16", "plain", 1, 2048, 16384, 16, 4, 128, 64, ragged=False),
        # one new token of one request over a short cache, in 4 bits
        _attention("mxfp4_777", "bf16", "mxfp4", 1, 1, 777, 8, 8, 64, 16),
        # as paged_32k, in 4 bits
        _attention("mxfp4_32k", "bf16", "mxfp4", 16, 1, 32768, 32, 8, 128, 64, cap=30.0),
        # five drafted tokens of each of 48 requests over caches of middle length
        _attention("mxfp4_drafts_4k", "bf16", "mxfp4", 48, 5, 4096, 16, 4, 128, 32),
        # as paged_prompt_16k, in 4 bits
        _attention("mxfp4_prompt_16k", "bf16", "mxfp4", 1, 2048, 16384, 16, 4, 128, 64, ragged=False),
        # fp32 queries over a cache of 4 bits, a few tokens each, odd sizes and a learned bias by distance
        _attention("mxfp4_5001_f32", "f32", "mxfp4", 3, 7, 5001, 12, 4, 96, 16, mask="prefix", buckets=32, distance=128),
        # a long request on its way to another machine
        _read("read_32k_mxfp4", "bf16", "mxfp4", 1, 32768, 8, 128, 64),
        # what two short requests hold, fp32
        _read("read_2x101_f32", "f32", "plain", 2, 101, 4, 72, 16),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_ROWS = 8192 * 48 * 128
_MOST_READ = 32768 * 8 * 128
_MOST_CACHE = 16 * 32768 * 8 * 128
_MOST_SCORES = 16 * 2048 * 16384


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "prompt", "read"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    kind = rng.choice(["plain", "mxfp4", "mxfp4"])
    dim = rng.choice([8 * rng.randint(2, 16), 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    wide = 1 if dtype == "bf16" else 2
    while True:
        if op == "append":
            requests = _log_int(rng, 1, 256)
            tokens = rng.choice([1, _log_int(rng, 1, 8192)])
            axes = rng.choice([1, 1, 2, 3])
            rot = rng.choice([dim // (2 * axes) * (2 * axes), max(1, dim // (4 * axes)) * (2 * axes)])
            case = _append("", dtype, kind, requests, tokens, heads, kv, dim, rot, axes, rng.random() < 0.5,
                           rng.random() < 0.6, page, rng.choice([32, 4096, 1 << 20]), rng.choice([0, 0, tokens // 5]))
            fits = requests * tokens * (heads + 2 * kv) * dim * wide <= _MOST_ROWS
        elif op == "read":
            case = _read("", dtype, kind, _log_int(rng, 1, 16), _log_int(rng, 1, 32768), kv, dim, page)
            fits = case["requests"] * case["tokens"] * kv * dim * wide <= _MOST_READ
        else:
            mask, cap = rng.choice(["none", "causal", "causal", "prefix"]), rng.choice([0.0, 0.0, 15.0, 50.0])
            buckets, distance = rng.choice([(0, 0), (0, 0), (0, 0), (32, 128), (16, _log_int(rng, 20, 500))])
            batch, len_k = _log_int(rng, 1, 48), _log_int(rng, 1, 32768)
            len_q = rng.choice([1, 1, 1, 2, 5, 9]) if op == "attention" else _log_int(rng, 16, 2048)
            case = _attention("", dtype, kind, batch, min(len_q, len_k), len_k, heads, kv, dim, page, mask, cap, buckets,
                              distance, rng.random() < 0.8)
            fits = batch * len_k * kv * dim * wide <= _MOST_CACHE
            fits = fits and batch * heads * case["len_q"] * len_k * wide * wide <= _MOST_SCORES
        if fits:
            return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------------------
# What follows from the case alone
# ---------------------------------------------------------------------------
def _lengths(c):
    """Tokens of each request that its cache holds, the new ones among them."""
    n = c["len_k"]
    if not c["ragged"]:
        return [n] * c["batch"]
    return [max(c["len_q"], n - (b * 5 % 16) * n // 20 - b % 3) for b in range(c["batch"])]


def _prefixes(c):
    return [(c["len_k"] // 4 + 7 * b) % (c["len_k"] + 1) for b in range(c["batch"])]


def _bytes_of(c):
    return 2 if c["dtype"] == "bf16" else 4


def _row_bytes(c):
    """Bytes of a token's key (or value) of one head in the cache."""
    return -(-c["dim"] // 32) * 17 if c["kind"] == "mxfp4" else c["dim"] * _bytes_of(c)


def work(c):
    e = _bytes_of(c)
    if c["op"] == "append":
        t = c["requests"] * (c["tokens"] - c["padded"])
        h, kv, d = c["heads"], c["kv_heads"], c["dim"]
        read = t * (h + 2 * kv) * d * e + t * (4 * c["axes"] + 8) + 4 * c["rot"] + (8 * d if c["norm"] else 0)
        back = 2 * t * kv * (_row_bytes(c) + d * e) if c["kind"] == "mxfp4" else 0  # out of the pages, as values
        return {"bytes": read + t * h * d * e + 2 * t * kv * _row_bytes(c) + back, "flops": 8 * t * (h + kv) * d}
    if c["op"] == "read":
        rows = c["requests"] * c["tokens"]
        return {"bytes": rows * (8 + 2 * c["kv_heads"] * (_row_bytes(c) + c["dim"] * e)), "flops": 0}
    lengths = _lengths(c)
    nq = c["batch"] * c["len_q"] * c["heads"]
    pairs = 0
    for length, prefix in zip(lengths, _prefixes(c)):
        for i in range(c["len_q"]):
            seen = length
            if c["mask"] != "none":
                seen = min(length, max(length - c["len_q"] + i + 1, prefix if c["mask"] == "prefix" else 0))
            pairs += seen
    cache = 2 * sum(lengths) * c["kv_heads"] * _row_bytes(c) + 4 * sum(-(-n // c["page"]) for n in lengths)
    return {"bytes": 2 * nq * c["dim"] * e + 4 * nq + cache, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---------------------------------------------------------------------------
# The cache's layout: pages [kv_heads, page tokens] of rows on 16 bytes each; in 4 bits a head's rows (16 bytes for 32
# features, feature 2 i in the low half of byte i), then its scales (a byte for 32 features, 127 + exponent)
# ---------------------------------------------------------------------------
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _grid(like):
    half = torch.tensor(_GRID, dtype=like, device=DEV)
    return torch.cat((half, -half))


def _row_values(c):
    e = _bytes_of(c)
    return -(-c["dim"] * e // 16) * 16 // e


def _quantised(x):
    """Rows [..., dim] of 64-bit values: codes [..., groups, 32] in 0..15 and exponents [..., groups]."""
    groups = -(-x.shape[-1] // 32)
    x = torch.nn.functional.pad(x, (0, groups * 32 - x.shape[-1])).unflatten(-1, (groups, 32))
    top, power = torch.frexp(x.abs().amax(-1))
    power = torch.where(top > 0.875, power - 2, power - 3).clamp(-120, 125)
    power = torch.where(top == 0, torch.full_like(power, -120), power)
    y = torch.ldexp(x.abs(), -power.unsqueeze(-1))
    code = torch.zeros(y.shape, dtype=torch.uint8, device=DEV)
    for at, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (y >= at) if up else (y > at)  # a value half way goes to the even code
    return code + (x < 0).to(torch.uint8) * 8, power


def _packed(code, power, pool, page, slot):
    """Writes rows [n, kv_heads, ...] into pool [pages, kv_heads, block bytes] at (page, slot)."""
    groups, tokens = power.shape[-1], pool.shape[-1] // (power.shape[-1] * 17)
    rows = pool[..., :tokens * groups * 16].unflatten(-1, (tokens, groups * 16))
    scales = pool[..., tokens * groups * 16:].unflatten(-1, (tokens, groups))
    rows[page, :, slot] = (code[..., 0::2] | code[..., 1::2] << 4).flatten(-2)
    scales[page, :, slot] = (power + 127).to(torch.uint8)


def _unpacked(c, pool, page, slot, like):
    """Rows [..., kv_heads, dim] of the tokens at (page, slot), as the values that they stand for."""
    if c["kind"] == "plain":
        return pool[page, :, slot][..., :c["dim"]].to(like)
    groups = -(-c["dim"] // 32)
    rows = pool[..., :c["page"] * groups * 16].unflatten(-1, (c["page"], groups * 16))[page, :, slot].unflatten(-1, (groups, 16))
    scales = pool[..., c["page"] * groups * 16:].unflatten(-1, (c["page"], groups))[page, :, slot]
    code = torch.stack((rows & 15, rows >> 4), -1).flatten(-2)
    values = _grid(like)[code.int()] * torch.ldexp(torch.ones((), dtype=like, device=DEV), scales.int() - 127).unsqueeze(-1)
    return values.flatten(-2)[..., :c["dim"]]


def _pool(c, pages):
    if c["kind"] == "plain":
        dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
        return torch.zeros(pages, c["kv_heads"], c["page"], _row_values(c), dtype=dtype, device=DEV)
    return torch.zeros(pages, c["kv_heads"], c["page"] * -(-c["dim"] // 32) * 17, dtype=torch.uint8, device=DEV)


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------
def _table(g, counts):
    """Page numbers [requests, most pages], scattered over the pool as a running server leaves them; -1 past the end."""
    width, total = max(counts), sum(counts)
    order = torch.randperm(total + 3, generator=g, device=DEV)[:total].to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
    used = torch.arange(width, device=DEV) < torch.tensor(counts, device=DEV)[:, None]
    table[used] = order
    return table, total + 3


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(to)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    def fill(pages):  # pages of keys and values as appends left them
        for name in ("k_pool", "v_pool"):
            s[name] = _pool(c, pages)
            for first in range(0, pages, 4096 * 64 // c["page"]):  # in parts: 64-bit values of a whole cache are many
                part = s[name][first:first + 4096 * 64 // c["page"]]
                x = normal(part.shape[0], c["page"], kv, dim, to=torch.float32)
                if c["kind"] == "plain":
                    part[..., :dim] = x.transpose(1, 2).to(dtype)
                else:
                    code, power = _quantised(x.double().flatten(0, 1))
                    at = torch.arange(part.shape[0], device=DEV).repeat_interleave(c["page"])
                    _packed(code, power, part, at, torch.arange(c["page"], device=DEV).repeat(part.shape[0]))

    s, kv, dim = {"case": c}, c["kv_heads"], c["dim"]
    if c["op"] == "read":
        n, each = c["requests"], c["tokens"]
        s["table"], pages = _table(g, [-(-each // c["page"])] * n)
        fill(pages)
        s["request"] = torch.arange(n, device=DEV, dtype=torch.int32).repeat_interleave(each)
        s["place"] = torch.arange(each, device=DEV, dtype=torch.int32).repeat(n)
        return s
    h = c["heads"]
    if c["op"] == "append":
        n, each = c["requests"], c["tokens"]
        held = [(11 * r) % 40 for r in range(n)]  # tokens that the requests have already
        s["table"], pages = _table(g, [-(-(held[r] + each) // c["page"]) for r in range(n)])
        s.update(k_pool=_pool(c, pages), v_pool=_pool(c, pages))
        qkv = normal(n * each, h + 2 * kv, dim, std=1.3)  # as the projection leaves it
        s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], eps=1e-6)
        if c["norm"]:
            s.update(q_weight=normal(dim, std=0.2, mean=1.0, to=torch.float32),
                     k_weight=normal(dim, std=0.2, mean=1.0, to=torch.float32))
        s["pos"] = torch.randint(0, c["far"], (n * each, c["axes"]), generator=g, device=DEV, dtype=torch.int32)
        per = max(1, c["rot"] // 2 // c["axes"])
        base = 10000.0 if c["far"] <= 8192 else 500000.0
        s["freq"] = base ** (-(torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64) % per) / per)
        s["request"] = torch.arange(n, device=DEV, dtype=torch.int32).repeat_interleave(each)
        place = torch.arange(each, device=DEV, dtype=torch.int32) + ints(held)[:, None]
        if c["padded"]:
            place[:, each - c["padded"]:] = -1
        s["place"] = place.flatten()
        return s
    b, lq = c["batch"], c["len_q"]
    lengths = _lengths(c)
    s["table"], pages = _table(g, [max(1, -(-n // c["page"])) for n in lengths])
    fill(pages)
    s.update(q=normal(b, lq, h, dim), scale=dim ** -0.5, k_len=ints(lengths), q_start=ints([n - lq for n in lengths]))
    if c["mask"] == "prefix":
        s["prefix"] = ints(_prefixes(c))
    if c["buckets"]:
        far = torch.arange(-c["distance"], c["distance"] + 1, device=DEV).abs().double()
        near = (c["buckets"] - 1) * torch.log1p(far) / math.log1p(c["distance"])
        s["bucket"] = near.round().to(torch.int32)
        s["bias"] = normal(c["buckets"], h, to=torch.float32)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _turned(s, x, weight, like):
    """Rows [tokens, heads, dim] normalised and turned, in `like`; angles of far positions in 64 bits."""
    c, r = s["case"], s["case"]["rot"]
    x = x.to(like)
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * weight.to(like)
    per = max(1, r // 2 // c["axes"])
    angle = s["pos"].double().repeat_interleave(per, dim=1)[:, :r // 2] * s["freq"]
    cos, sin = angle.cos().to(like)[:, None], angle.sin().to(like)[:, None]
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _places(s):
    """Page and slot of every token that is one, and which these are."""
    live = s["place"] >= 0
    place = s["place"][live].long()
    page = s["table"][s["request"][live].long(), place // s["case"]["page"]].long()
    return live, page, place % s["case"]["page"]


def _plain_append(s):
    c, t = s["case"], s["q"].dtype
    live, page, slot = _places(s)
    got = {"q_out": torch.zeros_like(s["q"])}
    got["q_out"][live] = _turned(s, s["q"], s.get("q_weight"), torch.float32).to(t)[live]
    if c["kind"] == "plain":
        k = _turned(s, s["k"], s.get("k_weight"), torch.float32)[live].to(t)
        s["k_pool"][page, :, slot, :c["dim"]] = k
        s["v_pool"][page, :, slot, :c["dim"]] = s["v"][live]
        got.update(k_pool=s["k_pool"], v_pool=s["v_pool"])
        return got
    k = _turned(s, s["k"], s.get("k_weight"), torch.float64)[live]  # which of two codes: 64 bits
    _packed(*_quantised(k), s["k_pool"], page, slot)
    _packed(*_quantised(s["v"][live].double()), s["v_pool"], page, slot)
    for name in ("k", "v"):
        got[name] = torch.zeros(s[name].shape, dtype=t, device=DEV)
        got[name][live] = _unpacked(c, s[name + "_pool"], page, slot, torch.float32).to(t)
    return got


def _plain_read(s):
    c, (_, page, slot) = s["case"], _places(s)
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    return {n: _unpacked(c, s[n + "_pool"], page, slot, torch.float32).to(dtype) for n in ("k", "v")}


def _plain_attention(s):
    c = s["case"]
    b, lq, lk, h, kv, dim = (c[n] for n in ("batch", "len_q", "len_k", "heads", "kv_heads", "dim"))
    j = torch.arange(lk, device=DEV)
    slot = (j % c["page"]).expand(b, lk)
    page = s["table"].long()[:, j // c["page"]].clamp(min=0)
    held = j < s["k_len"][:, None]
    gone = ~held[:, :, None, None]
    k = _unpacked(c, s["k_pool"], page, slot, torch.float32).masked_fill(gone, 0).transpose(1, 2).contiguous()
    v = _unpacked(c, s["v_pool"], page, slot, torch.float32).masked_fill(gone, 0).transpose(1, 2).contiguous()
    q = s["q"].float().transpose(1, 2).reshape(b, kv, h // kv * lq, dim)
    x = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, h, lq, lk)
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    pos = s["q_start"][:, None] + torch.arange(lq, device=DEV)
    if c["buckets"]:
        at = (j - pos[:, :, None]).clamp(-c["distance"], c["distance"]) + c["distance"]
        x = x + s["bias"][s["bucket"].long()[at]].permute(0, 3, 1, 2)
    seen = held[:, None, :]
    if c["mask"] == "causal":
        seen = seen & (j <= pos[:, :, None])
    elif c["mask"] == "prefix":
        seen = seen & ((j <= pos[:, :, None]) | (j < s["prefix"][:, None, None]))
    x = x.masked_fill(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(x - top)
    del x
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p.view(b, kv, h // kv * lq, lk), v).view(b, h, lq, dim).transpose(1, 2)
    return {"out": out.to(s["q"].dtype), "lse": (torch.log(total) + top).squeeze(-1)}


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


def _cache(nn, s):
    c = s["case"]
    return nn.NnCache(kind=nn.NN_CACHE_MXFP4 if c["kind"] == "mxfp4" else nn.NN_CACHE_PLAIN, page_tokens=c["page"],
                      pages=s["k_pool"].shape[0], requests=s["table"].shape[0], table_pages=s["table"].shape[1],
                      table=_ptr(s["table"]), k=_ptr(s["k_pool"]), v=_ptr(s["v_pool"]))


def _append_call(s):
    """What a program keeps beside its inputs: the descriptions of the calls, and outputs."""
    nn, c = _package(), s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    dtype = nn.NN_BF16 if c["dtype"] == "bf16" else nn.NN_F32
    r = {"L": nn.lib(), "cache": _cache(nn, s), "q_out": torch.zeros(q.shape, dtype=q.dtype, device=DEV)}
    r["args"] = nn.NnCacheAppend(
        rope=nn.NnQkNormRope(
            dtype=dtype, tokens=q.shape[0], heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["dim"], rot_dim=c["rot"],
            axes=c["axes"], interleaved=int(c["interleaved"]), eps=s["eps"], q_stride=q.stride()[:2],
            k_stride=k.stride()[:2], q_out_stride=r["q_out"].stride()[:2], q_weight=_ptr(s.get("q_weight")),
            k_weight=_ptr(s.get("k_weight")), pos=_ptr(s["pos"]), freq=_ptr(s["freq"])),
        norm=int(c["norm"]), v_stride=v.stride()[:2], request=_ptr(s["request"]), place=_ptr(s["place"]))
    if c["kind"] == "mxfp4":
        r.update(_read_call(s))
    return r


def _read_call(s):
    nn, c = _package(), s["case"]
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    # rows that are no tokens stay as they are
    k, v = (torch.zeros(s["place"].shape[0], c["kv_heads"], c["dim"], dtype=dtype, device=DEV) for _ in range(2))
    return {"L": nn.lib(), "cache": _cache(nn, s), "k": k, "v": v, "read": nn.NnCacheRead(
        dtype=nn.NN_BF16 if c["dtype"] == "bf16" else nn.NN_F32, tokens=k.shape[0], kv_heads=c["kv_heads"],
        head_dim=c["dim"], k_stride=k.stride()[:2], v_stride=v.stride()[:2], request=_ptr(s["request"]),
        place=_ptr(s["place"]))}


def _own_append(s):
    if "call" not in s:
        s["call"] = _append_call(s)
    r = s["call"]
    L, stream = r["L"], torch.cuda.current_stream().cuda_stream
    L.launch_cache_append(_ptr(r["q_out"]), _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), r["args"], r["cache"], stream)
    got = {"q_out": r["q_out"]}
    if s["case"]["kind"] == "plain":
        got.update(k_pool=s["k_pool"], v_pool=s["v_pool"])
    else:
        L.launch_cache_read(_ptr(r["k"]), _ptr(r["v"]), r["read"], r["cache"], stream)
        got.update(k=r["k"], v=r["v"])
    return got


def _own_read(s):
    if "call" not in s:
        s["call"] = _read_call(s)
    r = s["call"]
    r["L"].launch_cache_read(_ptr(r["k"]), _ptr(r["v"]), r["read"], r["cache"], torch.cuda.current_stream().cuda_stream)
    return {"k": r["k"], "v": r["v"]}


def _attention_call(s):
    nn, c = _package(), s["case"]
    L = nn.lib()
    q = s["q"]
    r = {"L": L, "cache": _cache(nn, s), "out": torch.empty(q.shape, dtype=q.dtype, device=DEV),
         "lse": torch.empty(c["batch"], c["heads"], c["len_q"], device=DEV)}
    r["args"] = nn.NnAttention(
        dtype=nn.NN_BF16 if c["dtype"] == "bf16" else nn.NN_F32, batch=c["batch"], len_q=c["len_q"], len_k=c["len_k"],
        heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["dim"], scale=s["scale"], softcap=c["cap"],
        mask={"none": nn.NN_MASK_NONE, "causal": nn.NN_MASK_CAUSAL, "prefix": nn.NN_MASK_PREFIX}[c["mask"]],
        buckets=c["buckets"], max_distance=c["distance"], q_stride=q.stride()[:3], out_stride=r["out"].stride()[:3],
        q_start=_ptr(s["q_start"]), k_len=_ptr(s["k_len"]), prefix=_ptr(s.get("prefix")), bucket=_ptr(s.get("bucket")),
        bias=_ptr(s.get("bias")))
    floats = L.nnhip_cache_attention_workspace(r["args"], r["cache"])
    r["workspace"] = torch.zeros(max(1, floats), dtype=torch.float32, device=DEV)
    return r


def _own_attention(s):
    if "call" not in s:
        s["call"] = _attention_call(s)
    r = s["call"]
    r["L"].launch_cache_attention_forward(_ptr(r["out"]), _ptr(r["lse"]), _ptr(s["q"]), r["args"], r["cache"],
                                          _ptr(r["workspace"]), torch.cuda.current_stream().cuda_stream)
    return {"out": r["out"], "lse": r["lse"]}


def run(s):
    if s["case"]["op"] == "append":
        return _own_append(s) if own else _plain_append(s)
    if s["case"]["op"] == "read":
        return _own_read(s) if own else _plain_read(s)
    return _own_attention(s) if own else _plain_attention(s)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _nearest(x):
    """Rows [..., dim] as the nearest values that 4 bits hold with the least exponent whose grid reaches them."""
    values = torch.tensor([v for v in _GRID] + [-v for v in _GRID[1:]], dtype=torch.float64, device=DEV)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=DEV)  # even codes first: they win at equal distance
    got = torch.zeros_like(x)
    for first in range(0, x.shape[-1], 32):
        block = x[..., first:first + 32]
        top = block.abs().amax(-1, keepdim=True)
        exponent = torch.ceil(torch.log2(top / 7)).nan_to_num(neginf=-120.0).clamp(-120, 125)
        # the logarithm may be a rounding off: settle it by what the exponent means
        exponent = torch.where(top > 7 * torch.exp2(exponent), exponent + 1, exponent)
        exponent = torch.where((top <= 7 * torch.exp2(exponent - 1)) & (exponent > -120), exponent - 1, exponent)
        y = block.abs() * torch.exp2(-exponent)
        far = (y.unsqueeze(-1) - values[order]).abs()
        got[..., first:first + 32] = values[order][far.argmin(-1)] * torch.exp2(exponent) * block.sign()
    return got


def _exact_turned(s, x, weight):
    """Each pair as a complex number, turned by e^(i angle)."""
    c, r = s["case"], s["case"]["rot"]
    x = x.double()
    if c["norm"]:
        x = x / (x.square().sum(-1, keepdim=True) / c["dim"] + s["eps"]).sqrt() * weight.double()
    order = torch.arange(r, device=DEV)
    order = order.view(-1, 2) if c["interleaved"] else order.view(2, -1).t()
    axis = torch.arange(r // 2, device=DEV) // max(1, r // 2 // c["axes"])
    angle = s["pos"].double()[:, axis] * s["freq"]
    z = torch.complex(x[..., order[:, 0]], x[..., order[:, 1]]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.clone()
    x[..., order[:, 0]], x[..., order[:, 1]] = z.real, z.imag
    return x


def _exact_append(s):
    c = s["case"]
    dead = (s["place"] < 0)[:, None, None]
    got = {"q_out": _exact_turned(s, s["q"], s.get("q_weight")).masked_fill(dead, 0)}
    k, v = _exact_turned(s, s["k"], s.get("k_weight")), s["v"].double()
    if c["kind"] == "mxfp4":
        got.update(k=torch.cat([_nearest(x) for x in k.split(1024)]).masked_fill(dead, 0),
                   v=torch.cat([_nearest(x) for x in v.split(1024)]).masked_fill(dead, 0))
        return got
    for name, rows in (("k_pool", k), ("v_pool", v)):
        pool = s[name].double()
        flat = pool.transpose(1, 2).reshape(-1, c["kv_heads"], pool.shape[-1])  # a row for every slot of the pool
        live = torch.nonzero(s["place"] >= 0).flatten()
        place = s["place"][live].long()
        at = s["table"].long()[s["request"][live].long(), place // c["page"]] * c["page"] + place % c["page"]
        flat[at, :, :c["dim"]] = rows[live]
        got[name] = flat.view(pool.shape[0], c["page"], c["kv_heads"], -1).transpose(1, 2)
    return got


def _exact_cache(s, name, b, length):
    """Keys (or values) [kv_heads, length, dim] of request b, page by page."""
    c, pool = s["case"], s[name]
    pages = s["table"][b, :-(-length // c["page"])].long()
    got = pool[pages]
    if c["kind"] == "plain":
        rows = got[..., :c["dim"]].double()
    else:
        groups, tokens = -(-c["dim"] // 32), c["page"]
        code = got[..., :tokens * groups * 16].view(-1, c["kv_heads"], tokens, groups, 16)
        scale = got[..., tokens * groups * 16:].view(-1, c["kv_heads"], tokens, groups, 1)
        parts = []
        for nibble in (code % 16, code // 16):
            step, half = (nibble % 8).double(), nibble // 8
            size = torch.where(step < 4, step / 2, torch.where(step < 6, step - 2, 2 * step - 8))
            parts.append(size * (1 - 2 * half.double()) * torch.exp2(scale.double() - 127))
        rows = torch.stack(parts, -1).reshape(got.shape[0], c["kv_heads"], tokens, groups * 32)[..., :c["dim"]]
    return rows.transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :length]


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "append":
        return _exact_append(s)
    if c["op"] == "read":
        rows = {n: [_exact_cache(s, n + "_pool", r, c["tokens"]) for r in range(c["requests"])] for n in ("k", "v")}
        return {n: torch.cat([x.transpose(0, 1) for x in rows[n]]) for n in rows}
    b, lq, h, kv = (c[n] for n in ("batch", "len_q", "heads", "kv_heads"))
    got = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV),
           "lse": torch.empty(b, h, lq, dtype=torch.float64, device=DEV)}
    for n in range(b):
        length, start = int(s["k_len"][n]), int(s["q_start"][n])
        k, v = _exact_cache(s, "k_pool", n, length), _exact_cache(s, "v_pool", n, length)
        key, place = torch.arange(length, device=DEV), torch.arange(lq, device=DEV) + start
        hidden = torch.zeros(lq, length, dtype=torch.bool, device=DEV)
        if c["mask"] != "none":
            hidden = key[None, :] > place[:, None]
            if c["mask"] == "prefix":
                hidden &= key[None, :] >= int(s["prefix"][n])
        for m in range(h):
            score = s["q"][n, :, m].double() @ k[m * kv // h].t() * s["scale"]
            if c["cap"]:
                score = torch.tanh(score / c["cap"]) * c["cap"]
            if c["buckets"]:
                far = (key[None, :] - place[:, None]).clamp(-c["distance"], c["distance"]) + c["distance"]
                score = score + s["bias"][:, m].double()[s["bucket"].long()[far]]
            score[hidden] = -math.inf
            lse = torch.logsumexp(score, 1)
            got["lse"][n, m] = lse
            got["out"][n, :, m] = torch.nan_to_num(torch.exp(score - lse[:, None]), nan=0.0) @ v[m * kv // h]
    return got
