"""The paged cache in 64-bit numpy: its layout, its 4 bits, and what its tests share.

Tolerances are those of attention_ref.py.  Codes of 4 bits have none: a value goes to the nearest
size, and 64 bits on both sides differ by some 2^-50 of it, so that only a value that near to a
border may go either way.
"""
from __future__ import annotations

import numpy as np

from attention_ref import Tensor, from_bf16, ints, rounded, to_bf16

SIZES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5])


def exponents(x):
    """Least e of -120..125 with max|x| <= 7 2^e over the last axis; 128 where a value is not finite."""
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
    fine = np.isfinite(x).all(-1)
    fraction, power = np.frexp(np.where(fine, top, 0))  # 7 is 0.875 * 2^3
    e = np.where(top == 0, -120, np.clip(power - np.where(fraction > 0.875, 2, 3), -120, 125))
    return np.where(fine, e, 128)


def codes(x):
    """Rows [..., dim] as codes [..., groups, 32], exponents [..., groups] and each value's distance to a border in its units."""
    groups = -(-x.shape[-1] // 32)
    x = np.concatenate([x, np.zeros(x.shape[:-1] + (groups * 32 - x.shape[-1],))], -1).reshape(x.shape[:-1] + (groups, 32))
    e = exponents(x)
    y = np.abs(np.where(e[..., None] < 128, x, 0)) * 2.0 ** -np.where(e < 128, e, 0)[..., None].astype(np.float64)
    code = np.zeros(x.shape, np.uint8)
    for i, border in enumerate(BORDERS):  # half way: the even code
        code += (y >= border) if i % 2 else (y > border)
    near = np.abs(y[..., None] - BORDERS).min(-1)
    return code | ((x < 0) * 8).astype(np.uint8), e, near


def unpacked(code, e, dim):
    value = SIZES[code & 7] * np.where(code & 8, -1.0, 1.0) * 2.0 ** e[..., None].astype(np.float64)
    value = np.where(e[..., None] == 128, np.nan, value)
    return value.reshape(code.shape[:-2] + (-1,))[..., :dim]


class Cache:
    """Pools on the device with a host image of their bytes, and a table.

    `counts`: pages of each request; the pages lie in the pools in a shuffled order.  What no test
    writes is 0xA5 bytes."""

    def __init__(self, nn, L, rng, kind, dtype, kv_heads, dim, page_tokens, counts, spare=2, width=None):
        self.nn, self.L, self.kind, self.dtype, self.kv, self.dim, self.tokens = nn, L, kind, dtype, kv_heads, dim, page_tokens
        e = 2 if dtype == "bf16" else 4
        self.groups = -(-dim // 32) if kind == "mxfp4" else 0
        self.row = 16 * self.groups if self.groups else -(-dim * e // 16) * 16
        self.block = page_tokens * (self.row + self.groups)
        self.pages = sum(counts) + spare
        width = max(counts) if width is None else width
        self.table = np.full((len(counts), width), -1, np.int32)
        order = rng.permutation(self.pages)
        for r, n in enumerate(counts):
            self.table[r, :n] = order[:n]
            order = order[n:]
        self.bytes = {n: np.full((self.pages, kv_heads, self.block), 0xA5, np.uint8) for n in ("k", "v")}
        self.dev = {n: L.alloc(-(-self.bytes[n].size // 4) + 4) for n in ("k", "v")}
        self.table_dev = ints(L, self.table)
        self.args = nn.NnCache(kind=nn.NN_CACHE_MXFP4 if self.groups else nn.NN_CACHE_PLAIN, page_tokens=page_tokens,
                               pages=self.pages, requests=len(counts), table_pages=width, table=self.table_dev.p,
                               k=self.dev["k"].p, v=self.dev["v"].p)
        assert L.nnhip_cache_page_bytes(self.args, self.nn_dtype(), kv_heads, dim) == kv_heads * self.block
        self.upload()

    def nn_dtype(self):
        return self.nn.NN_BF16 if self.dtype == "bf16" else self.nn.NN_F32

    def upload(self):
        for n, x in self.bytes.items():
            raw = x.ravel()
            self.dev[n].upload(np.concatenate([raw, np.zeros(-raw.size % 4, np.uint8)]).view(np.float32))

    def download(self, name):
        raw = self.dev[name].download().view(np.uint8)
        return raw[:self.bytes[name].size].reshape(self.bytes[name].shape)

    def where(self, request, place):
        """(page, slot) of a token, or None where there is none."""
        i = place // self.tokens
        if place < 0 or not 0 <= request < self.table.shape[0] or i >= self.table.shape[1]:
            return None
        page = self.table[request, i]
        return (int(page), place % self.tokens) if 0 <= page < self.pages else None

    def put(self, name, at, rows):
        """Rows [kv, dim] into the host image, as an append leaves them; gives the least distance to a border."""
        page, slot = at
        to = self.bytes[name][page]
        if not self.groups:
            row = np.zeros((self.kv, self.row // (2 if self.dtype == "bf16" else 4)), np.float32)
            row[:, :self.dim] = rows
            raw = to_bf16(row).reshape(row.shape) if self.dtype == "bf16" else row
            to[:, slot * self.row:(slot + 1) * self.row] = raw.view(np.uint8)
            return np.inf
        code, e, near = codes(rows)
        code = code.reshape(self.kv, -1)
        to[:, slot * self.row:(slot + 1) * self.row] = code[:, 0::2] | code[:, 1::2] << 4
        at = self.tokens * self.row + slot * self.groups
        to[:, at:at + self.groups] = e + 127
        return near.min()

    def get(self, name, at, image=None):
        """Row [kv, dim] of a slot as the values that it stands for."""
        page, slot = at
        block = (self.bytes[name] if image is None else image)[page]
        raw = np.ascontiguousarray(block[:, slot * self.row:(slot + 1) * self.row])
        if not self.groups:
            x = from_bf16(raw.view(np.uint16)) if self.dtype == "bf16" else raw.view(np.float32)
            return x[:, :self.dim].astype(np.float64)
        at = self.tokens * self.row + slot * self.groups
        code = np.stack([raw & 15, raw >> 4], -1).reshape(self.kv, self.groups, 32)
        return unpacked(code, block[:, at:at + self.groups].astype(np.int64) - 127, self.dim)

    def fill(self, rng, lengths, spoil=True):
        """Normal keys and values for the first lengths[r] tokens of each request; behind them, to the
        end of their pages, what nothing may read (NaN, or scales and codes that are)."""
        for r, n in enumerate(lengths):
            for i, page in enumerate(self.table[r]):
                here = min(max(n - i * self.tokens, 0), self.tokens)
                if not 0 <= page < self.pages or not (here or spoil):
                    continue
                for name in ("k", "v"):
                    x = np.full((self.tokens, self.kv, self.dim), np.nan)
                    x[:here] = rounded(rng.standard_normal((here, self.kv, self.dim)), self.dtype)
                    self._put_page(name, page, x if spoil else x[:here])
        self.upload()

    def _put_page(self, name, page, x):
        """The first rows [n, kv, dim] of a page."""
        to, n = self.bytes[name][page], len(x)
        if not self.groups:
            e = 2 if self.dtype == "bf16" else 4
            row = np.zeros((self.kv, n, self.row // e), np.float32)
            row[..., :self.dim] = x.transpose(1, 0, 2)
            raw = to_bf16(row).reshape(row.shape) if self.dtype == "bf16" else row
            to[:, :n * self.row] = raw.reshape(self.kv, -1).view(np.uint8)
            return
        code, e, _ = codes(x.transpose(1, 0, 2))
        code = code.reshape(self.kv, n, -1)
        to[:, :n * self.row] = (code[..., 0::2] | code[..., 1::2] << 4).reshape(self.kv, -1)
        at = self.tokens * self.row
        to[:, at:at + n * self.groups] = (e + 127).reshape(self.kv, -1)

    def _page(self, name, page):
        """The rows [page tokens, kv, dim] of a page."""
        block = self.bytes[name][page]
        raw = np.ascontiguousarray(block[:, :self.tokens * self.row])
        if not self.groups:
            x = from_bf16(raw.view(np.uint16)) if self.dtype == "bf16" else raw.view(np.float32)
            return x.reshape(self.kv, self.tokens, -1)[..., :self.dim].astype(np.float64).transpose(1, 0, 2)
        code = np.stack([raw & 15, raw >> 4], -1).reshape(self.kv, self.tokens, self.groups, 32)
        e = block[:, self.tokens * self.row:].astype(np.int64).reshape(self.kv, self.tokens, self.groups) - 127
        return unpacked(code, e, self.dim).transpose(1, 0, 2)

    def rows(self, name, request, length):
        """[length, kv, dim] of a request, zeros where there is no page; and which tokens have one."""
        got, held = np.zeros((length, self.kv, self.dim)), np.zeros(length, bool)
        for first in range(0, length, self.tokens):
            at = self.where(request, first)
            if at is not None:
                got[first:first + self.tokens] = self._page(name, at[0])[:length - first]
                held[first:first + self.tokens] = True
        return got, held


__all__ = ["Cache", "Tensor", "codes", "exponents", "ints", "rounded", "unpacked", "SIZES"]
