"""Rotary positions, the paged 4-bit cache and attention over it restated in numpy, 64
bits: the oracle of those operations (the reference has no counterpart).

Formulas: rotary embeddings with linear and by-part (YaRN) interpolation; MXFP4 of
oracle/mx_numpy.py; softmax attention with a causal mask and a sliding window, one
sequence, token and head after another.
"""
from __future__ import annotations

import math

import numpy as np

from . import mx_numpy as MX


# ---- rotary positions --------------------------------------------------------------
def frequencies(dim, base=10000.0, scale=1.0, extrapolate=0.0, beta_fast=32.0, beta_slow=1.0,
                original=0, factors=None) -> np.ndarray:
    """Radians a position of each pair."""
    out = np.zeros(dim // 2, dtype=np.longdouble)
    for i in range(dim // 2):
        f = np.longdouble(base) ** (np.longdouble(-2 * i) / dim)
        if factors is not None:
            f /= np.longdouble(np.float32(factors[i]))
        w = 0.0
        if extrapolate > 0:
            def pair_of(turns):
                return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
            low = max(0, math.floor(pair_of(beta_fast)))
            high = min(dim - 1, math.ceil(pair_of(beta_slow)))
            w = extrapolate * (1 - min(1.0, max(0.0, (i - low) / max(0.001, high - low))))
        out[i] = f * (scale * (1 - np.longdouble(w)) + w)
    return out


def rotate(x, positions, freq, halves, magnitude=1.0) -> np.ndarray:
    """tokens x heads x head_dim values, the first 2 len(freq) of a head turned."""
    y = np.array(x, dtype=np.float64)
    n = len(freq)
    a = np.asarray(positions, dtype=np.longdouble)[:, None] * freq[None, :]
    a = np.asarray(np.fmod(a, 2 * np.arccos(np.longdouble(-1))), dtype=np.float64)
    c, s = (np.cos(a) * magnitude)[:, None, :], (np.sin(a) * magnitude)[:, None, :]
    first = slice(0, n) if halves else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if halves else slice(1, 2 * n, 2)
    u, v = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = u * c - v * s, u * s + v * c
    return y


# ---- pages ---------------------------------------------------------------------------
def pack_page(codes, scales, values) -> np.ndarray:
    """A head's part of a page: rows x dim / 2 bytes of codes, rows x dim / 32 scales."""
    rows, half = codes.shape
    out = np.zeros(codes.size + scales.size, dtype=np.uint8)
    for r in range(rows):
        for d in range(0, half, 4):  # four bytes at a time
            at = (r // 4) * 4 * half + d * 4 + r % 4 * 4 if values else r * half + d
            out[at:at + 4] = codes[r, d:d + 4]
        for b in range(scales.shape[1]):
            at = (r // 4) * 4 * scales.shape[1] + b * 4 + r % 4 if values \
                else r * scales.shape[1] + b
            out[codes.size + at] = scales[r, b]
    return out


def unpack_page(page, rows, dim, values) -> tuple[np.ndarray, np.ndarray]:
    """Codes and scales of a head's part of a page."""
    half, blocks = dim // 2, dim // 32
    c, s = page[:rows * half], page[rows * half:rows * (half + blocks)]
    if values:
        c = c.reshape(rows // 4, half // 4, 4, 4).transpose(0, 2, 1, 3)
        s = s.reshape(rows // 4, blocks, 4).transpose(0, 2, 1)
    return c.reshape(rows, half).copy(), s.reshape(rows, blocks).copy()


class Cache:
    """Pages of keys and values, on the host, with what they hold before they are written."""

    def __init__(self, n_pages, page_size, heads, dim, fill=0xFF):
        self.n_pages, self.page_size, self.heads, self.dim = n_pages, page_size, heads, dim
        size = page_size * dim // 32 * 17
        self.k = np.full((n_pages, heads, size), fill, dtype=np.uint8)
        self.v = np.full((n_pages, heads, size), fill, dtype=np.uint8)

    def there(self, table, seq, pos):
        """The page of a position, or None."""
        if pos < 0 or pos // self.page_size >= table.shape[1]:
            return None
        page = int(table[seq, pos // self.page_size])
        return page if 0 <= page < self.n_pages else None

    def _bytes(self, row, values):
        """Where a row's codes (by dword) and scales are in a head's part of a page."""
        half, blocks = self.dim // 2, self.dim // 32
        d, b = np.arange(half), np.arange(blocks)
        if values:
            code = (row // 4) * 4 * half + d // 4 * 16 + row % 4 * 4 + d % 4
            scale = (row // 4) * 4 * blocks + b * 4 + row % 4
        else:
            code, scale = row * half + d, row * blocks + b
        return code, self.page_size * half + scale

    def write(self, table, seq, pos, k, v):
        """heads x dim values of one token."""
        page = self.there(table, seq, pos)
        if page is None:
            return
        for pages, x, values in ((self.k, k, False), (self.v, v, True)):
            codes, scales = MX.quantize(x)
            code, scale = self._bytes(pos % self.page_size, values)
            pages[page][:, code] = codes
            pages[page][:, scale] = scales

    def row(self, table, seq, pos, values):
        """heads x dim values of one token, None where its page is not there."""
        page = self.there(table, seq, pos)
        if page is None:
            return None
        held = (self.v if values else self.k)[page]
        code, scale = self._bytes(pos % self.page_size, values)
        return MX.decode(held[:, code], held[:, scale])


def places(starts, lengths, n_tokens):
    """(sequence, position) of each token of a batch, None for those of no sequence."""
    out = [None] * n_tokens
    for s in range(len(lengths)):
        for t in range(starts[s], starts[s + 1]):
            out[t] = (s, int(lengths[s]) - int(starts[s + 1]) + t)
    return out


def attention(q, cache, starts, lengths, table, scale, window=0):
    """(y, bound) of tokens x heads x dim queries; y is NaN-free only where what a row sees
    is.  bound: first-order error of each output, in units that attention_bound uses."""
    tokens, heads, dim = q.shape
    per = heads // cache.heads
    y = np.zeros(q.shape)
    terms = np.zeros((4,) + q.shape)
    at = places(starts, lengths, tokens)
    rows = {}
    for t in range(tokens):
        if at[t] is None:
            y[t] = np.nan  # not written
            continue
        seq, pos = at[t]
        first = max(0, pos - window + 1) if window else 0
        keys = [j for j in range(first, min(pos, int(lengths[seq]) - 1) + 1)
                if cache.there(table, seq, j) is not None]
        if not keys:
            continue
        for j in keys:
            if (seq, j) not in rows:
                rows[seq, j] = (cache.row(table, seq, j, False), cache.row(table, seq, j, True))
        K = np.stack([rows[seq, j][0] for j in keys])  # keys x kv heads x dim
        V = np.stack([rows[seq, j][1] for j in keys])
        for h in range(heads):
            k, v, x = K[:, h // per], V[:, h // per], q[t, h].astype(np.float64)
            s = scale * (k @ x)
            with np.errstate(invalid="ignore"):
                w = np.exp(s - s.max())
                w = w / w.sum()
                y[t, h] = w @ v
                # of a key's score: the sum of its products, and its size
                d_sum = scale * (np.abs(k) @ np.abs(x))
                d_size = np.abs(s) + np.abs(s).max() + 16
                a = w[:, None] * np.abs(v)
                terms[0, t, h] = (w * d_sum) @ np.abs(v) + (w @ d_sum) * a.sum(0)
                terms[1, t, h] = (w * d_size) @ np.abs(v) + (w @ d_size) * a.sum(0)
                terms[2, t, h] = a.sum(0)
                terms[3, t, h] = a.sum(0) * len(keys)
    return y, terms


def attention_bound(terms, dim, weight_rounding):
    """What y may be off before its own rounding.  A score is dim products (exact, with up to
    three terms of q) added in f32 by instructions that may truncate: 3 dim 2^-23 of the
    sum of their magnitudes; its product with scale and log2 e, each rounded once, and the
    exponential's argument: 3 2^-23 of its size and the maximum's (which is within 2^8 of
    the largest); an exponential of 2^-22; weights rounded by weight_rounding; sums of as
    many terms as there are keys, of the weights and of the weighted values: 2^-22 a term."""
    return (3 * dim * 2.0 ** -23 * terms[0] + 3 * 2.0 ** -23 * terms[1]
            + (weight_rounding + 2.0 ** -20) * terms[2] + 2.0 ** -22 * terms[3])
