"""Rotary positions and the 8-bit paged cache restated in 64-bit numpy, for their tests.

Independent of the library.  Codes are kept as the numbers they are (int8 whole numbers, e4m3 values).
"""
import math

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}
BLOCK = 16


def frequencies(rot, theta=10000.0, scaling=None, factor=1.0, low=1.0, high=32.0, original=0, factors=None):
    """Radians a position of each pair, by the header's definition."""
    got = []
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot) / (factors[i] if factors else 1.0)
        if scaling == "linear":
            f /= factor
        elif scaling == "llama3":
            r = (original * f / (2 * math.pi) - low) / (high - low)
            r = min(1.0, max(0.0, r))
            f = f * r + f / factor * (1 - r)
        elif scaling == "yarn":
            first, last = (rot * math.log(original / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (high, low))
            first, last = max(0, math.floor(first)), min(rot - 1, math.ceil(last))
            r = 1 - min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = f * r + f / factor * (1 - r)
        got.append(f)
    return np.array(got)


def rotate(x, positions, freq, interleaved=False, magnitude=1.0):
    """x [n, heads, hd] f64 with its first 2 len(freq) dimensions turned at positions [n]."""
    n = len(freq)
    a = np.asarray(positions, np.float64)[:, None, None] * freq
    c, s = magnitude * np.cos(a), magnitude * np.sin(a)
    y = x.astype(np.float64).copy()
    at = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    lo, hi = x[..., at[0]].astype(np.float64), x[..., at[1]].astype(np.float64)
    y[..., at[0]], y[..., at[1]] = lo * c - hi * s, lo * s + hi * c
    return y


def rounded(y, kind):
    """Values in steps -> the codes nearest to them, ties to even; inf to the largest, NaN to 0."""
    y = np.clip(np.where(np.isnan(y), 0.0, y), -TOP[kind], TOP[kind])
    if kind == "int8":
        return np.rint(y)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -30))), -6) - 3)
    return np.rint(y / step) * step


def least(values, kind):
    """The least exponent, at least -126, with which the finite values fit."""
    top = np.abs(np.where(np.isfinite(values), values, 0.0)).max(initial=0.0)
    e = -126
    if top > 0:
        e = max(e, math.frexp(top / TOP[kind])[1] - 1)
        while top > TOP[kind] * 2.0 ** e:
            e += 1
    return e


def e4m3_value(byte):
    """e4m3 bytes as numbers."""
    b = np.asarray(byte).astype(np.int64)
    exp, man = b >> 3 & 15, b & 7
    v = np.where(exp > 0, (8 + man) * 2.0 ** (exp - 10.0), man * 2.0 ** -9)
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


class Pool:
    """codes k [pages, heads, page, hd], v [pages, heads, hd, page], exponents [pages, heads, page / 16]."""

    def __init__(self, pages, heads, hd, page, kind):
        self.page, self.kind = page, kind
        self.k, self.v = np.zeros((pages, heads, page, hd)), np.zeros((pages, heads, hd, page))
        self.ke, self.ve = (np.full((pages, heads, page // BLOCK), -127) for _ in range(2))

    def _block(self, codes, exps, at, off, x):
        """codes [16, hd] (a view) of a block, exps[at] its exponent; x [n, hd] from place off on."""
        e = least(x, self.kind)
        if off:
            e = max(e, exps[at])
            codes[:off] = rounded(codes[:off] * 2.0 ** (exps[at] - float(e)), self.kind)
        with np.errstate(invalid="ignore"):
            codes[off:off + len(x)] = rounded(x * 2.0 ** -float(e), self.kind)
        exps[at] = e

    def write(self, slots, k, v):
        """Rows k, v [n, heads, hd] f64 into slots, a run of a block at a time."""
        i = 0
        while i < len(slots):
            off, n = slots[i] % BLOCK, 1
            while i + n < len(slots) and slots[i + n] == slots[i] + n and off + n < BLOCK:
                n += 1
            pg, first = slots[i] // self.page, slots[i] % self.page - off
            for h in range(k.shape[1]):
                at = (pg, h, first // BLOCK)
                self._block(self.k[pg, h, first:first + BLOCK], self.ke, at, off, k[i:i + n, h])
                self._block(self.v[pg, h, :, first:first + BLOCK].T, self.ve, at, off, v[i:i + n, h])
            i += n

    def values(self, table_row, length):
        """(k, v) [length, heads, hd] of a sequence."""
        ks, vs = [], []
        for p in range(length):
            pg, o = table_row[p // self.page], p % self.page
            ks.append(self.k[pg, :, o] * 2.0 ** self.ke[pg, :, o // BLOCK, None].astype(np.float64))
            vs.append(self.v[pg, :, :, o] * 2.0 ** self.ve[pg, :, o // BLOCK, None].astype(np.float64))
        return np.array(ks), np.array(vs)
