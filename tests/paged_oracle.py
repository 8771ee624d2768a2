"""The paged operators restated in plain Python and 64-bit numpy, for their tests.

Independent of the library: the page table as Python lists, and the attention of one step by
its formula, a sequence and a head at a time.
"""
import math

import numpy as np


class Pages:
    """The page table's state and calls, as include/unillm_hip_paged.h defines them."""

    def __init__(self, max_seqs, max_pages, n_pages, page):
        self.page, self.max_pages, self.max_seqs = page, max_pages, max_seqs
        self.table = [[] for _ in range(max_seqs)]
        self.lens = [0] * max_seqs
        self.stack = list(range(n_pages - 1, -1, -1))

    def extend(self, ids, news):
        cu, slots, positions = [0], [], []
        for i, n in zip(ids, news):
            if i < 0:
                cu.append(cu[-1])
                continue
            for p in range(self.lens[i], self.lens[i] + n):
                if p % self.page == 0:
                    self.table[i].append(self.stack.pop())
                slots.append(self.table[i][p // self.page] * self.page + p % self.page)
                positions.append(p)
            self.lens[i] += n
            cu.append(cu[-1] + n)
        return cu, slots, positions

    def truncate(self, ids, lens):
        for i, n in reversed(list(zip(ids, lens))):
            if i < 0:
                continue
            while len(self.table[i]) > -(-n // self.page):
                self.stack.append(self.table[i].pop())
            self.lens[i] = n

    def block_table(self):
        t = np.full((self.max_seqs, self.max_pages), -1, np.int32)
        for i, row in enumerate(self.table):
            t[i, :len(row)] = row
        return t


def rotate(x, positions, theta):
    """x [n, heads, hd] f64 rotated (half-split) at positions [n]."""
    half = x.shape[-1] // 2
    inv = float(np.float32(theta)) ** (-np.arange(half, dtype=np.float64) / half)
    a = np.asarray(positions, np.float64)[:, None, None] * inv
    lo, hi = x[..., :half], x[..., half:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)], -1)


def attend(q, k, v, positions, window=0, sinks=0):
    """One sequence: q [n, H, hd] rotated, k and v [L, KVH, hd] as stored, all f64 ->
    (out [n, H, hd], bound [n, H, hd] of an f32 evaluation's error).

    The bound, with u = 2^-24.  A score is a sum of hd products over any order, each product
    exact in the parts' sums or rounded once: off by at most (hd + 8) u sum |q_d k_d| / sqrt(hd)
    (8: the scalings of q, the parts' remainders and the sums' joining); its exponential by that
    much again in relation, plus 4 u |s| for the difference from the maximum in units of log2 e
    and 8 u for the exponential itself.  A weight's error enters the numerator and the
    denominator once each; both are sums of L terms, off by at most L u more, and the
    products, rescalings and the quotient add at most 64 u.  Everything is relative to
    sum w |v| / sum w.
    """
    n, H, hd = q.shape
    G = H // k.shape[1]
    out, bound = np.zeros((n, H, hd)), np.zeros((n, H, hd))
    j = np.arange(k.shape[0])
    for t, p in enumerate(positions):
        seen = j <= p
        if window > 0:
            seen &= (j > p - window) | (j < sinks)
        for h in range(H):
            kk, vv = k[seen, h // G], v[seen, h // G]
            s = kk @ q[t, h] / math.sqrt(hd)
            size = float((np.abs(kk) @ np.abs(q[t, h])).max()) / math.sqrt(hd)
            w = np.exp(s - s.max())
            out[t, h] = w @ vv / w.sum()
            terms = 2 * ((hd + 8) * size + 4 * float(np.abs(s).max()) + 8) + 2 * len(s) + 64
            bound[t, h] = terms * 2.0 ** -24 * (w @ np.abs(vv)) / w.sum()
    return out, bound
