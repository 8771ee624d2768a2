"""How far the values that an 8-bit cache holds are from those it was given, by the bounds its header states, and how far
that takes attention from the same over the unquantised rows.

With s the step of the block as it is, 2^(byte - 127), and x a value (a key after its rotation):
int8.  Written, a value is off by half the step of then.  Each growth multiplies the step by two or more and rounds the
code anew, off by half the new step: s / 2 (1 + 1/2 + 1/4 + ..) < s in all; s / 2 if the block has not grown since.
e4m3.  Codes have 4 significant bits, down to multiples of 2^-9: a value is off by 2^-4 |x|, or by 2^-10 of the step where
that is more.  A growth lowers a code's exponent and is exact until the code is below 2^-6; from there on as int8's: less
than 2^-9 s in all.
Attention.  Scores move by at most d = max_j sum_i |q_i| e_ji / sqrt(hd), e the keys' bounds, so weights by factors within
e^(+-2d): |out' - out| <= e^2d sum w e_v + (e^2d - 1) sum w |v|, w the unquantised rows' weights, sum w = 1.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv8_write import KINDS, ints
from unillm_amd import PagedKvCache8, PageTable

pytestmark = pytest.mark.gpu


def bound(x, step, kind, grown=True):
    """Of values x [..], steps alike."""
    if kind == "int8":
        return step * (1.0 if grown else 0.5) + 0 * x
    return np.abs(x) * 2.0 ** -4 + step * (2.0 ** -9 if grown else 2.0 ** -10)


class Given:
    """A cache, and the rows that sequence 0 was given."""

    def __init__(self, kind, heads, hd, page):
        self.table = PageTable(2, 64, 70, page, 512)
        self.cache = PagedKvCache8(heads, hd, 70, page, KINDS[kind])
        self.kind, self.rows = kind, np.zeros((0, 2, heads, hd))

    def append(self, kv):
        self.table.extend(ints([0]), ints([len(kv)]))
        self.cache.append(self.table, kv)
        self.rows = np.concatenate([self.rows, kv.double().cpu().numpy().reshape(len(kv), *self.rows.shape[1:])])

    def held(self):
        """(values, steps [n, 2, heads, 1]) of all positions."""
        n, page = len(self.rows), self.cache.page_size
        got = self.cache.read(self.table, ints([0]), ints([0]), ints([0, n]), n)
        self.table.check()
        pages = self.table.block_table[0, :-(-n // page)].tolist()
        exps = [torch.stack([e[p] for p in pages]).cpu().numpy().astype(int) for e in (self.cache.k_exp, self.cache.v_exp)]
        at = np.arange(n)
        steps = np.stack([2.0 ** (e[at // page, :, at % page // 16] - 127.0) for e in exps], 1)
        return np.stack([x.double().cpu().numpy() for x in got], 1), steps[..., None]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("sizes", [(1,) * 48, (3,) * 16, (5, 1, 1, 30, 2, 1, 1, 1, 6), (48,)])
def test_held_values(kind, hd, page, sizes):
    gen = torch.Generator(device="cuda").manual_seed(len(sizes))
    g = Given(kind, 2, hd, page)
    for i, n in enumerate(sizes):  # (within a block magnitudes grow, by 1.5 a step: most appends make its step larger)
        x = torch.randn(n, 4 * hd, device="cuda", generator=gen) * 1.5 ** (i % 16)
        x[:, ::5] = torch.round(x[:, ::5] * 8) / 8  # ties
        g.append(x)
    held, steps = g.held()
    off, most = np.abs(held - g.rows), bound(g.rows, steps, kind, len(sizes) > 1)
    assert (off <= most).all(), (off / most).max()
    # and not by less: one rounding alone would not reach this far
    assert len(sizes) < 48 or kind != "int8" or (off > 0.5 * steps).any()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("at_once", [True, False])
def test_attention_over_the_unquantised_rows(kind, at_once):
    heads, hd, n = 2, 64, 100
    gen = torch.Generator(device="cuda").manual_seed(8)
    g = Given(kind, heads, hd, 16)
    kv = torch.randn(n, 2 * heads * hd, device="cuda", generator=gen)
    for a in range(0, n, n if at_once else 1):
        g.append(kv[a:a + (n if at_once else 1)])
    q = torch.randn(n if at_once else 1, heads * hd, device="cuda", generator=gen)
    out = g.cache.attention(g.table, q, heads).double().cpu().numpy().reshape(-1, heads, hd)
    _, steps = g.held()
    e = bound(g.rows, steps, kind, not at_once)
    q = q.double().cpu().numpy().reshape(-1, heads, hd)
    for r in range(len(q)):
        seen = n - len(q) + r + 1
        for h in range(heads):
            k, v, ek, ev = (x[:seen, w, h] for x in (g.rows, e) for w in (0, 1))
            s = k @ q[r, h] / math.sqrt(hd)
            w = np.exp(s - s.max())
            w /= w.sum()
            d = (ek @ np.abs(q[r, h])).max() / math.sqrt(hd)
            most = math.exp(2 * d) * (w @ ev) + (math.exp(2 * d) - 1) * (w @ np.abs(v))
            assert (np.abs(out[r, h] - w @ v) <= most * (1 + 1e-4)).all()
