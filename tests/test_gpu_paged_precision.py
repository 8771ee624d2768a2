"""Paged attention where one key takes almost all of a row's weight and its value is nothing (an
attention sink): the output is made of weights far below the largest.

A score here is a product of two dimensions (q and the keys lie in the plane of the slowest
rotation), so an f32 evaluation of it is off by 2 u of the sum of its two products' sizes from
the products and sums, and 8 u from q's scalings and rotation (u = 2^-24).  With `size` the most
of that over the keys, a weight is off by 10 size u, 4 |s| u for the exponent's own rounding and 8 u for
the exponential, in relation; once in the numerator and once in the denominator.  Both are sums
of L terms (L u each), and rescalings and the quotient add 64 u: the bound of `evaluate`, relative
to sum w |v| / sum w in each dimension.  Where a 16-bit pool's weights are held in two parts of
f16, what a row loses by them is allowed 2^-16 of its largest output besides.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from paged_oracle import rotate  # noqa: E402
from unillm_amd import PagedKvCache, PageTable  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
PAGE = 16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def evaluate(q, k, v, p, window, sinks):
    """One row: q [hd] rotated, k and v [L, hd], f64 -> (out [hd], bound [hd] of an f32 evaluation)."""
    j = np.arange(k.shape[0])
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    k, v = k[seen], v[seen]
    s = k @ q / math.sqrt(q.size)
    size = float((np.abs(k) @ np.abs(q)).max()) / math.sqrt(q.size)
    w = np.exp(s - s.max())
    out = w @ v / w.sum()
    terms = 2 * (10 * size + 4 * float(np.abs(s).max()) + 8) + 2 * len(s) + 64
    return out, terms * 2.0 ** -24 * (w @ np.abs(v)) / w.sum()


# dominant key: first, in the midst, last before the new tokens; gap: of its score, in nats
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("ctx,where,window,sinks", [(3, 0, 0, 0), (40, 0, 0, 0), (40, 39, 0, 0),
                                                    (2000, 0, 0, 0), (2000, 1111, 0, 0), (2000, 0, 300, 4)])
def test_a_dominant_key_of_no_value(dtype, hd, new, ctx, where, window, sinks):
    g = torch.Generator().manual_seed(ctx + where + hd)
    H, n_pages = 2, -(-(ctx + new) // PAGE) + 1
    for gap in (8.0, 12.0, 16.0, 20.0, 30.0, 70.0):
        table = PageTable(1, n_pages, n_pages, PAGE, max(ctx, new))
        cache = PagedKvCache(1, hd, n_pages, PAGE, dtype)
        table.extend(ints([0]), ints([ctx]))
        pages = table.block_table[0, :-(-ctx // PAGE)].long()
        i, half = hd // 2 - 1, hd // 2
        q = torch.zeros(H, hd)
        q[:, i] = math.sqrt(hd)                      # score of a key: its element i, nearly
        k = torch.zeros(ctx, hd)
        k[:, i] = torch.rand(ctx, generator=g) - 0.5
        k[where, i] = gap
        v = torch.rand(ctx, hd, generator=g)
        v[where] = 0.0
        at, off = pages[torch.arange(ctx) // PAGE], torch.arange(ctx, device="cuda") % PAGE
        cache.k[at, 0, off] = k.to(dtype).cuda()
        cache.v[at, 0, :, off] = v.to(dtype).cuda()
        table.extend(ints([0]), ints([new]))
        qkv = torch.zeros(new, H + 2, hd)
        qkv[:, :H] = q
        qkv[:, H + 1] = torch.rand(new, hd, generator=g)
        out = cache.attention(table, qkv.view(new, -1).cuda(), H, window=window, sinks=sinks)
        table.check()
        pages = table.block_table[0].long()
        full = torch.arange(ctx + new, device="cuda")
        kk = cache.k[pages[full // PAGE], 0, full % PAGE].double().cpu().numpy()
        vv = cache.v[pages[full // PAGE], 0, :, full % PAGE].double().cpu().numpy()
        got = out.view(new, H, hd).double().cpu().numpy()
        for t in sorted({0, new // 2, new - 1}):
            turned = rotate(q.double().numpy()[None], [ctx + t], 10000.0)[0]
            for h in range(H):
                want, bound = evaluate(turned[h], kk, vv, ctx + t, window, sinks)
                if dtype == torch.float16:
                    bound = bound + 2.0 ** -16 * np.abs(want).max()
                err = np.abs(got[t, h] - want)
                assert (err <= bound).all(), (gap, t, h, float((err / bound).max()),
                                              float(err.max() / np.abs(want).max()))
