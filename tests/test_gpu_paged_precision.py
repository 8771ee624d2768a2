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
from test_gpu_paged_attention import Step  # noqa: E402
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


# pieces of more keys than 2048: 128 kv heads' tiles leave few pieces to each.  The dominant key's value is
# nothing, or so little that a row is done again, or is not; where it is not, 2^-27 a key is allowed.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rho", [0.0, 1 / 1000, 1 / 300])
def test_a_dominant_key_before_many_others(dtype, rho):
    g = torch.Generator().manual_seed(5)
    heads, hd, ctx, new = 128, 64, 9000, 70
    n_pages = -(-(ctx + new) // PAGE)
    for gap in (14.0, 20.0, 30.0):
        table = PageTable(1, n_pages, n_pages, PAGE, ctx)
        cache = PagedKvCache(heads, hd, n_pages, PAGE, dtype)
        table.extend(ints([0]), ints([ctx]))
        pages = table.block_table[0].long()
        i = hd // 2 - 1
        q = torch.zeros(hd)
        q[i] = math.sqrt(hd)
        k = torch.zeros(ctx, hd)
        k[:, i] = torch.rand(ctx, generator=g) - 0.5
        k[0, i] = 2 * gap                      # (0.36 of it is the score at these positions)
        v = torch.rand(ctx, hd, generator=g)
        v[0] *= rho
        at, off = pages[torch.arange(ctx, device="cuda") // PAGE], torch.arange(ctx, device="cuda") % PAGE
        cache.k[at, :, off] = k.to(dtype).cuda()[:, None].expand(ctx, heads, hd)
        cache.v[at, :, :, off] = v.to(dtype).cuda()[:, None].expand(ctx, heads, hd)
        table.extend(ints([0]), ints([new]))
        qkv = torch.zeros(new, 3 * heads, hd)
        qkv[:, :heads] = q
        qkv[:, 2 * heads:] = torch.rand(new, 1, hd, generator=g)
        out = cache.attention(table, qkv.view(new, -1).cuda(), heads).view(new, heads, hd)
        table.check()
        pages = table.block_table[0].long()  # (with those of the new tokens)
        full = torch.arange(ctx + new, device="cuda")
        kk = cache.k[pages[full // PAGE], 5, full % PAGE].double().cpu().numpy()
        vv = cache.v[pages[full // PAGE], 5, :, full % PAGE].double().cpu().numpy()
        for t in (0, new - 1):
            turned = rotate(q.double().numpy()[None, None], [ctx + t], 10000.0)[0, 0]
            want, bound = evaluate(turned, kk, vv, ctx + t, 0, 0)
            if dtype == torch.float16:
                bound = bound + (ctx + new) * 2.0 ** -27 * np.abs(want).max()
            for h in (0, 5, 127):
                err = np.abs(out[t, h].double().cpu().numpy() - want)
                assert (err <= bound).all(), (gap, t, h, float((err / bound).max()),
                                              float(err.max() / np.abs(want).max()))


# Normwise, on ordinary scores and on wide ones: the worst-case bounds above are a thousand times what an
# f32 evaluation is off by.  The kernels' errors are independent roundings as that one's are, of 2^-23 at
# most each for q and the weights (2^-24 there) and 2^-24 for sums: three times its error, and 2^-21 for the
# cases where it is lucky.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(8, 2, 64), (4, 1, 128), (3, 1, 256)])
@pytest.mark.parametrize("factor", [1.0, 3.0])
def test_errors_are_an_f32_evaluations(dtype, H, KVH, hd, factor):
    s = Step(dtype, H, KVH, hd, 32, [0, 3000, 700, 5000, 60], [130, 1, 70, 90, 3], seed=hd)
    s.qkv[:, :H * hd] *= factor
    for window, sinks in ((0, 0), (500, 4)):
        out = s.call(window, sinks).view(-1, H, hd).double().cpu()
        k, v = (x.double().cpu().numpy() for x in (s.cache.k, s.cache.v))
        first, off, plain_off, size = 0, 0.0, 0.0, 0.0
        for b, (c, n) in enumerate(zip(s.ctx, s.new)):
            rows = s.qkv[first:first + n].double().cpu().numpy().reshape(n, -1, hd)
            q = torch.from_numpy(rotate(rows[:, :H], np.arange(c, c + n), s.theta))
            kk, vv = (torch.from_numpy(x).repeat_interleave(H // KVH, 1) for x in s.sequence(b, k, v))
            p, j = torch.arange(c, c + n)[:, None, None], torch.arange(c + n)
            seen = j <= p
            if window:
                seen = seen & ((j > p - window) | (j < sinks))
            got = []
            for t in (torch.float64, torch.float32):
                scores = torch.einsum("nhd,jhd->nhj", q.to(t), kk.to(t)) / math.sqrt(hd)
                w = torch.softmax(scores.masked_fill(~seen, -math.inf), -1)
                got.append(torch.einsum("nhj,jhd->nhd", w, vv.to(t)).double())
            want, plain = got
            off += (out[first:first + n] - want).square().sum().item()
            plain_off += (plain - want).square().sum().item()
            size += want.square().sum().item()
            first += n
        err, plain = math.sqrt(off / size), math.sqrt(plain_off / size)
        assert err <= 3 * plain + 2.0 ** -21, (err, plain)
