"""Paged attention on the GPU against its 64-bit restatement (paged_oracle.attend).

Tolerances: paged_oracle.attend's bound, element by element.  Where k or v is held in 16 bits,
the restatement reads the pool as the call left it, and the pool itself is compared with the
rotated keys rounded once (equal, but for values whose f64 rotations in two libraries straddle
a rounding boundary: one unit in the last place on at most one in 100000).
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from paged_oracle import attend, rotate  # noqa: E402
from unillm_amd import HipError, PagedKvCache, PageTable  # noqa: E402
from unillm_amd._capi import ERR_INVALID_ARG, ERR_UNSUPPORTED  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Step:
    """A table whose sequences hold ctx tokens on scattered pages, a pool of random values, and
    a step of `new` tokens: what the call gets and what it should give."""

    def __init__(self, dtype, H, KVH, hd, page, ctx, new, seed=0, theta=10000.0, pad=0, scale=1.0,
                 spare=0):
        g = torch.Generator().manual_seed(seed)
        n = len(ctx)
        need = sum(-(-(c + x) // page) for c, x in zip(ctx, new))
        self.n_pages = need + 3
        self.H, self.KVH, self.hd, self.page, self.theta = H, KVH, hd, page, theta
        self.ctx, self.new, self.dtype = ctx, new, dtype
        rows = sum(new) + pad
        self.table = PageTable(n + 2 + spare, max(-(-(c + x) // page) for c, x in zip(ctx, new)) + 1,
                               self.n_pages, page, max(rows, 1, sum(ctx)))
        self.table.free_pages.copy_(torch.randperm(self.n_pages, generator=g).to(torch.int32))
        self.ids = torch.randperm(n + 2, generator=g)[:n].to(torch.int32).cuda()
        if sum(ctx):
            self.table.extend(self.ids, ints(ctx))
        self.table.extend(self.ids, ints(new))
        self.table.check()
        k = torch.randn((self.n_pages, KVH, page, hd), generator=g) * scale
        v = torch.randn((self.n_pages, KVH, hd, page), generator=g)
        self.qkv = (torch.randn((rows, (H + 2 * KVH) * hd), generator=g)).cuda()
        self.cache = PagedKvCache(KVH, hd, self.n_pages, page, dtype, theta,
                                  k=k.to(dtype).cuda(), v=v.to(dtype).cuda())

    def sequence(self, b, k, v):
        """Sequence b's keys and values [L, KVH, hd] out of pools k and v (numpy)."""
        L = self.ctx[b] + self.new[b]
        pages = self.table.block_table[int(self.ids[b])].cpu().numpy()[:-(-L // self.page)]
        kk = k[pages].transpose(0, 2, 1, 3).reshape(-1, self.KVH, self.hd)[:L]
        vv = v[pages].transpose(0, 3, 1, 2).reshape(-1, self.KVH, self.hd)[:L]
        return kk, vv

    def check(self, out, window=0, sinks=0, seqs=None):
        H, KVH, hd = self.H, self.KVH, self.hd
        k, v = (t.double().cpu().numpy() for t in (self.cache.k, self.cache.v))
        x = self.qkv.double().cpu().numpy()
        o = out.double().cpu().numpy()
        first = 0
        for b, (c, n) in enumerate(zip(self.ctx, self.new)):
            if n and (seqs is None or b in seqs):
                pos = np.arange(c, c + n)
                rows = x[first:first + n].reshape(n, H + 2 * KVH, hd)
                q = rotate(rows[:, :H], pos, self.theta)
                kk, vv = self.sequence(b, k, v)
                # the new keys and values, rounded once
                for got, true in ((kk[c:], rotate(rows[:, H:H + KVH], pos, self.theta)),
                                  (vv[c:], rows[:, H + KVH:])):
                    want = torch.from_numpy(true).float().to(self.dtype).double().numpy()
                    off = got != want
                    if self.dtype != torch.float32:
                        assert off.sum() <= 1e-5 * off.size + 1
                    eps = torch.finfo(self.dtype).eps
                    assert (np.abs(got - want) <= eps * np.abs(want) + 1e-37).all()
                ref, bound = attend(q, kk, vv, pos, window, sinks)
                err = np.abs(o[first:first + n].reshape(n, H, hd) - ref)
                assert np.isfinite(err).all()
                assert (err <= bound + 1e-30).all(), (b, float((err / (bound + 1e-30)).max()))
            first += n

    def call(self, window=0, sinks=0, **kw):
        out = self.cache.attention(self.table, self.qkv, self.H, window=window, sinks=sinks, **kw)
        self.table.check()
        return out


HEADS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (7, 1, 64), (6, 2, 256), (16, 1, 128), (32, 1, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS)
def test_one_token_a_sequence(dtype, H, KVH, hd):
    ctx = [0, 1, 15, 16, 17, 31, 32, 63, 64, 100, 257, 700]
    s = Step(dtype, H, KVH, hd, 16, ctx, [1] * len(ctx), seed=H)
    s.check(s.call())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS)
def test_ragged_chunks(dtype, H, KVH, hd):
    s = Step(dtype, H, KVH, hd, 32, [0, 0, 5, 63, 200, 31, 130], [1, 40, 3, 65, 0, 2, 129], seed=H + 1)
    s.check(s.call())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_page_sizes(dtype, page):
    s = Step(dtype, 4, 2, 64, page, [0, page - 1, page, 300], [page + 1, 2, 1, 70], seed=page)
    s.check(s.call())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (16, 0), (33, 4), (64, 37), (100, 64),
                                          (127, 200), (5000, 4), (1 << 40, 1 << 40)])
def test_windows_and_sinks(dtype, window, sinks):
    s = Step(dtype, 8, 2, 64, 16, [0, 3, 40, 129, 300, 511], [70, 1, 5, 1, 33, 1], seed=window % 1000)
    s.check(s.call(window, sinks), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,window,sinks", [(128, 0, 0), (64, 200, 4), (256, 0, 0)])
def test_long_sequences(dtype, hd, window, sinks):
    s = Step(dtype, 4, 1, hd, 64, [5000, 777, 9001], [1, 90, 4], seed=hd)
    s.check(s.call(window, sinks), window, sinks)


# query rows of an entry on both sides of the tiles' sizes: 16 (narrow), 64 (the last narrow
# entry), waves of 32 and tiles of 128 and 256 (wide)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_row_counts(dtype, hd):
    new = [15, 16, 17, 63, 64, 65, 95, 97, 128, 129, 255, 256, 257, 290]
    s = Step(dtype, 1, 1, hd, 16, [0, 3, 20, 0, 1, 0, 40, 9, 0, 2, 0, 31, 0, 64], new, seed=hd)
    s.check(s.call())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd,new", [(7, 1, 64, 41), (6, 2, 128, 130), (5, 1, 256, 60), (16, 1, 64, 20)])
def test_groups_that_divide_no_tile(dtype, H, KVH, hd, new):
    s = Step(dtype, H, KVH, hd, 32, [100, 0, 517], [new, new + 3, 7], seed=new)
    s.check(s.call())
    s.check(s.call(77, 5), 77, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 256)])
def test_chunks_behind_long_prefixes(dtype, hd, page):
    # the keys of a tile in pieces, on more pages than one read of page ids
    s = Step(dtype, 2, 1, hd, page, [20011, 0, 9000], [70, 1, 3], seed=page)
    s.check(s.call())
    s.check(s.call(5000, 100), 5000, 100)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_tiles_than_one_scan(dtype):
    # 300 entries of 70 rows (wide) and 300 of one, the plan's lists past 256 of each
    r = np.random.RandomState(5)
    new = [70 if i % 2 else 1 for i in range(600)]
    s = Step(dtype, 1, 1, 64, 16, [int(c) for c in r.randint(0, 90, 600)], new, seed=6)
    s.check(s.call(), seqs={0, 1, 255, 256, 257, 511, 513, 598, 599})


@pytest.mark.parametrize("hd", [64, 256])
def test_the_most_sequences(hd):
    # 8192 entries, the most of a table, in an order of their own
    g = torch.Generator().manual_seed(2)
    n, page = 8192, 16
    table = PageTable(n, 2, 2 * n, page, 3 * n)
    cache = PagedKvCache(1, hd, 2 * n, page, torch.bfloat16)
    ids = torch.randperm(n, generator=g).to(torch.int32).cuda()
    one = torch.ones(n, dtype=torch.int32, device="cuda")
    qkv = [torch.randn(n, 3 * hd, generator=g).cuda() for _ in range(3)]
    for x in qkv:
        table.extend(ids, one)
        out = cache.attention(table, x, 1)
    table.check()
    assert (table.seq_lens == 3).all()
    rows = [x.double().cpu().numpy().reshape(n, 3, hd) for x in qkv]
    for b in range(0, n, 1000):
        k = np.stack([torch.from_numpy(rotate(x[b:b + 1, 1:2], [t], 10000.0)).bfloat16().double().numpy()[0]
                      for t, x in enumerate(rows)])
        v = np.stack([torch.from_numpy(x[b, 2:3]).bfloat16().double().numpy() for x in rows])
        ref, bound = attend(rotate(rows[2][b:b + 1, :1], [2], 10000.0), k, v, [2])
        # (a key on a rounding boundary may be a unit off: 2^-8 of the scores' terms)
        assert (np.abs(out[b].double().cpu().numpy() - ref[0, 0]) <= bound[0, 0] + 2.0 ** -8).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences(dtype):
    r = np.random.RandomState(3)
    n = 300
    ctx = [int(c) for c in r.randint(0, 40, n)]
    new = [int(c) for c in r.randint(0, 4, n)]
    s = Step(dtype, 2, 1, 64, 16, ctx, new, seed=5)
    s.check(s.call(), seqs=set(range(0, 300, 7)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 6, 80])
def test_what_masked_places_hold_does_not_matter(dtype, new):
    ctx = [0, 40, 333]
    bad = float("nan")
    for window, sinks, value in ((0, 0, bad), (50, 3, bad), (50, 3, float("inf"))):
        s = Step(dtype, 4, 2, 64, 16, ctx, [new] * 3, seed=9)
        clean = s.call(window, sinks).clone()
        s.check(clean, window, sinks)
        k, v = s.cache.k, s.cache.v
        held = torch.zeros(s.n_pages, 16, dtype=torch.bool)
        for b, c in enumerate(ctx):
            pages = s.table.block_table[int(s.ids[b])].tolist()
            for j in range(c + new):
                # seen by the sequence's first new token: with a window, later ones see less
                if not window or j > c + new - 1 - window or j < sinks:
                    held[pages[j // 16], j % 16] = True
        dirty = (~held).cuda()
        k.masked_fill_(dirty[:, None, :, None], value)
        v.masked_fill_(dirty[:, None, None, :], value)
        out = s.call(window, sinks)
        # only the last token of each sequence sees none of them for certain
        last = np.cumsum(s.new) - 1
        assert torch.isfinite(out[last]).all()
        if not window or new == 1:
            assert torch.isfinite(out).all()
            first = 0
            err = (out - clean).abs().max().item()
            assert err <= 2.0 ** -24 * 4096, (first, err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [2, 70])
def test_infinite_and_nan_keys_and_values_that_are_seen(dtype, new):
    # a NaN key: every row that sees it is NaN, the rows before it are not; an infinite value: the
    # rows that see it have that sign of infinity in its dimension, and no other
    s = Step(dtype, 4, 2, 64, 16, [20, 50], [new, new], seed=2)
    clean = s.call().clone()
    W = s.H * s.hd
    s.qkv[1, W:W + 64] = float("nan")  # sequence 0's second new key, kv head 0
    out = s.call()
    o, c = out.view(-1, 4, 64), clean.view(-1, 4, 64)
    assert torch.isnan(o[1:new, :2]).all()
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[new:]).all()
    assert torch.isfinite(o[:new, 2:]).all()
    tol = 4096 * 2.0 ** -24
    assert (o[0] - c[0]).abs().max() <= tol and (o[new:] - c[new:]).abs().max() <= tol
    s = Step(dtype, 4, 2, 64, 16, [20, 50], [new, new], seed=2)
    s.qkv[new, W + 2 * 64 + 64 + 5] = -float("inf")  # sequence 1's first new value, kv head 1, d 5
    o = s.call().view(-1, 4, 64)
    assert (o[new:, 2:, 5] == -float("inf")).all()
    o[new:, 2:, 5] = 0
    assert torch.isfinite(o).all()
    mask = torch.ones_like(o, dtype=torch.bool)
    mask[new:, 2:, 5] = False
    assert ((o - c).abs()[mask] <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [3, 90])
def test_non_finite_values_where_keys_are_in_pieces(dtype, new):
    # a sequence long enough to be dealt out: NaN and infinities in its first page are seen without
    # a window and hidden behind one; both ways every piece's rows are right
    s = Step(dtype, 4, 2, 64, 16, [6000, 10], [new, new], seed=12)
    whole, windowed = s.call().clone(), s.call(300, 2).clone()
    page = int(s.table.block_table[int(s.ids[0]), 0])
    s.cache.v[page, 0, 7, 3] = float("inf")   # key 3, kv head 0, dimension 7
    s.cache.k[page, 1, 5, 9] = float("nan")   # key 5, kv head 1
    out = s.call().view(-1, 4, 64)
    assert (out[:new, :2, 7] == float("inf")).all() and torch.isnan(out[:new, 2:]).all()
    assert torch.isfinite(out[new:]).all()
    tol = 4096 * 2.0 ** -24
    assert (out[:new, :2, :7] - whole.view(-1, 4, 64)[:new, :2, :7]).abs().max() <= tol
    assert (s.call(300, 2) - windowed).abs().max() <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [1e-4, 30.0])
def test_flat_and_peaked_scores(dtype, scale):
    s = Step(dtype, 4, 2, 128, 16, [0, 90, 400], [33, 1, 20], seed=7, scale=scale)
    s.check(s.call())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [1e-30, 1e-3, 3e4])
def test_queries_of_any_size(dtype, factor):
    # tiny, and so large that one key takes all the weight
    s = Step(dtype, 4, 2, 64, 16, [50], [20], seed=8)
    s.qkv[:, :4 * 64] *= factor
    s.check(s.call())


@pytest.mark.parametrize("dtype", TYPES)
def test_padded_rows_are_left(dtype):
    s = Step(dtype, 4, 2, 64, 16, [10, 40, 0], [1, 30, 0], pad=9, seed=3)
    s.qkv[31:] = float("nan")
    out = torch.full((40, 4 * 64), -7.0, device="cuda")
    s.call(out=out)
    assert (out[31:] == -7).all()
    s.check(out)


def test_row_strides():
    s = Step(torch.float16, 4, 2, 64, 16, [10, 40], [1, 30], seed=3)
    plain = s.call().clone()
    wide = torch.full((31, 4 * 64 + 4 * 64 + 20), -7.0, device="cuda")
    wide[:, 4:4 + 8 * 64] = s.qkv
    out = torch.full((31, 4 * 64 + 8), -7.0, device="cuda")
    s.qkv = wide[:, 4:4 + 8 * 64]
    got = s.call(out=out[:, 4:4 + 256])
    assert torch.equal(got, plain)
    assert (out[:, :4] == -7).all() and (out[:, -4:] == -7).all()


def test_results_repeat_bit_for_bit():
    for dtype in TYPES:
        s = Step(dtype, 8, 2, 128, 16, [3000, 0, 50], [1, 200, 17], seed=4)
        a = s.call().clone()
        assert torch.equal(a, s.call())


def test_without_a_plan_the_rows_are_nan_and_nothing_is_appended():
    s = Step(torch.float16, 4, 2, 64, 16, [10, 40], [1, 30], seed=3)
    k = s.cache.k.clone()
    s.table.truncate(s.ids, ints([10, 40]))
    out = s.cache.attention(s.table, s.qkv, 4)
    with pytest.raises(HipError, match="without a plan") as e:
        s.table.check()
    assert e.value.status == ERR_INVALID_ARG
    assert torch.isnan(out).all() and torch.equal(k, s.cache.k)
    s.table.extend(s.ids, ints([1, 30]))
    # fewer rows than the plan has
    out = s.cache.attention(s.table, s.qkv[:30], 4)
    with pytest.raises(HipError, match="fewer rows"):
        s.table.check()
    assert torch.isnan(out).all() and torch.equal(k, s.cache.k)
    s.check(s.call())


@pytest.mark.parametrize("new", [1, 40])
def test_a_bad_page_makes_its_rows_nan(new):
    # the kernels' own bounds checks: a page id that the pool does not have is never read
    s = Step(torch.float16, 4, 2, 64, 16, [100, 40], [new, new], seed=3)
    keep = s.table.block_table[int(s.ids[0]), 2].item()
    for page in (-1, s.n_pages, 1 << 30, -(1 << 31)):
        s.table.block_table[int(s.ids[0]), 2] = page
        out = s.cache.attention(s.table, s.qkv, 4)
        with pytest.raises(HipError, match="not one that its calls leave"):
            s.table.check()
        assert torch.isnan(out[:new]).all()
        s.check(out, seqs={1})
    s.table.block_table[int(s.ids[0]), 2] = keep
    s.check(s.call())


def test_arguments_are_checked():
    s = Step(torch.float16, 4, 2, 64, 16, [10], [3], seed=3)
    a = s.cache.attention
    for bad in (s.qkv.double(), s.qkv.cpu(), s.qkv[:, :-1], s.qkv.t().contiguous().t(), s.qkv[0]):
        with pytest.raises(RuntimeError):
            a(s.table, bad, 4)
    for kw, text in ((dict(window=-1), "window >= 0"), (dict(sinks=2), "without a window"),
                     (dict(window=4, sinks=-1), "sinks >= 0")):
        with pytest.raises(HipError, match=text):
            a(s.table, s.qkv, 4, **kw)
    with pytest.raises(RuntimeError):
        a(s.table, s.qkv, 3)
    with pytest.raises(RuntimeError):
        a(s.table, s.qkv, 4, out=torch.empty(2, 256, device="cuda"))
    big = torch.zeros(4, 8 * 64 + 1, device="cuda")
    with pytest.raises(HipError, match="16-byte aligned|multiples of 4"):
        a(s.table, big[:3, 1:], 4)
    flat = torch.zeros(3 * 8 * 64 + 8, device="cuda")
    with pytest.raises(HipError, match="share memory"):
        a(s.table, flat[:3 * 512].view(3, 512), 4, out=flat[8:8 + 3 * 256].view(3, 256))
    with pytest.raises(HipError, match="n_tokens"):
        a(s.table, torch.zeros(200, 512, device="cuda"), 4)
    other = PagedKvCache(2, 64, s.n_pages, 32, torch.float16)
    with pytest.raises(HipError, match="pages of"):
        other.attention(s.table, s.qkv, 4)
    assert a(s.table, s.qkv[:0], 4).shape == (0, 256)
    many = PageTable(1, 1, s.n_pages, 16, 1 << 20)
    with pytest.raises(HipError, match="2\\^30"):
        s.cache.reserve(many, 1 << 20, 1024)
    with pytest.raises(RuntimeError):
        PagedKvCache(2, 64, 4, 16, torch.float64)
    with pytest.raises(RuntimeError):
        PagedKvCache(2, 64, 4, 16, torch.float16, k=torch.zeros(4, 2, 16, 64, device="cuda").half())
    with pytest.raises(RuntimeError):
        PagedKvCache(2, 64, 4, 16, torch.float16, k=torch.zeros(4, 2, 16, 64, device="cuda"),
                     v=torch.zeros(4, 2, 64, 16, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,hd,rows", [((8, 2), 128, 4), ((4, 4), 64, 24)])
def test_captured_steps_replay_at_other_lengths(dtype, heads, hd, rows):
    # one graph of a whole step, replayed with other requests and lengths, eager calls between
    H, KVH = heads
    g = torch.Generator().manual_seed(1)
    table = PageTable(6, 40, 150, 16, 64)
    cache = PagedKvCache(KVH, hd, 150, 16, dtype)
    eager_table = PageTable(6, 40, 150, 16, 64)
    eager = PagedKvCache(KVH, hd, 150, 16, dtype)
    ids, news = ints([0, 1, 2, 3]), ints([1, 1, 1, 1])
    qkv = torch.randn(rows, (H + 2 * KVH) * hd, generator=g).cuda()
    out = torch.zeros(rows, H * hd, device="cuda")
    side = torch.cuda.Stream()
    cache.reserve(table, rows, H, stream=side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        table.extend(ids, news)
        cache.attention(table, qkv, H, out=out)
        cache.attention(table, qkv, H, window=30, sinks=2, out=out)
    r = np.random.RandomState(0)
    for step in range(10):
        i = r.permutation(6)[:4].tolist()
        n = (r.multinomial(rows, [0.4, 0.3, 0.2, 0.1]) if rows > 4 else np.ones(4, int)).tolist()
        if step % 4 == 3:
            i[1] = -1
        ids.copy_(ints(i))
        news.copy_(ints(n))
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        out.fill_(-3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        eager_table.extend(ids, news)
        want = torch.full_like(out, -3.0)
        eager.attention(eager_table, qkv, H, window=30, sinks=2, out=want)
        assert (out - want).abs().max() <= 4096 * 2.0 ** -24
        assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)
    table.check()
    eager_table.check()


def test_capture_refuses_to_grow_the_workspace():
    # (250000 rows of head_dim 256 keep 256 MB of cosines and sines: more than other tests leave)
    n = 250000
    table, cache = PageTable(1, 1, 2, 16, n), PagedKvCache(1, 256, 2, 16)
    qkv, out = torch.zeros(n, 768, device="cuda"), torch.zeros(n, 256, device="cuda")
    ids, one = ints([0]), ints([1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        table.extend(ids, one)
        with pytest.raises(HipError) as e:
            cache.attention(table, qkv, 1, out=out)
        assert e.value.status == ERR_UNSUPPORTED
        with pytest.raises(HipError, match="captured") as e:
            table.check()
        assert e.value.status == ERR_UNSUPPORTED
    graph.replay()
    torch.cuda.synchronize()
    table.check()
    assert table.seq_lens[0].item() == 1


def test_captured_attention_reads_the_current_plan():
    s = Step(torch.float16, 32, 4, 128, 16, [9000, 3], [1, 1], seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty(2, 32 * 128, device="cuda")
    s.cache.reserve(s.table, 2, 32, stream=side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.cache.attention(s.table, s.qkv, 32, out=out)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        s.check(out)


def test_two_streams_at_once():
    # tables and pools of their own, a stream each, interleaved calls
    steps = [Step(t, 8, 2, 128, 16, [2000, 30, 0], [1, 20, 64], seed=i) for i, t in enumerate(TYPES)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    outs = [[] for _ in steps]
    for _ in range(4):
        for s, st, o in zip(steps, streams, outs):
            o.append(s.cache.attention(s.table, s.qkv, 8, stream=st))
    torch.cuda.synchronize()
    for s, o in zip(steps, outs):
        s.check(o[0])
        for x in o[1:]:
            assert torch.equal(x, o[0])


def test_positions_past_31_bits_of_bytes():
    # pages at the end of a pool of more than 2^32 bytes (and 2^31 elements) of K and V each
    KVH, hd, page = 8, 128, 256
    n_pages = (1 << 32) // (KVH * hd * page * 2) + 70
    table = PageTable(2, 8, n_pages, page, 600)
    table.free_pages.copy_(torch.arange(n_pages - 1, -1, -1, dtype=torch.int32).flip(0))
    cache = PagedKvCache(KVH, hd, n_pages, page, torch.float16)
    g = torch.Generator().manual_seed(1)
    table.extend(ints([1]), ints([520]))
    assert table.block_table[1, 0].item() == n_pages - 1
    qkv = torch.randn(520, (8 + 16) * hd, generator=g).cuda()
    big = cache.attention(table, qkv, 8)
    table.check()
    small_table = PageTable(2, 8, 4, page, 600)
    small = PagedKvCache(KVH, hd, 4, page, torch.float16)
    small_table.extend(ints([1]), ints([520]))
    assert torch.equal(big, small.attention(small_table, qkv, 8))
    table.truncate(ints([1]), ints([519]))
    small_table.truncate(ints([1]), ints([519]))
    table.extend(ints([1]), ints([1]))
    small_table.extend(ints([1]), ints([1]))
    assert torch.equal(cache.attention(table, qkv[:1], 8), small.attention(small_table, qkv[:1], 8))


def test_results_of_a_side_stream_outlive_it():
    # the output is the side stream's memory, used and freed on the current one
    s = Step(torch.float16, 4, 2, 64, 16, [30, 5], [1, 9], seed=2)
    want = s.call().clone()
    side = torch.cuda.Stream()
    for _ in range(5):
        side.wait_stream(torch.cuda.current_stream())
        out = s.cache.attention(s.table, s.qkv, 4, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        got = out + 0.0
        del out
        assert torch.equal(got, want)
