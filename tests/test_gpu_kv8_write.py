"""PagedKvCache8.append and read against the 64-bit oracle: codes and exponents bit for bit."""
import numpy as np
import pytest
import torch

from kv8_oracle import Pool, e4m3_value, frequencies, rotate
from unillm_amd import HipError, PagedKvCache8, PageTable, Rope

pytestmark = pytest.mark.gpu

MAX = float(np.finfo(np.float32).max)
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def codes(t):
    """A pool's codes as numbers."""
    raw = t.view(torch.uint8).cpu().numpy()
    return raw.view(np.int8).astype(np.float64) if t.dtype == torch.int8 else e4m3_value(raw)


def same(cache, pool):
    assert np.array_equal(cache.k_exp.cpu().numpy().astype(int) - 127, pool.ke)
    assert np.array_equal(cache.v_exp.cpu().numpy().astype(int) - 127, pool.ve)
    assert np.array_equal(codes(cache.k), pool.k)
    assert np.array_equal(codes(cache.v), pool.v)


class Run:
    """A table, a cache and the oracle's pool, stepped together."""

    def __init__(self, kind, heads, hd, page, n_pages=64, max_seqs=8, rope=None, freq=None, interleaved=False,
                 magnitude=1.0, max_tokens=600):
        self.table = PageTable(max_seqs, n_pages, n_pages, page, max_tokens)
        self.cache = PagedKvCache8(heads, hd, n_pages, page, KINDS[kind], rope)
        self.pool = Pool(n_pages, heads, hd, page, kind)
        self.heads, self.hd, self.rot = heads, hd, (freq, interleaved, magnitude)

    def step(self, ids, news, kv, again=False):
        n = sum(news)
        self.table.extend(ints(ids), ints(news))
        self.cache.append(self.table, kv)
        if again:
            self.cache.append(self.table, kv)
        x = kv[:n].double().cpu().numpy().reshape(n, 2, self.heads, self.hd)
        k, (freq, inter, m) = x[:, 0], self.rot
        if freq is not None:
            with np.errstate(invalid="ignore"):
                k = rotate(k, self.table.positions[:n].tolist(), freq, inter, m).astype(np.float32).astype(np.float64)
        self.pool.write(self.table.slots[:n].tolist(), k, x[:, 1])


def steps(run, kind_seed, sizes, spread=6.0):
    """Steps of ragged batches, whose rows' magnitudes differ by 2^spread and more."""
    gen = torch.Generator(device="cuda").manual_seed(kind_seed)
    for i, (ids, news) in enumerate(sizes):
        n = sum(news)
        scale = torch.exp2(spread * torch.randn(n, 1, device="cuda", generator=gen))
        kv = torch.randn(n, 2 * run.heads * run.hd, device="cuda", generator=gen) * scale
        run.step(ids, news, kv, again=i % 2 == 1)
        run.table.check()
        same(run.cache, run.pool)


SIZES = [([0, 1, 2], [1, 5, 40]), ([2, 0, 3], [1, 1, 17]), ([0, 1, 2, 3], [1, 1, 1, 1]), ([1, 0], [30, 3]),
         ([0, 1, 2, 3], [1, 1, 1, 1]), ([3, 2, 1, 0], [2, 16, 0, 100]), ([4, 0], [16, 15])]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("heads,hd,page", [(1, 64, 16), (3, 128, 32), (2, 256, 64), (5, 64, 256), (2, 128, 128)])
def test_steps_bit_for_bit(kind, heads, hd, page):
    steps(Run(kind, heads, hd, page), 1, SIZES)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,rot,interleaved,scaling", [(64, 64, False, None), (128, 128, True, None), (128, 40, False, "llama3"),
                                                        (256, 64, True, "yarn"), (256, 256, False, "linear"), (64, 8, True, None)])
def test_rotated_keys(kind, hd, rot, interleaved, scaling):
    more = dict(factor=8.0, low=1.0, high=4.0, original=64) if scaling else {}
    rope = Rope(hd, rotary_dim=rot, interleaved=interleaved, scaling=scaling, **more)
    m = 0.1 * np.log(8.0) + 1 if scaling == "yarn" else 1.0
    run = Run(kind, 2, hd, 32, rope=rope, freq=frequencies(rot, scaling=scaling, **more), interleaved=interleaved, magnitude=m)
    rope.close()  # (its frequencies were copied)
    steps(run, 2, SIZES, spread=2.0)


@pytest.mark.parametrize("kind", list(KINDS))
def test_many_rows_in_one_step(kind):
    """Rows past 512: workgroups of 16 rows; blocks that begin and end anywhere."""
    run = Run(kind, 3, 64, 16, n_pages=128, max_tokens=1500)
    steps(run, 3, [([0, 1, 2], [7, 1, 12]), ([0, 1, 2, 3, 4], [333, 1, 250, 90, 1]), ([4, 3, 1], [301, 301, 301])])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("heads,hd", [(9, 64), (18, 64), (34, 64), (33, 128), (32, 256)])
def test_decoding_rows_among_chunks(kind, heads, hd):
    """Workgroups of 4, 8 and 16 rows (by rows times heads), each with runs of one row and of several."""
    rope = Rope(hd, interleaved=True)
    run = Run(kind, heads, hd, 16, n_pages=300, max_seqs=90, rope=rope, freq=frequencies(hd), interleaved=True, max_tokens=700)
    small = [(i, 1 + (i * 7 % 11 == 0) * 2) for i in range(80)]
    first = [(i, 1 + i % 5) for i in range(80)] + [(80, 200)]
    mixed = small[:30] + [(80, 170)] + small[30:] + [(81, 250)]
    steps(run, 11, [([i for i, _ in e], [n for _, n in e]) for e in (first, mixed, mixed)], spread=2.0)


def test_a_table_of_8192_sequences():
    """The plan's LDS is the largest there; entries in any order."""
    run = Run("int8", 1, 64, 16, n_pages=600, max_seqs=8192, max_tokens=600)
    ids = [(i * 37) % 8192 for i in range(500)]
    steps(run, 12, [(ids, [1] * 500), (ids[::-1], [1] * 500)])


@pytest.mark.parametrize("kind", list(KINDS))
def test_every_growth_of_an_exponent(kind):
    """A block whose positions each need twice the last one's step, and more; values on ties."""
    run = Run(kind, 1, 64, 16, n_pages=4)
    base = torch.arange(128, device="cuda").float() - 63.5
    for p in range(32):
        run.step([0], [1], (base * 2.0 ** (p if p < 20 else 40 - p))[None].contiguous())
        same(run.cache, run.pool)


@pytest.mark.parametrize("kind,top", [("int8", 127.0), ("e4m3", 448.0)])
def test_exponents_at_their_borders(kind, top):
    run = Run(kind, 1, 64, 16, n_pages=40, max_seqs=40)
    values = [0.0, top, np.nextafter(np.float32(top), np.float32(np.inf)), np.nextafter(np.float32(top), np.float32(0)),
              MAX, -MAX, 1.1754944e-38, 1e-45, top * 2.0 ** -126, top * 2.0 ** -127, 2.0 ** -126,
              -top, 1.0, 2.0 ** 127, 0.5 * 2.0 ** -126]
    for i, v in enumerate(values):
        kv = torch.zeros(1, 128, device="cuda")
        kv[0, 3], kv[0, 100] = float(v), float(v)
        kv[0, 5], kv[0, 101] = float(v) / 3, -float(v) / 7
        run.step([i], [1], kv)
    run.table.check()
    same(run.cache, run.pool)


def test_every_e4m3_value_and_tie():
    """All e4m3 values, the ties between them and their neighbours, in one block."""
    v = np.sort(np.unique(np.abs(e4m3_value(np.arange(127)))))
    mid = ((v[1:] + v[:-1]) / 2).astype(np.float32)
    x = np.concatenate([v.astype(np.float32), mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1000))])
    x = np.concatenate([x, -x])
    run = Run("e4m3", 1, 64, 16, n_pages=4)
    kv = torch.zeros(16, 128, device="cuda")
    kv.view(-1)[:len(x)] = torch.from_numpy(x).cuda()
    run.step([0], [16], kv)
    same(run.cache, run.pool)


@pytest.mark.parametrize("kind", list(KINDS))
def test_values_that_are_not_finite(kind):
    """Held as the largest code or 0, counted for no exponent, reported; other rows are untouched by them."""
    run = Run(kind, 2, 64, 16)
    kv = torch.randn(20, 256, device="cuda")
    kv[3, 7], kv[5, 200], kv[18, 0] = float("inf"), float("nan"), float("-inf")
    kv[19] = float("nan")
    run.step([0], [20], kv)
    same(run.cache, run.pool)
    with pytest.raises(HipError, match="not finite"):
        run.table.check()
    run.table.check()


def test_what_stands_past_the_step_stays():
    """Stale codes of a taken-back position, other pages and padding rows are left as they were."""
    run = Run("int8", 2, 64, 32)
    steps(run, 5, [([0, 1], [40, 10])])
    run.table.truncate(ints([0]), ints([37]))
    run.table.extend(ints([0, -1]), ints([1, 5]))
    kv = torch.randn(6, 256, device="cuda")
    run.cache.append(run.table, kv)  # rows past the plan's one are padding
    x = kv[:1].double().cpu().numpy().reshape(1, 2, 2, 64)
    run.pool.write(run.table.slots[:1].tolist(), x[:, 0], x[:, 1])
    same(run.cache, run.pool)


def test_strided_rows_another_stream_and_replays():
    table, s = PageTable(4, 16, 32, 16, 64), torch.cuda.Stream()
    fused = torch.randn(12, 64 * 10, device="cuda")
    kv = fused[:, 128:128 + 256]
    a, b = (PagedKvCache8(2, 64, 32, 16, torch.int8, Rope(64)) for _ in range(2))
    table.extend(ints([2, 0]), ints([3, 9]))
    a.append(table, kv.contiguous())
    s.wait_stream(torch.cuda.current_stream())
    b.append(table, kv, stream=s)
    s.synchronize()
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_exp, b.k_exp), (a.v_exp, b.v_exp)):
        assert torch.equal(x, y)
    ids, news = ints([2, 0]), ints([1, 1])
    g = torch.cuda.CUDAGraph()
    small = kv[:2].contiguous()
    with torch.cuda.graph(g, stream=s):
        table.extend(ids, news)
        a.append(table, small)
    for i in range(4):
        small.normal_()
        g.replay()  # extends, and writes a
        b.append(table, small)
        torch.cuda.synchronize()
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.k_exp, b.k_exp)
    table.check()
    assert table.seq_lens.tolist() == [13, 0, 7, 0]


def test_without_a_plan_nothing_is_written():
    table = PageTable(2, 8, 8, 16, 64)
    cache = PagedKvCache8(1, 64, 8, 16)
    kv = torch.randn(4, 128, device="cuda")
    cache.append(table, kv)
    with pytest.raises(HipError, match="without a plan"):
        table.check()
    table.extend(ints([0]), ints([5]))
    cache.append(table, kv)
    with pytest.raises(HipError, match="fewer rows"):
        table.check()
    assert not cache.k.any() and not cache.v.any() and not cache.k_exp.any()


# ---- reading back ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,hd,page", [(1, 64, 16), (3, 128, 32), (2, 256, 256)])
def test_read_back(kind, dtype, heads, hd, page):
    run = Run(kind, heads, hd, page)
    steps(run, 7, SIZES, spread=1.0)
    lens = run.table.seq_lens.tolist()
    entries = [(2, 0, lens[2]), (0, 5, 1), (1, 15, 2), (-1, 3, 4), (3, 1, 3), (0, 0, 0), (2, 7, 33), (4, 15, 1)]
    cu = np.concatenate([[0], np.cumsum([n for _, _, n in entries])]).tolist()
    k, v = run.cache.read(run.table, ints([e[0] for e in entries]), ints([e[1] for e in entries]), ints(cu), cu[-1] + 3,
                          dtype=dtype)
    run.table.check()
    rows = run.table.block_table.cpu().numpy()
    for (i, start, n), at in zip(entries, cu):
        if i < 0 or n == 0:
            continue
        for got, want in zip((k, v), run.pool.values(rows[i], lens[i])):
            want = torch.from_numpy(want[start:start + n]).to(dtype)  # rounded once
            assert torch.equal(got[at:at + n].cpu(), want)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("heads,hd,n", [(1, 64, 20011), (2, 128, 9001), (4, 64, 8200)])
def test_read_of_many_rows(kind, heads, hd, n):
    """Workgroups of 16, 32 and 64 rows; some rows are not their sequence's."""
    table = PageTable(3, 2000, 2000, 16, 20600)
    cache = PagedKvCache8(heads, hd, 2000, 16, KINDS[kind])
    table.extend(ints([1, 0]), ints([n - 37, 500]))
    kv = torch.randn(n - 37 + 500, 2 * heads * hd, device="cuda")
    cache.append(table, kv)
    k, v = cache.read(table, ints([1, 2, 0, 1]), ints([3, 0, 490, 0]), ints([0, n - 40, n - 30, n - 17, n]), n,
                      dtype=torch.bfloat16)
    with pytest.raises(HipError, match="does not hold"):
        table.check()
    whole_k, whole_v = cache.read(table, ints([0, 1]), ints([0, 0]), ints([0, 500, 500 + n - 37]), 500 + n - 37)
    table.check()
    for got, whole, x in ((k, whole_k, kv[:, :heads * hd]), (v, whole_v, kv[:, heads * hd:])):
        assert torch.equal(got[:n - 40], whole[503:].bfloat16())
        assert torch.isnan(got[n - 40:n - 30]).all() and torch.isnan(got[n - 20:n - 17]).all()
        assert torch.equal(got[n - 30:n - 20], whole[490:500].bfloat16())
        assert torch.equal(got[n - 17:], whole[500:517].bfloat16())
        # (and the values are those that were written, to half a step: 1/127 of a block's largest at most, or 2^-4 of itself)
        y, x = whole[500:].flatten(1), x[:n - 37]
        top = x.abs().max()
        assert ((y - x).abs() <= (top / 127 if kind == "int8" else x.abs() * 2.0 ** -4 + top * 2.0 ** -16)).all()


def test_read_outside_a_sequence():
    run = Run("int8", 2, 64, 16)
    steps(run, 8, [([0, 1], [20, 3])])
    out = run.cache.read(run.table, ints([0, 1, 9, 0]), ints([18, 0, 0, -1]), ints([0, 4, 7, 8, 10]), 12)
    with pytest.raises(HipError, match="does not hold"):
        run.table.check()
    want = run.pool.values(run.table.block_table.cpu().numpy()[0], 20)
    for got, w in zip(out, want):
        got = got.cpu().double().numpy()
        assert np.array_equal(got[:2], w[18:]) and np.isnan(got[2:4]).all() and np.isfinite(got[4:7]).all()
        assert np.isnan(got[7]).all() and np.isnan(got[8]).all() and np.array_equal(got[9], w[0])


def test_read_of_a_page_that_is_none():
    run = Run("e4m3", 1, 64, 16)
    steps(run, 9, [([0], [40])])
    run.table.block_table[0, 1] = 1 << 20
    k, v = run.cache.read(run.table, ints([0]), ints([0]), ints([0, 40]), 40)
    with pytest.raises(HipError, match="page id"):
        run.table.check()
    assert torch.isnan(k[16:32]).all() and torch.isfinite(k[:16]).all() and torch.isfinite(v[32:]).all()


def test_a_request_moved_to_another_table():
    """Read back in f32 and written anew on other pages: the values are the same ones."""
    run = Run("int8", 2, 128, 16)
    steps(run, 10, [([3], [150])], spread=0.5)
    k, v = run.cache.read(run.table, ints([3]), ints([0]), ints([0, 150]), 150)
    table, cache = PageTable(2, 8, 9, 64, 200), PagedKvCache8(2, 128, 9, 64)
    table.extend(ints([1]), ints([150]))
    cache.append(table, torch.cat([k.flatten(1), v.flatten(1)], 1))
    k2, v2 = cache.read(table, ints([1]), ints([0]), ints([0, 150]), 150)
    assert torch.equal(k, k2) and torch.equal(v, v2)
