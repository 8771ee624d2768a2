"""PagedKvCache8.attention against its formula in 64 bits, over the values that the cache holds.

The cache's codes and exponents are read as they are (test_gpu_kv8_write.py holds the writes to the
oracle, bit for bit), so tolerances are those of an f32 evaluation, paged_oracle.attend's bound.  q is
rotated in f64 and rounded to f32 (2^-24 of its pair, within the bound's terms for q's scalings), and
held in two f16 parts: 2^-22 of an element, and 2^-39 of the row's largest where that is more.  The
bound counts hd + 8 roundings of 2^-24 a product, of which fewer than hd happen in sums of hd
products of 8 or 16 at a time, so the parts' 4 are within it.

To it comes f32's range: a weight is e^(s - top) against the largest, 1, and below f32's least normal
number, 2^-126, it (or one of its parts) may be 0 in any f32 evaluation, so that an output whose large
weights' values are all 0 may lose 2^-126 of the largest value for each key (scores 87 and more below the
largest; the first run of the exponents' test found a true output of 1e-83 there).

And, for entries of more than 64 query rows a kv head (hd 128: 96, hd 64: 144), the loss that the header states: their weights
(times a power of two) are held in two f16 parts, against 2^11 for the row's largest, so each is off by
2^-25 at most beyond 2^-22 of itself, and a sum over K keys of codes up to C by K C 2^-25.  A row whose
largest sum is below min(K, 2048) C 2^-9 is done again in f32; the others' loss is thus at most 2^-16 max(1,
K / 2048) of a piece's largest sum, which is at most the row's largest sum of |weight x value|.
"""
import numpy as np
import pytest
import torch

from kv8_oracle import e4m3_value, frequencies, rotate
from paged_oracle import attend
from unillm_amd import HipError, PagedKvCache8, PageTable, Rope

pytestmark = pytest.mark.gpu

KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def values(cache, row, length):
    """(k, v) [length, heads, hd] f64 of a sequence, from the pool's bytes."""
    def codes(t):
        raw = t.view(torch.uint8).cpu().numpy()
        return raw.view(np.int8).astype(np.float64) if t.dtype == torch.int8 else e4m3_value(raw)

    pages = [p for p in row if p >= 0][:-(-length // cache.page_size)]
    ke, ve = (np.exp2(e.cpu().numpy()[pages].astype(np.float64) - 127) for e in (cache.k_exp, cache.v_exp))
    k = codes(cache.k[pages]) * np.repeat(ke, 16, 2)[..., None]
    v = codes(cache.v[pages]).swapaxes(2, 3) * np.repeat(ve, 16, 2)[..., None]
    return tuple(x.swapaxes(1, 2).reshape(-1, x.shape[1], x.shape[3])[:length] for x in (k, v))


def expect(cache, table, q, H, entries, freq=None, interleaved=False, window=0, sinks=0):
    """(out, bound) for rows q [n, H hd] of the plan's entries (sequence, rows)."""
    rows, lens = table.block_table.cpu().numpy(), table.seq_lens.tolist()
    outs, bounds, at = [], [], 0
    for i, n in entries:
        if i < 0 or n == 0:
            continue
        x = q[at:at + n].double().cpu().numpy().reshape(n, H, cache.head_dim)
        pos = np.arange(lens[i] - n, lens[i])
        if freq is not None:
            x = rotate(x, pos, freq, interleaved)
        k, v = values(cache, rows[i], lens[i])
        o, b = attend(x, k, v, pos, window, sinks)
        if n * (H // cache.n_kv_heads) > {64: 144, 128: 96, 256: 64}[cache.head_dim]:
            sums = attend(x, k, np.abs(v), pos, window, sinks)[0].max(-1, keepdims=True)
            b = b + 2.0 ** -16 * max(1, len(v) / 2048) * sums
        outs.append(o)
        bounds.append(b + len(v) * 2.0 ** -126 * np.abs(v).max())
        at += n
    return np.concatenate(outs), np.concatenate(bounds)


def close(got, want, bound):
    y = got.double().cpu().numpy().reshape(want.shape)
    worst = (np.abs(y - want) / bound).max()
    assert worst <= 1


def fill(cache, table, lens, gen, scale=1.0, spread=0.0):
    """Sequences 0, 1, .. with so many tokens each; rows' magnitudes differ by 2^spread."""
    width = 2 * cache.n_kv_heads * cache.head_dim
    for i, n in enumerate(lens):
        for a in range(0, n, table.max_tokens):
            m = min(n - a, table.max_tokens)
            table.extend(ints([i]), ints([m]))
            kv = torch.randn(m, width, device="cuda", generator=gen) * scale
            if spread:
                kv *= torch.exp2(spread * torch.randn(m, 1, device="cuda", generator=gen))
            cache.append(table, kv)
    table.check()


def make(kind, KVH, hd, page, lens, max_tokens=600, rope=None, seed=0, room=4000, **more):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = -(-(max(lens) + room) // page)
    pages = sum(-(-n // page) for n in lens) + room // page * 2 + len(lens) + 4
    table = PageTable(len(lens) + 2, need, pages, page, max_tokens)
    cache = PagedKvCache8(KVH, hd, pages, page, KINDS[kind], rope)
    cache.k.view(torch.uint8).fill_(0xFF)  # what was never written: for e4m3 NaN
    cache.v.view(torch.uint8).fill_(0x7F)
    cache.k_exp.fill_(255)
    cache.v_exp.fill_(255)
    fill(cache, table, lens, gen, **more)
    return table, cache, gen


def step(table, cache, gen, H, entries, fused, **call):
    """One step: rows of the entries appended and attended, in one call or in two; q's rows and the outputs."""
    ids, news = [i for i, _ in entries], [n for _, n in entries]
    table.extend(ints(ids), ints(news))
    n = sum(n for i, n in entries if i >= 0)
    qkv = torch.randn(n, (H + 2 * cache.n_kv_heads) * cache.head_dim, device="cuda", generator=gen)
    q = qkv[:, :H * cache.head_dim]
    if fused:
        out = cache.attention(table, qkv, H, **call)
    else:
        cache.append(table, qkv[:, H * cache.head_dim:])
        out = cache.attention(table, q, H, **call)
    table.check()
    return q, out


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("KVH,G,hd,page", [(2, 4, 128, 16), (1, 1, 64, 32), (4, 1, 128, 64), (1, 7, 256, 16),
                                           (2, 8, 64, 256), (1, 20, 128, 128), (3, 2, 256, 32)])
def test_decode_steps(kind, fused, KVH, G, hd, page):
    lens = [1, 15, 16, 17, 63, 64, 65, 300, 1111]
    table, cache, gen = make(kind, KVH, hd, page, lens, rope=Rope(hd, interleaved=True))
    freq = frequencies(hd)
    entries = [(i, 1) for i in (8, 0, 3, 2, 1, 4, 7, 6, 5)] + [(9, 1)]
    q, out = step(table, cache, gen, KVH * G, entries, fused)
    close(out, *expect(cache, table, q, KVH * G, entries, freq, True))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("KVH,G,hd,page,entries", [
    (2, 4, 64, 16, [(0, 3), (1, 5), (2, 1), (3, 16)]),
    (1, 1, 128, 32, [(0, 100), (1, 1), (2, 257)]),
    (2, 2, 128, 64, [(3, 130), (2, 31), (-1, 0), (1, 33)]),
    (1, 8, 256, 16, [(1, 70), (0, 9)]),
    (1, 5, 64, 128, [(2, 300), (0, 1), (3, 77), (1, 29)]),
    (4, 1, 256, 32, [(3, 129), (0, 64), (1, 65)])])
def test_chunks(kind, KVH, G, hd, page, entries):
    table, cache, gen = make(kind, KVH, hd, page, [5, 40, 200, 77], rope=Rope(hd, rotary_dim=hd // 2))
    q, out = step(table, cache, gen, KVH * G, entries, True)
    close(out, *expect(cache, table, q, KVH * G, entries, frequencies(hd // 2)))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,G", [(64, 4), (128, 1), (256, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (16, 4), (64, 37), (100, 0), (250, 70), (5000, 4)])
def test_windows_and_sinks(kind, hd, G, window, sinks):
    table, cache, gen = make(kind, 1, hd, 16, [10, 333, 700, 64])
    entries = [(2, 1), (0, 20), (1, 90), (3, 1)]
    q, out = step(table, cache, gen, G, entries, True, window=window, sinks=sinks)
    close(out, *expect(cache, table, q, G, entries, window=window, sinks=sinks))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("spread", [3.0, 12.0])
def test_blocks_of_very_different_exponents(kind, spread):
    table, cache, gen = make(kind, 2, 128, 16, [900, 70, 33], spread=spread)
    entries = [(0, 1), (1, 40), (2, 60)]
    q, out = step(table, cache, gen, 4, entries, True)
    close(out, *expect(cache, table, q, 4, entries))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("gap", [16.0, 30.0, 60.0])
@pytest.mark.parametrize("n", [1, 144, 145])
def test_a_dominant_key_of_no_value(kind, gap, n):
    """One key takes almost all the weight and has a value of nothing: what the others give is kept."""
    table, cache, gen = make(kind, 1, 64, 16, [400])
    # key 7 of unit direction, scaled so that q . k7 / 8 = gap; the others orthogonal to it
    cache.k.zero_()
    cache.k_exp.fill_(127)
    table2 = table  # (one sequence: rewrite all of it)
    table2.truncate(ints([0]), ints([0]))
    table2.extend(ints([0]), ints([400]))
    kv = torch.randn(400, 128, device="cuda", generator=gen)
    kv[:, 0] = 0.0
    kv[7, :64] = 0.0
    kv[7, 0] = 8.0
    kv[7, 64:] = 0.0
    cache.append(table2, kv)
    table2.extend(ints([0]), ints([n]))
    new = torch.randn(n, 64 * 3, device="cuda", generator=gen)
    new[:, 0] = gap
    new[:, 1:64] *= 0.05
    new[:, 64] = 0.0
    out = cache.attention(table2, new, 1)
    table2.check()
    close(out, *expect(cache, table2, new[:, :64], 1, [(0, n)]))


def test_the_same_plan_again_gives_the_same_bits():
    table, cache, gen = make("int8", 2, 128, 16, [700, 1500, 3])
    q, out = step(table, cache, gen, 8, [(0, 1), (1, 60), (2, 1)], False)
    for _ in range(3):
        assert torch.equal(cache.attention(table, q, 8), out)


def test_long_sequences_dealt_out_in_pieces():
    table, cache, gen = make("e4m3", 1, 128, 128, [30000, 20], max_tokens=4096)
    entries = [(0, 2), (1, 1)]
    q, out = step(table, cache, gen, 4, entries, True)
    close(out, *expect(cache, table, q, 4, entries))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,G,ctx,n", [(128, 2, 5000, 70), (64, 3, 3000, 130), (256, 1, 2500, 140)])
def test_long_chunks_dealt_out_in_pieces(kind, hd, G, ctx, n):
    table, cache, gen = make(kind, 1, hd, 64, [ctx, 9], max_tokens=4096, rope=Rope(hd))
    entries = [(1, 1), (0, n)]
    q, out = step(table, cache, gen, G, entries, True)
    close(out, *expect(cache, table, q, G, entries, frequencies(hd)))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("n", [1, 90, 150])
def test_values_of_zero_and_a_few_that_are_not(kind, n):
    """All values 0: outputs 0.  Then one block's are not, which few weights reach."""
    table, cache, gen = make(kind, 1, 64, 16, [200])
    table.truncate(ints([0]), ints([0]))
    table.extend(ints([0]), ints([200]))
    kv = torch.randn(200, 128, device="cuda", generator=gen)
    kv[:, 64:] = 0.0
    cache.append(table, kv)
    table.extend(ints([0]), ints([n]))
    qkv = torch.randn(n, 192, device="cuda", generator=gen)
    qkv[:, 128:] = 0.0
    assert not cache.attention(table, qkv, 1).any()
    table.truncate(ints([0]), ints([200]))
    table.extend(ints([0]), ints([n]))
    qkv[0, 128:] = 1e-3 * torch.randn(64, device="cuda", generator=gen)
    out = cache.attention(table, qkv, 1)
    table.check()
    close(out, *expect(cache, table, qkv[:, :64], 1, [(0, n)]))


def test_a_step_on_a_table_of_8192_sequences():
    gen = torch.Generator(device="cuda").manual_seed(3)
    table = PageTable(8192, 8, 9000, 16, 9000)
    cache = PagedKvCache8(1, 64, 9000, 16, torch.float8_e4m3fn)
    ids = torch.randperm(8192, device="cuda", generator=gen).to(torch.int32)
    table.extend(ids, torch.ones_like(ids))
    qkv = torch.randn(8192, 64 * 4, device="cuda", generator=gen)
    out = cache.attention(table, qkv, 2)
    table.check()
    # a token alone has its own value
    k, v = cache.read(table, ids, torch.zeros_like(ids), torch.arange(8193, device="cuda", dtype=torch.int32), 8192)
    assert torch.equal(out.view(8192, 2, 64), v.expand(8192, 2, 64))


def test_padding_rows_and_strides():
    table, cache, gen = make("int8", 2, 64, 16, [30, 50])
    table.extend(ints([1, -1, 0]), ints([2, 3, 1]))
    wide = torch.randn(9, 800, device="cuda", generator=gen)
    qkv = wide[:7, 16:16 + 64 * 8]
    hold = torch.full((9, 300), 5.0, device="cuda")
    out = hold[:7, 8:8 + 256]
    assert cache.attention(table, qkv, 4, out=out) is out
    table.check()
    close(out[:3], *expect(cache, table, qkv[:3, :256], 4, [(1, 2), (0, 1)]))
    assert (out[3:] == 5).all() and (hold[:, :8] == 5).all() and (hold[:, 264:] == 5).all() and (hold[7:] == 5).all()


def test_queries_that_are_not_finite():
    table, cache, gen = make("int8", 1, 64, 16, [100, 100, 100])
    table.extend(ints([0, 1, 2]), ints([1, 1, 1]))
    qkv = torch.randn(3, 64 * 4, device="cuda", generator=gen)
    qkv[0, 3], qkv[1, 70] = float("nan"), float("inf")
    out = cache.attention(table, qkv, 2)
    table.check()  # (k and v are finite)
    assert torch.isnan(out[0, :64]).all() and torch.isfinite(out[0, 64:]).all() and torch.isfinite(out[2]).all()
    qkv[1, 70] = 0.0
    want, bound = expect(cache, table, qkv[:, :128], 2, [(0, 1), (1, 1), (2, 1)])
    got = out.double().cpu().numpy().reshape(3, 2, 64)
    keep = np.array([[False, True], [True, False], [True, True]])
    assert (np.abs(got - want)[keep] <= bound[keep]).all()


def test_scores_past_f32():
    """Scores that overflow f32 to one infinity: NaN, as the formula in f32 gives; other rows are not touched."""
    table, cache, gen = make("int8", 1, 64, 16, [20, 20], scale=1e20)
    table.extend(ints([0, 1]), ints([1, 1]))
    q = torch.randn(2, 64, device="cuda", generator=gen)
    q[0] *= 1e25
    q[1] = 0.0
    cache.append(table, torch.randn(2, 128, device="cuda", generator=gen))
    out = cache.attention(table, q, 1)
    assert torch.isnan(out[0]).all()
    want, bound = expect(cache, table, q[1:], 1, [(1, 1)])
    close(out[1:], want, bound)


def test_a_bad_page_makes_its_rows_nan():
    table, cache, gen = make("e4m3", 2, 64, 16, [100, 100])
    table.block_table[0, 2] = -5
    q, out = None, None
    table.extend(ints([0, 1]), ints([1, 1]))
    q = torch.randn(2, 256, device="cuda", generator=gen)
    cache.append(table, torch.randn(2, 256, device="cuda", generator=gen))
    out = cache.attention(table, q, 4)
    with pytest.raises(HipError, match="page id"):
        table.check()
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_without_a_plan_rows_are_nan():
    table, cache, gen = make("int8", 1, 64, 16, [20])
    table.truncate(ints([0]), ints([18]))
    out = cache.attention(table, torch.randn(3, 64 * 2, device="cuda"), 2)
    assert torch.isnan(out).all()
    with pytest.raises(HipError, match="without a plan"):
        table.check()
    table.extend(ints([0]), ints([4]))
    assert torch.isnan(cache.attention(table, torch.randn(3, 64 * 2, device="cuda"), 2)).all()
    with pytest.raises(HipError, match="fewer rows"):
        table.check()


def test_serving_run_eager_captured_and_on_streams():
    """Prompts, chunks, drafts taken back and decode steps of two layers, replayed from a graph beside eager calls."""
    KVH, H, hd, page = 2, 6, 64, 16
    table = PageTable(6, 40, 150, page, 256)
    rope = Rope(hd, interleaved=True, scaling="linear", factor=2.0)
    layers = [PagedKvCache8(KVH, hd, 150, page, t, rope) for t in KINDS.values()]
    freq = frequencies(hd, scaling="linear", factor=2.0)
    gen = torch.Generator(device="cuda").manual_seed(4)

    def eager(entries):
        ids, news = [i for i, _ in entries], [n for _, n in entries]
        table.extend(ints(ids), ints(news))
        for c in layers:
            qkv = torch.randn(sum(news), (H + 2 * KVH) * hd, device="cuda", generator=gen)
            out = c.attention(table, qkv, H)
            close(out, *expect(c, table, qkv[:, :H * hd], H, entries, freq, True))
        table.check()

    eager([(0, 37), (1, 5)])
    eager([(0, 1), (1, 1), (2, 130)])
    eager([(0, 4), (1, 4), (2, 1)])
    table.truncate(ints([0, 1]), ints([39, 8]))  # drafts taken back
    s = torch.cuda.Stream()
    ids, news = ints([0, 1, 2]), ints([1, 1, 1])
    qkvs = [torch.randn(3, (H + 2 * KVH) * hd, device="cuda") for _ in layers]
    outs = [torch.empty(3, H * hd, device="cuda") for _ in layers]
    for c in layers:
        c.reserve(table, 3, H, stream=s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        table.extend(ids, news)
        for c, x, o in zip(layers, qkvs, outs):
            c.attention(table, x, H, out=o)
    for i in range(20):  # across page and block borders
        for x in qkvs:
            x.normal_(generator=gen)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        table.check()
        if i % 4 == 3:
            for c, x, o in zip(layers, qkvs, outs):
                close(o, *expect(c, table, x[:, :H * hd], H, [(0, 1), (1, 1), (2, 1)], freq, True))
            table.release(ints([1]))
            eager([(1, 6)])
    s.wait_stream(torch.cuda.current_stream())
    aside = layers[0].attention(table, torch.ones(6, H * hd, device="cuda"), H, stream=s)
    s.synchronize()
    assert torch.equal(aside, layers[0].attention(table, torch.ones(6, H * hd, device="cuda"), H))


@pytest.mark.parametrize("kind,KVH,hd", [("int8", 8, 256), ("e4m3", 16, 128), ("int8", 32, 64)])
def test_pages_past_4_gib_of_a_pool(kind, KVH, hd):
    """The same rows on pages from 8200 on (512 KiB each, 4.3 GB before them) and on the first ones: the same bits."""
    page, H, got = 256, 2 * KVH, []
    for before in (8200, 0):
        table = PageTable(3, 8200, before + 12, page, 1 << 22)
        cache = PagedKvCache8(KVH, hd, before + 12, page, KINDS[kind], Rope(hd))
        if before:
            table.extend(ints([2]), ints([before * page]))
        gen = torch.Generator(device="cuda").manual_seed(hd)
        outs = [step(table, cache, gen, H, entries, True)[1]
                for entries in ([(0, 700), (1, 40)], [(0, 1), (1, 300)], [(1, 1), (0, 20)], [(0, 1), (1, 1)])]
        held = [p for p in table.block_table[:2].flatten().tolist() if p >= 0]
        assert len(held) >= 5 and min(held) >= before
        outs += cache.read(table, ints([0, 1]), ints([3, 0]), ints([0, 700, 1000]), 1000)
        table.check()
        got.append(outs)
        del table, cache
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_capture_without_a_workspace_is_refused():
    table, cache, gen = make("int8", 1, 64, 16, [20])
    table.extend(ints([0]), ints([1]))
    s = torch.cuda.Stream()
    x = torch.randn(500, 64 * 40, device="cuda")
    with pytest.raises(HipError, match="kv8_reserve"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            cache.attention(table, x, 40, out=torch.empty_like(x), stream=s)


def test_refusals():
    table, cache, gen = make("int8", 2, 64, 16, [20])
    table.extend(ints([0]), ints([2]))
    qkv = torch.randn(2, 64 * 8, device="cuda")
    for bad in (qkv.half(), qkv.cpu(), qkv[:, :300], qkv.t(), qkv[0]):
        with pytest.raises(RuntimeError, match="qkv"):
            cache.attention(table, bad, 4)
    with pytest.raises(RuntimeError, match="multiples of 4"):
        cache.attention(table, torch.randn(2, 64 * 8 + 2, device="cuda")[:, :64 * 8], 4)
    with pytest.raises(RuntimeError, match="aligned"):
        cache.attention(table, torch.randn(2, 64 * 8 + 4, device="cuda")[:, 1:1 + 64 * 8], 4)
    with pytest.raises(RuntimeError, match="n_heads"):
        cache.attention(table, torch.randn(2, 64 * 7, device="cuda"), 3)
    with pytest.raises(RuntimeError, match="window"):
        cache.attention(table, qkv, 4, sinks=3)
    with pytest.raises(RuntimeError, match="n_tokens"):
        cache.attention(table, torch.randn(700, 64 * 8, device="cuda"), 4)
    both = torch.randn(4, 64 * 8, device="cuda")
    with pytest.raises(RuntimeError, match="share memory with qkv"):
        cache.attention(table, both[:2], 4, out=both[1:3, :256])
    with pytest.raises(RuntimeError, match="pages of"):
        cache.attention(PageTable(2, 4, 8, 16, 16), qkv, 4)
    with pytest.raises(RuntimeError, match="kv must be"):
        cache.append(table, qkv)
    inside = cache.k.view(torch.uint8).view(-1)[:2 * 256 * 4].view(torch.float32).view(2, 256)
    with pytest.raises(RuntimeError, match="share memory with the pool"):
        cache.append(table, inside)
    with pytest.raises(RuntimeError, match="dtype"):
        cache.read(table, ints([0]), ints([0]), ints([0, 1]), 1, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="cu_rows"):
        cache.read(table, ints([0]), ints([0]), ints([0]), 1)
    with pytest.raises(RuntimeError, match="n_rows"):
        cache.read(table, ints([0]), ints([0]), ints([0, 1]), -1)
    for change in (dict(dtype=torch.float16), dict(head_dim=96), dict(page_size=24), dict(rope=Rope(128)),
                   dict(rope=Rope(64, rotary_dim=20)), dict(k=torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.int8))):
        with pytest.raises(RuntimeError):
            PagedKvCache8(**{**dict(n_kv_heads=2, head_dim=64, n_pages=4, page_size=16), **change})
    closed = Rope(64)
    closed.close()
    with pytest.raises(RuntimeError, match="closed"):
        PagedKvCache8(2, 64, 4, 16, rope=closed)
    with pytest.raises(RuntimeError, match="NULL"):
        closed.apply(torch.zeros(1, 1, 64, device="cuda"), ints([0]))
    mem = [torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.int8), torch.zeros(4, 2, 1, device="cuda", dtype=torch.uint8)]
    with pytest.raises(RuntimeError, match="share memory"):
        PagedKvCache8(2, 64, 4, 16, k=mem[0], v=mem[0].view(4, 2, 64, 16), k_exp=mem[1], v_exp=mem[1].clone())
