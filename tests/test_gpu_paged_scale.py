"""Paged attention of more work than the kernels' first rounds hold: workgroups that take several wide
items one after the other, and plans of several scans whose entries are dealt out in pieces."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged_attention import TYPES, Step  # noqa: E402
from unillm_amd import HipError  # noqa: E402

pytestmark = pytest.mark.gpu


# 700 entries of 72 rows on 8 kv heads: 5600 wide items on a grid of 16 workgroups a CU (4096 of 256)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_workgroups_that_take_several_wide_items(dtype, hd):
    r = np.random.RandomState(hd)
    n = 700
    s = Step(dtype, 64, 8, hd, 16, [int(c) for c in r.randint(0, 150, n)], [9] * n, seed=hd + 1)
    out = s.call()
    s.check(out, seqs={0, 1, 100, 255, 256, 511, 512, 513, 580, 640, 698, 699})
    # a bad page in some of them reaches no other item of the same workgroups
    plain = out.clone()
    hurt = [0, 3, 57, 300, 690]
    for b in hurt:
        s.table.block_table[int(s.ids[b]), 0] = -1
    again = s.cache.attention(s.table, s.qkv, 64)
    with pytest.raises(HipError, match="not one that its calls leave"):
        s.table.check()
    rows = torch.zeros(9 * n, dtype=torch.bool, device="cuda")
    for b in hurt:
        rows[9 * b:9 * b + 9] = True
    assert torch.isnan(again[rows]).all()
    assert torch.equal(again[~rows], plain[~rows])


# entries that see so many more keys than the others that they are dealt out, before and after the
# plan's first scan of 256 tiles; up to 4 wide tiles a CU, pieces by the search, and more
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,longs", [(600, {1: 20011, 4: 9000, 300: 12000, 515: 10007, 520: 15000, 598: 9999, 599: 16000}),
                                     (2300, {2: 12000, 7: 9001, 1000: 11000, 2099: 14000, 2200: 10001, 2299: 17000})])
def test_pieces_past_one_scan(dtype, n, longs):
    r = np.random.RandomState(n)
    ctx = [longs.get(i, int(c)) for i, c in enumerate(r.randint(0, 60, n))]
    new = [70 if i % 2 else 1 for i in range(n)]
    s = Step(dtype, 1, 1, 64, 16, ctx, new, seed=n)
    s.check(s.call(), seqs=set(longs) | {0, 3, 255, 257, 511, 513, n - 3})
    s.check(s.call(4000, 5), 4000, 5, seqs=set(longs) | {3, 513})


# more narrow tiles than one scan, most of them in two pieces, on two kv heads
@pytest.mark.parametrize("dtype", TYPES)
def test_small_tiles_in_pieces_of_several_heads(dtype):
    n = 300
    ctx = [700 + 13 * (i % 50) for i in range(n)]
    s = Step(dtype, 8, 2, 64, 64, ctx, [2] * n, seed=11)
    s.check(s.call(), seqs={0, 1, 2, 49, 150, 254, 255, 256, 257, 298, 299})
