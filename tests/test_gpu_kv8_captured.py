"""A whole step of an 8-bit cache captured into one graph, read-back among it, and replayed between eager steps of other
sequences: every replay gives the bits of the same calls made eagerly on a second table and cache."""
import pytest
import torch

from test_gpu_kv8_write import KINDS, ints
from unillm_amd import PagedKvCache8, PageTable, Rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,new", [(64, [1, 3]), (128, [100, 1]), (256, [1, 70])])
def test_a_step_with_its_read_back(kind, hd, new):
    KVH, H, page, n = 2, 4, 16, sum(new)
    rope = Rope(hd, interleaved=True)
    sides = [(PageTable(4, 60, 150, page, 256), PagedKvCache8(KVH, hd, 150, page, KINDS[kind], rope)) for _ in range(2)]
    ids, news, starts, cu = ints([2, 0]), ints(new), ints([5, 0]), ints([0, 9, 19])
    kv, q = torch.randn(n, 2 * KVH * hd, device="cuda"), torch.randn(n, H * hd, device="cuda")

    def step(table, cache):
        table.extend(ids, news)
        cache.append(table, kv)
        out = cache.attention(table, q, H)
        return [out, *cache.read(table, ids, starts, cu, 19, dtype=torch.bfloat16)]

    def other(table, cache):  # a step of sequences 1 and 3, the same on both sides
        table.extend(ints([1, 3]), ints([5, 2]))
        x = torch.linspace(-1, 1, 7 * (H + 2 * KVH) * hd, device="cuda").view(7, -1)
        return [cache.attention(table, x, H)]

    for table, cache in sides:
        table.extend(ids, ints([20, 17]))
        cache.append(table, torch.linspace(-2, 2, 37 * 2 * KVH * hd, device="cuda").view(37, -1))
        other(table, cache)
    s = torch.cuda.Stream()
    sides[0][1].reserve(sides[0][0], n, H, stream=s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = step(*sides[0])
    for i in range(5):
        kv.normal_()
        q.normal_()
        torch.cuda.synchronize()
        g.replay()
        want = step(*sides[1])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        assert all(torch.equal(*(other(*side)[0] for side in sides)) for _ in range(2))
    for table, cache in sides:
        table.check()
    for name in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(*(getattr(c, name).view(torch.uint8) for _, c in sides))
