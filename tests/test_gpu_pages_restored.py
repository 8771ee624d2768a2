"""A page table whose state the caller has restored, with page ids that are no pages: an extend that
would take one is refused, and changes nothing but its rows' slots; a sequence's own pages are the
attention's to check."""
import pytest

torch = pytest.importorskip("torch")

from unillm_amd import ERR_INVALID_ARG, HipError, PagedKvCache, PageTable  # noqa: E402

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def state(t):
    return [x.clone() for x in (t.block_table, t.seq_lens, t.free_pages, t.n_free)]


def refused(table, ids, news, rows):
    before = state(table)
    table.slots.fill_(7)
    table.extend(ints(ids), ints(news))
    with pytest.raises(HipError, match="not one that its calls leave") as e:
        table.check()
    assert e.value.status == ERR_INVALID_ARG
    for x, was in zip(state(table), before):
        assert torch.equal(x, was)
    assert not table.cu_tokens[:len(ids) + 1].any()
    assert (table.slots[:rows] == -1).all() and (table.slots[rows:] == 7).all()


# the bad id: first, in the midst, last of the pages to be popped; more of them than a workgroup's threads
@pytest.mark.parametrize("page", [-1, 4000, 1 << 30, -(1 << 31)])
@pytest.mark.parametrize("pages,at", [(1, 0), (3, 0), (3, 1), (3, 2), (700, 0), (700, 300), (700, 699)])
def test_a_free_page_that_is_none(page, pages, at):
    table = PageTable(5, 800, 800, 16, 16 * 800)
    table.extend(ints([1]), ints([20]))
    n = table.n_free.item()
    good = table.free_pages[n - 1 - at].item()
    table.free_pages[n - 1 - at] = page
    refused(table, [3, 1], [16 * pages - 1, 12], 16 * pages + 11)  # (1's tokens: the rest of its page)
    # with no page the id is not reached: it stays where it is
    table.extend(ints([1]), ints([12]))
    table.check()
    table.free_pages[n - 1 - at] = good
    table.extend(ints([3, 1]), ints([16 * pages - 1, 0]))
    table.check()
    assert table.n_free.item() == n - pages and table.seq_lens.tolist() == [0, 32, 0, 16 * pages - 1, 0]


@pytest.mark.parametrize("new", [1, 40])
def test_a_sequences_own_page_that_is_none(new):
    # checked by the attention, as those before it are: the step stands, its tokens on that page have no
    # slots, their rows are NaN and the check reports it once
    table, cache = PageTable(3, 8, 16, 16, 100), PagedKvCache(1, 64, 16, 16, torch.float32)
    qkv = torch.randn(2 * new, 3 * 64, generator=torch.Generator().manual_seed(0)).cuda()
    table.extend(ints([1, 2]), ints([20, 5]))
    good = table.block_table[1, 1].item()
    for page in (-1, 16, 1 << 30):
        table.block_table[1, 1] = page
        table.extend(ints([1, 2]), ints([new, new]))
        table.check()
        last = min(new, 12)
        assert (table.slots[:last] == -1).all() and (table.slots[last:2 * new] >= 0).all()
        out = cache.attention(table, qkv, 1)
        with pytest.raises(HipError, match="not one that its calls leave"):
            table.check()
        assert torch.isnan(out[:new]).all() and torch.isfinite(out[new:]).all()
        table.truncate(ints([2, 1]), ints([5, 20]))
        table.check()
    table.block_table[1, 1] = good
    table.extend(ints([1, 2]), ints([new, new]))
    assert torch.isfinite(cache.attention(table, qkv, 1)).all()
    table.check()


def test_a_refused_step_appends_nothing_and_may_be_retried():
    table, cache = PageTable(2, 4, 8, 16, 64), PagedKvCache(1, 64, 8, 16, torch.float32)
    qkv = torch.randn(20, 3 * 64, generator=torch.Generator().manual_seed(0)).cuda()
    table.extend(ints([1]), ints([20]))
    want = cache.attention(table, qkv, 1).clone()
    k = cache.k.clone()
    table.release(ints([1]))
    table.free_pages[6] = 8
    table.extend(ints([1]), ints([20]))
    out = cache.attention(table, qkv, 1)
    with pytest.raises(HipError, match="not one that its calls leave"):
        table.check()
    assert torch.isnan(out).all() and torch.equal(cache.k, k)
    table.free_pages[6] = 1
    table.extend(ints([1]), ints([20]))
    assert torch.equal(cache.attention(table, qkv, 1), want)
    table.check()
