"""The page table on the GPU against its plain Python restatement: integers, equal exactly."""
import random

import pytest

torch = pytest.importorskip("torch")

from paged_oracle import Pages  # noqa: E402
from unillm_amd import ERR_INVALID_ARG, HipError, PageTable  # noqa: E402
from unillm_amd._capi import ERR_OUT_OF_MEMORY  # noqa: E402

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def same_state(table, model):
    n = len(model.stack)
    assert table.n_free.item() == n
    assert table.free_pages[:n].tolist() == model.stack
    assert table.seq_lens.tolist() == model.lens
    assert (table.block_table.cpu().numpy() == model.block_table()).all()


def pair(max_seqs, max_pages, n_pages, page, max_tokens):
    return (PageTable(max_seqs, max_pages, n_pages, page, max_tokens),
            Pages(max_seqs, max_pages, n_pages, page))


def extend(table, model, ids, news):
    table.extend(ints(ids), ints(news))
    cu, slots, positions = model.extend(ids, news)
    assert table.cu_tokens[:len(cu)].tolist() == cu
    assert table.slots[:len(slots)].tolist() == slots
    assert table.positions[:len(slots)].tolist() == positions
    table.check()


# one entry to thousands (more than one scan of 256), one token to more than a workgroup's share
@pytest.mark.parametrize("page,max_seqs,most,steps", [
    (16, 1, 40, 6), (16, 7, 1, 40), (32, 300, 9, 6), (64, 300, 70, 4), (128, 5, 3000, 4),
    (256, 64, 300, 4), (16, 2500, 20, 3), (16, 8192, 5, 2)])
def test_random_steps_equal_the_restatement(page, max_seqs, most, steps):
    r = random.Random(page * max_seqs + most)
    max_pages = -(-most * steps // page) + 1
    n_pages = max_seqs * max_pages
    table, model = pair(max_seqs, max_pages, n_pages, page, max_seqs * most)
    for step in range(steps):
        n = r.randint(1, max_seqs)
        ids = r.sample(range(max_seqs), n)
        extend(table, model, ids, [r.randint(0, most) for _ in ids])
        same_state(table, model)
        back = r.sample(range(max_seqs), r.randint(1, max_seqs))
        lens = [r.randint(0, model.lens[i]) for i in back]
        table.truncate(ints(back), ints(lens))
        model.truncate(back, lens)
        same_state(table, model)
    gone = r.sample(range(max_seqs), (max_seqs + 1) // 2)
    table.release(ints(gone))
    model.truncate(gone, [0] * len(gone))
    same_state(table, model)
    table.check()


def test_truncate_undoes_extend():
    table, model = pair(9, 20, 150, 16, 500)
    extend(table, model, [3, 1, 8], [40, 16, 1])
    before = [t.clone() for t in (table.block_table, table.seq_lens, table.free_pages, table.n_free)]
    lens = table.seq_lens[[1, 8, 0, 3]].to(torch.int32)
    ids = ints([1, 8, 0, 3])
    table.extend(ids, ints([33, 15, 100, 9]))
    table.truncate(ids, lens)
    for t, was in zip((table.block_table, table.seq_lens, table.free_pages, table.n_free), before):
        assert torch.equal(t, was)
    table.check()


def test_padding_entries_take_nothing():
    table, model = pair(6, 4, 20, 16, 64)
    extend(table, model, [-1, 4, -7, 0, -1], [99, 17, -5, 16, 3])
    table.truncate(ints([-1, 4]), ints([50, 1]))
    model.truncate([-1, 4], [0, 1])
    same_state(table, model)
    table.check()


def test_an_empty_batch_is_an_empty_step():
    table, model = pair(2, 4, 8, 16, 8)
    extend(table, model, [], [])
    table.release(ints([]))
    same_state(table, model)


def test_rows_past_the_step_are_left():
    table, model = pair(4, 4, 16, 16, 100)
    table.slots.fill_(-77)
    table.positions.fill_(-78)
    extend(table, model, [2, 0], [3, 20])
    assert (table.slots[23:] == -77).all() and (table.positions[23:] == -78).all()


@pytest.mark.parametrize("ids,news,status,text", [
    ([0, 6], [1, 1], ERR_INVALID_ARG, "past max_seqs"),
    ([3, 0, 3], [1, 1, 0], ERR_INVALID_ARG, "twice in one batch"),
    ([0, 1], [1, -1], ERR_INVALID_ARG, "negative number"),
    ([0, 1], [2, 50], ERR_INVALID_ARG, "longer than max_pages"),
    ([0, 2, 3, 4], [64, 64, 64, 9], ERR_INVALID_ARG, "more than max_tokens"),
    # more pages than the pool has, and more than it has free
    ([0, 2, 3, 4], [64, 49, 49, 1], ERR_OUT_OF_MEMORY, "too few free pages"),
    ([0, 2, 3], [64, 64, 32], ERR_OUT_OF_MEMORY, "too few free pages"),
])
def test_a_failing_extend_changes_nothing(ids, news, status, text):
    table, model = pair(6, 4, 12, 16, 200)
    extend(table, model, [5, 1], [17, 15])
    table.extend(ints(ids), ints(news))
    same_state(table, model)
    assert not table.cu_tokens[:len(ids) + 1].any()
    with pytest.raises(HipError, match=text) as e:
        table.check()
    assert e.value.status == status
    table.check()  # reported once
    extend(table, model, [0, 5], [30, 1])
    same_state(table, model)


@pytest.mark.parametrize("ids,lens,text", [
    ([5, 1], [3, 16], "truncate outside"), ([5, 1], [-1, 3], "truncate outside"),
    ([5, 5], [3, 3], "twice"), ([6], [0], "past max_seqs")])
def test_a_failing_truncate_changes_nothing(ids, lens, text):
    table, model = pair(6, 4, 12, 16, 200)
    extend(table, model, [5, 1], [17, 15])
    table.truncate(ints(ids), ints(lens))
    same_state(table, model)
    with pytest.raises(HipError, match=text):
        table.check()


def test_sums_past_31_bits_are_refused():
    # 600 entries of 2^22 tokens: their sum wraps 2^31 before the last of them
    table, model = pair(600, 1 << 16, 300, 256, 1 << 22)
    table.extend(ints(list(range(600))), ints([1 << 22] * 600))
    with pytest.raises(HipError, match="more than max_tokens"):
        table.check()
    same_state(table, model)


def test_a_restored_state_that_is_none_is_refused():
    table, model = pair(4, 4, 12, 16, 64)
    extend(table, model, [1], [20])
    table.seq_lens[1] = 65  # past max_pages pages
    table.extend(ints([1]), ints([1]))
    with pytest.raises(HipError, match="not one that its calls leave"):
        table.check()
    table.seq_lens[1] = 20
    table.n_free[0] = 13  # more free pages than there are
    for call in (lambda: table.extend(ints([1]), ints([1])), lambda: table.release(ints([1]))):
        call()
        with pytest.raises(HipError, match="not one that its calls leave"):
            table.check()
    table.n_free[0] = 10
    table.free_pages[9] = 4000  # no such page
    table.extend(ints([1]), ints([13]))
    with pytest.raises(HipError, match="not one that its calls leave"):
        table.check()
    assert table.slots[:13].tolist()[12] == -1


def test_clear_and_restore():
    table, model = pair(5, 6, 30, 16, 64)
    extend(table, model, [4, 2], [33, 20])
    saved = [t.clone() for t in (table.block_table, table.seq_lens, table.free_pages, table.n_free)]
    table.clear()
    same_state(table, Pages(5, 6, 30, 16))
    for t, was in zip((table.block_table, table.seq_lens, table.free_pages, table.n_free), saved):
        t.copy_(was)
    extend(table, model, [2, 0], [13, 1])
    same_state(table, model)


def test_replayed_steps_read_lengths_on_the_device():
    table, model = pair(8, 32, 200, 16, 40)
    ids, news = ints([3, 0, -1, 6]), ints([1, 1, 1, 1])
    gone = ints([-1, -1])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        table.release(gone)
        table.extend(ids, news)
    r = random.Random(4)
    for step in range(12):
        i, n = r.sample(range(-1, 8), 4), [r.randint(0, 9) for _ in range(4)]
        g = r.sample(range(-1, 8), 2) if step % 3 == 2 else [-1, -1]
        ids.copy_(ints(i))
        news.copy_(ints(n))
        gone.copy_(ints(g))
        graph.replay()
        model.truncate(g, [0, 0])
        cu, slots, positions = model.extend(i, n)
        assert table.cu_tokens[:5].tolist() == cu
        assert table.slots[:len(slots)].tolist() == slots
        assert table.positions[:len(slots)].tolist() == positions
        same_state(table, model)
    table.check()


def test_arguments_are_checked():
    table = PageTable(4, 4, 12, 16, 64)
    for ids, lens in ((torch.zeros(2, dtype=torch.int32), ints([1, 1])),
                      (ints([0, 1]).long(), ints([1, 1])), (ints([0, 1]), ints([1, 1]).long()),
                      (ints([[0, 1]]), ints([1, 1])), (ints([0, 9, 1, 9])[::2], ints([1, 1])),
                      (ints([0, 1]), ints([1]))):
        for call in (table.extend, table.truncate):
            with pytest.raises(RuntimeError):
                call(ids, lens)
    with pytest.raises(HipError, match="n_seqs 5 outside"):
        table.extend(ints([0, 1, 2, 3, -1]), ints([1, 1, 1, 1, 1]))


def test_calls_on_a_side_stream():
    table, model = pair(300, 8, 900, 16, 3000)
    side = torch.cuda.Stream()
    ids, news = ints(list(range(299, -1, -1))), ints([7] * 300)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        table.extend(ids, news, stream=side)
        model.extend(list(range(299, -1, -1)), [7] * 300)
    table.check(stream=side)
    same_state(table, model)
