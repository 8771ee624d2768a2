"""Page-table calls whose ids or lengths are the table's own arrays: seq_lens may be, others are refused."""
import pytest

torch = pytest.importorskip("torch")

from paged_oracle import Pages  # noqa: E402
from test_gpu_pages import ints, pair, same_state  # noqa: E402
from unillm_amd import ERR_INVALID_ARG, HipError, PageTable  # noqa: E402

pytestmark = pytest.mark.gpu


# one entry a thread, and several: an entry's length is another entry's new one
@pytest.mark.parametrize("n", [3, 64, 257, 1000, 3000])
def test_truncate_to_other_sequences_lengths(n):
    table, model = pair(n + 1, 4, 4 * (n + 1), 16, 64 * (n + 1))
    lens = [1 + 60 * i // n for i in range(n + 1)]  # (no smaller than the one before)
    table.extend(ints(list(range(n + 1))), ints(lens))
    model.extend(list(range(n + 1)), lens)
    ids = list(range(1, n + 1))
    table.truncate(ints(ids), table.seq_lens[:n])
    model.truncate(ids, lens[:n])
    same_state(table, model)
    table.check()


@pytest.mark.parametrize("n", [5, 700])
def test_extend_by_other_sequences_lengths(n):
    table, model = pair(n, 8, 8 * n, 16, 128 * n)
    lens = [1 + i % 40 for i in range(n)]
    ids = list(range(n - 1, -1, -1))
    table.extend(ints(ids), ints(lens))
    model.extend(ids, lens)
    table.extend(ints(ids), table.seq_lens)
    model.extend(ids, list(model.lens))
    same_state(table, model)
    table.check()


def test_ids_that_are_lengths():
    # sequences 0, 1, 2 of 2, 0 and 1 tokens: a release by those numbers
    table, model = pair(3, 4, 12, 16, 64)
    table.extend(ints([0, 2]), ints([2, 1]))
    model.extend([0, 2], [2, 1])
    table.release(table.seq_lens[:2])
    model.truncate([2, 0], [0, 0])
    same_state(table, model)
    table.check()


def test_the_tables_other_arrays_are_refused():
    table = PageTable(4, 4, 12, 16, 64)
    table.extend(ints([0, 1]), ints([20, 5]))
    table.check()
    model = Pages(4, 4, 12, 16)
    model.extend([0, 1], [20, 5])
    two = ints([0, 1])
    own = (table.block_table[0, :2], table.free_pages[:2], table.cu_tokens[:2], table.slots[:2],
           table.positions[62:], table._mem[-8:].view(torch.int32),
           table._mem[table.seq_lens.data_ptr() - table._mem.data_ptr() + 12:][:8].view(torch.int32))
    for t in own:
        for call in (lambda: table.extend(two, t), lambda: table.extend(t, two),
                     lambda: table.truncate(two, t), lambda: table.truncate(t, two), lambda: table.release(t)):
            with pytest.raises(HipError, match="must not lie in the table") as e:
                call()
            assert e.value.status == ERR_INVALID_ARG
    same_state(table, model)
    other = PageTable(4, 4, 12, 16, 64)  # (another table's arrays are as good as any)
    other.extend(two, ints([3, 3]))
    table.extend(two, other.seq_lens[:2])
    model.extend([0, 1], [3, 3])
    same_state(table, model)
    table.check()
