"""PagedKvCache8.attention where a step has many rows, heads or entries, against its formula in 64 bits (the bounds of
test_gpu_kv8_attention.py): queries turned 4 and 16 rows and several heads a workgroup, plans of more than 256 tiles."""
import pytest
import torch

from kv8_oracle import frequencies
from test_gpu_kv8_attention import KINDS, close, expect, make, step
from unillm_amd import Rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("KVH,G,entries", [
    (3, 7, [(0, 1), (2, 380), (1, 60), (3, 59)]),   # 500 rows of 21 heads: 4 rows and 2 heads a workgroup
    (9, 7, [(2, 1), (0, 510), (3, 1), (1, 88)]),    # 600 of 63: 16 and 2, and one of one head
    (2, 1, [(1, 513), (0, 300)])])                  # 16 rows, one head
def test_many_rows_and_heads(kind, KVH, G, entries):
    table, cache, gen = make(kind, KVH, 64, 32, [40, 17, 5, 100], max_tokens=900, rope=Rope(64, interleaved=True))
    q, out = step(table, cache, gen, KVH * G, entries, KVH != 2)
    close(out, *expect(cache, table, q, KVH * G, entries, frequencies(64), True))


@pytest.mark.parametrize("kind", list(KINDS))
def test_more_than_256_narrow_tiles(kind):
    """310 entries of a few rows, one of them on 9000 keys, which is dealt out in pieces."""
    lens = [1 + i * 7 % 40 for i in range(310)]
    lens[17] = 9000
    table, cache, gen = make(kind, 1, 64, 16, lens, max_tokens=9000, rope=Rope(64), room=64)
    entries = [(i * 37 % 310, 1 + i % 3) for i in range(310)]
    q, out = step(table, cache, gen, 2, entries, True)
    close(out, *expect(cache, table, q, 2, entries, frequencies(64)))


@pytest.mark.parametrize("kind", list(KINDS))
def test_more_than_256_wide_tiles(kind):
    """260 entries of 65 query rows of one kv head."""
    lens = [1 + i * 5 % 23 for i in range(260)]
    table, cache, gen = make(kind, 1, 256, 16, lens, max_tokens=1500, rope=Rope(256), room=64)
    entries = [(i * 7 % 260, 5) for i in range(260)]
    q, out = step(table, cache, gen, 13, entries, True)
    close(out, *expect(cache, table, q, 13, entries, frequencies(256)))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,G", [(64, 145), (64, 300), (128, 97), (256, 130)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 5)])
def test_many_heads_on_one(kind, hd, G, window, sinks):
    """Single tokens of so many heads on one kv head that they are wide tiles' rows, beside a few of several tokens."""
    table, cache, gen = make(kind, 1, hd, 32, [300, 1, 40], rope=Rope(hd, rotary_dim=hd // 2))
    entries = [(1, 1), (0, 2), (2, 1)]
    q, out = step(table, cache, gen, G, entries, True, window=window, sinks=sinks)
    close(out, *expect(cache, table, q, G, entries, frequencies(hd // 2), window=window, sinks=sinks))
