"""PagedKvCache8.attention that appends first: what it writes, against the 64-bit oracle, bit for bit.

(append by itself is another kernel: test_gpu_kv8_write.py.)
"""
import numpy as np
import pytest
import torch

from kv8_oracle import frequencies
from test_gpu_kv8_write import KINDS, SIZES, Run, ints, same, steps
from unillm_amd import Rope

pytestmark = pytest.mark.gpu


class Fused(Run):
    """Run whose steps are one attention call on q, k and v; the rows' k and v are what steps() makes."""

    def __init__(self, *args, group=2, **more):
        super().__init__(*args, **more)
        self.heads_q = group * self.heads

    def step(self, ids, news, kv, again=False):
        cache, run = self.cache, self

        class Appends:  # (takes the append's place within Run.step)
            def append(self, table, kv):
                q = torch.randn(len(kv), run.heads_q * run.hd, device="cuda")
                cache.attention(table, torch.cat([q, kv], 1), run.heads_q)

        self.cache = Appends()
        try:
            super().step(ids, news, kv, again)
        finally:
            self.cache = cache


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("heads,hd,page,group", [(1, 64, 16, 1), (3, 128, 32, 4), (2, 256, 64, 7), (5, 64, 256, 2)])
def test_steps_bit_for_bit(kind, heads, hd, page, group):
    steps(Fused(kind, heads, hd, page, group=group), 1, SIZES)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd,rot,interleaved,scaling", [(64, 64, False, None), (128, 128, True, None), (128, 40, False, "llama3"),
                                                        (256, 64, True, "yarn"), (256, 256, False, "linear")])
def test_rotated_keys(kind, hd, rot, interleaved, scaling):
    more = dict(factor=8.0, low=1.0, high=4.0, original=64) if scaling else {}
    rope = Rope(hd, rotary_dim=rot, interleaved=interleaved, scaling=scaling, **more)
    m = 0.1 * np.log(8.0) + 1 if scaling == "yarn" else 1.0
    run = Fused(kind, 2, hd, 32, rope=rope, freq=frequencies(rot, scaling=scaling, **more), interleaved=interleaved, magnitude=m)
    steps(run, 2, SIZES, spread=2.0)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("heads,hd,rotated", [(9, 64, True), (18, 64, False), (34, 64, True), (33, 128, False), (32, 256, True)])
def test_decoding_rows_among_chunks(kind, heads, hd, rotated):
    """Workgroups of 2, 4, 8 and 16 rows, several heads to one, runs of one row and of several."""
    rope = Rope(hd, interleaved=True) if rotated else None
    run = Fused(kind, heads, hd, 16, n_pages=300, max_seqs=90, rope=rope, freq=frequencies(hd) if rotated else None,
                interleaved=True, max_tokens=700, group=1)
    small = [(i, 1 + (i * 7 % 11 == 0) * 2) for i in range(80)]
    first = [(i, 1 + i % 5) for i in range(80)] + [(80, 200)]
    mixed = small[:30] + [(80, 170)] + small[30:] + [(81, 250)]
    steps(run, 11, [([i for i, _ in e], [n for _, n in e]) for e in (first, mixed, mixed)], spread=2.0)


@pytest.mark.parametrize("kind", list(KINDS))
def test_a_prompt(kind):
    """Rows past 512, whose queries are turned 16 rows a workgroup, behind the plan and before the writes."""
    run = Fused(kind, 4, 64, 16, n_pages=200, max_tokens=1500, rope=Rope(64), freq=frequencies(64), group=8)
    steps(run, 3, [([0, 1], [900, 301]), ([1, 2, 0], [1, 700, 33])], spread=2.0)


def test_rows_inside_wider_ones_and_padding():
    run = Fused("int8", 2, 64, 16, rope=Rope(64), freq=frequencies(64))
    table, cache = run.table, run.cache
    wide = torch.randn(9, 1000, device="cuda")
    table.extend(ints([3, -1, 0]), ints([4, 2, 1]))
    cache.attention(table, wide[:, 20:20 + 8 * 64], 4)  # (four of the rows are padding)
    kv = wide[:5, 20 + 4 * 64:20 + 8 * 64].contiguous()
    other = Run("int8", 2, 64, 16, rope=Rope(64), freq=frequencies(64))
    other.step([3, 0], [4, 1], kv)
    assert torch.equal(other.table.slots[:5], table.slots[:5])
    same(cache, other.pool)
