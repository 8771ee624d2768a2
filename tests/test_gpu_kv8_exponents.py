"""PagedKvCache8 on exponents that only a caller's pool holds, bytes 0 and 255 (which count as 1 and 254) and 254:
an append behind held positions against the 64-bit oracle, bit for bit."""
import numpy as np
import pytest
import torch

from kv8_oracle import e4m3_value
from test_gpu_kv8_write import KINDS, Run, ints, same

pytestmark = pytest.mark.gpu

HELD = 5  # positions of a block before the append


def held_codes(run, page, byte):
    """Random codes and this exponent into a page's first block, in the cache and the oracle's pool."""
    gen = np.random.default_rng(byte)
    for t, exps, codes, ours, block in ((run.cache.k, run.cache.k_exp, run.pool.k, run.pool.ke, np.s_[:, :16]),
                                        (run.cache.v, run.cache.v_exp, run.pool.v, run.pool.ve, np.s_[:, :, :16])):
        shape = codes[page][block].shape
        if run.pool.kind == "int8":
            raw = gen.integers(-127, 128, shape).astype(np.int8).view(np.uint8)
            codes[page][block] = raw.view(np.int8)
        else:
            raw = (gen.integers(0, 127, shape) + 128 * gen.integers(0, 2, shape)).astype(np.uint8)
            codes[page][block] = e4m3_value(raw)
        t.view(torch.uint8)[page][block] = torch.from_numpy(raw).cuda()
        exps[page, :, 0] = byte
        ours[page, :, 0] = min(max(byte, 1), 254) - 127


@pytest.mark.parametrize("kind,top", [("int8", 127.0), ("e4m3", 448.0)])
@pytest.mark.parametrize("byte,e", [(0, -126), (0, -125), (0, -122), (1, -126), (1, -125), (253, 126), (254, 127), (255, 127),
                                    (254, -3), (255, -126)])
@pytest.mark.parametrize("seqs,n", [(1, 1), (6, 1), (1, 3), (3, 11)])
@pytest.mark.parametrize("hd", [64, 256])
def test_append_behind_held_codes(kind, top, byte, e, seqs, n, hd):
    """New values that need the step 2^e, or for large ones f32's largest, behind codes of this byte."""
    run = Run(kind, 2, hd, 32, n_pages=2 * seqs, max_seqs=seqs)
    ids = list(range(seqs))
    run.table.extend(ints(ids), ints([HELD] * seqs))
    for page in run.table.block_table[:, 0].tolist():
        held_codes(run, page, byte)
    gen = torch.Generator(device="cuda").manual_seed(e)
    # (ties among them: multiples of half a step; above 2^126 f32 ends at 2^128)
    kv = torch.randint(-255, 256, (seqs * n, 4 * hd), device="cuda", generator=gen).float() / 256
    kv = kv * 2.0 ** 64 * 2.0 ** 63 * 2 if e >= 126 else kv * (top * 2.0 ** e)
    kv = kv.clamp(-3.4e38, 3.4e38)
    kv[:, ::4] = torch.randint(-3, 4, kv[:, ::4].shape, device="cuda", generator=gen).float() * (0.5 * 2.0 ** min(e, 126))
    if e < 126:
        kv[:, ::hd] = top * 2.0 ** e
    run.step(ids, [n] * seqs, kv, again=True)
    run.table.check()
    same(run.cache, run.pool)
