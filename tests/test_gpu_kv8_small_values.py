"""PagedKvCache8.attention over values of very different powers of two.  Values times 2^p have the same codes and
exponents p higher, so outputs must be the same bits, p higher, wherever f32 holds both; and they keep the bounds of
test_gpu_kv8_attention.py."""
import pytest
import torch

from test_gpu_kv8_attention import KINDS, close, expect, ints, make

pytestmark = pytest.mark.gpu

CTX = 700


def attended(kind, hd, n, power, gap):
    """n rows behind CTX keys whose values are of size 2^power; gap: key 7 draws so many nats and its value is 0.
    -> (out, (64-bit out, bound))"""
    table, cache, gen = make(kind, 1, hd, 16, [CTX], max_tokens=2000)
    table.truncate(ints([0]), ints([0]))
    table.extend(ints([0]), ints([CTX]))
    kv = torch.randn(CTX, 2 * hd, device="cuda", generator=gen)
    new = torch.randn(n, 3 * hd, device="cuda", generator=gen)
    kv[:, hd:] *= 2.0 ** power
    new[:, 2 * hd:] *= 2.0 ** power
    if gap:
        kv[:, 0] = 0.0
        kv[7] = 0.0
        kv[7, 0] = 8.0
        new[:, 0] = gap * hd ** 0.5 / 8.0
        new[:, 1:hd] *= 0.05
        new[:, hd] = 0.0
    cache.append(table, kv)
    table.extend(ints([0]), ints([n]))
    out = cache.attention(table, new, 1)
    table.check()
    return out, expect(cache, table, new[:, :hd], 1, [(0, n)])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 20, 200])
@pytest.mark.parametrize("gap", [0.0, 9.0, 13.0, 16.0])
def test_a_power_of_two_of_the_values(kind, hd, n, gap):
    """The same bits, where also a quotient's remainder, 2^-24 of an output of 2^-30 of the values, is a normal number."""
    out, want = attended(kind, hd, n, 0, gap)
    close(out, *want)
    for power in (-70, 30):
        got, want = attended(kind, hd, n, power, gap)
        close(got, *want)
        assert torch.equal(torch.ldexp(got, torch.tensor(-power, device="cuda")), out), power


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 20, 200])
@pytest.mark.parametrize("gap", [0.0, 9.0, 16.0])
@pytest.mark.parametrize("power", [-115, -100, 100, 115])
def test_values_near_the_ends(kind, hd, n, power, gap):
    close(*(lambda out, want: (out, *want))(*attended(kind, hd, n, power, gap)))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gap", [11.0, 13.0])
@pytest.mark.parametrize("power", [-100, -105])
def test_rows_of_small_values_are_done_again_as_others(kind, hd, gap, power):
    """A chunk's rows beside a sink (wide tiles): those that are done again in f32 at the one size are at the other, by
    the same steps.  What comes below f32's normal numbers, at most each of the 900 products and sums, is off by 2^-150,
    2^-140 in all; a quotient's last bit may turn besides."""
    out, _ = attended(kind, hd, 200, 0, gap)
    got, want = attended(kind, hd, 200, power, gap)
    close(got, *want)
    off = (torch.ldexp(got.double(), torch.tensor(-power, device="cuda")) - out).abs()
    assert (off <= 2.0 ** (-140 - power) + 2.0 ** -23 * out.abs()).all(), float((off / out.abs().amax()).max())
