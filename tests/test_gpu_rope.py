"""Rope.apply against 64-bit rotations: layouts, parts of heads, scalings, types, strides, positions.

Tolerance: a row's own rounding (half a step, relative to the value) after products that are off by
2^-50 of the pair's size at most.  The angle p f is formed in f64: off by 2^-52 of itself, which at
position 2^20 is 2^-32 turns of a radian; with the frequency's own error, taken as 2^-50 p absolutely.
"""
import numpy as np
import pytest
import torch

from kv8_oracle import frequencies, rotate
from unillm_amd import Rope

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SCALED = {None: {}, "linear": dict(factor=4.0), "llama3": dict(factor=8.0, low=1.0, high=4.0, original=8192),
          "yarn": dict(factor=16.0, low=1.0, high=32.0, original=4096)}


def check(got, x, positions, freq, interleaved, magnitude=1.0):
    rot = 2 * len(freq)
    host = x.double().cpu().numpy()
    want = rotate(host, positions, freq, interleaved, magnitude)
    size = np.zeros_like(host)
    a, b = ((slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot)))
    pair = np.hypot(host[..., a], host[..., b]) * abs(magnitude)
    size[..., a], size[..., b] = pair, pair
    p = np.abs(np.asarray(positions, np.float64))[:, None, None]
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[x.dtype]
    # (16-bit rows round through f32: its half step besides)
    off = EPS[x.dtype] * np.abs(want) + size * (2.0 ** -50 * (p + 4) + (2.0 ** -24 if x.dtype != torch.float32 else 0)) + tiny
    y = got.double().cpu().numpy()
    assert (np.abs(y - want) <= off).all(), np.abs(y - want).max()
    assert np.array_equal(y[..., rot:], host[..., rot:])  # what does not turn stays, bit for bit


@pytest.mark.parametrize("dtype", list(EPS))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,hd,rot", [(1, 1, 2, 2), (1, 64, 128, 128), (3, 5, 64, 64), (7, 3, 80, 20),
                                            (33, 2, 96, 94), (5, 9, 256, 2), (300, 1, 512, 512), (4100, 2, 64, 32),
                                            (2, 300, 10, 6), (9001, 1, 128, 128)])
def test_shapes_and_types(dtype, interleaved, n, heads, hd, rot):
    torch.manual_seed(n + hd)
    x = torch.randn(n, heads, hd, device="cuda").to(dtype)
    pos = torch.randint(0, 1 << 20, (n,), device="cuda", dtype=torch.int32)
    rope = Rope(hd, rotary_dim=rot, interleaved=interleaved)
    before = x.clone()
    out = rope.apply(x, pos)
    assert torch.equal(x, before)
    check(out, x, pos.tolist(), frequencies(rot), interleaved)


@pytest.mark.parametrize("dtype", list(EPS))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,hd,rot", [(1, 1, 3, 2), (5, 3, 5, 4), (40, 2, 511, 2), (9, 7, 65, 64)])
def test_heads_of_odd_sizes(dtype, interleaved, n, heads, hd, rot):
    torch.manual_seed(hd)
    x = torch.randn(n, heads, hd, device="cuda").to(dtype)
    pos = torch.randint(0, 1 << 20, (n,), device="cuda", dtype=torch.int32)
    rope = Rope(hd, rotary_dim=rot, interleaved=interleaved)
    hold = torch.full((n, heads * hd + 3), 7.0, device="cuda", dtype=dtype)
    check(rope.apply(x, pos, out=hold[:, 1:-2].unflatten(1, (heads, hd))), x, pos.tolist(), frequencies(rot), interleaved)
    assert (hold[:, [0, -2, -1]] == 7).all()
    assert torch.equal(rope.apply(x, pos, out=x), hold[:, 1:-2].unflatten(1, (heads, hd)))


@pytest.mark.parametrize("scaling", list(SCALED))
@pytest.mark.parametrize("interleaved", [False, True])
def test_scalings(scaling, interleaved):
    x = torch.randn(50, 4, 128, device="cuda")
    pos = torch.arange(0, 50 * 2500, 2500, device="cuda", dtype=torch.int32)
    rope = Rope(128, rotary_dim=96, theta=500000.0, interleaved=interleaved, scaling=scaling, **SCALED[scaling])
    f = frequencies(96, 500000.0, scaling, **SCALED[scaling])
    check(rope.apply(x, pos), x, pos.tolist(), f, interleaved,
          0.1 * np.log(16.0) + 1 if scaling == "yarn" else 1.0)


def test_freq_factors_and_magnitude():
    factors = [1.0 + 0.25 * i for i in range(32)]
    x = torch.randn(6, 2, 64, device="cuda")
    pos = torch.tensor([0, 1, 2, 100, 9999, 65535], device="cuda", dtype=torch.int32)
    rope = Rope(64, freq_factors=factors, magnitude=1.5)
    check(rope.apply(x, pos), x, pos.tolist(), frequencies(64, factors=factors), False, 1.5)


@pytest.mark.parametrize("dtype", list(EPS))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pad,lead", [(0, 0), (1, 0), (1, 1), (2, 4), (8, 8), (24, 3)])
def test_rows_inside_wider_ones(dtype, interleaved, pad, lead):
    """Slices of fused projections, at any alignment, into slices of others."""
    n, heads, hd = 40, 3, 64
    wide = torch.randn(n * (heads * hd + pad) + lead, device="cuda").to(dtype)
    x = wide[lead:].view(n, heads * hd + pad)[:, :heads * hd].unflatten(1, (heads, hd))
    hold = torch.full((n, heads * hd + 2 * pad + 6), 7.0, device="cuda", dtype=dtype)
    out = hold[:, pad:pad + heads * hd].unflatten(1, (heads, hd))
    pos = torch.randint(0, 5000, (n,), device="cuda", dtype=torch.int32)
    rope = Rope(hd, rotary_dim=48, interleaved=interleaved)
    assert rope.apply(x, pos, out=out).data_ptr() == out.data_ptr()
    check(out, x, pos.tolist(), frequencies(48), interleaved)
    rest = torch.ones(hold.shape[1], dtype=torch.bool)
    rest[pad:pad + heads * hd] = False
    assert (hold[:, rest.cuda()] == 7).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_back(interleaved):
    x = torch.randn(100, 4, 128, device="cuda")
    pos = torch.randint(0, 100000, (100,), device="cuda", dtype=torch.int32)
    rope = Rope(128, rotary_dim=64, interleaved=interleaved)
    y = x.clone()
    assert rope.apply(y, pos, out=y) is y
    assert torch.equal(y, rope.apply(x, pos))
    rope.apply(y, -pos, out=y)  # turned back
    # each turn rounds once, half a step of a value no larger than its pair
    pair = torch.maximum(x.abs(), x.abs().amax(-1, keepdim=True))
    assert ((y - x).abs() <= 2 * 2.0 ** -24 * 1.5 * pair).all()


def test_positions_at_the_ends():
    x = torch.randn(4, 1, 64, device="cuda")
    pos = torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)
    y = Rope(64).apply(x, pos)
    assert torch.equal(y[0], x[0])
    check(y, x, pos.tolist(), frequencies(64), False)


def test_non_finite_values_stay_in_their_pairs():
    x = torch.randn(3, 2, 64, device="cuda")
    x[1, 0, 5], x[2, 1, 40] = float("nan"), float("inf")
    y = Rope(64).apply(x, torch.tensor([1, 2, 3], device="cuda", dtype=torch.int32))
    bad = ~torch.isfinite(y)
    assert bad.sum() == 4 and bad[1, 0, 5] and bad[1, 0, 37] and bad[2, 1, 40] and bad[2, 1, 8]


def test_empty_calls():
    rope = Rope(64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert rope.apply(torch.empty(0, 4, 64, device="cuda"), none).shape == (0, 4, 64)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert rope.apply(torch.empty(1, 0, 64, device="cuda"), one).shape == (1, 0, 64)


def test_captured_and_on_another_stream():
    x = torch.randn(64, 8, 128, device="cuda").bfloat16()
    pos = torch.arange(64, device="cuda", dtype=torch.int32)
    out = torch.empty_like(x)
    rope = Rope(128, interleaved=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rope.apply(x, pos, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            rope.apply(x, pos, out=out)
    torch.cuda.synchronize()
    for shift in (0, 700, 70000):
        pos.copy_(torch.arange(64, device="cuda", dtype=torch.int32) + shift)
        x.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rope.apply(x, pos))
        s.wait_stream(torch.cuda.current_stream())
        aside = rope.apply(x, pos, stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(out, aside)


def test_refusals():
    rope = Rope(64)
    x = torch.randn(4, 2, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (x.double(), x.cpu(), x[:, :, :32], x.transpose(0, 1), x[0], x[:1].expand(4, 2, 64)):
        with pytest.raises(RuntimeError):
            rope.apply(bad, pos[:bad.shape[0]])
    for bad in (pos.long(), pos.cpu(), pos[:3], torch.zeros(8, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(RuntimeError, match="positions"):
            rope.apply(x, bad)
    for bad in (x.half(), x[:3], torch.empty(4, 64, 2, device="cuda").transpose(1, 2)):
        with pytest.raises(RuntimeError, match="out"):
            rope.apply(x, pos, out=bad)
    flat = torch.randn(5, 2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        rope.apply(flat[:4], pos, out=flat[1:])
    with pytest.raises(RuntimeError, match="positions"):
        rope.apply(x, x.view(-1)[:4].view(torch.int32), out=x)
