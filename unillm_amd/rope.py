"""Rope: rotary positions of rows of heads.

The caches of attention.py and paged.py rotate whole heads, half-split, by themselves (the reference's
apply_rope_with_offset, crates/runtime/src/models_v2/llama.rs:827-883).  Rope is for what they do not
cover: the interleaved order (q and k of GGUF Llama files), part of a head, frequencies scaled for
long contexts; PagedKvCache8 takes one.
"""
from __future__ import annotations

import ctypes

import torch

from . import _capi
from .paged import _check, _hold, _stream_ptr

_TYPES = {torch.float32: _capi.F32, torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}
_SCALINGS = {None: 0, "linear": 1, "llama3": 2, "yarn": 3}


def _empty(shape: tuple, dtype: torch.dtype, device: torch.device, stream: torch.cuda.Stream | None) -> torch.Tensor:
    """An output's memory, that `stream` may write at once: its own.  (The current stream's without a
    context around it, which takes 2 us.)"""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        out = torch.empty(shape, dtype=dtype, device=device)
    out.record_stream(torch.cuda.current_stream(device))
    return out


class Rope:
    """Frequencies f_i = theta^(-2 i / rotary_dim) / freq_factors[i] of the pairs of a head's first
    rotary_dim dimensions: i and i + rotary_dim / 2, or interleaved 2 i and 2 i + 1.

    scaling "linear": f / factor.  "llama3", "yarn": f (r + (1 - r) / factor), r a ramp from 0 to 1
    between `low` and `high` turns over the `original` context, by the turns (llama3) or by the pair's
    number (yarn).  magnitude: of the turned pairs; None: 0.1 ln(factor) + 1 for yarn, else 1.
    """

    def __init__(self, head_dim: int, rotary_dim: int | None = None, theta: float = 10000.0,
                 interleaved: bool = False, scaling: str | None = None, factor: float = 1.0,
                 low: float = 1.0, high: float = 32.0, original: int = 0,
                 freq_factors: list[float] | None = None, magnitude: float | None = None):
        self._h = None
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if scaling not in _SCALINGS:
            raise RuntimeError(f"Rope: scaling {scaling!r} (want None, 'linear', 'llama3' or 'yarn')")
        if magnitude is not None and not magnitude:
            raise RuntimeError("Rope: a magnitude of 0")
        factors = None
        if freq_factors is not None:
            if len(freq_factors) != rotary_dim // 2:
                raise RuntimeError(f"Rope: {len(freq_factors)} freq_factors for {rotary_dim // 2} pairs")
            factors = (ctypes.c_double * len(freq_factors))(*map(float, freq_factors))
        h = ctypes.c_void_p()
        _check(_capi.lib().unillm_hip_rope_create(head_dim, rotary_dim, int(interleaved), float(theta),
                                                  _SCALINGS[scaling], float(factor), float(low), float(high),
                                                  original, factors, float(magnitude or 0.0), ctypes.byref(h)))
        self._h = h
        self._apply = _capi.lib().unillm_hip_rope_apply
        self._device = torch.device("cuda", torch.cuda.current_device())  # (the library's, made current)
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, interleaved

    def apply(self, x: torch.Tensor, positions: torch.Tensor, out: torch.Tensor | None = None,
              stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """x [n, heads, head_dim] of f32, f16 or bf16, each row's heads contiguous (a slice of fused
        projections is fine), turned at int32 positions [n] -> out, a new tensor, one given, or x
        itself (in place).  A negative position turns back, if the magnitude is 1."""

        kind = _TYPES.get(x.dtype)
        if kind is None or not self._rows(x):
            raise RuntimeError(f"Rope.apply: x must be an f32, f16 or bf16 [n, heads, {self.head_dim}] tensor on "
                               f"{self._device} with contiguous heads")
        n, heads, _ = x.shape
        if (positions.dtype != torch.int32 or positions.get_device() != self._device.index
                or positions.shape != (n,) or not positions.is_contiguous()):
            raise RuntimeError(f"Rope.apply: positions must be {n} contiguous int32 on {self._device}")
        if out is None:
            out = _empty((n, heads, self.head_dim), x.dtype, self._device, stream)
        elif out.dtype != x.dtype or out.shape != x.shape or not self._rows(out):
            raise RuntimeError("Rope.apply: out must be as x, with contiguous heads")
        if n == 0 or heads == 0:
            return out
        if stream is not None:
            _hold(stream, x, positions, out)
        width = heads * self.head_dim
        one = n == 1  # (a single row's stride means nothing)
        status = self._apply(self._h, kind, x.data_ptr(), width if one else x.stride(0), n, heads,
                             positions.data_ptr(), out.data_ptr(), width if one else out.stride(0),
                             _stream_ptr(stream, self._device))
        if status:
            _check(status)
        return out

    def _rows(self, t: torch.Tensor) -> bool:
        """Whether t is rows of contiguous heads, apart by what they take at least."""
        if t.dim() != 3 or t.get_device() != self._device.index:
            return False
        (n, heads, hd), (a, b, c) = t.shape, t.stride()
        return hd == self.head_dim and (n == 0 or heads == 0 or (
            c == 1 and (heads == 1 or b == hd) and (n == 1 or a >= heads * hd)))

    def close(self) -> None:
        if self._h is not None and self._h.value:
            _capi.lib().unillm_hip_rope_destroy(self._h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
