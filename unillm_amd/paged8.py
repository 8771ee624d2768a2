"""PagedKvCache8: a paged KV cache held in 8 bits, half the bytes of an f16 one.

It stands where PagedKvCache (paged.py) does: one for each layer on a PageTable, one ``attention`` a
layer and step.  A code is an int8 or an e4m3 float; 16 positions of a kv head share a power of two.
"""
from __future__ import annotations

import ctypes

import torch

from . import _capi
from .paged import PageTable, _check, _hold, _stream_ptr
from .rope import Rope, _empty

_KV8_TYPES = {torch.int8: _capi.KV8_INT8, torch.float8_e4m3fn: _capi.KV8_E4M3}
_OUT_TYPES = {torch.float32: _capi.F32, torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}
BLOCK = 16  # positions to an exponent


class PagedKvCache8:
    """One layer's pool: codes ``k`` [n_pages, n_kv_heads, page_size, head_dim] and ``v`` [n_pages,
    n_kv_heads, head_dim, page_size] (keys contiguous) of dtype int8 or float8_e4m3fn, and ``k_exp``,
    ``v_exp`` [n_pages, n_kv_heads, page_size / 16] of uint8: a code c of a block with byte b stands
    for c 2^(b - 127).  All four given, or allocated zeroed.  rope: how q and k are rotated (its
    frequencies are copied), or None: they come rotated."""

    def __init__(self, n_kv_heads: int, head_dim: int, n_pages: int, page_size: int,
                 dtype: torch.dtype = torch.int8, rope: Rope | None = None,
                 k: torch.Tensor | None = None, v: torch.Tensor | None = None,
                 k_exp: torch.Tensor | None = None, v_exp: torch.Tensor | None = None,
                 device: torch.device | str | None = None):
        self._h = None
        if dtype not in _KV8_TYPES:
            raise RuntimeError(f"PagedKvCache8: dtype {dtype} (want int8 or float8_e4m3fn)")
        if rope is not None and rope._h is None:
            raise RuntimeError("PagedKvCache8: the rope is closed")
        parts = [k, v, k_exp, v_exp]
        if any((p is None) != (k is None) for p in parts):
            raise RuntimeError("PagedKvCache8: give all of k, v, k_exp and v_exp, or none")
        exps = (n_pages, n_kv_heads, page_size // BLOCK)
        shapes = ((n_pages, n_kv_heads, page_size, head_dim), (n_pages, n_kv_heads, head_dim, page_size), exps, exps)
        types = (dtype, dtype, torch.uint8, torch.uint8)
        if k is None:
            parts = [torch.zeros(s, dtype=torch.uint8, device=device or "cuda").view(t)
                     for s, t in zip(shapes, types)]
            torch.cuda.current_stream(parts[0].device).synchronize()  # zeroed for every stream
        for name, p, s, t in zip(("k", "v", "k_exp", "v_exp"), parts, shapes, types):
            if tuple(p.shape) != s or p.dtype != t or not p.is_cuda or not p.is_contiguous():
                raise RuntimeError(f"PagedKvCache8: {name} must be a contiguous {t} device tensor of shape {list(s)}")
            if p.device != parts[0].device:
                raise RuntimeError("PagedKvCache8: buffers on different devices")
        h = ctypes.c_void_p()
        _check(_capi.lib().unillm_hip_paged_kv8_create(
            _KV8_TYPES[dtype], n_kv_heads, head_dim, n_pages, page_size, rope._h if rope is not None else None,
            *[p.data_ptr() for p in parts], ctypes.byref(h)))
        self._h = h
        self.k, self.v, self.k_exp, self.v_exp = parts
        self._lib = _capi.lib()
        self.dtype, self._device = dtype, parts[0].device
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.n_pages, self.page_size = n_pages, page_size

    def _rows(self, what: str, name: str, t: torch.Tensor, *widths: int) -> int:
        """The width of t, f32 rows of one of these on the cache's device."""
        if (t.dtype != torch.float32 or t.get_device() != self._device.index or t.dim() != 2
                or t.shape[1] not in widths or not (t.stride(1) == 1 or t.numel() == 0)):
            raise RuntimeError(f"{what}: {name} must be an f32 [n, {' or '.join(map(str, widths))}] tensor on "
                               f"{self._device} with contiguous rows")
        return t.shape[1]

    def _on(self, what: str, table: PageTable) -> None:
        if table._device != self._device:
            raise RuntimeError(f"{what}: the table is on another device")

    def _held(self, stream: torch.cuda.Stream | None, table: PageTable, *tensors: torch.Tensor) -> None:
        if stream is not None:
            _hold(stream, *tensors, self.k, self.v, self.k_exp, self.v_exp, table._mem)

    def reserve(self, table: PageTable, n_tokens: int, n_heads: int,
                stream: torch.cuda.Stream | None = None) -> None:
        """Grow the stream's workspace for attention of up to n_tokens rows, so that it can be
        captured into a HIP graph."""
        _check(_capi.lib().unillm_hip_paged_kv8_reserve(self._h, table._h, n_tokens, n_heads,
                                                        _stream_ptr(stream, self._device)))

    def append(self, table: PageTable, kv: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
        """kv [n, 2 n_kv_heads head_dim], keys then values of the plan's rows (and of padding after
        them), into the rows' slots: keys rotated, each block's exponent grown to what they need."""
        self._on("8-bit paged append", table)
        width = self._rows("8-bit paged append", "kv", kv, 2 * self.n_kv_heads * self.head_dim)
        n = kv.shape[0]
        self._held(stream, table, kv)
        _check(self._lib.unillm_hip_paged_kv8_append(self._h, table._h, kv.data_ptr(),
                                                     width if n <= 1 else kv.stride(0), n,
                                                     _stream_ptr(stream, self._device)))

    def attention(self, table: PageTable, qkv: torch.Tensor, n_heads: int, window: int = 0,
                  sinks: int = 0, out: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """qkv [n, (n_heads + 2 n_kv_heads) head_dim] (the fused projections of the plan's rows, and
        of padding after them), k and v appended first, or q alone [n, n_heads head_dim] -> out
        [n, n_heads head_dim].  window > 0: a token sees the last `window` positions, its own among
        them, and the first `sinks`.  Rows past the plan's last are left as they were."""
        what, owidth = "8-bit paged attention", n_heads * self.head_dim
        self._on(what, table)
        width = self._rows(what, "qkv", qkv, owidth + 2 * self.n_kv_heads * self.head_dim, owidth)
        n = qkv.shape[0]
        if out is None:
            out = _empty((n, owidth), torch.float32, self._device, stream)
        else:
            self._rows(what, "out", out, owidth)
            if out.shape[0] != n:
                raise RuntimeError(f"{what}: out must have {n} rows")
        self._held(stream, table, qkv, out)
        one = n <= 1  # (a single row's stride means nothing)
        _check(self._lib.unillm_hip_paged_kv8_attention(
            self._h, table._h, qkv.data_ptr(), width if one else qkv.stride(0), n, n_heads, int(width != owidth),
            window, sinks, out.data_ptr(), owidth if one else out.stride(0), _stream_ptr(stream, self._device)))
        return out

    def read(self, table: PageTable, seq_ids: torch.Tensor, starts: torch.Tensor, cu_rows: torch.Tensor,
             n_rows: int, dtype: torch.dtype = torch.float32,
             stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The cached keys (rotated, as they are held) and values of stretches of sequences: entry b,
        sequence seq_ids[b] from position starts[b] on, is rows cu_rows[b] .. cu_rows[b + 1] - 1 of k
        and v [n_rows, n_kv_heads, head_dim].  Rows past the last entry's, and of entries with
        negative ids, are not written; rows outside a sequence are NaN, and ``PageTable.check``
        raises."""
        what = "8-bit paged read"
        self._on(what, table)
        if dtype not in _OUT_TYPES:
            raise RuntimeError(f"{what}: dtype {dtype} (want float32, float16 or bfloat16)")
        B = seq_ids.numel()
        for name, t, size in (("seq_ids", seq_ids, B), ("starts", starts, B), ("cu_rows", cu_rows, B + 1)):
            if (t.dtype != torch.int32 or t.get_device() != self._device.index or t.shape != (size,)
                    or not t.is_contiguous()):
                raise RuntimeError(f"{what}: {name} must be {size} contiguous int32 on {self._device}")
        if n_rows < 0:
            raise RuntimeError(f"{what}: n_rows {n_rows}")
        shape = (n_rows, self.n_kv_heads, self.head_dim)
        k, v = _empty(shape, dtype, self._device, stream), _empty(shape, dtype, self._device, stream)
        self._held(stream, table, seq_ids, starts, cu_rows)
        _check(self._lib.unillm_hip_paged_kv8_read(
            self._h, table._h, seq_ids.data_ptr(), starts.data_ptr(), cu_rows.data_ptr(), B, n_rows,
            _OUT_TYPES[dtype], k.data_ptr(), v.data_ptr(), self.n_kv_heads * self.head_dim,
            _stream_ptr(stream, self._device)))
        return k, v

    def close(self) -> None:
        if self._h is not None and self._h.value:
            _capi.lib().unillm_hip_paged_kv8_destroy(self._h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
