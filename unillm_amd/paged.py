"""PageTable and PagedKvCache: many sequences on one pool of KV-cache pages.

A serving step is one ``PageTable.extend`` (room for every request's new tokens) and then one
``PagedKvCache.attention`` a layer.  KvCache (attention.py) holds one sequence in one buffer;
here sequences share a pool of pages, and requests' lengths stay on the device, so a step can
be captured and replayed.  The reference declares such a cache without a device behind it
(crates/kv/src/gpu_memory.rs:110, 154-300).  Torch supplies device memory and the current
stream; the work runs in libunillm_hip.so.
"""
from __future__ import annotations

import ctypes

import torch

from . import _capi
from ._capi import HipError

_KV_TYPES = {torch.float32: _capi.F32, torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}


def _stream_ptr(stream: torch.cuda.Stream | None, device: torch.device) -> int:
    """The stream given, or the device's current one (read as the handle alone: 0.1 us, where
    making a Stream object takes 3 of a table call's 8)."""
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(device.index)


def _hold(stream: torch.cuda.Stream | None, *tensors: torch.Tensor | None) -> None:
    """Tensors used on a stream other than the current one are not reused before it is done."""
    if stream is None:
        return
    for t in tensors:
        if t is not None and stream != torch.cuda.current_stream(t.device):
            t.record_stream(stream)


def _check(status: int) -> None:
    if status != _capi.OK:
        raise HipError(status, _capi.last_error())


class PageTable:
    """Which page holds which positions of which sequence, and the current step's plan.

    Sequences are numbered 0 .. max_seqs - 1.  ``block_table`` [max_seqs, max_pages],
    ``seq_lens`` [max_seqs], ``free_pages`` [n_pages] and ``n_free`` [1] are its state (int32
    device tensors; copied out and back they save and restore it); ``cu_tokens``
    [max_seqs + 1], ``slots`` and ``positions`` [max_tokens] are the last extend's plan, to be
    read only.  Calls on one table are ordered by the caller (one stream, or events).
    """

    def __init__(self, max_seqs: int, max_pages: int, n_pages: int, page_size: int, max_tokens: int,
                 device: torch.device | str | None = None):
        self._h = None
        n = ctypes.c_size_t()
        _check(_capi.lib().unillm_hip_page_table_bytes(max_seqs, max_pages, n_pages, page_size,
                                                       max_tokens, ctypes.byref(n)))
        self._mem = torch.empty(n.value, dtype=torch.uint8, device=device or "cuda")
        self._device = self._mem.device
        torch.cuda.current_stream(self._device).synchronize()  # the storage is free to write
        h = ctypes.c_void_p()
        _check(_capi.lib().unillm_hip_page_table_create(max_seqs, max_pages, n_pages, page_size,
                                                        max_tokens, self._mem.data_ptr(),
                                                        ctypes.byref(h)))
        self._h = h
        self.max_seqs, self.max_pages, self.n_pages = max_seqs, max_pages, n_pages
        self.page_size, self.max_tokens = page_size, max_tokens
        at = [ctypes.c_void_p() for _ in range(7)]
        _check(_capi.lib().unillm_hip_page_table_buffers(h, *[ctypes.byref(p) for p in at]))

        def part(p, *shape):
            off, ints = p.value - self._mem.data_ptr(), 1
            for s in shape:
                ints *= s
            return self._mem[off:off + 4 * ints].view(torch.int32).view(shape)

        self.block_table = part(at[0], max_seqs, max_pages)
        self.seq_lens = part(at[1], max_seqs)
        self.free_pages = part(at[2], n_pages)
        self.n_free = part(at[3], 1)
        self.cu_tokens = part(at[4], max_seqs + 1)
        self.slots = part(at[5], max_tokens)
        self.positions = part(at[6], max_tokens)

    def _entries(self, what: str, ids: torch.Tensor, lens: torch.Tensor | None) -> int:
        for name, t in (("seq_ids", ids), ("lengths", lens)):
            if t is not None and (t.dtype != torch.int32 or t.device != self._device
                                  or t.dim() != 1 or not t.is_contiguous()):
                raise RuntimeError(f"{what}: {name} must be a contiguous int32 vector on "
                                   f"{self._device}")
        if lens is not None and lens.numel() != ids.numel():
            raise RuntimeError(f"{what}: {ids.numel()} ids and {lens.numel()} lengths")
        return ids.numel()

    def extend(self, seq_ids: torch.Tensor, new_lens: torch.Tensor,
               stream: torch.cuda.Stream | None = None) -> None:
        """Room for new_lens[b] more tokens of sequence seq_ids[b], and the step's plan.  Each
        sequence at most once; an entry with a negative id is padding.  What fails on the
        device (no free page) leaves the table as it was, and ``check`` raises it."""
        n = self._entries("extend", seq_ids, new_lens)
        _hold(stream, seq_ids, new_lens, self._mem)
        _check(_capi.lib().unillm_hip_page_table_extend(
            self._h, seq_ids.data_ptr(), new_lens.data_ptr(), n, _stream_ptr(stream, self._device)))

    def truncate(self, seq_ids: torch.Tensor, lens: torch.Tensor,
                 stream: torch.cuda.Stream | None = None) -> None:
        """Sequence seq_ids[b] keeps its first lens[b] tokens (0 <= lens[b] <= its length); the
        pages past them are free again, as before the extend that took them.  Ends the plan."""
        n = self._entries("truncate", seq_ids, lens)
        _hold(stream, seq_ids, lens, self._mem)
        _check(_capi.lib().unillm_hip_page_table_truncate(
            self._h, seq_ids.data_ptr(), lens.data_ptr(), n, _stream_ptr(stream, self._device)))

    def release(self, seq_ids: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
        """Finished requests: all their pages are free again."""
        n = self._entries("release", seq_ids, None)
        _hold(stream, seq_ids, self._mem)
        _check(_capi.lib().unillm_hip_page_table_truncate(
            self._h, seq_ids.data_ptr(), None, n, _stream_ptr(stream, self._device)))

    def clear(self, stream: torch.cuda.Stream | None = None) -> None:
        """No sequence holds a token, every page is free."""
        _hold(stream, self._mem)
        _check(_capi.lib().unillm_hip_page_table_clear(self._h, _stream_ptr(stream, self._device)))

    def check(self, stream: torch.cuda.Stream | None = None) -> None:
        """Waits for the stream and raises the first call since the last check that failed on
        the device."""
        _check(_capi.lib().unillm_hip_page_table_check(self._h, _stream_ptr(stream, self._device)))

    def close(self) -> None:
        if self._h is not None and self._h.value:
            _capi.lib().unillm_hip_page_table_destroy(self._h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedKvCache:
    """One layer's pool: ``k`` [n_pages, n_kv_heads, page_size, head_dim] and ``v`` [n_pages,
    n_kv_heads, head_dim, page_size] (keys contiguous) of dtype f32, f16 or bf16; given, or
    allocated zeroed."""

    def __init__(self, n_kv_heads: int, head_dim: int, n_pages: int, page_size: int,
                 dtype: torch.dtype = torch.float16, rope_theta: float = 10000.0,
                 k: torch.Tensor | None = None, v: torch.Tensor | None = None,
                 device: torch.device | str | None = None):
        self._h = None
        if dtype not in _KV_TYPES:
            raise RuntimeError(f"PagedKvCache: dtype {dtype} (want float32, float16 or bfloat16)")
        if (k is None) != (v is None):
            raise RuntimeError("PagedKvCache: give both k and v, or neither")
        shapes = ((n_pages, n_kv_heads, page_size, head_dim), (n_pages, n_kv_heads, head_dim, page_size))
        if k is None:
            k, v = (torch.zeros(s, dtype=dtype, device=device or "cuda") for s in shapes)
            torch.cuda.current_stream(k.device).synchronize()  # zeroed for every stream
        for name, t, s in (("k", k, shapes[0]), ("v", v, shapes[1])):
            if tuple(t.shape) != s or t.dtype != dtype or not t.is_cuda or not t.is_contiguous():
                raise RuntimeError(f"PagedKvCache: {name} must be a contiguous {dtype} device "
                                   f"tensor of shape {list(s)}")
        if k.device != v.device:
            raise RuntimeError("PagedKvCache: k and v on different devices")
        h = ctypes.c_void_p()
        _check(_capi.lib().unillm_hip_paged_kv_create(_KV_TYPES[dtype], n_kv_heads, head_dim, n_pages,
                                                      page_size, float(rope_theta), k.data_ptr(),
                                                      v.data_ptr(), ctypes.byref(h)))
        self._h = h
        self.k, self.v, self.dtype, self._device = k, v, dtype, k.device
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.n_pages, self.page_size = n_pages, page_size

    def reserve(self, table: PageTable, n_tokens: int, n_heads: int,
                stream: torch.cuda.Stream | None = None) -> None:
        """Grow the stream's workspace for calls of up to n_tokens rows, so that they can be
        captured into a HIP graph."""
        _check(_capi.lib().unillm_hip_paged_attention_reserve(self._h, table._h, n_tokens, n_heads,
                                                              _stream_ptr(stream, self._device)))

    def attention(self, table: PageTable, qkv: torch.Tensor, n_heads: int, window: int = 0,
                  sinks: int = 0, out: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """qkv [n, (n_heads + 2 n_kv_heads) head_dim] (the fused projections of the plan's rows,
        and of padding after them) -> out [n, n_heads head_dim]; k and v go to the rows' slots.
        window > 0: a token sees the last `window` positions, its own among them, and the first
        `sinks`.  Rows past the plan's last are left as they were."""
        width, owidth = (n_heads + 2 * self.n_kv_heads) * self.head_dim, n_heads * self.head_dim

        def rows(t, w):
            return (t.dtype == torch.float32 and t.device == self._device and t.dim() == 2
                    and t.shape[1] == w and (t.stride(1) == 1 or t.numel() == 0))

        if table._device != self._device:
            raise RuntimeError("paged attention: the table is on another device")
        if not rows(qkv, width):
            raise RuntimeError(f"paged attention: qkv must be an f32 [n, {width}] tensor on "
                               f"{self._device} with contiguous rows")
        n = qkv.shape[0]
        if out is None:  # (memory that `stream` may write at once: its own)
            with torch.cuda.stream(stream):
                out = torch.empty(n, owidth, dtype=torch.float32, device=self._device)
            if stream is not None:
                out.record_stream(torch.cuda.current_stream(self._device))
        elif not rows(out, owidth) or out.shape[0] != n:
            raise RuntimeError(f"paged attention: out must be an f32 [{n}, {owidth}] tensor on "
                               f"{self._device} with contiguous rows")
        _hold(stream, qkv, out, self.k, self.v, table._mem)
        one = n <= 1  # (a single row's stride means nothing)
        _check(_capi.lib().unillm_hip_paged_attention(
            self._h, table._h, qkv.data_ptr(), width if one else qkv.stride(0), n, n_heads, window,
            sinks, out.data_ptr(), owidth if one else out.stride(0), _stream_ptr(stream, self._device)))
        return out

    def close(self) -> None:
        if self._h is not None and self._h.value:
            _capi.lib().unillm_hip_paged_kv_destroy(self._h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
