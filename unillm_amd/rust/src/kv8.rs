//! Rotary positions and the paged KV cache held in 8 bits (`include/unillm_hip_kv8.h`).
//!
//! * [`Rope`] turns rows of heads: half-split or interleaved, part of a head, scaled frequencies.
//! * [`PagedKvCache8`] stands where [`PagedKvCache`](crate::PagedKvCache) does, on a
//!   [`PageTable`], in half an f16 pool's bytes.

use std::ffi::{c_int, c_void};
use std::ptr;

use crate::{check, to_i64, PageTable, Result};

/// The C ABI (`include/unillm_hip_kv8.h`).
#[allow(non_camel_case_types)]
pub mod sys {
    use std::ffi::{c_int, c_void};

    use crate::sys::unillm_page_table;

    /// Opaque rotary positions.
    #[repr(C)]
    pub struct unillm_rope {
        _private: [u8; 0],
    }
    /// Opaque pool of one layer's KV pages in 8 bits.
    #[repr(C)]
    pub struct unillm_paged_kv8 {
        _private: [u8; 0],
    }

    pub const UNILLM_ROPE_HALF: c_int = 0;
    pub const UNILLM_ROPE_INTERLEAVED: c_int = 1;
    pub const UNILLM_ROPE_SCALE_NONE: c_int = 0;
    pub const UNILLM_ROPE_SCALE_LINEAR: c_int = 1;
    pub const UNILLM_ROPE_SCALE_LLAMA3: c_int = 2;
    pub const UNILLM_ROPE_SCALE_YARN: c_int = 3;
    pub const UNILLM_KV8_INT8: c_int = 1;
    pub const UNILLM_KV8_E4M3: c_int = 2;

    extern "C" {
        pub fn unillm_hip_rope_create(head_dim: i64, rotary_dim: i64, layout: c_int, theta: f64,
                                      scaling: c_int, factor: f64, low: f64, high: f64,
                                      original: i64, freq_factors: *const f64, magnitude: f64,
                                      out: *mut *mut unillm_rope) -> c_int;
        pub fn unillm_hip_rope_destroy(r: *mut unillm_rope) -> c_int;
        pub fn unillm_hip_rope_apply(r: *const unillm_rope, type_: c_int, x_dev: *const c_void,
                                     x_stride: i64, n: i64, n_heads: i64,
                                     positions_dev: *const i32, out_dev: *mut c_void,
                                     out_stride: i64, stream: *mut c_void) -> c_int;
        pub fn unillm_hip_paged_kv8_create(kv_type: c_int, n_kv_heads: i64, head_dim: i64,
                                           n_pages: i64, page_size: i64, rope: *const unillm_rope,
                                           k_dev: *mut c_void, v_dev: *mut c_void,
                                           k_exp_dev: *mut c_void, v_exp_dev: *mut c_void,
                                           out: *mut *mut unillm_paged_kv8) -> c_int;
        pub fn unillm_hip_paged_kv8_destroy(c: *mut unillm_paged_kv8) -> c_int;
        pub fn unillm_hip_paged_kv8_buffers(c: *const unillm_paged_kv8, k: *mut *mut c_void,
                                            v: *mut *mut c_void, k_exp: *mut *mut c_void,
                                            v_exp: *mut *mut c_void, bytes: *mut usize,
                                            exp_bytes: *mut usize) -> c_int;
        pub fn unillm_hip_paged_kv8_append(c: *mut unillm_paged_kv8, t: *const unillm_page_table,
                                           kv_dev: *const f32, kv_stride: i64, n_tokens: i64,
                                           stream: *mut c_void) -> c_int;
        pub fn unillm_hip_paged_kv8_attention(c: *mut unillm_paged_kv8, t: *const unillm_page_table,
                                              qkv_dev: *const f32, qkv_stride: i64, n_tokens: i64,
                                              n_heads: i64, append: c_int, window: i64, sinks: i64,
                                              out_dev: *mut f32, out_stride: i64,
                                              stream: *mut c_void) -> c_int;
        pub fn unillm_hip_paged_kv8_reserve(c: *const unillm_paged_kv8, t: *const unillm_page_table,
                                            n_tokens: i64, n_heads: i64, stream: *mut c_void) -> c_int;
        pub fn unillm_hip_paged_kv8_read(c: *const unillm_paged_kv8, t: *const unillm_page_table,
                                         seq_ids_dev: *const i32, starts_dev: *const i32,
                                         cu_rows_dev: *const i32, n_seqs: i64, n_rows: i64,
                                         out_type: c_int, k_out_dev: *mut c_void,
                                         v_out_dev: *mut c_void, out_stride: i64,
                                         stream: *mut c_void) -> c_int;
    }
}

/// How a [`Rope`]'s frequencies are scaled; `low` and `high` in turns over the `original` context.
#[derive(Debug, Clone, Copy, PartialEq)]
pub enum Scaling {
    None,
    Linear { factor: f64 },
    Llama3 { factor: f64, low: f64, high: f64, original: usize },
    Yarn { factor: f64, low: f64, high: f64, original: usize },
}

/// Rotary positions of heads of head_dim elements, the first rotary_dim of which turn.
pub struct Rope {
    r: *mut sys::unillm_rope,
    rotary_dim: usize,
}

unsafe impl Send for Rope {}

impl Rope {
    /// freq_factors: empty, or rotary_dim / 2 divisors of the frequencies (a GGUF file's `rope_freqs`).
    /// magnitude 0: the scaling's own.
    pub fn new(head_dim: usize, rotary_dim: usize, interleaved: bool, theta: f64, scaling: Scaling,
               freq_factors: &[f64], magnitude: f64) -> Result<Self> {
        let (kind, factor, low, high, original) = match scaling {
            Scaling::None => (sys::UNILLM_ROPE_SCALE_NONE, 1.0, 0.0, 0.0, 0),
            Scaling::Linear { factor } => (sys::UNILLM_ROPE_SCALE_LINEAR, factor, 0.0, 0.0, 0),
            Scaling::Llama3 { factor, low, high, original } => {
                (sys::UNILLM_ROPE_SCALE_LLAMA3, factor, low, high, original)
            }
            Scaling::Yarn { factor, low, high, original } => {
                (sys::UNILLM_ROPE_SCALE_YARN, factor, low, high, original)
            }
        };
        if !freq_factors.is_empty() && freq_factors.len() != rotary_dim / 2 {
            return Err(crate::invalid(format!("rope: {} freq_factors for rotary_dim {rotary_dim}",
                                              freq_factors.len())));
        }
        let factors = if freq_factors.is_empty() { ptr::null() } else { freq_factors.as_ptr() };
        let layout = if interleaved { sys::UNILLM_ROPE_INTERLEAVED } else { sys::UNILLM_ROPE_HALF };
        let mut r = ptr::null_mut();
        check(unsafe {
            sys::unillm_hip_rope_create(to_i64(head_dim, "head_dim")?, to_i64(rotary_dim, "rotary_dim")?,
                                        layout, theta, kind, factor, low, high,
                                        to_i64(original, "original")?, factors, magnitude, &mut r)
        })?;
        Ok(Self { r, rotary_dim })
    }

    pub fn rotary_dim(&self) -> usize {
        self.rotary_dim
    }

    /// n rows of n_heads heads of `qtype` (`crate::sys::UNILLM_QTYPE_F32`, `_F16` or `_BF16`) turned at
    /// `positions`, `_stride` elements apart; `out` may be `x` (in place, the same stride).
    ///
    /// # Safety
    /// `x`, `positions` (n i32) and `out` point to device memory of those sizes; `stream` is a HIP
    /// stream of the library's device, or null.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn apply_raw(&self, qtype: c_int, x: *const c_void, x_stride: usize, n: usize,
                            n_heads: usize, positions: *const i32, out: *mut c_void,
                            out_stride: usize, stream: *mut c_void) -> Result<()> {
        check(sys::unillm_hip_rope_apply(self.r, qtype, x, to_i64(x_stride, "x_stride")?, to_i64(n, "n")?,
                                         to_i64(n_heads, "n_heads")?, positions, out,
                                         to_i64(out_stride, "out_stride")?, stream))
    }
}

impl Drop for Rope {
    fn drop(&mut self) {
        unsafe {
            sys::unillm_hip_rope_destroy(self.r);
        }
    }
}

/// One layer's pool of KV pages in 8 bits, `sys::UNILLM_KV8_INT8` or `_E4M3`.
pub struct PagedKvCache8 {
    c: *mut sys::unillm_paged_kv8,
}

unsafe impl Send for PagedKvCache8 {}

impl PagedKvCache8 {
    /// rope: how q and k are rotated (copied), or None: they come rotated.
    pub fn new(kv_type: c_int, n_kv_heads: usize, head_dim: usize, n_pages: usize,
               page_size: usize, rope: Option<&Rope>) -> Result<Self> {
        let mut c = ptr::null_mut();
        let rope = rope.map_or(ptr::null(), |r| r.r as *const _);
        check(unsafe {
            sys::unillm_hip_paged_kv8_create(kv_type, to_i64(n_kv_heads, "n_kv_heads")?,
                                             to_i64(head_dim, "head_dim")?,
                                             to_i64(n_pages, "n_pages")?,
                                             to_i64(page_size, "page_size")?, rope, ptr::null_mut(),
                                             ptr::null_mut(), ptr::null_mut(), ptr::null_mut(), &mut c)
        })?;
        Ok(Self { c })
    }

    /// Grows `stream`'s workspace for attention of up to n_tokens rows (before a graph capture).
    pub fn reserve(&self, table: &PageTable, n_tokens: usize, n_heads: usize,
                   stream: *mut c_void) -> Result<()> {
        check(unsafe {
            sys::unillm_hip_paged_kv8_reserve(self.c, table.as_ptr(), to_i64(n_tokens, "n_tokens")?,
                                              to_i64(n_heads, "n_heads")?, stream)
        })
    }

    /// Keys and values of the plan's rows, kv [n_tokens, 2 n_kv_heads head_dim], into their slots.
    ///
    /// # Safety
    /// `kv` points to device memory of that size, 16-byte aligned; `stream` is a HIP stream of the
    /// library's device, or null.
    pub unsafe fn append_raw(&mut self, table: &PageTable, kv: *const f32, kv_stride: usize,
                             n_tokens: usize, stream: *mut c_void) -> Result<()> {
        check(sys::unillm_hip_paged_kv8_append(self.c, table.as_ptr(), kv, to_i64(kv_stride, "kv_stride")?,
                                               to_i64(n_tokens, "n_tokens")?, stream))
    }

    /// Attention of the plan's rows: append: qkv [n_tokens, (n_heads + 2 n_kv_heads) head_dim], k and v
    /// appended first; else q alone [n_tokens, n_heads head_dim] -> out [n_tokens, n_heads head_dim].
    ///
    /// # Safety
    /// `qkv` and `out` point to device memory of those sizes, 16-byte aligned, not overlapping;
    /// `stream` is a HIP stream of the library's device, or null.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn attention_raw(&mut self, table: &PageTable, qkv: *const f32, qkv_stride: usize,
                                n_tokens: usize, n_heads: usize, append: bool, window: usize,
                                sinks: usize, out: *mut f32, out_stride: usize,
                                stream: *mut c_void) -> Result<()> {
        check(sys::unillm_hip_paged_kv8_attention(self.c, table.as_ptr(), qkv,
                                                  to_i64(qkv_stride, "qkv_stride")?,
                                                  to_i64(n_tokens, "n_tokens")?,
                                                  to_i64(n_heads, "n_heads")?, append as c_int,
                                                  to_i64(window, "window")?, to_i64(sinks, "sinks")?, out,
                                                  to_i64(out_stride, "out_stride")?, stream))
    }

    /// Cached keys and values: sequence `seq_ids[b]` from position `starts[b]` on into rows `cu_rows[b]` ..
    /// `cu_rows[b + 1]` - 1 of the outputs (either may be null), of `qtype`.
    ///
    /// # Safety
    /// `seq_ids` and `starts` point to n_seqs i32, `cu_rows` to n_seqs + 1, `k_out` and `v_out` to n_rows
    /// rows of out_stride elements, 16-byte aligned, in device memory; `stream` is a HIP stream of
    /// the library's device, or null.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn read_raw(&self, table: &PageTable, seq_ids: *const i32, starts: *const i32,
                           cu_rows: *const i32, n_seqs: usize, n_rows: usize, qtype: c_int,
                           k_out: *mut c_void, v_out: *mut c_void, out_stride: usize,
                           stream: *mut c_void) -> Result<()> {
        check(sys::unillm_hip_paged_kv8_read(self.c, table.as_ptr(), seq_ids, starts, cu_rows,
                                             to_i64(n_seqs, "n_seqs")?, to_i64(n_rows, "n_rows")?, qtype,
                                             k_out, v_out, to_i64(out_stride, "out_stride")?, stream))
    }
}

impl Drop for PagedKvCache8 {
    fn drop(&mut self) {
        unsafe {
            sys::unillm_hip_paged_kv8_destroy(self.c);
        }
    }
}
