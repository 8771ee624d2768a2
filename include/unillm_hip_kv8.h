/*
 * unillm_hip_kv8.h -- C ABI of rotary positions and of the paged KV cache held in 8 bits.
 * Part of unillm_hip.h (its conventions: status, errors, streams, ownership), which includes it.
 *
 * The reference rotates whole heads, half-split (crates/runtime/src/models_v2/llama.rs:827-883),
 * and holds its caches in f32 (crates/runtime/src/kv_cache.rs:28-150); GGUF files of Llama models
 * hold q and k in the interleaved order, and other families rotate part of a head or scale the
 * frequencies for long contexts.
 */
#ifndef UNILLM_HIP_KV8_H
#define UNILLM_HIP_KV8_H

#include <stddef.h>
#include <stdint.h>

#include "unillm_hip_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct unillm_rope unillm_rope;
typedef struct unillm_paged_kv8 unillm_paged_kv8;

/* Which dimensions are pair i of a head's first rotary_dim: i and i + rotary_dim / 2, or 2 i and
 * 2 i + 1. */
#define UNILLM_ROPE_HALF 0
#define UNILLM_ROPE_INTERLEAVED 1

/* How a pair's frequency f = theta^(-2 i / rotary_dim) / freq_factors[i] is scaled; a ramp r goes from
 * 0 to 1 between `low` and `high`, numbers of turns over the `original` context, 0 < low < high:
 * LINEAR f / factor; LLAMA3 f (r + (1 - r) / factor), r by the turns original f / (2 pi); YARN the
 * same with r by the pair's number, between those that make `high` and `low` turns,
 * rotary_dim log(original / (2 pi turns)) / (2 log theta), rounded down and up and cut to
 * [0, rotary_dim - 1]. */
#define UNILLM_ROPE_SCALE_NONE 0
#define UNILLM_ROPE_SCALE_LINEAR 1
#define UNILLM_ROPE_SCALE_LLAMA3 2
#define UNILLM_ROPE_SCALE_YARN 3

/* What a code of the cache is: a signed byte (-127 .. 127), or an e4m3 float (to 448). */
#define UNILLM_KV8_INT8 1
#define UNILLM_KV8_E4M3 2

/* Rotary positions of heads of head_dim (2 .. 512) elements, of which the first rotary_dim (even, 2 ..
 * head_dim) turn.  theta > 1 (finite).  factor >= 1 where a scaling takes it; low, high and original
 * (> 0) where LLAMA3 or YARN do; what a scaling does not take is not looked at.  freq_factors:
 * rotary_dim / 2 positive host values (a GGUF file's rope_freqs) that leave no frequency past 2^20,
 * or NULL: 1.  magnitude: of the turned pairs, finite; 0: the scaling's own (YARN 0.1 ln factor + 1,
 * else 1). */
int unillm_hip_rope_create(int64_t head_dim, int64_t rotary_dim, int layout, double theta, int scaling,
                           double factor, double low, double high, int64_t original,
                           const double* freq_factors, double magnitude, unillm_rope** out);
int unillm_hip_rope_destroy(unillm_rope* r);
/* n rows of n_heads heads each, of type UNILLM_QTYPE_F32, _F16 or _BF16, x_stride and out_stride
 * elements from row to row (at least n_heads head_dim, at most 2^27): each turned at its position
 * positions_dev[row], rounded once.  A negative position turns back (where the magnitude is 1).
 * Pointers aligned to their elements; faster where 16 bytes divide pointers, strides and
 * rotary_dim / 2 (interleaved: rotary_dim).  out_dev is x_dev (with the same stride: in place), or
 * the stretches of memory from the rows' first element to their last do not overlap; out_dev does not
 * overlap positions_dev. */
int unillm_hip_rope_apply(const unillm_rope* r, int type_, const void* x_dev, int64_t x_stride, int64_t n,
                          int64_t n_heads, const int32_t* positions_dev, void* out_dev,
                          int64_t out_stride, void* stream);

/* One layer's pool in 8 bits: K codes [n_pages][n_kv_heads][page_size][head_dim], V codes [n_pages]
 * [n_kv_heads][head_dim][page_size] (keys contiguous), and for each block of 16 positions and kv head a
 * power of two, k_exp and v_exp [n_pages][n_kv_heads][page_size / 16]: a code c of a block with byte
 * b stands for c 2^(b - 127) (b 0 and 255, which no append leaves, count as 1 and 254).  Shapes as unillm_hip_paged_kv_create's.  rope:
 * how q and k are rotated, of this head_dim and a rotary_dim that is a multiple of 8 (copied, need not
 * outlive the call), or NULL: not at all (they come rotated).  The four buffers are the caller's,
 * 16-byte aligned, not overlapping, and outlive the handle; all NULL: the library allocates them
 * (zeroed). */
int unillm_hip_paged_kv8_create(int kv_type, int64_t n_kv_heads, int64_t head_dim, int64_t n_pages,
                                int64_t page_size, const unillm_rope* rope, void* k_dev, void* v_dev,
                                void* k_exp_dev, void* v_exp_dev, unillm_paged_kv8** out);
int unillm_hip_paged_kv8_destroy(unillm_paged_kv8* c);
/* Its buffers, and the bytes of k (and of v) and of k_exp (and of v_exp); any out-pointer may be NULL. */
int unillm_hip_paged_kv8_buffers(const unillm_paged_kv8* c, void** k, void** v, void** k_exp,
                                 void** v_exp, size_t* bytes, size_t* exp_bytes);

/* The keys and values of the rows of t's plan into their slots.  kv_dev: n_tokens rows of 2 n_kv_heads
 * head_dim f32 (k, v projections), kv_stride floats apart (a multiple of 4; 16-byte aligned,
 * overlapping neither pool nor table).  Keys are rotated at their positions first (to f32).  Of each
 * block that gets new positions: its exponent becomes the least, at least -126, with which the new
 * values' largest magnitude is at most 127 (e4m3: 448) steps, and no less than it was if the
 * block holds positions before them; if it grows, their codes are rounded anew, each growth
 * doubling the step at least.  New values are rounded to nearest even.  So of a block whose step is s an
 * int8 value is off by at most s / 2, and by less than s where the block grew after it was written; an
 * e4m3 one by at most 2^-4 of itself or 2^-10 s, whichever is more, and where the block grew by 2^-4 of
 * itself and less than 2^-9 s.  What a block holds past the step's last position stays.  What is
 * not finite is held as the largest code (an infinity) or as 0 (NaN), counts for no exponent, and is
 * reported by unillm_hip_page_table_check.  Exponents do not shrink when positions are taken back
 * (truncate) and written again within a block.  If the table has no plan, or one of more than n_tokens
 * rows, nothing is written and the check reports it.  A call made again on the same plan and rows
 * changes nothing. */
int unillm_hip_paged_kv8_append(unillm_paged_kv8* c, const unillm_page_table* t, const float* kv_dev,
                                int64_t kv_stride, int64_t n_tokens, void* stream);

/* The attention of one layer for the rows of t's plan, as unillm_hip_paged_attention's: its shapes,
 * strides, window and sinks, and what becomes of other rows and of a table without a plan, over this
 * cache's values.  append 1: qkv_dev's rows are q, k, v, and k and v are appended first; append 0: they are q
 * alone (n_heads head_dim floats), and the rows' keys and values are there already.  f32's precision:
 * q is held to 22 bits, an element 2^-17 below its row's largest to fewer, 2^-39 of that one; weights are
 * held whole where an entry has up to 64 query rows a kv head (hd 128: 96, hd 64: 144).  A row of a longer entry may be off
 * by 2^-16 of its largest sum of |weight x value| besides, 2^-27 a key where it sees more than 2048, if keys
 * of almost no value in their blocks take almost all of its weight.  Rows of a longer entry that would be off by
 * more are done again, by a wave each that reads all its keys: behind an attention sink of no value, where the
 * other keys' weighted values come to less than 1/512 of the largest code at the sink's weight, a chunk takes tens of
 * times as long. */
int unillm_hip_paged_kv8_attention(unillm_paged_kv8* c, const unillm_page_table* t,
                                   const float* qkv_dev, int64_t qkv_stride, int64_t n_tokens,
                                   int64_t n_heads, int append, int64_t window, int64_t sinks,
                                   float* out_dev, int64_t out_stride, void* stream);
/* Grow `stream`'s workspace to what such calls of up to n_tokens rows need on this table (the queries' bytes
 * once more, and some 100 MB at most), so they can be captured into a HIP graph
 * (unillm_hip_attention_reserve).  Graphs captured on one stream share it, with each other and with
 * eager calls there: replay them on that stream.  (append and read need none.) */
int unillm_hip_paged_kv8_reserve(const unillm_paged_kv8* c, const unillm_page_table* t,
                                 int64_t n_tokens, int64_t n_heads, void* stream);

/* The cached values of stretches of sequences, as they are held (keys rotated): entry b < n_seqs is
 * sequence seq_ids_dev[b] from position starts_dev[b] on, rows cu_rows_dev[b] .. cu_rows_dev[b + 1]
 * - 1 of the outputs (cu_rows_dev[0] 0, not falling).  k_out_dev, v_out_dev: n_rows rows of n_kv_heads
 * head_dim elements of out_type (UNILLM_QTYPE_F32, _F16 or _BF16; 16-byte aligned, one of them may be
 * NULL), out_stride elements apart, a multiple of 16 bytes, overlapping nothing else of the call.
 * n_rows at most 2^26.  Rows past the last entry's are left as they were, and an entry with a
 * negative id is padding, whose rows are; a row outside its sequence, of an id past max_seqs or on a
 * page that is none is NaN, and the check reports it. */
int unillm_hip_paged_kv8_read(const unillm_paged_kv8* c, const unillm_page_table* t,
                              const int32_t* seq_ids_dev, const int32_t* starts_dev,
                              const int32_t* cu_rows_dev, int64_t n_seqs, int64_t n_rows, int out_type,
                              void* k_out_dev, void* v_out_dev, int64_t out_stride, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* UNILLM_HIP_KV8_H */
