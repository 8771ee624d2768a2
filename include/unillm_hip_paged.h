/*
 * unillm_hip_paged.h -- C ABI of the paged KV cache: many sequences on one pool of pages.
 * Part of unillm_hip.h (its conventions: status, errors, streams, ownership), which includes it.
 *
 * A page holds page_size positions of one layer's K and V.  A page table says which page
 * holds which positions of which sequence, for all layers; each layer has a pool of its own
 * (unillm_paged_kv) under the same page ids.  A serving step is one extend (room for every
 * request's new tokens, and the step's plan), then one unillm_hip_paged_attention a layer.
 * The reference declares such a cache and never backs it with device memory
 * (crates/kv/src/gpu_memory.rs:110, 154-300); its runtime holds one sequence at a time.
 *
 * The table lives in device memory and every call on it is asynchronous: requests' ids and
 * lengths are read on the device, so a step can be captured into a HIP graph and replayed
 * with other lengths.  What only the device can find (a pool that ran out) leaves the table
 * as it was and the step without a plan; unillm_hip_page_table_check reports it.  Calls on
 * one table, and the attention calls that read it, must be ordered (one stream, or events).
 */
#ifndef UNILLM_HIP_PAGED_H
#define UNILLM_HIP_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct unillm_page_table unillm_page_table;
typedef struct unillm_paged_kv unillm_paged_kv;

/* Device bytes of a table for max_seqs sequences (1 .. 8192) of up to max_pages pages each
 * (1 .. 2^22), on a pool of n_pages pages of page_size positions (16, 32, 64, 128 or 256;
 * n_pages * page_size and max_pages * page_size below 2^31), and steps of up to max_tokens
 * new tokens in all (1 .. 2^22). */
int unillm_hip_page_table_bytes(int64_t max_seqs, int64_t max_pages, int64_t n_pages,
                                int64_t page_size, int64_t max_tokens, size_t* bytes);
/* A table without tokens, every page free.  storage_dev: that many device bytes, 256-byte
 * aligned, which must outlive the handle; NULL: the library allocates.  Synchronises. */
int unillm_hip_page_table_create(int64_t max_seqs, int64_t max_pages, int64_t n_pages,
                                 int64_t page_size, int64_t max_tokens, void* storage_dev,
                                 unillm_page_table** out);
int unillm_hip_page_table_destroy(unillm_page_table* t);
/* The table's parts in device memory (any out-pointer may be NULL).  block_table[max_seqs]
 * [max_pages] page ids (-1: none), seq_lens[max_seqs], free_pages[n_pages] (a stack, its top
 * at n_free - 1) and n_free[1] are its state: copied out and back they save and restore it.
 * (Of these only seq_lens may itself be passed to extend or truncate.)
 * The last extend's plan, to be read only: cu_tokens[max_seqs + 1] (entry b's rows are
 * cu_tokens[b] .. cu_tokens[b + 1] - 1), and per row slots (page * page_size + offset) and
 * positions. */
int unillm_hip_page_table_buffers(const unillm_page_table* t, int32_t** block_table,
                                  int32_t** seq_lens, int32_t** free_pages, int32_t** n_free,
                                  int32_t** cu_tokens, int32_t** slots, int32_t** positions);
/* Forget every sequence: all pages free, no plan. */
int unillm_hip_page_table_clear(unillm_page_table* t, void* stream);
/* Room for new_lens_dev[b] >= 0 more tokens of sequence seq_ids_dev[b], b < n_seqs <=
 * max_seqs, and the step's plan: pages from the top of the free stack, entries in order, the
 * step's rows entry after entry.  A sequence may be in a batch once; an entry with a negative
 * id is padding (no tokens, its length not read).  Rows of slots and positions past the
 * step's last are left as they were.  A restored free_pages with an id that is no page among those
 * to be taken fails the call like a pool that ran out, and its rows' slots become -1; such an id in a
 * sequence's own row of block_table is the attention's to find. */
int unillm_hip_page_table_extend(unillm_page_table* t, const int32_t* seq_ids_dev,
                                 const int32_t* new_lens_dev, int64_t n_seqs, void* stream);
/* Sequence seq_ids_dev[b] keeps its first lens_dev[b] tokens (0 <= lens_dev[b] <= its length;
 * lens_dev NULL: none, the request is done); its further pages are free again, in the order
 * that undoes an extend.  The step's plan ends with it: extend before the next attention. */
int unillm_hip_page_table_truncate(unillm_page_table* t, const int32_t* seq_ids_dev,
                                   const int32_t* lens_dev, int64_t n_seqs, void* stream);
/* Waits for `stream` and reports the first extend / truncate / attention since the last check
 * that failed on the device (UNILLM_ERR_INVALID_ARG with a message; UNILLM_ERR_OUT_OF_MEMORY
 * where the pool had too few free pages).  UNILLM_ERR_UNSUPPORTED while `stream` is captured. */
int unillm_hip_page_table_check(unillm_page_table* t, void* stream);

/* One layer's pool: K [n_pages][n_kv_heads][page_size][head_dim] and V [n_pages][n_kv_heads]
 * [head_dim][page_size] (keys contiguous) of kv_type UNILLM_QTYPE_F32, _F16 or _BF16;
 * head_dim 64, 128 or 256; n_kv_heads page_size head_dim and n_pages n_kv_heads below 2^31.
 * k_dev, v_dev: such buffers of the caller's, 16-byte aligned, not overlapping,
 * which must outlive the handle; both NULL: the library allocates them (zeroed). */
int unillm_hip_paged_kv_create(int kv_type, int64_t n_kv_heads, int64_t head_dim, int64_t n_pages,
                               int64_t page_size, float rope_theta, void* k_dev, void* v_dev,
                               unillm_paged_kv** out);
int unillm_hip_paged_kv_destroy(unillm_paged_kv* c);
/* Its buffers and the bytes of each (any out-pointer may be NULL). */
int unillm_hip_paged_kv_buffers(const unillm_paged_kv* c, void** k, void** v, size_t* bytes);

/* The attention of one layer for the rows of t's plan.  qkv_dev: n_tokens rows of (n_heads +
 * 2 n_kv_heads) head_dim f32 (q, k, v projections), qkv_stride floats apart; out_dev: n_tokens
 * rows of n_heads head_dim, out_stride apart (strides multiples of 4 floats, both 16-byte
 * aligned, overlapping neither each other nor the pool, out_dev nor the table); n_tokens at most
 * t's max_tokens, n_heads a multiple of n_kv_heads below 2^16, n_tokens n_heads below 2^30.  Each row's q and k are rotated at its position p (half-split RoPE; the angles
 * p theta^(-2 i / hd) are formed in f64, where unillm_hip_attention_decode takes them in f32), k
 * and v rounded once to the pool's type into the row's slot, and out = softmax(q k^T / sqrt(hd)) v
 * over the positions j <= p of its sequence, at f32's precision whatever the pool's type.  (f16:
 * q is held to 22 bits, an element 2^-17 below its row's largest to fewer, 2^-39 of that one; a
 * chunk's row may be off by 2^-16 of its largest output besides, 2^-27 a key where it sees more
 * than 2048, if keys of almost no value take almost all of its weight.)  window > 0: only j > p - window, and j < sinks (sliding window with
 * attention sinks; the reference's masks, crates/runtime/src/tensor_core.rs:1761-1781); window 0:
 * all, sinks 0.  What masked keys and values hold does not matter.
 * Rows past the step's last are left as they were; if the table has no plan, or one of more
 * than n_tokens rows, nothing is appended, all n_tokens rows become NaN, and the check reports
 * it.  A call may be made again on the same plan (each layer does). */
int unillm_hip_paged_attention(unillm_paged_kv* c, const unillm_page_table* t,
                               const float* qkv_dev, int64_t qkv_stride, int64_t n_tokens,
                               int64_t n_heads, int64_t window, int64_t sinks, float* out_dev,
                               int64_t out_stride, void* stream);
/* Grow `stream`'s workspace to what such calls of up to n_tokens rows need on this table, so
 * they can be captured into a HIP graph (as unillm_hip_attention_reserve). */
int unillm_hip_paged_attention_reserve(const unillm_paged_kv* c, const unillm_page_table* t,
                                       int64_t n_tokens, int64_t n_heads, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* UNILLM_HIP_PAGED_H */
