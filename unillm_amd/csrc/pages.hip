// pages.hip -- block tables, slot maps and positions of a serving step, built on the GPU from
// the requests' lengths (the page table of include/unillm_hip.h).
//
// State, all int32 in device memory: table[max_seqs][max_pages] (page of each block of
// page_size positions, -1 where none), lens[max_seqs], the stack of free pages (its top at
// n_free - 1) and the step's plan.  With ps the page size, held = ceil(len / ps):
//   extend: entry b of the batch (sequence id_b, n_b new tokens) needs ceil((len + n_b) / ps)
//     - held pages; with off the exclusive prefix sum of the needs, its page i is
//     free[n_free - 1 - (off_b + i)].  With cu the prefix sum of the n_b, token t of entry b
//     lies at row cu_b + t, position len + t, slot page * ps + position % ps.
//   truncate: the pages past the new length go back as free[n_free + F - 1 - (off_b + i)],
//     F of them in all, so a truncate to the old lengths undoes an extend exactly.
// Everything a call checks (ids in range and distinct, lengths, room, free pages and whether what it
// takes of them are pages) it checks before it writes, and a failing call leaves the state as it
// was: the step it leaves is empty and the first error is kept for unillm_hip_page_table_check.
// (The ids in sequences' own rows of a restored table are the attention's to check: a truncate puts
// them on the stack as they are, and no extend takes one that is no page.)
//
// One launch a call.  Every workgroup reads all entries and forms both prefix sums itself, in
// LDS, and then serves its share of the step's tokens (or freed pages): a thread finds its
// first token's entry by bisection in LDS and walks from there.  Nothing that a workgroup reads
// is written by another (new pages and tokens go where no entry's old ones are), but the
// lengths, n_free and the plan's header must wait until every workgroup has read them: the
// last one to arrive at a ticket writes those.  (A scan kernel and a fill kernel would be two
// launches of a step that is bound by launch latency.)
// Bound by latency: a few KB for a decode step.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "internal.hpp"

namespace unillm {
namespace {

constexpr int kThreads = 256;

// a + b of counts that are at most `cap`, cut off just past it: what a call has no room for stays
// so, and no sum wraps.
__device__ __forceinline__ int2 add_capped(int2 a, int2 b, int2 cap) {
    return make_int2(min(a.x + b.x, cap.x + 1), min(a.y + b.y, cap.y + 1));
}

// Sums of two counts over the workgroup's threads before this one, and all (tmp: 2 ints a wave).
__device__ __forceinline__ int2 block_scan2(int2 v, int2 cap, int2* tmp, int2* all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int2 s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int2 up = make_int2(__shfl_up(s.x, o, 64), __shfl_up(s.y, o, 64));
        if (lane >= o) s = add_capped(s, up, cap);
    }
    if (lane == 63) tmp[w] = s;
    const int2 left = make_int2(__shfl_up(s.x, 1, 64), __shfl_up(s.y, 1, 64));
    __syncthreads();
    int2 base = make_int2(0, 0), sum = base;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
        if (i < w) base = add_capped(base, tmp[i], cap);
        sum = add_capped(sum, tmp[i], cap);
    }
    *all = sum;
    return lane > 0 ? add_capped(base, left, cap) : base;
}

// The last workgroup of the launch to call this gets true (and clears the ticket).
__device__ __forceinline__ bool last_to_arrive(int* ticket) {
    __shared__ int last;
    __syncthreads();  // the workgroup's reads of the state are done
    if (threadIdx.x == 0) {
        const int n = (int)gridDim.x;
        last = n == 1 || __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        if (last && n > 1) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last != 0;
}

// Greatest b with key[b] <= x < key[b + 1] (key ascending, key[0] <= x < key[n]).
__device__ __forceinline__ int bisect(const int* key, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (key[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Both calls' first part: each entry's id (-1: a padding entry) and old length into LDS, the
// checks, and the prefix sums ca[0 .. B], cb[0 .. B] of tokens and pages.  Returns an error code
// (full: that of more pages than the pool has).
struct Entries {
    int* id;
    int* len;
    int* ca;
    int* cb;
};

// A thread takes neighbouring entries, 8 at a time with their loads in flight together, and the
// threads' sums are scanned once.
template <class F>
__device__ int scan_entries(const Entries& e, int B, const PageTable& t, const int* ids, const int* lens,
                            F&& counts, int* seen, int2* tmp, int* error, int full) {
    const int words = (t.max_seqs + 31) / 32;
    for (int i = threadIdx.x; i < words; i += kThreads) seen[i] = 0;
    if (threadIdx.x == 0) *error = 0;
    const int each = (B + kThreads - 1) / kThreads, b0 = (int)threadIdx.x * each, b1 = min(B, b0 + each);
    __syncthreads();
    const int top = t.max_pages * t.page_size;
    const int2 cap = make_int2(t.max_tokens, t.n_pages);
    int2 sum = make_int2(0, 0);
    int worst = 0;
    for (int c = b0; c < b1; c += 8) {
        int id[8], n[8], len[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            id[i] = c + i < b1 ? ids[c + i] : -1;
            n[i] = c + i < b1 && lens ? lens[c + i] : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) len[i] = id[i] >= 0 && id[i] < t.max_seqs ? t.lens[id[i]] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c + i >= b1) break;
            int2 v = make_int2(0, 0);
            int bad = 0;
            if (id[i] >= t.max_seqs) bad = kPagesBadId;
            else if (id[i] >= 0) {
                if (atomicOr(&seen[id[i] / 32], 1 << (id[i] % 32)) >> (id[i] % 32) & 1) bad = kPagesBadId;
                if (len[i] < 0 || len[i] > top) bad = kPagesBadState;
                else if (!bad) bad = counts(n[i], len[i], v);
            }
            worst = max(worst, bad);
            if (bad) v = make_int2(0, 0);
            e.id[c + i] = id[i] < t.max_seqs ? max(id[i], -1) : -1;
            e.len[c + i] = len[i];
            e.ca[c + i] = v.x;
            e.cb[c + i] = v.y;
            sum = add_capped(sum, v, cap);
        }
    }
    if (worst) atomicMax(error, worst);
    int2 all;
    int2 at = block_scan2(sum, cap, tmp, &all);
    for (int b = b0; b < b1; ++b) {  // counts to sums before
        const int2 v = make_int2(e.ca[b], e.cb[b]);
        e.ca[b] = at.x;
        e.cb[b] = at.y;
        at = add_capped(at, v, cap);
    }
    if (threadIdx.x == 0) {
        e.ca[B] = all.x;
        e.cb[B] = all.y;
    }
    __syncthreads();
    const int err = *error;
    return err ? err : all.x > t.max_tokens ? kPagesStepFull : all.y > t.n_pages ? full : 0;
}

// Page ids from the stack's top: four a load (past n_free within the part's 256 bytes), each thread its
// group of four of every 1024 downwards.  The first is requested before the entries are read.  (The look
// at them takes 0.4 us of 5.0 for 8 entries, 1.5 of 13.2 where 2048 entries take 4200 pages; four
// groups a thread requested ahead, 1.1 and 2.3.)
struct Popped {
    int4 first;
    int at;
    __device__ static int4 load(const PageTable& t, int i) {
        return i >= 0 ? *reinterpret_cast<const int4*>(t.free_pages + i) : make_int4(0, 0, 0, 0);
    }
    __device__ Popped(const PageTable& t, int n_free) {
        at = n_free > 0 && n_free <= t.n_pages ? ((n_free - 1) & ~3) - 4 * (int)threadIdx.x : -4;
        first = load(t, at);
    }
    // whether one of free_pages[lo .. n_free - 1] that this thread reads is no page
    __device__ bool bad(const PageTable& t, int lo, int n_free) const {
        auto none = [&](int4 x, int i) {
            const int id[4] = {x.x, x.y, x.z, x.w};
            bool any = false;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                any |= i + j >= lo && i + j < n_free && (unsigned)id[j] >= (unsigned)t.n_pages;
            return any;
        };
        bool any = none(first, at);
        for (int i = at - 4 * kThreads; i + 3 >= lo; i -= 16 * kThreads) {  // (four loads in flight)
            int4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = load(t, i - 4 * kThreads * k);
#pragma unroll
            for (int k = 0; k < 4; ++k) any |= none(x[k], i - 4 * kThreads * k);
        }
        return any;
    }
};

// dynamic LDS: id[B] | len[B] | ca[B + 1] | cb[B + 1] | seen[ceil(max_seqs / 32)]
__device__ __forceinline__ Entries entries_in(int* sm, int B, int** seen) {
    Entries e;
    e.id = sm;
    e.len = e.id + B;
    e.ca = e.len + B;
    e.cb = e.ca + B + 1;
    *seen = e.cb + B + 1;
    return e;
}

size_t entries_bytes(const PageTable& t, int64_t B) {
    return (size_t)(4 * B + 2 + (t.max_seqs + 31) / 32) * sizeof(int);
}

__global__ __launch_bounds__(kThreads) void extend_kernel(PageTable t, const int* ids, const int* news, int B) {
    extern __shared__ int sm[];
    __shared__ int2 tmp[kThreads / 64];
    __shared__ int error, no_page;
    int* seen;
    const Entries e = entries_in(sm, B, &seen);
    const int ps = t.page_size, shift = t.page_shift;
    const int n_free = t.counts[kPagesFree];
    if (threadIdx.x == 0) no_page = 0;
    Popped popped(t, n_free);
    int err = scan_entries(e, B, t, ids, news, [&](int n, int len, int2& v) {
        if (n < 0) return kPagesBadLength;
        if (n > t.max_pages * ps - len) return kPagesSeqFull;
        if (n > t.max_tokens) return kPagesStepFull;
        v.x = n;
        v.y = ((len + n + ps - 1) >> shift) - ((len + ps - 1) >> shift);
        return 0;
    }, seen, tmp, &error, kPagesNoPages);
    const int total = e.ca[B], pages = e.cb[B];
    if (!err && (n_free < 0 || n_free > t.n_pages)) err = kPagesBadState;
    if (!err && pages > n_free) err = kPagesNoPages;
    if (!err && pages > 0) {
        if (popped.bad(t, n_free - pages, n_free)) no_page = 1;
        __syncthreads();
        if (no_page) err = kPagesBadState;
    }
    if (no_page)  // (no slots for its rows)
        for (int r = (int)blockIdx.x * kThreads + (int)threadIdx.x; r < total; r += (int)gridDim.x * kThreads)
            t.slots[r] = -1;
    if (!err) {
        // four rows a thread at a time: a row's entry is the one before's or a later one
        const int stride = (int)gridDim.x * kThreads * 4;
        for (int r0 = ((int)blockIdx.x * kThreads + (int)threadIdx.x) * 4; r0 < total; r0 += stride) {
            int b = bisect(e.ca, B, r0);
            int4 at, page;
            int* pos = &at.x;
            int* pg = &page.x;
            bool fresh[4];
            int* entry[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = min(r0 + i, total - 1);
                while (r >= e.ca[b + 1]) ++b;
                const int len = e.len[b];
                pos[i] = len + r - e.ca[b];
                const int col = pos[i] >> shift, held = (len + ps - 1) >> shift;
                entry[i] = t.table + (int64_t)e.id[b] * t.max_pages + col;
                fresh[i] = col >= held;
                pg[i] = *(fresh[i] ? t.free_pages + (n_free - 1 - (e.cb[b] + col - held)) : entry[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (fresh[i] && (pos[i] & (ps - 1)) == 0) *entry[i] = pg[i];  // (the page's first token)
                // (a sequence's own page that is none: no slot, and the attention reports it)
                pg[i] = (unsigned)pg[i] < (unsigned)t.n_pages ? pg[i] * ps + (pos[i] & (ps - 1)) : -1;
            }
            if (r0 + 4 <= total) {
                *reinterpret_cast<int4*>(t.slots + r0) = page;
                *reinterpret_cast<int4*>(t.positions + r0) = at;
            } else {
                for (int i = 0; r0 + i < total; ++i) t.slots[r0 + i] = pg[i], t.positions[r0 + i] = pos[i];
            }
        }
    }
    if (!last_to_arrive(&t.counts[kPagesTicket])) return;
    for (int b = threadIdx.x; b <= B; b += kThreads) t.cu[b] = err ? 0 : e.ca[b];
    for (int b = threadIdx.x; b < B; b += kThreads) {
        const int id = e.id[b], n = e.ca[b + 1] - e.ca[b];
        t.step_ids[b] = id;
        t.step_lens[b] = err || id < 0 ? 0 : e.len[b] + n;
        if (!err && id >= 0) t.lens[id] = e.len[b] + n;
    }
    if (threadIdx.x == 0) {
        if (!err) t.counts[kPagesFree] = n_free - pages;
        else atomicCAS(&t.counts[kPagesError], 0, err);
        t.counts[kPagesStep] = err ? 0 : 1;
        t.counts[kPagesTokens] = err ? 0 : total;
        t.counts[kPagesEntries] = B;
    }
}

__global__ __launch_bounds__(kThreads) void truncate_kernel(PageTable t, const int* ids, const int* news,
                                                            int B) {
    extern __shared__ int sm[];
    __shared__ int2 tmp[kThreads / 64];
    __shared__ int error;
    int* seen;
    const Entries e = entries_in(sm, B, &seen);
    const int ps = t.page_size, shift = t.page_shift;
    const int n_free = t.counts[kPagesFree];
    int err = scan_entries(e, B, t, ids, news, [&](int n, int len, int2& v) {
        if (n < 0 || n > len) return kPagesBadLength;
        v.x = 0;
        v.y = ((len + ps - 1) >> shift) - ((n + ps - 1) >> shift);
        return 0;
    }, seen, tmp, &error, kPagesBadState);
    const int freed = e.cb[B];
    if (!err && (n_free < 0 || freed > t.n_pages - n_free)) err = kPagesBadState;
    if (!err) {
        const int stride = (int)gridDim.x * kThreads;
        for (int f = (int)blockIdx.x * kThreads + (int)threadIdx.x; f < freed; f += stride) {
            const int b = bisect(e.cb, B, f);
            const int held = (e.len[b] + ps - 1) >> shift;
            int* entry = t.table + (int64_t)e.id[b] * t.max_pages + held - (e.cb[b + 1] - f);
            t.free_pages[n_free + freed - 1 - f] = *entry;
            *entry = -1;
        }
    }
    if (!last_to_arrive(&t.counts[kPagesTicket])) return;
    // (the new lengths may lie among the table's own: all are read before one is written)
    for (int b = threadIdx.x; b < B; b += kThreads) e.len[b] = news ? news[b] : 0;
    __syncthreads();
    if (!err)
        for (int b = threadIdx.x; b < B; b += kThreads)
            if (e.id[b] >= 0) t.lens[e.id[b]] = e.len[b];
    if (threadIdx.x == 0) {
        if (!err) t.counts[kPagesFree] = n_free + freed;
        else atomicCAS(&t.counts[kPagesError], 0, err);
        t.counts[kPagesStep] = 0;  // the plan's slots may be free again
        t.counts[kPagesTokens] = 0;
    }
}

// Every sequence empty, every page free (page 0 on top), no step.
__global__ __launch_bounds__(kThreads) void clear_kernel(PageTable t) {
    const int64_t i0 = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t stride = (int64_t)gridDim.x * kThreads;
    for (int64_t i = i0; i < (int64_t)t.max_seqs * t.max_pages; i += stride) t.table[i] = -1;
    for (int64_t i = i0; i < t.n_pages; i += stride) t.free_pages[i] = (int)(t.n_pages - 1 - i);
    for (int64_t i = i0; i <= t.max_seqs; i += stride) {
        t.cu[i] = 0;
        if (i < t.max_seqs) t.lens[i] = 0, t.step_ids[i] = -1, t.step_lens[i] = 0;
    }
    for (int64_t i = i0; i < t.max_tokens; i += stride) t.slots[i] = -1, t.positions[i] = 0;
    if (i0 < kPagesCounts) t.counts[i0] = i0 == kPagesFree ? t.n_pages : 0;
}

unsigned groups(int64_t work, int64_t each) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((work + each - 1) / each,
                                                           device_info().cu_count));
}

hipError_t launch_entries(void (*kernel)(PageTable, const int*, const int*, int), const PageTable& t,
                          const int32_t* ids, const int32_t* lens, int64_t B, unsigned grid,
                          hipStream_t s) {
    const size_t lds = entries_bytes(t, B);
    kernel<<<grid, kThreads, lds, s>>>(t, ids, lens, (int)B);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_pages_clear(const PageTable& t, hipStream_t s) {
    const int64_t most = std::max<int64_t>((int64_t)t.max_seqs * t.max_pages,
                                           std::max<int64_t>(t.n_pages, t.max_tokens));
    clear_kernel<<<groups(most, 4 * kThreads), kThreads, 0, s>>>(t);
    return hipGetLastError();
}

// A workgroup serves 1024 rows at a time; the grid is for the most rows a step can hold.
hipError_t launch_pages_extend(const PageTable& t, const int32_t* ids, const int32_t* news,
                               int64_t B, hipStream_t s) {
    static const bool attr = hipFuncSetAttribute((const void*)extend_kernel,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 159 * 1024) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    return launch_entries(extend_kernel, t, ids, news, B, groups(t.max_tokens, 4 * kThreads), s);
}

// How many pages a call frees only the device knows: 256 a workgroup of at most what the
// batch's entries can hold.
hipError_t launch_pages_truncate(const PageTable& t, const int32_t* ids, const int32_t* lens,
                                 int64_t B, hipStream_t s) {
    static const bool attr = hipFuncSetAttribute((const void*)truncate_kernel,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 159 * 1024) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    const int64_t most = std::min<int64_t>(B * t.max_pages, t.n_pages);
    return launch_entries(truncate_kernel, t, ids, lens, B, groups(most, 4 * kThreads), s);
}

}  // namespace unillm
