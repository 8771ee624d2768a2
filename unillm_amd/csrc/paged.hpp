// paged.hpp -- what the attention kernels over paged KV caches share (paged.hip, paged8.hip): how a
// call's work is dealt out on the device, its pieces joined, and operands split into parts.
#pragma once

#include <hip/hip_runtime.h>

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "internal.hpp"
#include "split.hpp"

namespace unillm {
namespace {

typedef _Float16 f16_t;
struct bf16_t {
    uint16_t bits;
};

constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(f16_t v) { return (float)v; }
__device__ __forceinline__ float widen(bf16_t v) { return __uint_as_float((uint32_t)v.bits << 16); }
// An f32 value to the pool's type, to nearest even.  (Opaque first: the compiler would fold the
// conversion of a narrowed f64 into one from f64, and a key that is a tie in f32 would round
// otherwise than the f32 key does.)
template <class T>
__device__ __forceinline__ T narrow(float v) {
    asm volatile("" : "+v"(v));
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, f16_t>) return (f16_t)v;
    else return bf16_t{(uint16_t)(pack_bf16(v, 0.0f) & 0xFFFF)};
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// One piece of a call's work: the visits v0 .. v0 + nv - 1 of a tile of `rows` query rows
// (row r of an entry is head r % G of its token r / G, for each kv head).  Of a tile dealt out
// in S > 1 pieces this is piece s; its partial sums go to rows base + (g S + s) rows + r.
// An entry of up to kNarrowRows rows has narrow tiles, a longer one wide ones, each kind with
// a list and a kernel of its own.
struct Item {
    int first, ctx, len, id;  // of the entry: its first step row, tokens before the step and with it, sequence
    int row0, rows, v0, nv, base, s, S, pad;
};
// A tile dealt out, for the merge.
struct Split {
    int first, row0, rows, base, S, pad[3];
};

// What the kernels of a call share.
struct Call {
    const float* qkv;
    float* out;
    int64_t qstride, ostride;
    int n, H, KVH, G;
    int window, sinks;
    float2* turn;  // [n][hd / 2] cos, sin of each row's angles
    float2* ms;    // partial rows: maximum (log2), sum of the weights
    float* po;     // [hd] unnormalized sums
    int* redo_count;  // rows and heads (row H + head) whose products of parts came out non-finite
    int* redo;
    struct Kind {
        int tile_rows;  // most query rows of a tile
        int places;     // workgroups of the kind that the device holds
        int target;     // most pieces to deal the kind's work out in, over all kv heads, but for
                        // tiles' remainders; at least places
        int least;      // visits of the smallest piece
        int overhead;   // of a piece, in visits
        int row0;       // its first partial row
        int* head;      // [0] items, [1] splits
        Item* items;
        Split* splits;
    } kind[2];
};

constexpr int kNarrow = 0, kWide = 1;
// Most query rows of an entry (a kv head) for narrow tiles.  (8 entries on 4000 keys, 8 kv heads of 128,
// f16 / bf16 / f32, us: of 48 rows narrow 66 / 66 / 114, wide 84 / 123 / 159; of 80 rows 97 / 97 / 178
// and 82 / 125 / 162; of 112 rows 133 / 133 / 250 and 83 / 125 / 166.  One number for all types and
// widths: bf16 entries of 65 to about 100 rows are up to a fourth slower for it at hd 128, a tenth at
// hd 64 (68 rows: 64, narrow 56); at hd 256 wide is right from there on for each, 87 and 137.)
constexpr int kNarrowRows = 64;
constexpr int kTileRows = 16;    // query rows of a narrow tile
constexpr int kUnit = 32;        // keys of a narrow tile's visit
// Wide tiles: groups of four waves of 32 rows each (what the registers hold: two groups, one at
// hd 256), and keys of a visit.
template <class T, int D>
constexpr int kGroups = D < 256 ? 2 : 1;
template <class T, int D>
constexpr int kWideUnit = D == 64 || (sizeof(T) == 2 && D == 128) ? 64 : 32;

// Whether the step can run: a plan, of at most the call's rows.
__device__ __forceinline__ bool step_fits(const PageTable& t, int n) {
    return t.counts[kPagesStep] == 1 && t.counts[kPagesTokens] <= n;
}

// The call's outputs of a step that cannot run, a share of them a workgroup; the table's
// first error is kept.
__device__ void fail_call(const PageTable& t, const Call& a, int D, int group, int groups) {
    const int width = a.H * D;
    for (int64_t i = (int64_t)group * blockDim.x + threadIdx.x; i < (int64_t)a.n * width;
         i += (int64_t)groups * blockDim.x)
        a.out[i / width * a.ostride + i % width] = __builtin_nanf("");
    if (group == 0 && threadIdx.x == 0)
        atomicCAS(&t.counts[kPagesError], 0, t.counts[kPagesStep] == 1 ? kPagesRows : kPagesNoPlan);
}

// The blocks of U keys that rows at positions pmin .. pmax see between them, numbered as
// visits: those of the first `sinks` keys before the window's, then the window's.
template <int U>
struct Visits {
    int sink_blocks, first, count;
    __device__ Visits(int pmin, int pmax, int window, int sinks) {
        first = window > 0 ? max(0, pmin - window + 1) / U : 0;
        sink_blocks = window > 0 ? min((sinks + U - 1) / U, first) : 0;
        count = sink_blocks + pmax / U - first + 1;
    }
    __device__ int key(int v) const { return (v < sink_blocks ? v : first + v - sink_blocks) * U; }
};

// Inclusive sums of two values over 256 threads, and all (tmp: [4]).
__device__ __forceinline__ ulong2 block_scan(ulong2 v, ulong2* tmp, ulong2* all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_up(v.x, o, 64), y = __shfl_up(v.y, o, 64);
        if (lane >= o) v.x += x, v.y += y;
    }
    if (lane == 63) tmp[w] = v;
    __syncthreads();
    ulong2 base = {0, 0}, sum = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const ulong2 x = tmp[i];
        if (i < w) base.x += x.x, base.y += x.y;
        sum.x += x.x;
        sum.y += x.y;
    }
    __syncthreads();
    *all = sum;
    return ulong2{v.x + base.x, v.y + base.y};
}

// Deals one kind's work out (one workgroup): every entry's rows in equal tiles, every tile's visits of
// U keys in equal pieces of at most C, where C makes the kind's target of pieces over all kv
// heads.
// sm: LDS, for max_seqs entries each: tp (tiles before each entry, and all) | m | ctx.
// LIMIT: most rows of an entry for narrow tiles.
template <int U, int LIMIT = kNarrowRows>
__device__ void plan(const PageTable& t, const Call& a, int kind, int* sm) {
    __shared__ ulong2 tmp[4];
    __shared__ long long part[4];
    __shared__ int off[257], info[256][7];
    const Call::Kind& kd = a.kind[kind];
    const int tid = threadIdx.x, TR = kd.tile_rows;
    int *tp = sm, *ms = tp + t.max_seqs + 1, *ctxs = ms + t.max_seqs;
    // (entries' facts are requested with their number: the arrays hold max_seqs)
    const int b_first = min(tid, t.max_seqs - 1);
    int c0 = t.cu[b_first], c1 = t.cu[b_first + 1], held = t.step_lens[b_first];
    const int B = t.counts[kPagesEntries];
    int tiles = 0;
    if (tid == 0) tp[0] = 0;
    for (int b0 = 0; b0 < B; b0 += 256) {
        const int b = b0 + tid;
        int n = 0;
        if (b < B) {
            if (b0 > 0) c0 = t.cu[b], c1 = t.cu[b + 1], held = t.step_lens[b];
            const int m = c1 - c0, rows = m * a.G;
            ms[b] = m;
            ctxs[b] = held - m;
            if ((rows <= LIMIT) == (kind == kNarrow)) n = (rows + TR - 1) / TR;
        }
        ulong2 all;
        const ulong2 s = block_scan(ulong2{(uint64_t)n, 0}, tmp, &all);
        if (b < B) tp[b + 1] = tiles + (int)s.x;
        tiles += (int)all.x;
    }
    __syncthreads();
    struct Tile {
        int b, row0, rows, nv;
    };
    auto tile = [&](int i) {
        int lo = 0, hi = B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (tp[mid] <= i) lo = mid;
            else hi = mid;
        }
        // (wide: in whole waves of 32 rows; no tile comes out empty, as rows > (tiles - 1) TR)
        const int rows = ms[lo] * a.G, n = tp[lo + 1] - tp[lo];
        const int each = kind == kNarrow ? TR : ((rows + n - 1) / n + 31) / 32 * 32;
        Tile x{lo, (tp[lo + 1] - 1 - i) * each, 0, 0};  // (an entry's last, which sees the most keys, first)
        x.rows = min(each, rows - x.row0);
        const int last = x.row0 + x.rows - 1;
        x.nv = Visits<U>(ctxs[lo] + x.row0 / a.G, ctxs[lo] + last / a.G, a.window, a.sinks).count;
        return x;
    };
    Tile mine{0, 0, 0, 0};  // the thread's first
    if (tid < tiles) mine = tile(tid);
    long long sum = mine.nv;
    for (int i = tid + 256; i < tiles; i += 256) sum += tile(i).nv;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if ((tid & 63) == 0) part[tid >> 6] = sum;
    __syncthreads();
    sum = part[0] + part[1] + part[2] + part[3];
    // (In 32 bits where they hold it: 64-bit divisions are long.  No tile has more than 2^27
    // visits: so large a C is whole tiles.)
    const long long work = sum * a.KVH;
    auto equal = [&](int n) {
        const int C = work < 1 << 30 ? ((int)work + n - 1) / n
                                     : (int)min<long long>(1 << 28, (work + n - 1) / n);
        return max(kd.least, C);
    };
    auto pieces = [&](int nv, int C) { return (nv - 1) / C + 1; };
    // The lists' and the partial rows' room is what this C can need, and a larger one needs less.
    int C = equal(kd.target), longest = INT_MAX;
    // A piece for every place the device has, if tiles' remainders make no more of them: no piece
    // then waits for a place.  Otherwise (narrow) the larger number, whose second round is shorter.
    // (One token on 8192 keys, 8 kv heads of 128, f16: 25 us, with 3 pieces a CU 28; 32 sequences on 4096, hd
    // 256, f16: 114, 128; 8 entries of 48 rows on 4000 keys, hd 128, f16, where 2 a CU make 576: 77 us,
    // with 3 a CU 66.  Wide: 500 tokens behind 777, 8 heads on one of 256, f32, 223 pieces of 5 visits 83
    // us, by the search below 91; 145 of 8 visits 96, 117 of 10 105, 85 of 15 131.)
    bool fit = false;
    if ((kind == kWide || kd.places < kd.target) && (int64_t)tiles * a.KVH <= kd.places) {
        const int one_each = equal(kd.places);
        __shared__ int made;
        if (tid == 0) made = 0;
        __syncthreads();
        int n = mine.nv > 0 ? pieces(mine.nv, one_each) : 0;
        for (int i = tid + 256; i < tiles; i += 256) n += pieces(tile(i).nv, one_each);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
        if ((tid & 63) == 0 && n > 0) atomicAdd(&made, n);
        __syncthreads();
        fit = (int64_t)made * a.KVH <= kd.places;
        if (fit) C = one_each;
    }
    // Else wide, few tiles: of C0 = C, 5 / 4, 3 / 2 and 2 C0 and whole tiles the one of the shortest time, in
    // visits.  An item's own time is `overhead` visits, and as much again where its sums go
    // through memory.  Up to as many items as places take the largest one's time; up to twice as
    // many, the sum of an item's and of one that follows it, the sizes sorted: the last to find a
    // place of its own and the next, or the largest that is followed and the smallest; more, the
    // mean place's load and half an item.  (Three chunks among 24 sequences, bf16: 165 us with pieces of 18
    // visits, 272 for 256 places, whose small ones pair up; 195 with 15, 328 pieces; 191 with 22, 264; 207
    // with 30, 216.)
    if (!fit && kind == kWide && (int64_t)tiles * a.KVH <= 4 * (int64_t)kd.places) {
        const int C0 = C;
        constexpr int TRY = 5, BINS = 32;
        __shared__ int hist[TRY][BINS], split_made[TRY], top;
        __shared__ float times[TRY];
        for (int i = tid; i < TRY * BINS; i += 256) hist[i / BINS][i % BINS] = 0;
        if (tid < TRY) split_made[tid] = 0;
        if (tid == 0) top = 0;
        __syncthreads();
        auto candidate = [&](int k) {
            return k == 0 ? C0 : k == 1 ? C0 + C0 / 4 : k == 2 ? C0 + C0 / 2 : k == 3 ? 2 * C0 : INT_MAX / 2;
        };
        int my_top = mine.nv;
        for (int i = tid + 256; i < tiles; i += 256) my_top = max(my_top, tile(i).nv);
        if (my_top > 0) atomicMax(&top, my_top);
        __syncthreads();
        longest = top;
        const float bin = (float)(BINS - 1) / (float)longest;
        for (int i = tid; i < tiles; i += 256) {
            const int nv = i < 256 ? mine.nv : tile(i).nv;
#pragma unroll
            for (int k = 0; k < TRY; ++k) {
                const int S = pieces(nv, candidate(k));
                atomicAdd(&hist[k][min(BINS - 1, (int)((float)nv / (float)S * bin))], S);
                if (S > 1) atomicAdd(&split_made[k], S);
            }
        }
        __syncthreads();
        const int lane = tid & 63;
        for (int k = tid >> 6; k < TRY; k += 4) {  // a wave a candidate, a lane a bin
            const int places = max(1, kd.places / a.KVH), h = lane < BINS ? hist[k][lane] : 0;
            int upto = h;  // items of this size and larger
#pragma unroll
            for (int o = 1; o < BINS; o <<= 1) {
                const int x = __shfl_down(upto, o, 64);
                if (lane + o < BINS) upto += x;
            }
            const int n = __shfl(upto, 0, 64);
            const float ov = (float)kd.overhead * (1.0f + (float)split_made[k] / (float)n);
            const float item = (float)min(candidate(k), longest) + ov;
            float time = item;
            if (n > 2 * places) {
                time = fmaxf(item, ((float)sum + ov * (float)n) / (float)places + 0.5f * item);
            } else if (n > places) {
                auto size = [&](int rank) {  // of the item at this rank, the largest first
                    const uint64_t here = __ballot(lane < BINS && rank >= upto - h && rank < upto);
                    return (float)__builtin_ctzll(here | 1ull << 63) / bin;
                };
                time = fmaxf(item, 2.0f * ov + fmaxf(size(places - 1) + size(places),
                                                     size(2 * places - n) + size(n - 1)));
            }
            if (lane == 0) times[k] = time;
        }
        __syncthreads();
        float least_time = INFINITY;
        for (int k = 0; k < TRY; ++k)
            if (times[k] < least_time) {
                least_time = times[k];
                C = candidate(k);
            }
    }
    // Pieces in order of their size, in quarters of the largest, that first (and a tile's neighbours
    // beside it, whose keys are the same): what is dealt out last fills the gaps.  The four
    // ranks' numbers are 16 bits each of a scan's first value: pieces are at most target + tiles.
    const int largest = min(C, longest);
    auto rank = [&](int nv, int S) { return 3 - min(3, (int)(4 * (int64_t)(nv / S) / largest)); };
    int fill[4] = {0, 0, 0, 0};
    if (tiles > 256) {
        __shared__ int count[4];
        if (tid < 4) count[tid] = 0;
        __syncthreads();
        for (int i = tid; i < tiles; i += 256) {
            const int nv = tile(i).nv, S = pieces(nv, C);
            atomicAdd(&count[rank(nv, S)], S);
        }
        __syncthreads();
#pragma unroll
        for (int e = 1; e < 4; ++e) fill[e] = fill[e - 1] + count[e - 1];
    }
    int items = 0, splits = 0, rows = 0;
    for (int i0 = 0; i0 < tiles; i0 += 256) {
        const int i = i0 + tid;
        Tile x = mine;
        if (i0 > 0 && i < tiles) x = tile(i);
        const int S = i < tiles ? pieces(x.nv, C) : 0, rk = S > 0 ? rank(x.nv, S) : 0;
        const int want = S > 1 ? S * a.KVH * x.rows : 0;
        const int first = S > 0 ? t.cu[x.b] : 0, id = S > 0 ? t.step_ids[x.b] : 0;
        ulong2 all;
        const ulong2 n = block_scan(
            ulong2{(uint64_t)S << (16 * rk), (uint64_t)want << 16 | (S > 1 ? 1 : 0)}, tmp, &all);
        auto field = [](uint64_t v, int e) { return (int)(v >> (16 * e) & 0xFFFF); };
        if (tiles <= 256)
#pragma unroll
            for (int e = 1; e < 4; ++e) fill[e] = fill[e - 1] + field(all.x, e - 1);
        int at = 0, upto = 0, made = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (rk == e) at = fill[e] + field(n.x, e) - S;
            upto += field(n.x, e);
            made += field(all.x, e);
            fill[e] += field(all.x, e);
        }
        const int base = kd.row0 + rows + (int)(n.y >> 16) - want;
        off[tid + 1] = upto;
        if (tid == 0) off[0] = 0;
        const int v[7] = {x.b, x.row0, x.rows, x.nv, base, S, at};
#pragma unroll
        for (int e = 0; e < 7; ++e) info[tid][e] = v[e];
        if (want) kd.splits[splits + (int)(n.y & 0xFFFF) - 1] = {first, x.row0, x.rows, base, S, {}};
        if (S == 1)
            kd.items[at] = {first, ctxs[x.b], ctxs[x.b] + ms[x.b], id, x.row0, x.rows, 0, x.nv, base, 0, 1, 0};
        __syncthreads();
        if ((all.y & 0xFFFF) != 0)
            for (int k = tid; k < made; k += 256) {  // tiles in pieces: a thread a piece
                int lo = 0, hi = 256;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (off[mid] <= k) lo = mid;
                    else hi = mid;
                }
                const int* w = info[lo];
                const int s = k - off[lo], nv = w[3], Sw = w[5];
                if (Sw < 2) continue;
                const int v0 = (int)((int64_t)s * nv / Sw), v1 = (int)((int64_t)(s + 1) * nv / Sw);
                const int b = w[0], ctx = ctxs[b];
                kd.items[w[6] + s] = {t.cu[b], ctx, ctx + ms[b], t.step_ids[b], w[1], w[2],
                                      v0, v1 - v0, w[4], s, Sw, 0};
            }
        items += made;
        splits += (int)(all.y & 0xFFFF);
        rows += (int)(all.y >> 16);
        __syncthreads();
    }
    if (tid == 0) {
        kd.head[0] = items;
        kd.head[1] = splits;
    }
}

// 8 weights -> two f16 parts: the first cut off, what is left of up to 2^-10 rounded: 2^-22 of the weight, in
// either direction, and 2^-25 where that is more (one conversion a pair, one mixed-precision multiply-add a
// weight that takes the f16 back out, one conversion a pair).
__device__ __forceinline__ void halve_weights(const f32x8& v, u32x4 (&p)[2]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v[2 * j], v[2 * j + 1]));
        f32x2 lo;  // v - hi, exactly
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]"
            : "=v"(lo[0]) : "v"(hi), "v"(v[2 * j]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
            : "=v"(lo[1]) : "v"(hi), "v"(v[2 * j + 1]));
        p[0][j] = hi;
        p[1][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, f16x2));
    }
}

template <class T>
__device__ __forceinline__ f32x4 mfma16(u32x4 x, u32x4 y, f32x4 z) {
    if constexpr (std::is_same_v<T, f16_t>)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x),
                                                      __builtin_bit_cast(f16x8, y), z, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x),
                                                       __builtin_bit_cast(bf16x8, y), z, 0, 0, 0);
}

// The power of two that brings a row of magnitude at most amax into the f16 parts' range, and
// its inverse (1 where amax is 0 or not finite).
__device__ __forceinline__ float2 row_scale(float amax) {
    if (!(amax > 0.0f) || amax > 3.4e38f) return make_float2(1.0f, 1.0f);
    const int e = min(14 - ilogbf(amax), 126);
    return make_float2(ldexpf(1.0f, e), ldexpf(1.0f, -e));
}

__device__ __forceinline__ void redo_row(const Call& a, int64_t row, int h) {
    a.redo[atomicAdd(a.redo_count, 1)] = (int)row * a.H + h;
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T>
__device__ __forceinline__ f32x16 mfma32(u32x4 x, u32x4 y, f32x16 z) {
    if constexpr (std::is_same_v<T, f16_t>)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x),
                                                      __builtin_bit_cast(f16x8, y), z, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                       __builtin_bit_cast(bf16x8, y), z, 0, 0, 0);
}

// the wave's LDS stores before its reads after them
__device__ __forceinline__ void settle_wave() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The pieces of tiles dealt out, joined (the last kernel of a call): out = sum_s 2^(M_s - M) o_s /
// sum_s 2^(M_s - M) l_s over the pieces' (M_s, l_s, o_s); a piece in which a row sees no key has M_s = -inf, weight 0.  A
// workgroup per (16 rows of a tile, kv head), D / 4 threads to a row; where there are fewer rows
// than such groups, several share a row's pieces and meet in LDS.  A row with a piece of NaN sum
// is left: its output is written (a bad page), or it is one of the rows listed to be done again.
template <int D>
__device__ __forceinline__ void merge_pieces(const Call& a) {
    constexpr int W = D / 4, N = 256 / W;
    __shared__ f32x4 so[N][W];
    __shared__ float sl[N];
    const int ln = threadIdx.x % W, sub = threadIdx.x / W;
    const int nn = a.kind[kNarrow].head[1] * a.KVH;
    const int bl = a.kind[kWide].tile_rows / 16;
    const int nw = a.kind[kWide].head[1] * a.KVH * bl;
    for (int i = blockIdx.x; i < nn + nw; i += gridDim.x) {
        const bool wide = i >= nn;
        const int k = wide ? (i - nn) / bl : i;
        const int r0 = wide ? (i - nn) % bl * 16 : 0;
        const Split sp = a.kind[wide ? kWide : kNarrow].splits[k / a.KVH];
        const int g = k % a.KVH, rows = min(16, sp.rows - r0);
        if (rows <= 0 || sp.S < 2) continue;  // (uniform)
        int share = 1;
        while (share * 2 * rows <= N) share *= 2;
        const int per = N / share;  // rows at a time
        const int part = sub % share;
        const int64_t first = sp.first;
        for (int rb = 0; rb < rows; rb += per) {
            const int r = rb + sub / share;
            const bool live = r < rows;
            const int64_t p0 = (int64_t)sp.base + (int64_t)g * sp.S * sp.rows + r0 + min(r, rows - 1);
            float M = -INFINITY;
            for (int s = ln; s < sp.S; s += W) M = fmaxf(M, a.ms[p0 + (int64_t)s * sp.rows].x);
#pragma unroll
            for (int x = W / 2; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, W));
            float l = 0.0f;
            f32x4 o = 0.0f;
#pragma unroll 8
            for (int s = part; s < sp.S; s += share) {
                const int64_t p = p0 + (int64_t)s * sp.rows;
                const float2 x = a.ms[p];
                const f32x4 v = *reinterpret_cast<const f32x4*>(a.po + p * D + 4 * ln);
                const float f = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - M);
                l = fmaf(x.y, f, l);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], f, o[e]);
            }
            if (share > 1) {
                so[sub][ln] = o;
                if (ln == 0) sl[sub] = l;
                __syncthreads();
                if (part == 0)
                    for (int x = 1; x < share; ++x) {
                        o += so[sub + x][ln];
                        l += sl[sub + x];
                    }
                __syncthreads();
            }
            if (live && part == 0 && l == l) {
                const int rr = sp.row0 + r0 + r;
                *reinterpret_cast<f32x4*>(a.out + (first + rr / a.G) * a.ostride +
                                          (int64_t)(g * a.G + rr % a.G) * D + 4 * ln) = o / l;
            }
        }
    }
}

}  // namespace
}  // namespace unillm
