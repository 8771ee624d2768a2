// paged.hip -- attention of a serving step's new tokens over paged KV caches.
//
// For every row of the step's plan (token at position p of its sequence, pages.hip): q and k
// rotated at p, k and v rounded once to the pool's type T and stored in the row's slot, then
// per head h with kv head g = h / (H / KVH)
//   out = sum_j w_j v_j / sum_j w_j,  w_j = e^(q k_j / sqrt(hd) - max),
// over the positions j <= p of the sequence; with a window w > 0 only j > p - w, and j < sinks.
// The angles p theta^(-2 i / hd) are formed and reduced in f64 (at position 100000 their f32
// forms are 0.003 off), and k is rotated in f64, so its one rounding to T is the rounding of
// the true value; sums, maxima and quotients are f32.
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
template <int U>
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
            if ((rows <= kNarrowRows) == (kind == kNarrow)) n = (rows + TR - 1) / TR;
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

// The first kernel of a call.  Workgroups 0 and 1 deal the work out; each other one takes nr rows
// of the step and `heads` kv heads: the rows' rotations (kept in f32 for the queries), their
// keys rotated and stored, their values stored.  A V page runs along the keys, so where 8 rows
// are 8 neighbouring slots of a page, aligned (a prompt's rows, but for its ends), a thread
// stores a dimension's 8 values at once; other rows value by value.
// Bound by HBM where rows are many: 2048 rows of 32 kv heads of 128, f16, 100 MB in 21 us (65 with
// every value on its own, a row after the other); by latency and by the plan where they are few:
// 6 us for one row, 12 where three chunks of 24 entries are dealt out.
// nr is 16, or 4 of a step of up to 512 rows, whose workgroups are too few otherwise (a whole call of
// 512 such rows 45 us, 46 with 16 a workgroup; of 2048 rows 129 us, 145 with 4).
constexpr int kAppendRows = 16;

template <class T, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedKv c, PageTable t, Call a, int nr, int heads) {
    constexpr int HALF = D / 2, Q4 = HALF / 4, NR = kAppendRows;
    __shared__ double2 turn[NR][HALF];
    __shared__ int slots[NR + 14];  // of the rows from 7 before the workgroup's to 7 after
    extern __shared__ int plan_lds[];
    const int tid = threadIdx.x;
    const int bx = (int)blockIdx.x - 2, groups = (a.KVH + heads - 1) / heads;
    const int row0 = bx / groups * nr, g0 = bx % groups * heads;
    // (rows' slots and positions are requested with the plan's header: both arrays hold max_tokens)
    int slot = -1, pos = 0;
    if (bx >= 0 && tid < nr + 14) {
        const int row = row0 + tid - 7;
        if (row >= 0 && row < t.max_tokens) slot = t.slots[row];
    }
    if (bx >= 0 && tid < nr && row0 + tid < t.max_tokens) pos = t.positions[row0 + tid];
    if (!step_fits(t, a.n)) {
        if (blockIdx.x < 2 && tid < 2) a.kind[blockIdx.x].head[tid] = 0;
        if (blockIdx.x == 0 && tid == 0) *a.redo_count = 0;
        fail_call(t, a, D, blockIdx.x, gridDim.x);
        return;
    }
    if (blockIdx.x == 0 && tid == 0) *a.redo_count = 0;
    if (blockIdx.x == 0) return plan<kUnit>(t, a, kNarrow, plan_lds);
    if (blockIdx.x == 1) return plan<kWideUnit<T, D>>(t, a, kWide, plan_lds);
    const int total = t.counts[kPagesTokens];
    if (row0 >= total) return;
    const int rows = min(nr, total - row0);
    __shared__ int at[NR];
    if (tid < nr + 14) slots[tid] = row0 + tid - 7 < total ? slot : -1;
    if (tid < nr) at[tid] = pos;
    __syncthreads();
    // Row r is in a run of 8 if the row r - slot % 8 and the one 7 after it are 7 slots apart; the
    // runs that begin here and the rows in none, listed.
    __shared__ int list[2], run_rows[NR], one_rows[NR];
    if (tid < 64) {
        const int sl = tid < rows ? slots[tid + 7] : -1, s0 = tid - (sl & 7);
        const bool run = sl >= 0 && s0 >= -7 && s0 < nr && slots[s0 + 7] == (sl & ~7) &&
                         slots[s0 + 14] == (sl | 7);
        const uint64_t begins = __ballot(run && (sl & 7) == 0), ones = __ballot(sl >= 0 && !run);
        const uint64_t before = (1ull << tid) - 1;
        if (begins >> tid & 1) run_rows[__popcll(begins & before)] = tid;
        if (ones >> tid & 1) one_rows[__popcll(ones & before)] = tid;
        if (tid == 0) list[0] = __popcll(begins), list[1] = __popcll(ones);
    }
    for (int i = tid; i < rows * HALF; i += 256) {
        const int r = i / HALF, p = i % HALF;
        double sn, cs;
        sincospi((double)at[r] * c.freq[p], &sn, &cs);
        turn[r][p] = make_double2(cs, sn);
        if (g0 == 0) a.turn[(int64_t)(row0 + r) * HALF + p] = make_float2((float)cs, (float)sn);
    }
    __syncthreads();
    const int KVH = a.KVH, shift = c.page_shift;
    const int64_t ps = c.page_size;
    const int g1 = min(g0 + heads, KVH);
    const float* xk = a.qkv + (int64_t)row0 * a.qstride + (int64_t)a.H * D;
    const float* xv = xk + (int64_t)KVH * D;
    // keys: 4 dimensions and their partners a thread
    for (int i = tid; i < (g1 - g0) * rows * Q4; i += 256) {
        const int g = g0 + i / (rows * Q4), r = i / Q4 % rows, p = i % Q4 * 4;
        const int sl = slots[r + 7];
        const float* x = xk + r * a.qstride + (int64_t)g * D + p;
        const f32x4 u = *reinterpret_cast<const f32x4*>(x), w = *reinterpret_cast<const f32x4*>(x + HALF);
        struct alignas(4 * sizeof(T)) Four {
            T v[4];
        } lo, hi;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double2 z = turn[r][p + e];
            const double uu = u[e], ww = w[e];
            lo.v[e] = narrow<T>((float)(uu * z.x - ww * z.y));
            hi.v[e] = narrow<T>((float)(uu * z.y + ww * z.x));
        }
        if (sl < 0) continue;
        T* dst = static_cast<T*>(c.k) +
                 (((((int64_t)(sl >> shift) * KVH + g) << shift) + (sl & (ps - 1))) * D + p);
        *reinterpret_cast<Four*>(dst) = lo;
        *reinterpret_cast<Four*>(dst + HALF) = hi;
    }
    // values: a wave a task of 64 dimensions of a run or of a single row
    const int lane = tid & 63;
    constexpr int DG = D / 64;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_runs = list[0], n_ones = list[1];
    for (int i = wv; i < (g1 - g0) * n_runs * DG; i += 4) {
        const int g = g0 + i / (n_runs * DG), r = run_rows[i / DG % n_runs], d = i % DG * 64 + lane;
        const int sl = slots[r + 7];
        T* dst = static_cast<T*>(c.v) +
                 (((((int64_t)(sl >> shift) * KVH + g) * D + d) << shift) + (sl & (ps - 1)));
        const float* x = xv + r * a.qstride + (int64_t)g * D + d;
        struct alignas(16) Eight {
            T v[8];
        } y;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = x[e * a.qstride];
#pragma unroll
        for (int e = 0; e < 8; ++e) y.v[e] = narrow<T>(f[e]);
        *reinterpret_cast<Eight*>(dst) = y;
    }
    const int tasks = (g1 - g0) * n_ones * DG;
    for (int i0 = wv; i0 < tasks; i0 += 16) {
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // (four tasks' loads in flight)
            const int i = min(i0 + 4 * k, tasks - 1), g = g0 + i / (n_ones * DG), r = one_rows[i / DG % n_ones];
            x[k] = xv[r * a.qstride + (int64_t)g * D + i % DG * 64 + lane];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + 4 * k;
            if (i >= tasks) break;
            const int g = g0 + i / (n_ones * DG), d = i % DG * 64 + lane;
            const int sl = slots[one_rows[i / DG % n_ones] + 7];
            T* page = static_cast<T*>(c.v) + ((((int64_t)(sl >> shift) * KVH + g) * D + d) << shift);
            page[sl & (ps - 1)] = narrow<T>(x[k]);
        }
    }
}

// ---- products at f32's precision ------------------------------------------------------------
//
// The 16-bit matrix cores run 16 times the f32 ones.  A value held in f16 or bf16 is its own
// single part.  f32 values are sums of parts: against bf16 (and f32, itself three bf16 parts) three
// bf16 ones, all 24 bits; against f16 two f16 ones, 22 bits, where a power of two per query
// row brings q into range (its largest magnitude in [2^14, 2^15)) and the weights, at most
// 2^slack above their reference (below), are taken times 2^shift: parts down to 2^-24 then reach
// 2^-38 of a row's largest element and 2^-35 of the reference weight.  A weight is then off by
// 2^-36 of the reference's at most, and that is too much where the large weights' values are nothing
// (a key that takes all the attention, of value 0: with the others 16 nats below it the outputs
// were 1e-3 off).  Narrow tiles multiply a visit with a weight so small by bf16 parts, wide ones
// look at what came of them (below).
template <class T>
struct Parts;
template <>
struct Parts<f16_t> {
    static constexpr int K = 1, Q = 2, N = 2;
    static constexpr int ki[N] = {0, 0}, qi[N] = {1, 0};  // products, the large one last
    static constexpr float shift = 11.0f, slack = 4.0f;
};
template <>
struct Parts<bf16_t> {
    static constexpr int K = 1, Q = 3, N = 3;
    static constexpr int ki[N] = {0, 0, 0}, qi[N] = {2, 1, 0};
    static constexpr float shift = 0.0f, slack = 8.0f;
};
template <>
struct Parts<float> {
    static constexpr int K = 3, Q = 3, N = 6;
    static constexpr int ki[N] = {2, 0, 1, 1, 0, 0}, qi[N] = {0, 2, 1, 0, 1, 0};
    static constexpr float shift = 0.0f, slack = 8.0f;
};
// How far below a row's reference (log2) a weight held in two parts of f16 may be in a narrow tile's
// visit: 2^-20 of it is lost at most.  (32 sequences of 8192 keys, scores that make half of the visits
// and all of them such: 210 and 205 us, 201 with none.)
constexpr float kSpread = 16.0f;
// What a wide tile's row may lose by them, of its largest sum: 2^-16 over up to 2048 keys, 2^-27 a key
// over more (an f32 sum of as many terms may be off by 2^-24 a term).  A row loses so much where
// keys of values below 1/512 of V's largest have all but 1/512 of the weight.  (Five products a visit
// would be 7 for 4 in all, and most visits are such where scores spread; few rows are.)
constexpr float kLoss = 0x1p-16f;
constexpr int kLossKeys = 2048;

// 8 f32 -> the parts of a q or weight operand
template <class T>
__device__ __forceinline__ void split_q(const f32x8& v, u32x4 (&p)[Parts<T>::Q]) {
    if constexpr (std::is_same_v<T, f16_t>) {
        const f16x8 hi = __builtin_convertvector(v, f16x8);
        const f16x8 lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x8), f16x8);
        p[0] = __builtin_bit_cast(u32x4, hi);
        p[1] = __builtin_bit_cast(u32x4, lo);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t x, y, z;
            split2(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]), x, y, z);
            p[0][j] = x;
            p[1][j] = y;
            p[2][j] = z;
        }
    }
}

// 8 weights -> their parts.  f16: the first part cut off, what is left of up to 2^-10 rounded:
// 2^-22 of the weight, in either direction (one conversion a pair, one mixed-precision
// multiply-add a weight that takes the f16 back out, one conversion a pair).
template <class T>
__device__ __forceinline__ void split_w(const f32x8& v, u32x4 (&p)[Parts<T>::Q]) {
    if constexpr (std::is_same_v<T, f16_t>) {
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
    } else {
        split_q<T>(v, p);
    }
}

// 8 elements of the pool as loaded, and as an operand's parts
template <class T>
struct Raw {
    u32x4 w[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Raw<T> load8(const T* p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const u32x4*>(p)[i];
    return r;
}
template <class T>
__device__ __forceinline__ T element(const Raw<T>& r, int e) {
    return reinterpret_cast<const T*>(&r)[e];
}
template <class T>
__device__ __forceinline__ void split_k(const Raw<T>& r, u32x4 (&p)[Parts<T>::K]) {
    if constexpr (sizeof(T) == 2) {
        p[0] = r.w[0];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t x, y, z;
            split2(r.w[j / 2][j % 2 * 2], r.w[j / 2][j % 2 * 2 + 1], x, y, z);
            p[0][j] = x;
            p[1][j] = y;
            p[2][j] = z;
        }
    }
}

// 8 f16 values -> their two bf16 parts, exactly: 8 of the 11 bits and the rest
__device__ __forceinline__ void widen_f16(u32x4 r, u32x4 (&p)[2]) {
    const f32x8 v = __builtin_convertvector(__builtin_bit_cast(f16x8, r), f32x8);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[0][j] = pack_bf16(v[2 * j], v[2 * j + 1]);
        p[1][j] = pack_bf16(v[2 * j] - bf16_lo(p[0][j]), v[2 * j + 1] - bf16_hi(p[0][j]));
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

// Query row r of an entry (its first step row `first`): 1 / sqrt(D) and log2 e times the
// rotated dimensions d .. d + 7 (d a multiple of 8).
template <int D>
__device__ __forceinline__ f32x8 rotated8(const Call& a, int first, int g, int r, int d) {
    constexpr int HALF = D / 2;
    const int64_t row = first + r / a.G;
    const float* x = a.qkv + row * a.qstride + (int64_t)(g * a.G + r % a.G) * D;
    const float2* cs = a.turn + row * HALF + d % HALF;
    const float scale = kLog2e / sqrtf((float)D);
    const float* x0 = x + d % HALF;
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float u = x0[j], w = x0[j + HALF];
        const float2 z = cs[j];
        v[j] = (d < HALF ? u * z.x - w * z.y : u * z.y + w * z.x) * scale;
    }
    return v;
}

// ---- few query rows: keys stream through registers --------------------------------------------
//
// A workgroup takes an item of a tile of 16 query rows of a kv head, its four waves every fourth
// visit of 32 keys each.  Both products are formed transposed (16x16x32 MFMAs), so that each
// operand of the pool is a lane's own 16-byte load, used once and straight from its
// registers, and the weights never leave theirs:
//   S^T [32 keys][16 rows] = K . Q^T: operand row i of subtile t is key 8 (i / 4) + 4 t + i % 4,
//     so lane l holds, of row l % 16, the scores of the 8 keys 8 (l / 16) ..;
//   O^T [D][16 rows] += V^T . P^T: those 8 keys are the 8 the lane's B operand contracts, and
//     V^T's operand, of dimension l % 16 of each 16, is 8 neighbouring keys of a V page.
// A page id per 16 keys is read ahead into LDS; the next visit's keys are requested once this
// one's are used, its values likewise, so each has the other's products to arrive in.
// The reference that the weights' exponents are taken against follows a row's maximum only when
// some score passes it by 2^slack, so a visit needs no exchange between lanes; the sums of the
// weights stay per lane until the end.  Bound by HBM: 4 D bytes of a 16-bit pool a key (one GB of f16
// at hd 128, two sequences of up to 131040 keys: 177 us, 5.8 TB/s; 64 sequences, bf16, 596 MB: 109 us,
// 5.5 TB/s),
// and for short sequences by latency (one, of 4000 keys: 8 us).
template <class T, int D>
struct NarrowLds {
    static constexpr int NB = D / 32, OT = D / 16;
    static constexpr int IDS = 0;                                  // page ids of 256 visits
    static constexpr int STAT = IDS + 2048;                        // row scales, maxima, sums, flags
    static constexpr int Q = STAT + 1024;                          // q's parts [Q][NB][64][16 B]
    static constexpr int QBYTES = Parts<T>::Q * NB * 1024;
    static constexpr int O = Q;                                    // later the waves' sums [4][OT][64][16 B]
    static constexpr int OBYTES = 4 * OT * 1024;
    static constexpr int BYTES = Q + (QBYTES > OBYTES ? QBYTES : OBYTES);
};

template <class T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_narrow_kernel(PagedKv c, PageTable t, Call a) {
    using L = NarrowLds<T, D>;
    using P = Parts<T>;
    constexpr int NB = L::NB, OT = L::OT;
    constexpr bool kHoldQ = sizeof(T) == 2 && D < 256;  // q's parts in registers: where they fit
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int* ids = reinterpret_cast<int*>(lds + L::IDS);              // [2][256]
    float* rowmax = reinterpret_cast<float*>(lds + L::STAT);      // [16]
    float* wm = rowmax + 16;                                       // [4][16]
    float* wl = wm + 64;                                           // [4][16]
    int* flags = reinterpret_cast<int*>(wl + 64);                 // [0] a bad page, [1] rows to redo
    u32x4* qp = reinterpret_cast<u32x4*>(lds + L::Q);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, qd = lane >> 4;
    const int64_t ps = c.page_size;
    const int KVH = a.KVH, G = a.G;
    const int total = a.kind[kNarrow].head[0] * KVH;
    for (int idx = blockIdx.x; idx < total; idx += gridDim.x) {
        const Item it = a.kind[kNarrow].items[idx / KVH];
        const int g = idx % KVH;
        const int first = it.first, len = it.len, ctx = it.ctx;
        const int* pages = t.table + (int64_t)it.id * t.max_pages;
        const int pmin = ctx + it.row0 / G, pmax = ctx + (it.row0 + it.rows - 1) / G;
        const Visits<kUnit> vis(pmin, pmax, a.window, a.sinks);
        // q's parts: task (block, lane) as the B operand takes it
        constexpr int TASKS = (NB * 64 + 255) / 256;
        f32x8 qv[TASKS];
        __syncthreads();  // (the item before is done with the LDS)
        if (tid < 16) rowmax[tid] = 0.0f;
        if (tid < 2) flags[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
            const int f = i * 256 + tid, r = f % 16, d = f / 64 * 32 + f / 16 % 4 * 8;
            qv[i] = 0.0f;
            if (f < NB * 64 && r < it.rows) {
                qv[i] = rotated8<D>(a, first, g, it.row0 + r, d);
                float mx = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(qv[i][j]));
                if (std::is_same_v<T, f16_t>)  // (non-negative floats order as their bits)
                    atomicMax(reinterpret_cast<int*>(rowmax) + r, __float_as_int(mx));
            }
        }
        __syncthreads();
        float inv = 1.0f;  // of this lane's row
        if (std::is_same_v<T, f16_t>) inv = row_scale(rowmax[col]).y;
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
            const int f = i * 256 + tid;
            if (f < NB * 64) {
                if (std::is_same_v<T, f16_t>) qv[i] *= row_scale(rowmax[f % 16]).x;
                u32x4 p[P::Q];
                split_q<T>(qv[i], p);
#pragma unroll
                for (int q = 0; q < P::Q; ++q) qp[q * NB * 64 + f] = p[q];
            }
        }
        const int ppos = ctx + min(it.row0 + col, it.row0 + it.rows - 1) / G;  // the lane's row's position

        float ref = -INFINITY, l = 0.0f;
        f32x4 o[OT];
#pragma unroll
        for (int i = 0; i < OT; ++i) o[i] = 0.0f;
        u32x4 qh[kHoldQ ? P::Q : 1][NB];
        int ql = lane;
        auto q = [&](int i, int b) { return kHoldQ ? qh[kHoldQ ? i : 0][b] : qp[(i * NB + b) * 64 + ql]; };
        Raw<T> kr[2][NB], vr[OT];
        for (int seg = 0; seg < it.nv; seg += 256) {
            const int nseg = min(256, it.nv - seg);
            __syncthreads();
            for (int i = tid; i < 2 * nseg; i += 256) {  // the page of each 16 keys
                int j = vis.key(it.v0 + seg + i / 2) + i % 2 * 16;
                if (j >= len) j -= 16;  // (past the sequence: read the visit's first ones again)
                int pg = pages[j >> c.page_shift];
                if ((unsigned)pg >= (unsigned)c.n_pages) {
                    pg = 0;
                    flags[0] = 1;
                }
                ids[i % 2 * 256 + i / 2] = pg;
            }
            __syncthreads();
            if (kHoldQ && seg == 0)
#pragma unroll
                for (int i = 0; i < (kHoldQ ? P::Q : 0); ++i)
#pragma unroll
                    for (int b = 0; b < NB; ++b) qh[i][b] = qp[(i * NB + b) * 64 + lane];
            // element offsets of a 16-key half's K and V
            auto half = [&](int v, int hf, int64_t& page, int& off) {
                const int j = vis.key(it.v0 + seg + v);
                page = __builtin_amdgcn_readfirstlane(ids[hf * 256 + v]);
                off = (j + (j + hf * 16 < len ? hf * 16 : 0)) & (int)(ps - 1);
            };
            auto load_k = [&](int v) {
                int64_t p0, p1;
                int f0, f1;
                half(v, 0, p0, f0);
                half(v, 1, p1, f1);
                const int i = col / 4;
                const int64_t at = i >= 2 ? (p1 * KVH + g) * ps + f1 : (p0 * KVH + g) * ps + f0;
                const T* k = static_cast<const T*>(c.k) + (at + 8 * (i & 1) + col % 4) * D + 8 * qd;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int b = 0; b < NB; ++b) kr[s][b] = load8<T>(k + 4 * s * D + 32 * b);
            };
            auto load_v = [&](int v) {
                int64_t p0, p1;
                int f0, f1;
                half(v, 0, p0, f0);
                half(v, 1, p1, f1);
                const int64_t at = qd >= 2 ? (p1 * KVH + g) * D * ps + f1 : (p0 * KVH + g) * D * ps + f0;
                const T* x = static_cast<const T*>(c.v) + at + col * ps + 8 * (qd & 1);
#pragma unroll
                for (int i = 0; i < OT; ++i) vr[i] = load8<T>(x + i * 16 * ps);
            };
            if (wv < nseg) {
                load_k(wv);
                load_v(wv);
            }
            for (int v = wv; v < nseg; v += 4) {
                const int j0 = vis.key(it.v0 + seg + v);
                if (!kHoldQ) asm volatile("" : "+v"(ql));  // (not read ahead of the loop)
                f32x8 s;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    f32x4 hi = 0.0f, lo = 0.0f;  // (the small products in a sum of their own)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        u32x4 kp[P::K];
                        split_k<T>(kr[u][b], kp);
#pragma unroll
                        for (int i = 0; i < P::N - 1; ++i) lo = mfma16<T>(kp[P::ki[i]], q(P::qi[i], b), lo);
                        hi = mfma16<T>(kp[0], q(0, b), hi);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[4 * u + r] = hi[r] + lo[r];
                }
                if (v + 4 < nseg) load_k(v + 4);
                if (std::is_same_v<T, f16_t>) s *= inv;
                float low = s[0];  // (hidden keys' among them: their visit only takes longer)
#pragma unroll
                for (int r = 1; r < 8; ++r) low = fminf(low, s[r]);
                // masks, where some row of the tile does not see the whole visit
                const bool whole = j0 + kUnit - 1 <= pmin &&
                                   (a.window == 0 || j0 > pmax - a.window || j0 + kUnit <= a.sinks);
                if (!whole) {
                    const int at = ppos - j0 - 8 * qd, far = a.window > 0 ? at - a.window : INT_MIN;
                    const int sk = a.sinks - j0 - 8 * qd;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const bool hidden = (r > at) | ((r <= far) & (r >= sk));
                        s[r] = hidden ? -INFINITY : s[r];
                    }
                }
                float top = s[0];
#pragma unroll
                for (int r = 1; r < 8; ++r) top = fmaxf(top, s[r]);
                if (__any(top > ref + P::slack)) {
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float up = fmaxf(ref, top);
                    const float f = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - up);
                    l *= f;
#pragma unroll
                    for (int i = 0; i < OT; ++i) o[i] *= f;
                    ref = up;
                }
                const float from = ref == -INFINITY ? 0.0f : ref - P::shift;  // (all weights are 0 then)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    s[r] = __builtin_amdgcn_exp2f(s[r] - from);
                    l += s[r];
                }
                if (j0 + kUnit > len) {  // past the sequence's end a page holds anything
#pragma unroll
                    for (int i = 0; i < OT; ++i) {
                        constexpr int E = 4 / sizeof(T);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (j0 + 8 * qd + e >= len) {
                                uint32_t& w = reinterpret_cast<uint32_t*>(&vr[i])[e / E];
                                if constexpr (E == 1) w = 0;
                                else w &= e % 2 ? 0xFFFFu : 0xFFFF0000u;
                            }
                    }
                }
                if (std::is_same_v<T, f16_t> && __any(low < ref - kSpread)) {
                    // weights of any size: five products of three bf16 parts and two (and none is left below)
                    u32x4 p[3];
                    split_q<bf16_t>(s, p);
#pragma unroll
                    for (int i = 0; i < OT; ++i) {
                        u32x4 vp[2];
                        widen_f16(vr[i].w[0], vp);
                        o[i] = mfma16<bf16_t>(vp[1], p[1], o[i]);
                        o[i] = mfma16<bf16_t>(vp[0], p[2], o[i]);
                        o[i] = mfma16<bf16_t>(vp[1], p[0], o[i]);
                        o[i] = mfma16<bf16_t>(vp[0], p[1], o[i]);
                        o[i] = mfma16<bf16_t>(vp[0], p[0], o[i]);
                    }
                    s = 0.0f;
                }
                u32x4 p[P::Q];
                split_q<T>(s, p);
#pragma unroll
                for (int i = 0; i < OT; ++i) {
                    u32x4 vp[P::K];
                    split_k<T>(vr[i], vp);
#pragma unroll
                    for (int n = 0; n < P::N; ++n) o[i] = mfma16<T>(vp[P::ki[n]], p[P::qi[n]], o[i]);
                }
                if (v + 4 < nseg) load_v(v + 4);
            }
        }

        // the four waves' sums: scaled to one reference, added through LDS
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        __syncthreads();  // (q's parts are read)
        if (lane < 16) {
            wm[wv * 16 + lane] = ref;
            wl[wv * 16 + lane] = l;
        }
        __syncthreads();
        float top = wm[col];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, wm[w * 16 + col]);
        auto weight = [&](float r) { return r == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r - top); };
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum = fmaf(weight(wm[w * 16 + col]), wl[w * 16 + col], sum);
        const float mine = weight(ref);
        f32x4* ox = reinterpret_cast<f32x4*>(lds + L::O);
#pragma unroll
        for (int i = 0; i < OT; ++i) ox[(wv * OT + i) * 64 + lane] = o[i] * mine;
        __syncthreads();
        const bool whole = it.S == 1;
        const float inv_sum = 1.0f / sum;
        float chk = sum * 0.0f;
        f32x4 res[OT / 4];
#pragma unroll
        for (int i = 0; i < OT / 4; ++i) {
            const int ot = 4 * i + wv;
            f32x4 x = ox[ot * 64 + lane];
#pragma unroll
            for (int w = 1; w < 4; ++w) x += ox[(w * OT + ot) * 64 + lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // the quotient: the rounded product, corrected by its remainder
                const float y = x[r] * inv_sum;
                if (whole) x[r] = fmaf(fmaf(-y, sum, x[r]), inv_sum, y);
                chk = fmaf(x[r], 0.0f, chk);
            }
            res[i] = x;
        }
        const bool live = col < it.rows;
        if (live && chk != 0.0f) atomicOr(&flags[1], 1 << col);
        __syncthreads();
        const bool bad_page = flags[0] != 0;
        if (bad_page && tid == 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesBadState);
        if (live) {
            const bool again = !bad_page && (flags[1] >> col & 1);
            const int rr = it.row0 + col;
            const int64_t row = first + rr / G;
            const int h = g * G + rr % G;
            const int64_t piece = (int64_t)it.base + ((int64_t)g * it.S + it.s) * it.rows + col;
            // (a row with a bad page is NaN, whatever its other pieces hold)
            float* dst = whole || bad_page ? a.out + row * a.ostride + (int64_t)h * D : a.po + piece * D;
            if (!again)
#pragma unroll
                for (int i = 0; i < OT / 4; ++i)
                    *reinterpret_cast<f32x4*>(dst + (4 * i + wv) * 16 + 4 * qd) =
                        bad_page ? f32x4(__builtin_nanf("")) : res[i];
            if (wv == 0 && qd == 0) {
                if (again) redo_row(a, row, h);
                if (!whole)
                    a.ms[piece] = make_float2(top - P::shift, again || bad_page ? __builtin_nanf("") : sum);
            }
        }
    }
}

// ---- many query rows: tiles of keys shared through LDS -----------------------------------------
//
// A workgroup takes an item of a tile of up to 256 query rows of a kv head (128 at hd 256), 32 to
// each of its waves (32x32x16 MFMAs), and visits U keys at a time through LDS: K [U][2 D bytes] and V^T
// [D][2 U bytes] (of f32 three planes of parts each), 16-byte chunks XOR-swizzled so that the lanes
// a read serves together touch all banks.  As above both products are transposed, a lane's 16
// accumulators of a 32-key group are one row's scores of keys 16 k + 8 (l / 32) + 0 .. 7 (the row
// of K that operand row i reads is i with bits 2 and 3 exchanged), and those are the keys its
// operand of the second product contracts.
// Visit n is a matrix phase, p v of visit n - 1 and q k of visit n, and a vector phase, the
// weights of visit n; a barrier ends each.  The two groups of four waves, a wave of each on every
// SIMD, are a phase apart, so the matrix cores and the vector units are both at work (as two
// workgroups a CU they ran their phases together).  V of n - 1 and K of n share one of two
// LDS buffers; each group stores its half of the next pair in its vector phase, requested one
// visit before.
// Bound by the matrix cores, with Parts::N times the products of a 16-bit attention, and at hd 64
// by the vector units (a visit's weights 1400 to 1600 cycles, its products 1024).  At hd 128 in f16 a visit
// takes 3000 cycles of matrix phase, 2048 of them MFMAs back to back, the rest reads of LDS and the
// barriers.  A 2048-token prompt of 32 heads of 128, f16, 34 GFLOP in two parts: 100 us, 690 TFLOP/s
// of f16 products, where a large library product reaches 1066.
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

template <class T, int D>
struct WideLds {
    static constexpr int GR = kGroups<T, D>, NT = 256 * GR;
    static constexpr int U = kWideUnit<T, D>, KPARTS = Parts<T>::K;
    static constexpr int KROW = 2 * D, VROW = 2 * U;
    static constexpr int PLANE = U * KROW;                  // of K, and of V^T
    static constexpr int K = 0, V = KPARTS * PLANE, PAIR = 2 * V;
    // q's last part, where registers lack: held there the queries spill to memory (8 heads on one kv
    // head, 2000 tokens behind 8000, us: f32 hd 64 241 -> 222, 128 434 -> 395, 256 1418 -> 963; bf16
    // hd 256 740 -> 483, f16 428 -> 399, and 415 since V's magnitudes are looked at)
    static constexpr int QL = GR * PAIR;
    static constexpr bool kQl = D >= 128 || sizeof(T) == 4;
    // (from this block of 16 dimensions on: LDS is full)
    static constexpr int QL0 = sizeof(T) == 4 && D >= 128 ? 1 : 0;
    static constexpr int QREGS = Parts<T>::Q - (kQl ? 1 : 0);
    static constexpr int QROWS = 32 * D * 4;                // a wave's rows in f32, before and after
    static constexpr int USED = QL + (kQl ? NT / 64 * (D / 16 - QL0) * 1024 : 0), ROWS = NT / 64 * QROWS;
    static constexpr int STAT = USED > ROWS ? USED : ROWS;  // whether a page is bad, V's largest
    static constexpr int BYTES = STAT + 64 + 256;
    static constexpr int TASKS = U * D / 8 / NT;            // 8-element chunks of K (or V) a thread
    __device__ static uint32_t kslot(uint32_t r, uint32_t c) {
        return D >= 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
    }
    __device__ static uint32_t vslot(uint32_t d, uint32_t c) {
        return U == 64 ? c ^ ((d >> 1) & 7) : c ^ ((d >> 2) & 3);
    }
};

template <class T, int D>
__global__ __launch_bounds__((256 * kGroups<T, D>), (D == 256 ? 1 : 2)) void paged_wide_kernel(
    PagedKv c, PageTable t, Call a) {
    using L = WideLds<T, D>;
    using P = Parts<T>;
    constexpr int U = L::U, NB = D / 16, OT = D / 32, NG = U / 32, GR = L::GR, NT = L::NT;
    constexpr int LOG_D = D == 64 ? 6 : D == 128 ? 7 : 8;
    constexpr int KSTEP = NT * 8 / D, KROWS = 512 / D;  // keys between a thread's chunks, keys of a wave's
    constexpr int VGROUPS = U / 16;
    // A buffer's pair m - 2 was last read in the second group's matrix phase m - 2, so either group may
    // store its share of pair m in the two phases after: its matrix phase m - 1, or the vector
    // phase m - 1 (m - 2 in the second group).  The stores go with the shorter phase (f16: at hd 128
    // a matrix phase takes 3000 cycles, the weights 1470; at hd 64 1350 and 1600).
    constexpr bool kStoreEarly = GR == 2 && D == 64 && sizeof(T) == 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int* flags = reinterpret_cast<int*>(lds + L::STAT);  // [0] a bad page
    int* vtop = flags + 16;  // f16: [64] V's largest magnitudes (as bits), by lanes that staged them
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wv / 4;
    const int col = lane & 31, hf = lane >> 5;
    const int ps = c.page_size, shift = c.page_shift;
    const int KVH = a.KVH, G = a.G;
    const int kread = ((col & 16) | (col & 4) << 1 | (col & 8) >> 1 | (col & 3));  // operand row's key
    // where the lane's operand rows begin, chunk hf
    const uint32_t kat = kread * L::KROW + L::kslot(kread, hf) * 16;
    const uint32_t vat = col * L::VROW + L::vslot(col, hf) * 16;
    // its staging: offsets of its chunks of K and V from their group's first, and in a buffer
    const int kr0 = tid / (D / 8), vgroup = wv % VGROUPS;
    const uint32_t vd0 = wv / VGROUPS * (32 * L::TASKS) + lane / 2;
    const uint32_t klane = (uint32_t)(kr0 % 16 * D + tid % (D / 8) * 8);
    const uint32_t vlane = (vd0 << shift) + 8 * (lane & 1);
    const uint32_t kto = kr0 * L::KROW + L::kslot(kr0, tid % (D / 8)) * 16;
    const uint32_t vto = vd0 * L::VROW + L::vslot(vd0, 2 * vgroup + (lane & 1)) * 16;
    const int total = a.kind[kWide].head[0] * KVH;
    for (int idx = blockIdx.x; idx < total; idx += gridDim.x) {
        const Item it = a.kind[kWide].items[idx / KVH];
        const int g = idx % KVH;
        const int first = it.first, len = it.len, ctx = it.ctx;
        const int* pages = t.table + (int64_t)it.id * t.max_pages;
        const Visits<U> vis(ctx + it.row0 / G, ctx + (it.row0 + it.rows - 1) / G, a.window, a.sinks);
        // the wave's rows and their positions
        const int w0 = 32 * wv;
        const int wmin = ctx + (it.row0 + min(w0, it.rows - 1)) / G;
        const int wmax = ctx + (it.row0 + min(w0 + 31, it.rows - 1)) / G;
        const int myrow = it.row0 + min(w0 + col, it.rows - 1);  // (rows past the tile repeat its last)
        const int ppos = ctx + myrow / G;

        // Staging.  A wave's chunks of K are 8 dimensions of keys kr0 + i KSTEP of the visit each, of V 8
        // keys of dimensions vd0 + 32 i, all chunk i of one group of 16 keys and so of one page:
        // addresses are a uniform base and the lane's fixed offset.  A page id is read a pair ahead
        // of its request, that a pair ahead of its store.  Past the item's ends the nearest visit is
        // staged again, unused: with no branch around a load the waits count only what they need.
        Raw<T> sk[L::TASKS], sv[L::TASKS];
        int pk[L::TASKS], pv;
        bool bad_id = false;
        auto key_of = [&](int n) { return vis.key(it.v0 + max(0, min(n, it.nv - 1))); };
        // the keys of visits m - 1, m and m + 1 where pair m (V of m - 1, K of m) is fetched next, and
        // of V's visit in the pair fetched last
        int k0 = key_of(-1), k1 = key_of(0), k2 = key_of(1), kstored = k0;
        // (past the sequence: the visit's first group again)
        auto group_key = [&](int j0, int grp16) { return j0 + 16 * grp16 < len ? j0 + 16 * grp16 : j0; };
        auto sound = [&](int page) {  // (looked at when it is used: its load has a pair to arrive in)
            const uint32_t pg = (uint32_t)__builtin_amdgcn_readfirstlane(page);
            bad_id |= pg >= (uint32_t)c.n_pages;
            return min(pg, (uint32_t)c.n_pages - 1);
        };
        auto kgroup = [&](int i) { return (wv * KROWS + i * KSTEP) / 16; };
        const T* kbase = static_cast<const T*>(c.k) + ((int64_t)g << (shift + LOG_D));
        const T* vbase = static_cast<const T*>(c.v) + ((int64_t)g << (shift + LOG_D));
        const uint32_t page_elems = (uint32_t)KVH << (shift + LOG_D);
        auto read_pages = [&](int jk, int jv) {
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i) pk[i] = pages[group_key(jk, kgroup(i)) >> shift];
            pv = pages[group_key(jv, vgroup) >> shift];
        };
        auto fetch_k = [&](int i) {
            const uint32_t at = (uint32_t)group_key(k1, kgroup(i)) & (uint32_t)(ps - 1);
            sk[i] = load8<T>(kbase + ((uint64_t)sound(pk[i]) * page_elems + (at << LOG_D)) +
                             (klane + (KSTEP == 8 ? i % 2 * 8 * D : 0)));
        };
        auto fetch_v = [&] {
            const uint32_t at = (uint32_t)group_key(k0, vgroup) & (uint32_t)(ps - 1);
            const T* from = vbase + ((uint64_t)sound(pv) * page_elems + at);
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i) sv[i] = load8<T>(from + (32 * i << shift) + vlane);
        };
        auto fetch_pages = [&](int m) {  // of pair m + 1, after pair m's requests
            read_pages(k2, k1);
            kstored = k0;
            k0 = k1;
            k1 = k2;
            k2 = key_of(m + 2);
        };
        // pair m in four pieces, to go between MFMAs
        auto fetch_piece = [&](int m, int piece) {
            constexpr int HALF_T = (L::TASKS + 1) / 2;
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i)
                if (piece == (i < HALF_T ? 0 : 1)) fetch_k(i);
            if (piece == 2) fetch_v();
            if (piece == 3) fetch_pages(m);
        };
        auto fetch = [&](int m) {
#pragma unroll
            for (int piece = 0; piece < 4; ++piece) fetch_piece(m, piece);
        };
        auto store = [&](int m) {
            uint8_t* buf = lds + m % GR * L::PAIR;
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i) {
                u32x4 p[P::K];
                split_k<T>(sk[i], p);
                // (a chunk step of 8 rows turns bit 3 of the slot)
                const uint32_t at = (KSTEP == 8 && i % 2 ? kto ^ 128 : kto) + i * KSTEP * L::KROW;
#pragma unroll
                for (int x = 0; x < P::K; ++x) *reinterpret_cast<u32x4*>(buf + L::K + x * L::PLANE + at) = p[x];
            }
            const int left = len - kstored;  // keys of V's visit and on
            if (left < U) {                  // past the sequence's end a page holds anything
                constexpr int E = 4 / sizeof(T);
                const int mine = left - 16 * vgroup - 8 * (lane & 1);
#pragma unroll
                for (int i = 0; i < L::TASKS; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t& w = reinterpret_cast<uint32_t*>(&sv[i])[e / E];
                        const uint32_t keep = E == 1 ? 0u : e % 2 ? 0xFFFFu : 0xFFFF0000u;
                        w = e >= mine ? w & keep : w;
                    }
            }
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i) {
                u32x4 p[P::K];
                split_k<T>(sv[i], p);
#pragma unroll
                for (int x = 0; x < P::K; ++x)
                    *reinterpret_cast<u32x4*>(buf + L::V + x * L::PLANE + vto + 32 * i * L::VROW) = p[x];
                if constexpr (std::is_same_v<T, f16_t>) {
                    // (a chunk at a time behind its store: all before the stores costs hd 256 3 %, hd 64 3 % more)
                    u16x2 top = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, p[0][j] & 0x7FFF7FFFu));
                    atomicMax(&vtop[lane], max((int)top[0], (int)top[1]));
                }
            }
        };
        read_pages(k1, k0);
        fetch(0);

        u32x4 q[L::QREGS][NB];
        u32x4* ql = reinterpret_cast<u32x4*>(lds + L::QL) + (wv * (NB - L::QL0) - L::QL0) * 64 + lane;
        __syncthreads();  // (the item before is done with the LDS)
        if (tid == 0) flags[0] = 0;
        if (std::is_same_v<T, f16_t> && tid < 64) vtop[tid] = 0;
        float inv = 1.0f;
        // The wave's rows of q and of their rotations come whole rows at a time and through its own
        // part of the LDS: a lane's operand is 32 bytes of a row, and loaded so every request would
        // touch 32 lines (22000 cycles an item at hd 128 before, of 115000).
        u32x4 qfirst;
        {
            // (opaque lane numbers here and at the end: no address of these is kept through the visits)
            int el = lane;
            asm volatile("" : "+v"(el));
            constexpr int CH = D / 4, N = 32 * CH / 64;  // 16-byte chunks of a row, requests of 32 rows
            f32x4* own = reinterpret_cast<f32x4*>(lds + wv * L::QROWS);
            auto slot = [&](int r, int ch) { return r * CH + (ch ^ (r & (CH - 1 < 31 ? CH - 1 : 31))); };
            // (requests at once: with all 32 of hd 256 the compiler spills, tuples of four in two places,
            // and reads one back wrong)
            constexpr int NX = N < 16 ? N : 16;
            // (a lane's own row is `myrow`: its place is handed to the lanes that load it)
            auto rows = [&](const float* from, int64_t place) {
#pragma unroll
                for (int i0 = 0; i0 < N; i0 += NX) {
                    f32x4 x[NX];
#pragma unroll
                    for (int i = 0; i < NX; ++i)
                        x[i] = reinterpret_cast<const f32x4*>(
                            from + __shfl(place, ((i0 + i) * 64 + el) / CH, 64))[el % CH];
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < NX; ++i) own[slot(((i0 + i) * 64 + el) / CH, el % CH)] = x[i];
                    __builtin_amdgcn_sched_barrier(0);
                }
                settle_wave();
            };
            f32x8 r[NB];
            const int64_t myq = first + myrow / G;
            rows(a.qkv, myq * a.qstride + (int64_t)(g * G + myrow % G) * D);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const f32x4 v = own[slot(el % 32, 4 * b + 2 * (el / 32) + k)];
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[b][4 * k + j] = v[j];
                }
            settle_wave();
            rows(reinterpret_cast<const float*>(a.turn), myq * D);
            const float scale = kLog2e / sqrtf((float)D);
#pragma unroll
            for (int b = 0; b < NB / 2; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x4 v = own[slot(el % 32, 8 * b + 4 * (el / 32) + k)];  // two (cos, sin)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float uu = r[b][2 * k + j], ww = r[b + NB / 2][2 * k + j];
                        r[b][2 * k + j] = (uu * v[2 * j] - ww * v[2 * j + 1]) * scale;
                        r[b + NB / 2][2 * k + j] = (uu * v[2 * j + 1] + ww * v[2 * j]) * scale;
                    }
                }
            float up = 1.0f;
            if (std::is_same_v<T, f16_t>) {
                float amax = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(r[b][j]));
                amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
                const float2 sc = row_scale(amax);
                up = sc.x;
                inv = sc.y;
            }
            __syncthreads();  // (every wave is done with its rows: the buffers and q's last parts go there)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (std::is_same_v<T, f16_t>) r[b] *= up;
                u32x4 p[P::Q];
                split_q<T>(r[b], p);
#pragma unroll
                for (int i = 0; i < L::QREGS; ++i) q[i][b] = p[i];
                if (L::kQl && b < L::QL0) qfirst = p[P::Q - 1];
                else if (L::kQl) ql[b * 64] = p[P::Q - 1];
            }
        }
        float ref = -INFINITY, l = 0.0f;
        f32x16 o[OT];
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;

        store(0);
        fetch(1);
        __syncthreads();
        if (grp == 1) {  // (a phase behind)
            if (!kStoreEarly) {
                store(1);
                fetch(2);
            }
            __syncthreads();
        }
        // s = q k of visit n: operands read ahead of the MFMAs of the block before (chunk 2 b + hf of a
        // row: the swizzle is an XOR, so b's bits can be turned last).  Every wave forms all its
        // products, seen or not: the phase lasts as long as the longest wave's.
        f32x16 s[NG];
        auto scores = [&](int n) {
            const uint8_t* buf = lds + n % GR * L::PAIR;
            uint32_t ka = kat;  // (opaque: no address is kept across visits, nor 32 zeros)
            float zero = 0.0f;
            asm volatile("" : "+v"(ka), "+v"(zero));
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[u][e] = zero;
            u32x4 kp[2][NG][P::K], qx[2];
            auto read = [&](int b) {
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int x = 0; x < P::K; ++x)
                        kp[b % 2][u][x] = *reinterpret_cast<const u32x4*>(
                            buf + L::K + x * L::PLANE + 32 * u * L::KROW + (ka ^ 32 * b));
                if (L::kQl) qx[b % 2] = b < L::QL0 ? qfirst : ql[b * 64];
            };
            read(0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b + 1 < NB) read(b + 1);
                if (kStoreEarly && b % (NB / 4) == 0) fetch_piece(n + 2, b / (NB / 4));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < P::N; ++x)
#pragma unroll
                    for (int u = 0; u < NG; ++u) {
                        const u32x4 y = P::qi[x] < L::QREGS ? q[P::qi[x] < L::QREGS ? P::qi[x] : 0][b] : qx[b % 2];
                        s[u] = mfma32<T>(kp[b % 2][u][P::ki[x]], y, s[u]);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (kStoreEarly) store(1);
        scores(0);
        __syncthreads();  // the first matrix phase ends
        for (int n = 0;; ++n) {
            const int j0 = vis.key(it.v0 + n);
            u32x4 p[NG][2][P::Q];
            {
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < NG; ++u) {
                    const int ju = j0 + 32 * u;
                    const bool all = ju + 31 <= wmin &&
                                     (a.window == 0 || ju > wmax - a.window || ju + 32 <= a.sinks);
                    if (!all) {
                        const int at = ppos - ju - 8 * hf, far = a.window > 0 ? at - a.window : INT_MIN;
                        const int sk0 = a.sinks - ju - 8 * hf;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int j = 16 * (e / 8) + e % 8;
                            const bool hidden = (j > at) | ((j <= far) & (j >= sk0));
                            s[u][e] = hidden ? -INFINITY : s[u][e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
                }
                if (std::is_same_v<T, f16_t>) top *= inv;  // (a power of two)
                if (__any(top > ref + P::slack)) {
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float to = fmaxf(ref, top);
                    const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - to);
                    l *= f;
#pragma unroll
                    for (int i = 0; i < OT; ++i) o[i] *= f;
                    ref = to;
                }
                const float from = ref == -INFINITY ? 0.0f : ref - P::shift;
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        f32x8 w;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            w[e] = __builtin_amdgcn_exp2f(fmaf(s[u][8 * k + e], inv, -from));
                            l += w[e];
                        }
                        split_w<T>(w, p[u][k]);
                    }
            }
            if (!kStoreEarly) store(n + 1 + grp);
            __syncthreads();  // the vector phase ends
            // (where the matrix phase is the longer one, its wave goes first on the SIMD: three chunks
            // among 24 sequences, bf16, 169 us against 175; at hd 64, f16, 233 against 224)
            if (!kStoreEarly) __builtin_amdgcn_s_setprio(1);
            {
                // o += p v of visit n.  Step i: dimensions 32 (i % OT) .., keys of MFMA i / OT
                const uint8_t* buf = lds + (n + 1) % GR * L::PAIR;
                uint32_t va = vat;
                asm volatile("" : "+v"(va));
                u32x4 vp[2][P::K];
                auto read = [&](int i) {
#pragma unroll
                    for (int x = 0; x < P::K; ++x)
                        vp[i % 2][x] = *reinterpret_cast<const u32x4*>(
                            buf + L::V + x * L::PLANE + 32 * (i % OT) * L::VROW + (va ^ 32 * (i / OT)));
                };
                read(0);
#pragma unroll
                for (int i = 0; i < 2 * NG * OT; ++i) {
                    if (i + 1 < 2 * NG * OT) read(i + 1);
                    // (what is stored next is requested between the first MFMAs after the stores before)
                    if (!kStoreEarly && i % (NG * OT / 2) == 0) fetch_piece(n + 2 + grp, i / (NG * OT / 2));
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int x = 0; x < P::N; ++x)
                        o[i % OT] = mfma32<T>(vp[i % 2][P::ki[x]], p[i / OT / 2][i / OT % 2][P::qi[x]], o[i % OT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (n + 1 == it.nv) {
                __builtin_amdgcn_s_setprio(0);
                break;
            }
            if (kStoreEarly) store(n + 2);
            scores(n + 1);
            if (!kStoreEarly) __builtin_amdgcn_s_setprio(0);
            __syncthreads();  // the matrix phase ends
        }
        if (GR == 2) {  // (both groups pass 2 nv + 2 barriers from the first pair on)
            __syncthreads();
            if (grp == 0) __syncthreads();
        }
        if (bad_id) flags[0] = 1;
        __syncthreads();

        const bool whole = it.S == 1;
        const bool mine = w0 + col < it.rows;
        l += __shfl_xor(l, 32, 64);
        const float inv_l = 1.0f / l;
        float chk = l * 0.0f;
        if constexpr (std::is_same_v<T, f16_t>) {
            // Weights in two parts are off by up to 2^-25, and a row's sums by that times the item's keys and
            // V's largest magnitude: a row whose largest sum may have lost too much is done again.
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < OT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(o[i][e]));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            const float vmax = wave_max((float)__builtin_bit_cast(f16_t, (uint16_t)vtop[lane]));
            if (l > 0.0f && most * kLoss < vmax * ((float)min(it.nv * U, kLossKeys) * 0x1p-25f)) chk = 1.0f;
        }
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                // the quotient: the rounded product, corrected by its remainder
                const float y = o[i][e] * inv_l;
                if (whole) o[i][e] = fmaf(fmaf(-y, l, o[i][e]), inv_l, y);
                chk = fmaf(o[i][e], 0.0f, chk);
            }
        bool bad = mine && chk != 0.0f;
        bad |= (bool)__shfl_xor((int)bad, 32, 64);  // (both halves of a row)
        const bool bad_page = flags[0] != 0;
        if (bad_page && tid == 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesBadState);
        const bool again = mine && !bad_page && bad;
        const int64_t piece = (int64_t)it.base + ((int64_t)g * it.S + it.s) * it.rows;
        if (mine && hf == 0) {
            const int rr = it.row0 + w0 + col;
            if (again) redo_row(a, first + rr / G, g * G + rr % G);
            if (!whole)
                a.ms[piece + w0 + col] = make_float2(ref - P::shift, again || bad_page ? __builtin_nanf("") : l);
        }
        // whole rows out, through the wave's part of the LDS (a row with a bad page is NaN, whatever its
        // other pieces hold)
        const uint32_t skip = (uint32_t)__ballot(again);
        constexpr int CH = D / 4, N = 32 * CH / 64;
        int el = lane;
        asm volatile("" : "+v"(el));
        f32x4* own = reinterpret_cast<f32x4*>(lds + wv * L::QROWS);
        auto slot = [&](int r, int ch) { return r * CH + (ch ^ (r & (CH - 1 < 31 ? CH - 1 : 31))); };
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                own[slot(el % 32, 8 * i + 2 * u + el / 32)] =
                    f32x4{o[i][4 * u], o[i][4 * u + 1], o[i][4 * u + 2], o[i][4 * u + 3]};
        settle_wave();
        const bool direct = whole || bad_page;
        float* to = direct ? a.out : a.po;
        const int64_t place = direct ? (int64_t)(first + myrow / G) * a.ostride + (int64_t)(g * G + myrow % G) * D
                                     : (piece + w0 + col) * D;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (i * 64 + el) / CH;
            float* dst = to + __shfl(place, r, 64) + el % CH * 4;
            const f32x4 v = own[slot(r, el % CH)];
            if (w0 + r < it.rows && !(skip >> r & 1))
                *reinterpret_cast<f32x4*>(dst) = bad_page ? f32x4(__builtin_nanf("")) : v;
        }
    }
}

// One row and head by a wave, in plain f32: for rows whose products of parts came out non-finite
// (an infinity times a part that is 0, also where a mask hides it) or lost too much.  Bound by the
// latency of its loads: all rows of a 2048-token prompt of 32 heads of 128, f16, 5.0 ms (an infinite
// value in the first position; 0.37 where a NaN key ends each row early).  qf: LDS [D], the query;
// sc: LDS [64].  Lane el gets dimensions el + 64 i of out.
template <class T, int D>
__device__ void attend_row(const PagedKv& c, const Call& a, const int* pages, int row, int h, int p,
                           float* qf, float* sc, float (&acc)[D / 64]) {
    constexpr int U = 64;
    const int el = threadIdx.x & 63, g = h / a.G;
    const int64_t ps = c.page_size;
    auto settle = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    bool bad = false;
    auto page_of = [&](int j) {
        const int pg = pages[j >> c.page_shift];
        if ((unsigned)pg < (unsigned)c.n_pages) return (int64_t)pg;
        bad = true;
        return (int64_t)0;
    };
    settle();
    if (el < D / 8) {
        const f32x8 v = rotated8<D>(a, row, g, h % a.G, 8 * el);
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[8 * el + j] = v[j];
    }
    settle();
    float mx = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.0f;
    const Visits<U> vis(p, p, a.window, a.sinks);
    for (int v = 0; v < vis.count && !(l != l); ++v) {  // (a NaN sum stays one)
        const int j0 = vis.key(v);
        for (int i = 0; i < U / 8; ++i) {  // 8 lanes a key
            const int j = min(j0 + 8 * i + el / 8, p);
            const T* kr = static_cast<const T*>(c.k) +
                          ((page_of(j) * a.KVH + g) * ps + (j & (ps - 1))) * D + el % 8 * (D / 8);
            float dot = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 8; d += 8) {
                const Raw<T> x = load8<T>(kr + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = fmaf(widen(element<T>(x, e)), qf[el % 8 * (D / 8) + d + e], dot);
            }
            dot += __shfl_xor(dot, 1, 64);
            dot += __shfl_xor(dot, 2, 64);
            dot += __shfl_xor(dot, 4, 64);
            if (el % 8 == 0) sc[8 * i + el / 8] = dot;
        }
        settle();
        const int j = j0 + el;
        const bool seen = j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
        const float s = seen ? sc[el] : -INFINITY;
        const float mnew = fmaxf(mx, wave_max(s));
        const float alpha = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mnew);
        const float w = s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - mnew);
        l = l * alpha + wave_add(w);
        mx = mnew;
        settle();
        sc[el] = w;
        settle();
        const uint64_t mask = __ballot(seen);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) acc[i] *= alpha;
        for (int u = 0; u < U / 8; ++u) {
            if ((mask >> (8 * u) & 0xFF) == 0) continue;
            const int j8 = j0 + 8 * u;
            const T* vr = static_cast<const T*>(c.v) + (page_of(j8) * a.KVH + g) * D * ps + (j8 & (ps - 1));
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const Raw<T> x = load8<T>(vr + (el + 64 * i) * ps);
#pragma unroll
                for (int e = 0; e < 8; ++e)  // (a hidden key's value may be anything)
                    if (mask >> (8 * u + e) & 1) acc[i] = fmaf(sc[8 * u + e], widen(element<T>(x, e)), acc[i]);
            }
        }
        settle();
    }
    if (__any(bad)) l = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = l != l ? l : acc[i] / l;
}

// The last kernel of a call.  The pieces of a tile dealt out, joined: out = sum_s 2^(M_s - M) o_s /
// sum_s 2^(M_s - M) l_s over the pieces' (M_s, l_s, o_s); a piece in which a row sees no key has M_s = -inf, weight 0.  A
// workgroup per (16 rows of a tile, kv head), D / 4 threads to a row; where there are fewer rows
// than such groups, several share a row's pieces and meet in LDS.  A row with a piece of NaN sum
// is left: its output is written (a bad page), or it is one of the rows listed to be done again,
// which follow.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedKv c, PageTable t, Call a) {
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
    const int again = *a.redo_count;
    if (again == 0) return;
    __shared__ float rows[4][D + 64];
    const int wv = threadIdx.x / 64, B = t.counts[kPagesEntries];
    for (int i = (int)blockIdx.x * 4 + wv; i < again; i += (int)gridDim.x * 4) {
        const int row = a.redo[i] / a.H, h = a.redo[i] % a.H;
        int lo = 0, hi = B;  // its entry
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (t.cu[mid] <= row) lo = mid;
            else hi = mid;
        }
        const int p = t.step_lens[lo] - t.cu[lo + 1] + row;
        float acc[D / 64];
        attend_row<T, D>(c, a, t.table + (int64_t)t.step_ids[lo] * t.max_pages, row, h, p, rows[wv],
                         rows[wv] + D, acc);
        float* o = a.out + row * a.ostride + (int64_t)h * D + (threadIdx.x & 63);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[64 * e] = acc[e];
    }
}

// How a call's workspace is laid out, and its grids.
struct Layout {
    int64_t items[2], rows[2];
    size_t head_at[2], items_at[2], splits_at[2], turn_at, ms_at, po_at, count_at, redo_at, bytes;
};

// Workgroups of a kind that the device holds: wide one a CU, narrow by its registers.
int places(int kind, int64_t D) {
    return (kind == kWide || D == 256 ? 1 : D == 128 ? 2 : 3) * device_info().cu_count;
}
// Pieces a kind's work is dealt out in at most.
int target_pieces(int kind) { return (kind == kNarrow ? 3 : 1) * device_info().cu_count; }

int tile_rows(int kind, int64_t D) { return kind == kNarrow ? kTileRows : D < 256 ? 256 : 128; }

Layout layout(const PagedKv& c, const unillm_page_table& t, int64_t n, int64_t H) {
    const int64_t KVH = c.n_kv_heads, G = H / KVH, D = c.head_dim;
    Layout l;
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += ((size_t)bytes + 255) & ~(size_t)255;
        return here;
    };
    for (int k = 0; k < 2; ++k) {
        // tiles: an entry's last may be ragged (a wide entry has more than kNarrowRows rows).  A
        // tile of nv visits makes at most nv / C + 1 pieces, and the nv / C add up to target /
        // KVH; more than one piece, at most 2 nv / C.
        const int64_t entries = std::min<int64_t>(k == kNarrow ? n : n * G / (kNarrowRows + 1),
                                                  t.st.max_seqs);
        const int64_t tiles = n * G / tile_rows(k, D) + entries;
        const bool some = k == kNarrow || n * G > kNarrowRows;
        l.items[k] = some ? tiles + target_pieces(k) / KVH + 1 : 0;
        l.rows[k] = some ? 2 * (int64_t)target_pieces(k) * std::min<int64_t>(tile_rows(k, D), n * G) : 0;
        l.head_at[k] = take(2 * sizeof(int));
        l.items_at[k] = take(l.items[k] * (int64_t)sizeof(Item));
        l.splits_at[k] = take(tiles * (int64_t)sizeof(Split));
    }
    l.turn_at = take(n * D / 2 * (int64_t)sizeof(float2));
    l.ms_at = take((l.rows[0] + l.rows[1]) * (int64_t)sizeof(float2));
    l.po_at = take((l.rows[0] + l.rows[1]) * D * (int64_t)sizeof(float));
    // rows to do again: every (row, head), and again for each piece
    l.count_at = take(sizeof(int));
    l.redo_at = take((n * H + l.rows[0] + l.rows[1]) * (int64_t)sizeof(int));
    l.bytes = at;
    return l;
}

template <class T, int D>
hipError_t launch_typed(const PagedKv& c, const unillm_page_table& t, const Call& a, const Layout& l,
                        hipStream_t s) {
    using L = NarrowLds<T, D>;
    using LW = WideLds<T, D>;
    static const bool attr =
        hipFuncSetAttribute((const void*)paged_narrow_kernel<T, D>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, L::BYTES) == hipSuccess &&
        hipFuncSetAttribute((const void*)paged_wide_kernel<T, D>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, LW::BYTES) == hipSuccess &&
        hipFuncSetAttribute((const void*)paged_append_kernel<T, D>,
                            hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)((3 * kPagesMaxSeqs + 1) * sizeof(int))) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    // (the plan keeps three ints an entry in LDS)
    const size_t plan_lds = (size_t)(3 * t.st.max_seqs + 1) * sizeof(int);
    // kv heads a workgroup: one, or what makes four workgroups a CU
    const int nr = a.n <= 512 ? 4 : kAppendRows;
    const int64_t blocks = (a.n + nr - 1) / nr, most = 4 * device_info().cu_count;
    const int heads = (int)std::min<int64_t>(a.KVH, std::max<int64_t>(1, blocks * a.KVH / most));
    const int64_t append = blocks * ((a.KVH + heads - 1) / heads);
    paged_append_kernel<T, D><<<(unsigned)(2 + append), 256, plan_lds, s>>>(c, t.st, a, nr, heads);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (l.items[kWide] > 0) {
        const unsigned grid = (unsigned)std::min<int64_t>(l.items[kWide] * a.KVH, 4 * most);
        paged_wide_kernel<T, D><<<grid, LW::NT, LW::BYTES, s>>>(c, t.st, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const unsigned grid = (unsigned)std::min<int64_t>(l.items[kNarrow] * a.KVH, most);
    paged_narrow_kernel<T, D><<<grid, 256, L::BYTES, s>>>(c, t.st, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    paged_merge_kernel<T, D><<<(unsigned)std::min<int64_t>((l.rows[0] + l.rows[1]) / 2, most), 256, 0, s>>>(
        c, t.st, a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_type(const PagedKv& c, const unillm_page_table& t, const Call& a, const Layout& l,
                       hipStream_t s) {
    if (c.head_dim == 64) return launch_typed<T, 64>(c, t, a, l, s);
    if (c.head_dim == 128) return launch_typed<T, 128>(c, t, a, l, s);
    return launch_typed<T, 256>(c, t, a, l, s);
}

}  // namespace

hipError_t launch_paged_attention(const PagedKv& c, const unillm_page_table& t, const float* qkv,
                                  int64_t qstride, int64_t n, int64_t H, int64_t window,
                                  int64_t sinks, float* out, int64_t ostride, hipStream_t s) {
    const Layout l = layout(c, t, n, H);
    void* ws = nullptr;
    hipError_t e = stream_workspace(s, l.bytes, &ws, kPagedSlot);
    if (e != hipSuccess) return e;
    uint8_t* w = static_cast<uint8_t*>(ws);
    // a window or sinks past any position are all of them
    const int64_t far = (int64_t)1 << 30;
    Call a{qkv, out, qstride, ostride, (int)n, (int)H, (int)c.n_kv_heads, (int)(H / c.n_kv_heads),
           (int)std::min(window, far), (int)std::min(sinks, far),
           reinterpret_cast<float2*>(w + l.turn_at), reinterpret_cast<float2*>(w + l.ms_at),
           reinterpret_cast<float*>(w + l.po_at), reinterpret_cast<int*>(w + l.count_at),
           reinterpret_cast<int*>(w + l.redo_at), {}};
    for (int k = 0; k < 2; ++k)
        a.kind[k] = {tile_rows(k, c.head_dim), places(k, c.head_dim), target_pieces(k),
                     k == kNarrow ? 4 : 2, 5, k == kNarrow ? 0 : (int)l.rows[0],
                     reinterpret_cast<int*>(w + l.head_at[k]), reinterpret_cast<Item*>(w + l.items_at[k]),
                     reinterpret_cast<Split*>(w + l.splits_at[k])};
    if (c.type == UNILLM_QTYPE_F32) return launch_type<float>(c, t, a, l, s);
    if (c.type == UNILLM_QTYPE_F16) return launch_type<f16_t>(c, t, a, l, s);
    return launch_type<bf16_t>(c, t, a, l, s);
}

size_t paged_workspace_bytes(const PagedKv& c, const unillm_page_table& t, int64_t n, int64_t H) {
    return layout(c, t, n, H).bytes;
}

}  // namespace unillm
