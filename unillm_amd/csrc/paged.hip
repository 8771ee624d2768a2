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

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// One piece of a call's work: the visits v0 .. v0 + nv - 1 of a tile of `rows` query rows
// (row r of an entry is head r % G of its token r / G, for each kv head).  Of a tile dealt out
// in S > 1 pieces this is piece s; its partial sums go to rows base + (g S + s) rows + r.
struct Item {
    int entry, row0, rows, v0, nv, base, s, S;
};
// A tile dealt out, for the merge.
struct Split {
    int entry, row0, rows, base, S, pad[3];
};

// What the kernels of a call share.
struct Call {
    const float* qkv;
    float* out;
    int64_t qstride, ostride;
    int n, H, KVH, G;
    int window, sinks;
    int target;     // pieces to deal the call's work out in, over all kv heads
    int most_rows;  // partial rows there is room for
    int* head;      // [0] items, [1] splits
    Item* items;
    Split* splits;
    float2* turn;   // [n][hd / 2] cos, sin of each row's angles
    float2* ms;     // [most_rows] maximum (log2), sum of the weights
    float* po;      // [most_rows][hd] unnormalized sums
};

constexpr int kTileRows = 16;  // query rows of a tile
constexpr int kUnit = 32;      // keys of a visit

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

// Inclusive sums of two ints over 256 threads (tmp: [4]).
__device__ __forceinline__ int2 block_scan2(int2 v, int2* tmp) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(v.x, o, 64), y = __shfl_up(v.y, o, 64);
        if (lane >= o) v.x += x, v.y += y;
    }
    if (lane == 63) tmp[w] = v;
    __syncthreads();
    int2 base = make_int2(0, 0);
    for (int i = 0; i < w; ++i) base.x += tmp[i].x, base.y += tmp[i].y;
    __syncthreads();
    return make_int2(v.x + base.x, v.y + base.y);
}

// Deals the step's work out (one workgroup): every entry's rows in tiles of kTileRows, every
// tile's visits in equal pieces of at most C, where C makes a.target pieces over all kv heads.
// tp: LDS [entries + 1].
__device__ void plan(const PageTable& t, const Call& a, int* tp, int2* tmp) {
    const int tid = threadIdx.x, B = t.counts[kPagesEntries];
    int carry = 0;
    if (tid == 0) tp[0] = 0;
    for (int b0 = 0; b0 < B; b0 += 256) {
        const int b = b0 + tid;
        const int m = b < B ? t.cu[b + 1] - t.cu[b] : 0;
        const int2 s = block_scan2(make_int2((m * a.G + kTileRows - 1) / kTileRows, 0), tmp);
        if (b < B) tp[b + 1] = carry + s.x;
        __syncthreads();
        carry = tp[min(b0 + 256, B)];
    }
    const int tiles = carry;
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
        const int m = t.cu[lo + 1] - t.cu[lo], ctx = t.step_lens[lo] - m;
        Tile x{lo, (i - tp[lo]) * kTileRows, 0, 0};
        x.rows = min(kTileRows, m * a.G - x.row0);
        x.nv = Visits<kUnit>(ctx + x.row0 / a.G, ctx + (x.row0 + x.rows - 1) / a.G, a.window, a.sinks).count;
        return x;
    };
    // (visits of a call: below 2^31 / 32 keys a tile; their sum in f32 is exact enough to divide)
    float sum = 0.0f;
    for (int i = tid; i < tiles; i += 256) sum += (float)tile(i).nv;
    sum = wave_add(sum);
    __shared__ float part[4];
    __syncthreads();
    if ((tid & 63) == 0) part[tid >> 6] = sum;
    __syncthreads();
    const float all = (part[0] + part[1]) + (part[2] + part[3]);
    const int C = max(4, (int)ceilf(all * (float)a.KVH / (float)a.target));
    int items = 0, splits = 0, rows = 0;
    for (int i0 = 0; i0 < tiles; i0 += 256) {
        const int i = i0 + tid;
        Tile x{0, 0, 0, 0};
        int S = 0;
        if (i < tiles) {
            x = tile(i);
            S = (x.nv + C - 1) / C;
        }
        const int want = S > 1 ? S * a.KVH * x.rows : 0;
        const int2 r = block_scan2(make_int2(want, S > 1 ? 1 : 0), tmp);
        const int base = rows + r.x - want;
        if (S > 1 && base + want > a.most_rows) S = 1;  // (no room: whole)
        const int2 n = block_scan2(make_int2(S, 0), tmp);
        for (int s = 0; s < S; ++s) {
            const int v0 = (int)((int64_t)s * x.nv / S), v1 = (int)((int64_t)(s + 1) * x.nv / S);
            a.items[items + n.x - S + s] = {x.b, x.row0, x.rows, v0, v1 - v0, base, s, S};
        }
        if (want) a.splits[splits + r.y - 1] = {x.b, x.row0, x.rows, base, S, {}};
        __shared__ int last[3];
        if (tid == 255) {
            last[0] = n.x;
            last[1] = r.y;
            last[2] = r.x;
        }
        __syncthreads();
        items += last[0];
        splits += last[1];
        rows += last[2];
        __syncthreads();
    }
    if (tid == 0) {
        a.head[0] = items;
        a.head[1] = splits;
    }
}

// The first kernel of a call.  Workgroup 0 deals the work out; each other one takes R rows of
// the step: the rotation of their angles (kept for the queries), the keys rotated and stored,
// the values stored.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedKv c, PageTable t, Call a, int R) {
    constexpr int HALF = D / 2;
    __shared__ double2 turn[HALF];
    __shared__ int2 tmp[4];
    extern __shared__ int tp[];
    if (!step_fits(t, a.n)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) a.head[0] = a.head[1] = 0;
        fail_call(t, a, D, blockIdx.x, gridDim.x);
        return;
    }
    if (blockIdx.x == 0) {
        plan(t, a, tp, tmp);
        return;
    }
    const int total = t.counts[kPagesTokens];
    const int KVH = a.KVH;
    const int64_t ps = c.page_size;
    for (int r = 0; r < R; ++r) {
        const int row = ((int)blockIdx.x - 1) * R + r;
        if (row >= total) return;
        const int slot = t.slots[row];
        __syncthreads();
        if (threadIdx.x < HALF) {
            double sn, cs;
            sincospi((double)t.positions[row] * c.freq[threadIdx.x], &sn, &cs);
            turn[threadIdx.x] = make_double2(cs, sn);
            a.turn[(int64_t)row * HALF + threadIdx.x] = make_float2((float)cs, (float)sn);
        }
        __syncthreads();
        if (slot < 0) continue;
        const int64_t page = slot >> c.page_shift, off = slot & (c.page_size - 1);
        const float* xk = a.qkv + row * a.qstride + (int64_t)a.H * D;
        const float* xv = xk + (int64_t)KVH * D;
        for (int i = threadIdx.x; i < KVH * HALF; i += 256) {
            const int g = i / HALF, p = i % HALF;
            const double2 cs = turn[p];
            const double u = xk[g * D + p], v = xk[g * D + p + HALF];
            T* dst = static_cast<T*>(c.k) + ((page * KVH + g) * ps + off) * D;
            dst[p] = narrow<T>((float)(u * cs.x - v * cs.y));
            dst[p + HALF] = narrow<T>((float)(u * cs.y + v * cs.x));
        }
        for (int i = threadIdx.x; i < KVH * D; i += 256)
            static_cast<T*>(c.v)[(page * KVH * D + i) * ps + off] = narrow<T>(xv[i]);
    }
}

// ---- products at f32's precision ------------------------------------------------------------
//
// The 16-bit matrix cores run 16 times the f32 ones.  A value held in f16 or bf16 is its own
// single part.  f32 values are sums of parts: against bf16 (and f32, itself three bf16 parts) three
// bf16 ones, all 24 bits; against f16 two f16 ones, 22 bits, where a power of two per query
// row brings q into range (its largest magnitude in [2^14, 2^15)) and the weights, at most
// 2^8 above their reference (below), are taken times 2^7: parts down to 2^-24 then reach
// 2^-38 of a row's largest element and 2^-31 of the reference weight.
template <class T>
struct Parts;
template <>
struct Parts<f16_t> {
    static constexpr int K = 1, Q = 2, N = 2;
    static constexpr int ki[N] = {0, 0}, qi[N] = {1, 0};  // products, the large one last
    static constexpr float shift = 7.0f;
};
template <>
struct Parts<bf16_t> {
    static constexpr int K = 1, Q = 3, N = 3;
    static constexpr int ki[N] = {0, 0, 0}, qi[N] = {2, 1, 0};
    static constexpr float shift = 0.0f;
};
template <>
struct Parts<float> {
    static constexpr int K = 3, Q = 3, N = 6;
    static constexpr int ki[N] = {2, 0, 1, 1, 0, 0}, qi[N] = {0, 2, 1, 0, 1, 0};
    static constexpr float shift = 0.0f;
};

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

// One query row over an item's visits by a wave, in plain f32: for rows whose products of parts
// came out non-finite (an infinity times a part that is 0, or what a masked place holds).
// qf: LDS [D] for the query; sc: LDS [64].  Lane el gets dimensions el + 64 i of the
// unnormalized sum, with the maximum (log2) and the sum of the weights.
template <class T, int D, int U>
__device__ void attend_row(const PagedKv& c, const Call& a, const int* pages, const Visits<U>& vis,
                           const Item& it, int first, int ctx, int g, int r, float* qf, float* sc,
                           float& mx, float& l, float (&acc)[D / 64]) {
    const int el = threadIdx.x & 63;
    const int64_t ps = c.page_size;
    const int p = ctx + r / a.G;
    auto settle = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto page_of = [&](int j) {  // (ids out of range make the tile NaN elsewhere; never read)
        const int pg = pages[j >> c.page_shift];
        return (int64_t)((unsigned)pg < (unsigned)c.n_pages ? pg : 0);
    };
    settle();
    if (el < D / 8) {
        const f32x8 v = rotated8<D>(a, first, g, r, 8 * el);
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[8 * el + j] = v[j];
    }
    settle();
    mx = -INFINITY;
    l = 0.0f;
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.0f;
    for (int v = it.v0; v < it.v0 + it.nv; ++v) {
        const int j0 = vis.key(v);
        if (j0 > p) break;
        for (int i = 0; i < U / 8; ++i) {  // 8 lanes a key
            const int j = min(j0 + 8 * i + el / 8, p);
            const T* kr = static_cast<const T*>(c.k) +
                          ((page_of(j) * a.KVH + g) * ps + (j & (ps - 1))) * D + el % 8 * (D / 8);
            float dot = 0.0f;
            for (int d = 0; d < D / 8; ++d) dot = fmaf(widen(kr[d]), qf[el % 8 * (D / 8) + d], dot);
            dot += __shfl_xor(dot, 1, 64);
            dot += __shfl_xor(dot, 2, 64);
            dot += __shfl_xor(dot, 4, 64);
            if (el % 8 == 0) sc[8 * i + el / 8] = dot;
        }
        settle();
        const int j = j0 + el;
        const bool seen = el < U && j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
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
        for (int i = 0; i < D / 64; ++i) acc[i] *= alpha;
        for (int u = 0; u < U / 8; ++u) {
            if ((mask >> (8 * u) & 0xFF) == 0) continue;
            const int j8 = j0 + 8 * u;
            const T* vr = static_cast<const T*>(c.v) + (page_of(j8) * a.KVH + g) * D * ps + (j8 & (ps - 1));
            for (int e = 0; e < 8; ++e)
                if (mask >> (8 * u + e) & 1)
                    for (int i = 0; i < D / 64; ++i)
                        acc[i] = fmaf(sc[8 * u + e], widen(vr[(el + 64 * i) * ps + e]), acc[i]);
        }
        settle();
    }
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
// some score passes it by 2^8, so a visit needs no exchange between lanes; the sums of the
// weights stay per lane until the end.  Bound by HBM: 4 D bytes of a 16-bit pool a key.
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
    const int total = a.head[0] * KVH;
    for (int idx = blockIdx.x; idx < total; idx += gridDim.x) {
        const Item it = a.items[idx / KVH];
        const int g = idx % KVH;
        const int first = t.cu[it.entry], m = t.cu[it.entry + 1] - first;
        const int len = t.step_lens[it.entry], ctx = len - m;
        const int* pages = t.table + (int64_t)t.step_ids[it.entry] * t.max_pages;
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
                // masks, where some row of the tile does not see the whole visit
                const bool whole = j0 + kUnit - 1 <= pmin &&
                                   (a.window == 0 || j0 > pmax - a.window || j0 + kUnit <= a.sinks);
                if (!whole) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const int j = j0 + 8 * qd + r;
                        if (j > ppos || (a.window > 0 && j <= ppos - a.window && j >= a.sinks)) s[r] = -INFINITY;
                    }
                }
                float top = s[0];
#pragma unroll
                for (int r = 1; r < 8; ++r) top = fmaxf(top, s[r]);
                if (__any(top > ref + 8.0f)) {
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
                u32x4 p[P::Q];
                split_q<T>(s, p);
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
        const int redo = bad_page ? 0 : flags[1];
        if (bad_page) {
            sum = __builtin_nanf("");
            if (tid == 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesBadState);
        }
        const int r0 = it.row0 + col;
        const int64_t prow = (int64_t)it.base + ((int64_t)g * it.S + it.s) * it.rows + col;
        float* dst = whole ? a.out + (int64_t)(first + r0 / G) * a.ostride + (int64_t)(g * G + r0 % G) * D
                           : a.po + prow * D;
        if (live && !(redo >> col & 1)) {
#pragma unroll
            for (int i = 0; i < OT / 4; ++i)
                *reinterpret_cast<f32x4*>(dst + (4 * i + wv) * 16 + 4 * qd) =
                    bad_page ? f32x4(__builtin_nanf("")) : res[i];
            if (!whole && wv == 0 && qd == 0) a.ms[prow] = make_float2(top - P::shift, sum);
        }
        if (redo) {
            __syncthreads();
            float* qf = reinterpret_cast<float*>(lds + L::O) + wv * (D + 64);
            int left = redo, turn = 0;
            while (left) {
                const int r = __builtin_ctz(left);
                left &= left - 1;
                if (turn++ % 4 != wv) continue;
                float mx, sw, acc[D / 64];
                attend_row<T, D, kUnit>(c, a, pages, vis, it, first, ctx, g, it.row0 + r, qf, qf + D, mx, sw, acc);
                const int64_t pr = (int64_t)it.base + ((int64_t)g * it.S + it.s) * it.rows + r;
                const int rr = it.row0 + r;
                float* y = whole ? a.out + (int64_t)(first + rr / G) * a.ostride + (int64_t)(g * G + rr % G) * D
                                 : a.po + pr * D;
#pragma unroll
                for (int e = 0; e < D / 64; ++e) y[lane + 64 * e] = whole ? acc[e] / sw : acc[e];
                if (!whole && lane == 0) a.ms[pr] = make_float2(mx, sw);
            }
        }
    }
}

// The pieces of a tile dealt out, joined: out = sum_s 2^(M_s - M) o_s / sum_s 2^(M_s - M) l_s over the
// pieces' (M_s, l_s, o_s); a piece in which a row sees no key has M_s = -inf, weight 0.  A
// group of D / 4 threads per (tile, kv head, row).
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PageTable t, Call a) {
    constexpr int W = D / 4, N = 256 / W;
    const int d4 = threadIdx.x % W, sub = threadIdx.x / W;
    const int64_t per = (int64_t)a.KVH * kTileRows, total = (int64_t)a.head[1] * per;
    for (int64_t i = (int64_t)blockIdx.x * N + sub; i < total; i += (int64_t)gridDim.x * N) {
        const Split sp = a.splits[i / per];
        const int g = (int)(i % per) / kTileRows, r = (int)(i % kTileRows);
        if (r >= sp.rows || sp.S < 2) continue;
        const int64_t p0 = (int64_t)sp.base + (int64_t)g * sp.S * sp.rows + r;
        float M = -INFINITY;
        for (int s = 0; s < sp.S; ++s) M = fmaxf(M, a.ms[p0 + (int64_t)s * sp.rows].x);
        float l = 0.0f;
        f32x4 o = 0.0f;
        for (int s = 0; s < sp.S; ++s) {
            const int64_t p = p0 + (int64_t)s * sp.rows;
            const float2 x = a.ms[p];
            const float f = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - M);
            const f32x4 v = *reinterpret_cast<const f32x4*>(a.po + p * D + 4 * d4);
            l = fmaf(x.y, f, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], f, o[e]);
        }
        const int rr = sp.row0 + r;
        const int64_t row = t.cu[sp.entry] + rr / a.G;
        *reinterpret_cast<f32x4*>(a.out + row * a.ostride + (int64_t)(g * a.G + rr % a.G) * D + 4 * d4) = o / l;
    }
}

// How a call's workspace is laid out, and its grids.
struct Layout {
    int64_t items, most_rows;
    size_t items_at, splits_at, turn_at, ms_at, po_at, bytes;
};

// Pieces a call is dealt out in: four workgroups of four waves for every CU.
int target_pieces() { return 4 * device_info().cu_count; }

Layout layout(const PagedKv& c, const unillm_page_table& t, int64_t n, int64_t H) {
    const int64_t KVH = c.n_kv_heads, G = H / KVH, D = c.head_dim;
    Layout l;
    // tiles: an entry's last may be ragged.  A tile of nv visits makes at most nv / C + 1 pieces,
    // and the nv / C add up to target / KVH.
    const int64_t tiles = n * G / kTileRows + std::min<int64_t>(n, t.st.max_seqs);
    l.items = tiles + target_pieces() / KVH + 1;
    // a tile in more than one piece has at most 2 nv / C of them
    l.most_rows = 2 * (int64_t)target_pieces() * std::min<int64_t>(kTileRows, n * G);
    size_t at = 256;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += ((size_t)bytes + 255) & ~(size_t)255;
        return here;
    };
    l.items_at = take(l.items * (int64_t)sizeof(Item));
    l.splits_at = take(tiles * (int64_t)sizeof(Split));
    l.turn_at = take(n * D / 2 * (int64_t)sizeof(float2));
    l.ms_at = take(l.most_rows * (int64_t)sizeof(float2));
    l.po_at = take(l.most_rows * D * (int64_t)sizeof(float));
    l.bytes = at;
    return l;
}

template <class T, int D>
hipError_t launch_typed(const PagedKv& c, const unillm_page_table& t, const Call& a, const Layout& l,
                        hipStream_t s) {
    using L = NarrowLds<T, D>;
    static const bool attr =
        hipFuncSetAttribute((const void*)paged_narrow_kernel<T, D>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, L::BYTES) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    const int R = (int)std::max<int64_t>(1, std::min<int64_t>(16, a.n / 1024));
    // (the plan keeps a prefix sum of the entries in LDS)
    const size_t plan_lds = (size_t)(t.st.max_seqs + 1) * sizeof(int);
    paged_append_kernel<T, D><<<(unsigned)(1 + (a.n + R - 1) / R), 256, plan_lds, s>>>(c, t.st, a, R);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const unsigned grid = (unsigned)std::min<int64_t>(l.items * a.KVH, 1 << 16);
    paged_narrow_kernel<T, D><<<grid, 256, L::BYTES, s>>>(c, t.st, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const int64_t merged = (l.most_rows / 2 * (D / 4) + 255) / 256;
    paged_merge_kernel<D><<<(unsigned)std::min<int64_t>(merged, 4 * device_info().cu_count), 256, 0, s>>>(
        t.st, a);
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
    const Call a{qkv, out, qstride, ostride, (int)n, (int)H, (int)c.n_kv_heads, (int)(H / c.n_kv_heads),
                 (int)std::min(window, far), (int)std::min(sinks, far), target_pieces(),
                 (int)l.most_rows, reinterpret_cast<int*>(w), reinterpret_cast<Item*>(w + l.items_at),
                 reinterpret_cast<Split*>(w + l.splits_at), reinterpret_cast<float2*>(w + l.turn_at),
                 reinterpret_cast<float2*>(w + l.ms_at), reinterpret_cast<float*>(w + l.po_at)};
    if (c.type == UNILLM_QTYPE_F32) return launch_type<float>(c, t, a, l, s);
    if (c.type == UNILLM_QTYPE_F16) return launch_type<f16_t>(c, t, a, l, s);
    return launch_type<bf16_t>(c, t, a, l, s);
}

size_t paged_workspace_bytes(const PagedKv& c, const unillm_page_table& t, int64_t n, int64_t H) {
    return layout(c, t, n, H).bytes;
}

}  // namespace unillm
