// paged8.hip -- paged KV caches held in 8 bits: written, read back, attended.
//
// A pool's codes are int8 or e4m3, and 16 positions of a kv head share a power of two, so a code c of a
// block with byte b stands for c 2^(b - 127).  Powers of two: a block's exponent grows as further
// positions come, and its codes are rounded anew then.  Each growth at least doubles the step s, so an int8
// code's roundings add up to less than s however often it happens, s / 2 (1 + 1/2 + ..) (with the tightest step,
// growing by little each time, to several).  e4m3 codes have 4 significant bits, which a growth keeps until a code is
// below 2^-6: 2^-4 of the value, and less than 2^-9 s.  Values times a power of two, and codes rounded from them, are
// exact arithmetic: the same bits on every machine.
//
// Attention is that of paged.hip (its plan, pieces and merge are shared, paged.hpp):
//   out = sum_j w_j v_j / sum_j w_j,  w_j = e^(q k_j / sqrt(hd) - max).
// A code is exact in f16 and in bf16.  q k: codes in f16 against two f16 parts of q (22 bits), the block's
// power of two multiplied onto the scores.  w v: the weight times its block's power of two, in narrow tiles in
// three bf16 parts against codes in bf16, all 24 bits of it and of any size; in wide tiles, which the
// matrix cores bound, in two f16 parts against codes in f16.
#include <hip/hip_runtime.h>

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace unillm {
namespace {

constexpr int kBlock = 16;  // positions to an exponent
// Most query rows of an entry (a kv head) for narrow tiles.  (8 entries on 4000 keys, pages of 32, int8, us a call:
// hd 64, 8 kv heads, of 112 rows narrow 56, wide 64, of 160 rows 64 and 64; hd 128, 8 kv heads, of 80 rows 74 and
// 85, of 112 rows 90 and 86; hd 256, 4 kv heads, of 64 rows 67 and 84, of 80 rows 122 and 85.  e4m3 the
// same to 10 %.)
__host__ __device__ constexpr int narrow_rows(int64_t D) { return D == 64 ? 144 : D == 128 ? 96 : 64; }
struct Int8 {
    static constexpr float top = 127.0f, room = 127.0f / 128.0f;  // top = room 2^bits
    static constexpr int bits = 7;
};
struct E4m3 {
    static constexpr float top = 448.0f, room = 0.875f;
    static constexpr int bits = 9;
};

// The least byte with which values up to `top` fit.
template <class C>
__device__ __forceinline__ int least_exponent(float top) {
    if (!(top > 0.0f)) return 1;
    const int e = __builtin_amdgcn_frexp_expf(top) - C::bits + (__builtin_amdgcn_frexp_mantf(top) > C::room ? 1 : 0);
    return max(1, e + 127);
}
// A byte of the pool as the exponent it counts as (0 and 255, which no block is given, as 1 and 254).
__device__ __forceinline__ int counted(int b) { return min(max(b, 1), 254); }
// 2^(b - 127), and 2^(127 - b) of a counted b (of 254 a denormal, by which products are as exact)
__device__ __forceinline__ float power(int b) { return __uint_as_float((uint32_t)counted(b) << 23); }
__device__ __forceinline__ float inverse(int b) { return __uint_as_float(b < 254 ? (uint32_t)(254 - b) << 23 : 1u << 22); }

// Four values, in steps, as codes: to nearest even, infinities to the largest code, NaN to 0.
template <class C>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    auto cut = [](float v) { return v != v ? 0.0f : fminf(fmaxf(v, -C::top), C::top); };
    if constexpr (std::is_same_v<C, Int8>) {
        auto one = [&](float v) { return (uint32_t)(int)rintf(cut(v)) & 0xFF; };
        return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(cut(a), cut(b), 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cut(c), cut(d), w, true);
    }
}
template <class C, int E>
__device__ __forceinline__ float decode(uint32_t w) {
    if constexpr (std::is_same_v<C, Int8>) return (float)(int8_t)(w >> (8 * E) & 0xFF);
    else return __builtin_amdgcn_cvt_f32_fp8((int)w, E);
}
template <class C>
__device__ __forceinline__ f32x4 decode4(uint32_t w) {
    return f32x4{decode<C, 0>(w), decode<C, 1>(w), decode<C, 2>(w), decode<C, 3>(w)};
}
// Codes of a block whose step is 1 / f times as large now.
template <class C>
__device__ __forceinline__ uint32_t again4(uint32_t w, float f) {
    const f32x4 v = decode4<C>(w) * f;
    return encode4<C>(v[0], v[1], v[2], v[3]);
}

// A load of what is read once: it takes no place in the caches.  (32 sequences of 8192 keys, 8 kv heads of
// 128, pages of 32: 115 us a call, 139 with ordinary loads.  ONCE, below: whether V comes so.  A visit's 64 keys
// are half a line of V where a page is 128 positions or more, and the next wave reads the other half: on three
// sequences of 70001 to 100000 a call takes 117 us with ordinary loads of V there, 124 with these, 225 with
// these and neighbouring visits in one wave.  As two kernels: a branch around the loads costs 5 %.  The keys of an entry of
// more than one narrow tile are read again by the tiles' other items, and there these loads cost time: 80 sequences
// of up to 8750 keys, 32 heads on 8 of 128, e4m3, pages of 32, us a call with these and with ordinary loads: 16 rows
// an entry and kv head 87 and 91, 32 rows 142 and 120, 64 rows 248 and 195.)
template <class V>
__device__ __forceinline__ V once(const V* p) {
    return __builtin_nontemporal_load(p);
}

// ---- rows into their blocks -------------------------------------------------------------------
//
// Rows of consecutive slots in one block of 16 are a run: a wave writes a run of one kv head's keys, or
// values, whole, so no two waves meet in a block, and an exponent's byte is its own.
// Bound by HBM where rows are many: 4000 rows of 32 kv heads of 128, e4m3, 164 MB in 48 us, 3.4 TB/s (a copy 5.4:
// V goes out in 16-byte pieces of its lines); by the latency of dependent loads where they are few: 96 rows of 8
// heads 6 us.
constexpr int kWriteRows = 16;  // rows of a workgroup whose runs it takes, at most

template <int ROWS>
struct Runs {
    int slots[ROWS + 16];  // of row row0 - 1 + i, -1: none
    int first[ROWS], count[ROWS];  // those of several rows first
    int n, many, end;  // runs, those of several rows; rows from row0 on that they take in
};

// The runs that begin in rows row0 .. row0 + nr - 1, 64 at most (slot: of row row0 - 1 + threadIdx.x, up to nr +
// 16 of them).  All threads of the workgroup.
template <int ROWS>
__device__ __forceinline__ void find_runs(Runs<ROWS>& r, int slot, int nr) {
    static_assert(ROWS <= 64, "a wave looks at all");
    const int tid = threadIdx.x;
    if (tid < nr + 16) r.slots[tid] = slot;
    if (tid == 0) r.end = 0;
    __syncthreads();
    if (tid < 64) {
        const int sl = tid < nr ? r.slots[tid + 1] : -1;
        const bool begins = sl >= 0 && (r.slots[tid] + 1 != sl || sl % kBlock == 0);
        int n = begins ? 1 : 0;
        if (begins)
            while (sl % kBlock + n < kBlock && tid + 1 + n < nr + 16 && r.slots[tid + 1 + n] == sl + n) ++n;
        const uint64_t many = __ballot(n > 1), ones = __ballot(n == 1), before = (1ull << tid) - 1;
        if (begins) {
            const int at = n > 1 ? __popcll(many & before) : __popcll(many) + __popcll(ones & before);
            r.first[at] = tid;
            r.count[at] = n;
            atomicMax(&r.end, tid + n);
        }
        if (tid == 0) r.many = __popcll(many), r.n = __popcll(many | ones);
    }
    __syncthreads();
}

// The cosines and sines of `rows` rows (positions at: LDS), in turn [rows][R / 2], a row's pair p at (p % 4) R /
// 8 + p / 4: what lanes read together lies together.  A thread takes a pair of several rows; a position
// that follows the one before is that one's turn times a position's (f64, up to 7 times in a row: an angle off
// by 2^-50, where the position's product with the frequency has 2^-53 of itself; f64's sines are
// a third of a prompt's append otherwise: 4000 rows of 32 kv heads of 128, 61 us, 47 with no
// rotation at all).  All threads of the workgroup.
__device__ __forceinline__ void turns(const PagedKv8& c, const int* at, int rows, double2* turn) {
    const int pairs = c.rotary_dim / 2;
    if (pairs == 0) return;
    const int each = min(8, max(1, rows * pairs / 256)), sets = (rows + each - 1) / each;
    const double2* unit = reinterpret_cast<const double2*>(c.freq + pairs);
    for (int i = threadIdx.x; i < sets * pairs; i += 256) {
        const int p = i % pairs, r0 = i / pairs * each, to = p % 4 * (pairs / 4) + p / 4;
        const double f = c.freq[p];
        const double2 w = unit[p];
        double cs = 0.0, sn = 0.0;
        for (int r = r0; r < min(r0 + each, rows); ++r) {
            if (r > r0 && at[r] == at[r - 1] + 1) {
                const double x = cs * w.x - sn * w.y;
                sn = cs * w.y + sn * w.x;
                cs = x;
            } else {
                sincospi((double)at[r] * f, &sn, &cs);
            }
            turn[r * pairs + to] = make_double2(cs * c.magnitude, sn * c.magnitude);
        }
    }
    __syncthreads();
}

// Eight dimensions of a head, four at d0 and four at d1, that turn among themselves: unit u of D / 8.
struct Octet {
    f32x4 lo, hi;
};
__device__ __forceinline__ int2 octet_at(const PagedKv8& c, int u) {
    const int R = c.rotary_dim;
    if (c.layout == UNILLM_ROPE_HALF && 8 * u < R) return make_int2(4 * u, 4 * u + R / 2);
    return make_int2(8 * u, 8 * u + 4);
}
__device__ __forceinline__ Octet octet(const float* x, int2 d) {
    return Octet{once(reinterpret_cast<const f32x4*>(x + d.x)), once(reinterpret_cast<const f32x4*>(x + d.y))};
}
// It rotated, in f64, to f32.
__device__ __forceinline__ void rotate(const PagedKv8& c, Octet& o, int u, const double2* turn) {
    const int R = c.rotary_dim;
    if (8 * u >= R) return;
    double2 z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = turn[e * (R / 8) + u];
    auto pair = [](float& a, float& b, const double2& w) {
        const double x = a, y = b;
        a = (float)(x * w.x - y * w.y);
        b = (float)(x * w.y + y * w.x);
    };
    float a[4], b[4];
    if (c.layout == UNILLM_ROPE_HALF) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = o.lo[e], b[e] = o.hi[e];
            pair(a[e], b[e], z[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = o.lo[e], b[e] = o.hi[e];
        pair(a[0], a[1], z[0]);
        pair(a[2], a[3], z[1]);
        pair(b[0], b[1], z[2]);
        pair(b[2], b[3], z[3]);
    }
    o.lo = f32x4{a[0], a[1], a[2], a[3]};
    o.hi = f32x4{b[0], b[1], b[2], b[3]};
}

// A value's magnitude where it is finite, else 0 (and `odd` is set).
__device__ __forceinline__ float magnitude(float v, bool& odd) {
    const float m = fabsf(v);
    if (m < INFINITY) return m;
    odd = true;
    return 0.0f;
}

// A run's keys of kv head g (its first row's at x), into slots sl ..
template <class C, int D>
__device__ __forceinline__ void write_keys(const PagedKv8& c, const float* x, int64_t stride, int n, int sl, int g,
                                           const double2* turn, bool& odd) {
    constexpr int CH = D / 8, RP = 64 / CH, N = kBlock / RP;  // lanes a row, rows and passes
    const int lane = threadIdx.x & 63, u = lane % CH, sub = lane / CH;
    const int pairs = c.rotary_dim / 2, off = sl % kBlock;
    const int in_page = sl & ((int)c.page_size - 1);
    const int64_t head = (int64_t)(sl >> c.page_shift) * c.n_kv_heads + g;
    uint8_t* dst = c.k + ((head << c.page_shift) + in_page) * D;
    uint8_t* exps = c.k_exp + ((head << c.page_shift >> 4) + in_page / kBlock);
    const int had = off > 0 ? counted(*exps) : 0;
    const int2 d = octet_at(c, u);
    Octet v[N];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i].lo = v[i].hi = 0.0f;
        const int r = i * RP + sub;
        if (r < n) v[i] = octet(x + r * stride, d);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = i * RP + sub;
        if (r < n) rotate(c, v[i], u, turn + r * pairs);
        // (opaque: the keys are rows of f32 first, and rounded from there)
        asm volatile("" : "+v"(v[i].lo), "+v"(v[i].hi));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            top = fmaxf(top, magnitude(v[i].lo[e], odd));
            top = fmaxf(top, magnitude(v[i].hi[e], odd));
        }
    }
    const int b = max(least_exponent<C>(wave_max(top)), had);
    if (lane == 0) *exps = (uint8_t)b;
    const float inv = inverse(b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = i * RP + sub;
        if (r < n) {
            const f32x4 lo = v[i].lo * inv, hi = v[i].hi * inv;
            *reinterpret_cast<uint32_t*>(dst + r * D + d.x) = encode4<C>(lo[0], lo[1], lo[2], lo[3]);
            *reinterpret_cast<uint32_t*>(dst + r * D + d.y) = encode4<C>(hi[0], hi[1], hi[2], hi[3]);
        }
    }
    if (off > 0 && b > had) {
        const float f = power(127 + had - b);
        uint32_t* old = reinterpret_cast<uint32_t*>(dst - off * D);
        for (int i = lane; i < off * (D / 4); i += 64) old[i] = again4<C>(old[i], f);
    }
}

// A run's values.
template <class C, int D>
__device__ __forceinline__ void write_values(const PagedKv8& c, const float* x, int64_t stride, int n, int sl, int g,
                                             bool& odd) {
    constexpr int N = D / 64;  // neighbouring dimensions a lane
    struct alignas(4 * N) Dims {
        float v[N];
    };
    const int lane = threadIdx.x & 63, off = sl % kBlock;
    const int in_page = sl & ((int)c.page_size - 1);
    const int64_t head = (int64_t)(sl >> c.page_shift) * c.n_kv_heads + g;
    uint8_t* dst = c.v + ((head * D + N * lane) << c.page_shift) + in_page / kBlock * kBlock;
    uint8_t* exps = c.v_exp + ((head << c.page_shift >> 4) + in_page / kBlock);
    const int had = off > 0 ? counted(*exps) : 0;
    u32x4 old[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        old[j] = 0u;
        if (n < kBlock) old[j] = *reinterpret_cast<const u32x4*>(dst + ((int64_t)j << c.page_shift));
    }
    Dims v[kBlock];  // by position of the block
    float top = 0.0f;
#pragma unroll
    for (int p = 0; p < kBlock; ++p) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[p].v[j] = 0.0f;
        if (p >= off && p < off + n)
#pragma unroll
            for (int j = 0; j < N; ++j) v[p].v[j] = once(x + (p - off) * stride + N * lane + j);
    }
#pragma unroll
    for (int p = 0; p < kBlock; ++p)
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, magnitude(v[p].v[j], odd));
    const int b = max(least_exponent<C>(wave_max(top)), had);
    if (lane == 0) *exps = (uint8_t)b;
    const float inv = inverse(b), f = power(127 + had - b);
    const bool anew = off > 0 && b > had;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t fresh = encode4<C>(v[4 * i].v[j] * inv, v[4 * i + 1].v[j] * inv, v[4 * i + 2].v[j] * inv,
                                              v[4 * i + 3].v[j] * inv);
            uint32_t is_old = 0, is_new = 0;  // bytes of the word
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = 4 * i + e;
                if (p < off) is_old |= 0xFFu << (8 * e);
                else if (p < off + n) is_new |= 0xFFu << (8 * e);
            }
            const uint32_t kept = anew && is_old != 0 ? (again4<C>(old[j][i], f) & is_old) | (old[j][i] & ~is_old) : old[j][i];
            w[i] = (fresh & is_new) | (kept & ~is_new);
        }
        *reinterpret_cast<u32x4*>(dst + ((int64_t)j << c.page_shift)) = w;
    }
}

// Several runs of one row each (decoding requests'): their keys, each by the lanes of one row.
template <class C, int D>
__device__ __forceinline__ void write_one_keys(const PagedKv8& c, const float* kv, int64_t stride, const Runs<kWriteRows>& runs,
                                               int from, int n, int g, const double2* turn, bool& odd) {
    constexpr int CH = D / 8;  // lanes a row
    const int lane = threadIdx.x & 63, u = lane % CH;
    const int row = runs.first[from + min(lane / CH, n - 1)], sl = runs.slots[row + 1];
    const bool live = lane / CH < n;
    const int off = sl % kBlock, in_page = sl & ((int)c.page_size - 1);
    const int64_t head = (int64_t)(sl >> c.page_shift) * c.n_kv_heads + g;
    uint8_t* dst = c.k + ((head << c.page_shift) + in_page) * D;
    uint8_t* exps = c.k_exp + ((head << c.page_shift >> 4) + in_page / kBlock);
    const int2 d = octet_at(c, u);
    Octet v = octet(kv + row * stride + (int64_t)g * D, d);
    const int had = off > 0 ? counted(*exps) : 0;
    rotate(c, v, u, turn + row * (c.rotary_dim / 2));
    asm volatile("" : "+v"(v.lo), "+v"(v.hi));  // (rows of f32 first)
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        top = fmaxf(top, magnitude(v.lo[e], odd));
        top = fmaxf(top, magnitude(v.hi[e], odd));
    }
#pragma unroll
    for (int o = CH / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const int b = max(least_exponent<C>(top), had);
    if (!live) return;
    if (u == 0) *exps = (uint8_t)b;
    const float inv = inverse(b);
    const f32x4 lo = v.lo * inv, hi = v.hi * inv;
    *reinterpret_cast<uint32_t*>(dst + d.x) = encode4<C>(lo[0], lo[1], lo[2], lo[3]);
    *reinterpret_cast<uint32_t*>(dst + d.y) = encode4<C>(hi[0], hi[1], hi[2], hi[3]);
    if (off > 0 && b > had) {
        const float f = power(127 + had - b);
        uint32_t* old = reinterpret_cast<uint32_t*>(dst - off * D);
        for (int i = u; i < off * (D / 4); i += CH) old[i] = again4<C>(old[i], f);
    }
}

// The values of up to B of them.
template <class C, int D, int B>
__device__ __forceinline__ void write_one_values(const PagedKv8& c, const float* kv, int64_t stride, const Runs<kWriteRows>& runs,
                                                 int from, int n, int g, bool& odd) {
    constexpr int N = D / 64;  // neighbouring dimensions a lane
    struct alignas(4 * N) Dims {
        float v[N];
    };
    const int lane = threadIdx.x & 63;
    Dims v[B];
    int sl[B], had[B];
    int64_t head[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const int row = __builtin_amdgcn_readfirstlane(runs.first[from + min(i, n - 1)]);
        sl[i] = __builtin_amdgcn_readfirstlane(runs.slots[row + 1]);
        head[i] = (int64_t)(sl[i] >> c.page_shift) * c.n_kv_heads + g;
        v[i] = *reinterpret_cast<const Dims*>(kv + row * stride + (int64_t)(c.n_kv_heads + g) * D + N * lane);
        had[i] = c.v_exp[(head[i] << c.page_shift >> 4) + (sl[i] & ((int)c.page_size - 1)) / kBlock];
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
        if (i >= n) break;
        const int off = sl[i] % kBlock, in_page = sl[i] & ((int)c.page_size - 1);
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, magnitude(v[i].v[j], odd));
        const int was = off > 0 ? counted(had[i]) : 0;
        const int b = max(least_exponent<C>(wave_max(top)), was);
        if (lane == 0) c.v_exp[(head[i] << c.page_shift >> 4) + in_page / kBlock] = (uint8_t)b;
        uint8_t* dst = c.v + ((head[i] * D + N * lane) << c.page_shift) + in_page - off;
        const float inv = inverse(b);
        if (off > 0 && b > was) {  // (the codes before it, in the row's first words)
            const float f = power(127 + was - b);
            for (int j = 0; j < N; ++j)
                for (int w = 0; 4 * w < off; ++w) {
                    uint32_t* to = reinterpret_cast<uint32_t*>(dst + ((int64_t)j << c.page_shift)) + w;
                    const uint32_t x = *to, keep = off - 4 * w >= 4 ? 0xFFFFFFFFu : (1u << (8 * (off - 4 * w))) - 1;
                    *to = (again4<C>(x, f) & keep) | (x & ~keep);
                }
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
            dst[((int64_t)j << c.page_shift) + off] = (uint8_t)encode4<C>(v[i].v[j] * inv, 0.0f, 0.0f, 0.0f);
    }
}

// Consecutive numbers to workgroups of one XCD, which takes every eighth: neighbours share lines of a V page
// (1/8 of a line each at a page of 128), which each XCD's cache fetches for itself.
__device__ __forceinline__ int by_xcd(int i, int n) { return i % 8 * (n / 8) + i / 8; }

// What a call's first kernel does: `plan` workgroups deal the work out; then q_groups take q_rows query
// rows and q_heads heads each (rotated, times log2 e / sqrt(hd), f32, into q_out); the rest write the runs
// that begin in `rows` rows, of `heads` kv heads. An append does only the last of these: its kernel is
// compiled without the others (PLAN false: 400 B of LDS instead of 9 KB, and 4000 rotated rows of 32 heads of
// 128, e4m3, in 48.2 us instead of 49.5).
struct Prepare {
    const float *q, *kv;
    int64_t stride;  // of both
    float* q_out;
    int plan, q_groups, q_rows, q_heads, rows, heads, writes;  // writes: its workgroups, a multiple of 8
};

template <class C, int D, bool PLAN>
__global__ __launch_bounds__(256, D == 256 ? 3 : 4) void kv8_prepare_kernel(PagedKv8 c, PageTable t, Call a, Prepare p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ int at[2 * kWriteRows];
    double2* turn = reinterpret_cast<double2*>(lds);
    const int tid = threadIdx.x;
    const int KVH = (int)c.n_kv_heads, bx = (int)blockIdx.x - p.plan;
    const bool writes = bx >= p.q_groups;
    // the workgroup's rows and heads
    const int of = writes ? KVH : a.H, nr = writes ? p.rows : p.q_rows, each = writes ? p.heads : p.q_heads;
    const int groups = (of + each - 1) / each, wx = writes ? by_xcd(bx - p.q_groups, p.writes) : bx;
    const int row0 = wx / groups * nr, h0 = wx % groups * each, heads = min(each, of - h0);
    // (slots and positions are requested with the plan's header: both arrays hold max_tokens)
    int slot = -1, pos = 0;
    if (bx >= 0 && tid < nr + 16) {
        if (writes && row0 - 1 + tid >= 0 && row0 - 1 + tid < t.max_tokens) slot = t.slots[row0 - 1 + tid];
        if (row0 + tid < t.max_tokens) pos = t.positions[row0 + tid];
    }
    if (!step_fits(t, a.n)) {
        if (!PLAN) {
            if (blockIdx.x == 0 && tid == 0)
                atomicCAS(&t.counts[kPagesError], 0, t.counts[kPagesStep] == 1 ? kPagesRows : kPagesNoPlan);
            return;
        }
        if (blockIdx.x < 2 && tid < 2) a.kind[blockIdx.x].head[tid] = 0;
        if (blockIdx.x == 0 && tid == 0) *a.redo_count = 0;
        fail_call(t, a, D, blockIdx.x, gridDim.x);
        return;
    }
    if constexpr (PLAN)
        if (bx < 0) {
            if (blockIdx.x == 0 && tid == 0) *a.redo_count = 0;
            if (blockIdx.x == 0) return plan<64, narrow_rows(D)>(t, a, kNarrow, reinterpret_cast<int*>(lds));
            return plan<D == 256 ? 32 : 64, narrow_rows(D)>(t, a, kWide, reinterpret_cast<int*>(lds));
        }
    const int total = t.counts[kPagesTokens];
    if (row0 >= total) return;
    if (tid < nr + 16) at[tid] = pos;
    const int pairs = c.rotary_dim / 2;
    if (PLAN && !writes) {
        const int rows = min(nr, total - row0);
        __syncthreads();
        turns(c, at, rows, turn);
        const float scale = kLog2e / sqrtf((float)D);
        constexpr int CH = D / 8;
#pragma unroll 2
        for (int i = tid; i < rows * heads * CH; i += 256) {
            const int u = i % CH, h = h0 + i / CH % heads, r = i / CH / heads;
            const int2 d = octet_at(c, u);
            Octet o = octet(p.q + (row0 + r) * p.stride + (int64_t)h * D, d);
            rotate(c, o, u, turn + r * pairs);
            float* to = p.q_out + ((int64_t)(row0 + r) * a.H + h) * D;
            *reinterpret_cast<f32x4*>(to + d.x) = o.lo * scale;
            *reinterpret_cast<f32x4*>(to + d.y) = o.hi * scale;
        }
        return;
    }
    __shared__ Runs<kWriteRows> runs;
    find_runs(runs, row0 - 1 + tid < total ? slot : -1, nr);
    if (runs.n == 0) return;
    turns(c, at, runs.end, turn);
    bool odd = false;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* kv = p.kv + row0 * p.stride;
    constexpr int RP = 512 / D;  // one-row runs of a task of keys
    const int many = runs.many, ones = runs.n - many, batch = ones > 4 ? 4 : 1;
    const int k_tasks = (ones + RP - 1) / RP, tasks = 2 * many + k_tasks + (ones + batch - 1) / batch;
    for (int i = wv; i < tasks * heads; i += 4) {
        const int g = h0 + i % heads, task = i / heads;
        if (task < 2 * many) {
            const int r = __builtin_amdgcn_readfirstlane(runs.first[task / 2]);
            const int n = __builtin_amdgcn_readfirstlane(runs.count[task / 2]);
            const int sl = __builtin_amdgcn_readfirstlane(runs.slots[r + 1]);
            const float* x = kv + r * p.stride + (int64_t)g * D;
            if (task % 2 == 0) write_keys<C, D>(c, x, p.stride, n, sl, g, turn + r * pairs, odd);
            else write_values<C, D>(c, x + (int64_t)KVH * D, p.stride, n, sl, g, odd);
        } else if (task < 2 * many + k_tasks) {
            const int from = (task - 2 * many) * RP;
            write_one_keys<C, D>(c, kv, p.stride, runs, many + from, min(RP, ones - from), g, turn, odd);
        } else {
            const int from = (task - 2 * many - k_tasks) * batch;
            if (batch == 4) write_one_values<C, D, 4>(c, kv, p.stride, runs, many + from, min(4, ones - from), g, odd);
            else write_one_values<C, D, 1>(c, kv, p.stride, runs, many + from, 1, g, odd);
        }
    }
    if (__any(odd) && (tid & 63) == 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesNotFinite);
}

// ---- few query rows: keys stream through registers --------------------------------------------
//
// The narrow kernel of paged.hip on codes.  A workgroup takes an item of a tile of 16 query rows of a kv
// head, its four waves every fourth visit of 64 keys each; both products are formed transposed (16x16x32
// MFMAs), and each operand of the pool is a lane's own 16-byte load of codes, widened in its registers:
//   S^T: operand row i of subtile t (of four) is key 16 (i / 4) + 4 t + i % 4, so lane l holds, of query
//     row l % 16, the scores of the 16 keys of block l / 16 of the visit, and one exponent is all of theirs.  Its
//     16 bytes are dimensions 64 b + 16 (l / 16) .. of the key, 8 to each of two products;
//   O^T += V^T . P^T: its 16 bytes are those 16 keys' values of dimension l % 16 of each 16.
// Bound by HBM: 80 sequences of up to 9000, 8 kv heads of 128, pages of 32, e4m3, 441 MB in 84 us, 5.2 TB/s (a copy
// 5.4); widening int8 codes takes 540 vector instructions a visit beside 80 MFMAs, e4m3 320, and 32 sequences
// of 8192 take either at the same rate; for short sequences by latency (one of 1500 keys: 8 us).
template <int D>
struct Narrow8Lds {
    static constexpr int NB = D / 32, OT = D / 16;
    static constexpr int IDS = 0;                          // page ids of 256 visits, 4 each
    static constexpr int STAT = IDS + 4096;                // maxima, sums, flags
    static constexpr int Q = STAT + 1024;                  // q's parts [2][NB][64][16 B]
    static constexpr int QBYTES = 2 * NB * 1024;
    static constexpr int O = Q;                            // later the waves' sums [4][OT][64][16 B]
    static constexpr int OBYTES = 4 * OT * 1024;
    static constexpr int BYTES = Q + (QBYTES > OBYTES ? QBYTES : OBYTES);
};

// 8 codes -> f16 or bf16, exactly
template <class C>
__device__ __forceinline__ u32x4 codes_f16(uint32_t lo, uint32_t hi) {
    u32x4 r;
    if constexpr (std::is_same_v<C, Int8>) {
        // c + 128 as the low bits of 1024, less 1152
        const f16x2 base = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = (i < 2 ? lo : hi) ^ 0x80808080u;
            const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w, i % 2 ? 0x04030402u : 0x04010400u);
            r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - base);
        }
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    }
    return r;
}
template <class C>
__device__ __forceinline__ u32x4 codes_bf16(uint32_t lo, uint32_t hi) {
    u32x4 r;
    if constexpr (std::is_same_v<C, Int8>) {
        // (a whole number below 256 has no bits past bf16's: its upper half is it)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = i < 2 ? lo : hi;
            const float a = i % 2 ? decode<C, 2>(w) : decode<C, 0>(w), b = i % 2 ? decode<C, 3>(w) : decode<C, 1>(w);
            r[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        }
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    }
    return r;
}

// 8 f32 -> two f16 parts (22 bits), or three bf16 ones (all)
__device__ __forceinline__ void parts_f16(const f32x8& v, u32x4 (&p)[2]) {
    const f16x8 hi = __builtin_convertvector(v, f16x8);
    const f16x8 lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x8), f16x8);
    p[0] = __builtin_bit_cast(u32x4, hi);
    p[1] = __builtin_bit_cast(u32x4, lo);
}
__device__ __forceinline__ void parts_bf16(const f32x8& v, u32x4 (&p)[3]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t x, y, z;
        split2(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]), x, y, z);
        p[0][j] = x;
        p[1][j] = y;
        p[2][j] = z;
    }
}

// How far above the reference a weight may come before the reference follows (log2).
constexpr float kSlack = 8.0f;
// Narrow tiles' weights times their blocks' powers of two, and the sums of both, are held 2^kLift times as large, so
// that weights of small values keep their bits: with the least step, 2^-126, down to a weight of 2^-16 all of
// them.  (Of values past 2^80 or so the products are infinite: their rows are done again.)
constexpr int kLift = 32;
__device__ __forceinline__ float lifted(int b) { return __uint_as_float((uint32_t)min(max(b, 1) + kLift, 255) << 23); }

template <class C, int D, bool ONCE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv8_narrow_kernel(PagedKv8 c, PageTable t, Call a) {
    using L = Narrow8Lds<D>;
    constexpr int NB = L::NB, OT = L::OT, KB = D / 64, U = 64;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int* ids = reinterpret_cast<int*>(lds + L::IDS);               // [256][4]
    float* wm = reinterpret_cast<float*>(lds + L::STAT);           // [4][16]
    float* wl = wm + 64;                                            // [4][16]
    int* flags = reinterpret_cast<int*>(wl + 64);                  // [0] a bad page, [1] rows to redo
    u32x4* qp = reinterpret_cast<u32x4*>(lds + L::Q);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, qd = lane >> 4;
    const int ps = (int)c.page_size, shift = c.page_shift;
    const int KVH = a.KVH, G = a.G;
    const int total = a.kind[kNarrow].head[0] * KVH;
    for (int idx = blockIdx.x; idx < total; idx += gridDim.x) {
        const Item it = a.kind[kNarrow].items[idx / KVH];
        const int g = idx % KVH;
        const int first = it.first, len = it.len, ctx = it.ctx;
        const int* pages = t.table + (int64_t)it.id * t.max_pages;
        const int pmin = ctx + it.row0 / G, pmax = ctx + (it.row0 + it.rows - 1) / G;
        const Visits<U> vis(pmin, pmax, a.window, a.sinks);
        bool bad = false;
        auto read_ids = [&](int seg) {  // the page of each block of up to 256 visits
            for (int i = tid; i < 4 * min(256, it.nv - seg); i += 256) {
                int j = vis.key(it.v0 + seg + i / 4);
                if (j + i % 4 * kBlock < len) j += i % 4 * kBlock;  // (past the sequence: the visit's first again)
                int pg = pages[j >> shift];
                if ((unsigned)pg >= (unsigned)c.n_pages) {
                    pg = 0;
                    bad = true;
                }
                ids[i] = pg;
            }
        };
        // block x of visit v of a segment: its page and head, and its first key's place in the page
        auto block = [&](int seg, int v, int x, int64_t& head, int& off) {
            const int j = vis.key(it.v0 + seg + v);
            head = (int64_t)ids[4 * v + x] * KVH + g;
            off = (j + (j + x * kBlock < len ? x * kBlock : 0)) & (ps - 1);
        };
        u32x4 kr[4][KB], vr[OT];
        int ke = 0, ve = 0;
        auto load_k = [&](int seg, int v) {
            int64_t head;
            int off;
            block(seg, v, col / 4, head, off);
            const uint8_t* k = c.k + ((head << shift) + off + col % 4) * D + 16 * qd;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int b = 0; b < KB; ++b) kr[s][b] = once(reinterpret_cast<const u32x4*>(k + 4 * s * D + 64 * b));
            block(seg, v, qd, head, off);
            ke = c.k_exp[(head << shift >> 4) + off / kBlock];
        };
        auto load_v = [&](int seg, int v) {
            int64_t head;
            int off;
            block(seg, v, qd, head, off);
            const uint8_t* x = c.v + ((head * D + col) << shift) + off;
#pragma unroll
            for (int i = 0; i < OT; ++i) {
                const u32x4* from = reinterpret_cast<const u32x4*>(x + ((16 * i) << shift));
                vr[i] = ONCE ? once(from) : *from;
            }
            ve = c.v_exp[(head << shift >> 4) + off / kBlock];
        };
        // q's parts: task (product, lane) as the B operand takes it.  (Its requests and the page ids' go out
        // together, the first keys' and values' before its parts are formed.)
        constexpr int TASKS = (NB * 64 + 255) / 256;
        f32x8 qv[TASKS];
        float mx = 0.0f;
        __syncthreads();  // (the item before is done with the LDS)
        if (tid < 2) flags[tid] = 0;
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
            const int f = i * 256 + tid, r = f % 16, b = f / 64, d = b / 2 * 64 + f / 16 % 4 * 16 + b % 2 * 8;
            qv[i] = 0.0f;
            if (f < NB * 64 && r < it.rows) {
                const int rr = it.row0 + r;
                const f32x4* x = reinterpret_cast<const f32x4*>(
                    a.qkv + (first + rr / G) * a.qstride + (int64_t)(g * G + rr % G) * D + d);
                const f32x4 lo = x[0], hi = x[1];
#pragma unroll
                for (int j = 0; j < 8; ++j) qv[i][j] = j < 4 ? lo[j % 4] : hi[j % 4];
            }
        }
        read_ids(0);
#pragma unroll
        for (int i = 0; i < TASKS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(qv[i][j]));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (lane < 16) wm[wv * 16 + lane] = mx;
        __syncthreads();
        if (wv < min(256, it.nv)) {
            load_k(0, wv);
            load_v(0, wv);
        }
        const float2 size = row_scale(fmaxf(fmaxf(wm[col], wm[16 + col]), fmaxf(wm[32 + col], wm[48 + col])));
        const float inv = size.y;  // of this lane's row (and tasks': f % 16 is lane % 16)
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
            const int f = i * 256 + tid;
            if (f < NB * 64) {
                u32x4 p[2];
                parts_f16(qv[i] * size.x, p);
#pragma unroll
                for (int q = 0; q < 2; ++q) qp[q * NB * 64 + f] = p[q];
            }
        }
        __syncthreads();
        u32x4 q[2][NB];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) q[i][b] = qp[(i * NB + b) * 64 + lane];
        const int ppos = ctx + min(it.row0 + col, it.row0 + it.rows - 1) / G;  // the lane's row's position

        float ref = -INFINITY, l = 0.0f;
        f32x4 o[OT];
#pragma unroll
        for (int i = 0; i < OT; ++i) o[i] = 0.0f;
        for (int seg = 0; seg < it.nv; seg += 256) {
            const int nseg = min(256, it.nv - seg);
            if (seg > 0) {
                __syncthreads();
                read_ids(seg);
                __syncthreads();
                if (wv < nseg) {
                    load_k(seg, wv);
                    load_v(seg, wv);
                }
            }
            for (int v = wv; v < nseg; v += 4) {
                const int j0 = vis.key(it.v0 + seg + v);
                float s[16];
                const float times = inv * power(ke);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    f32x4 hi = 0.0f, lo = 0.0f;  // (the small products in a sum of their own)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const u32x4 w = kr[u][b / 2];
                        const u32x4 kp = codes_f16<C>(b % 2 ? w[2] : w[0], b % 2 ? w[3] : w[1]);
                        lo = mfma16<f16_t>(kp, q[1][b], lo);
                        hi = mfma16<f16_t>(kp, q[0][b], hi);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[4 * u + r] = (hi[r] + lo[r]) * times;
                }
                if (v + 4 < nseg) load_k(seg, v + 4);
                // masks, where some row of the tile does not see the whole visit
                const bool whole = j0 + U - 1 <= pmin &&
                                   (a.window == 0 || j0 > pmax - a.window || j0 + U <= a.sinks);
                if (!whole) {
                    const int at = ppos - j0 - 16 * qd, far = a.window > 0 ? at - a.window : INT_MIN;
                    const int sk = a.sinks - j0 - 16 * qd;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool hidden = (r > at) | ((r <= far) & (r >= sk));
                        s[r] = hidden ? -INFINITY : s[r];
                    }
                }
                float top = s[0];
#pragma unroll
                for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
                if (__any(top > ref + kSlack)) {
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float up = fmaxf(ref, top);
                    const float f = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - up);
                    l *= f;
#pragma unroll
                    for (int i = 0; i < OT; ++i) o[i] *= f;
                    ref = up;
                }
                const float from = ref == -INFINITY ? 0.0f : ref;  // (all weights are 0 then)
                const float step = lifted(ve);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = __builtin_amdgcn_exp2f(s[r] - from);
                    l += s[r];
                    s[r] *= step;
                }
                if (j0 + U > len) {  // past the sequence's end a page holds anything
                    const int left = len - j0 - 16 * qd;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int n = min(max(left - 4 * w, 0), 4);
                        const uint32_t keep = n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1;
#pragma unroll
                        for (int i = 0; i < OT; ++i) vr[i][w] &= keep;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f32x8 w;
#pragma unroll
                    for (int r = 0; r < 8; ++r) w[r] = s[8 * h + r];
                    u32x4 p[3];
                    parts_bf16(w, p);
#pragma unroll
                    for (int i = 0; i < OT; ++i) {
                        const u32x4 x = codes_bf16<C>(vr[i][2 * h], vr[i][2 * h + 1]);
                        o[i] = mfma16<bf16_t>(x, p[2], o[i]);
                        o[i] = mfma16<bf16_t>(x, p[1], o[i]);
                        o[i] = mfma16<bf16_t>(x, p[0], o[i]);
                    }
                }
                if (v + 4 < nseg) load_v(seg, v + 4);
            }
        }

        // the four waves' sums: scaled to one reference, added through LDS
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        l *= (float)(1ull << kLift);  // (as the sums of values)
        if (bad) flags[0] = 1;
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
                if (!whole) a.ms[piece] = make_float2(top, again || bad_page ? __builtin_nanf("") : sum);
            }
        }
    }
}

// ---- many query rows: tiles of keys shared through LDS -----------------------------------------
//
// The wide kernel of paged.hip on codes: an item of a tile of up to 256 query rows of a kv head (128 at
// hd 256), 32 to each wave (32x32x16 MFMAs), U keys at a time through LDS; two groups of four waves a phase
// apart, so that one's products run beside the other's softmax.  Codes are widened to f16 on their way into the
// LDS; their blocks' powers of two go beside them, K's for the scores, V's for the weights.
// A weight times its block's power of two is held in two f16 parts (four products a visit in all, where three
// bf16 parts make five: a prompt of 3001 tokens, 32 heads on 8 of 128, 200 us with those), taken against
// the row's largest weight times power of two so far, as 2^11: parts down to 2^-24 reach 2^-35 of it.  (A
// whole power of two apart from the weights' own reference, so that sums and weights are scaled alike, to the
// bit.)  What that may lose is looked at in the end.
// Bound by the matrix cores at hd 128 (3001 tokens behind 8000, 32 heads on 8, int8: 950 us, 980 TFLOP/s of
// products, where a large library product reaches 1152), by the vector units at hd 64 (750 over a call), and at hd 256 by
// having one wave a SIMD, whose products nothing overlaps (780).
constexpr int kWideShift = 11;
constexpr float kWideSlack = 4.0f;
// What a row may lose by the weights' parts, of its largest sum: 2^-16 over up to 2048 keys, 2^-27 a key over
// more (an f32 sum of as many terms may be off by 2^-24 a term).  A row loses so much where keys whose values
// are almost nothing in their blocks have all but 1/512 of the weight (an attention sink of value 0).
constexpr float kWideLoss = 0x1p-16f;
constexpr int kWideLossKeys = 2048;

template <int D>
struct Wide8Lds {
    static constexpr int GR = D < 256 ? 2 : 1, NT = 256 * GR;
    static constexpr int U = D == 256 ? 32 : 64;
    static constexpr int KROW = 2 * D, VROW = 2 * U;
    static constexpr int PLANE = U * KROW;                  // of K, and of V^T
    static constexpr int K = 0, V = PLANE, PAIR = 2 * PLANE;
    static constexpr int QL = GR * PAIR;                    // q's second part, where registers lack
    static constexpr bool kQl = D >= 128;
    static constexpr int QREGS = kQl ? 1 : 2;
    static constexpr int QROWS = 32 * D * 4;                // a wave's rows in f32, before and after
    static constexpr int USED = QL + (kQl ? NT / 64 * (D / 16) * 1024 : 0), ROWS = NT / 64 * QROWS;
    static constexpr int STAT = USED > ROWS ? USED : ROWS;  // whether a page is bad, K's powers of two
    static constexpr int BYTES = STAT + 64 + 128;
    static constexpr int TASKS = U * D / 8 / NT;            // 8-code chunks of K (or V) a thread
    __device__ static uint32_t kslot(uint32_t r, uint32_t c) {
        return D >= 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
    }
    __device__ static uint32_t vslot(uint32_t d, uint32_t c) {
        return U == 64 ? c ^ ((d >> 1) & 7) : c ^ ((d >> 2) & 3);
    }
};

template <class C, int D>
__global__ __launch_bounds__((256 * Wide8Lds<D>::GR), (D == 256 ? 1 : 2)) void kv8_wide_kernel(
    PagedKv8 c, PageTable t, Call a) {
    using L = Wide8Lds<D>;
    constexpr int U = L::U, NB = D / 16, OT = D / 32, NG = U / 32, GR = L::GR, NT = L::NT;
    constexpr int LOG_D = D == 64 ? 6 : D == 128 ? 7 : 8;
    constexpr int KSTEP = NT * 8 / D, KROWS = 512 / D;  // keys between a thread's chunks, keys of a wave's
    constexpr int VGROUPS = U / 16;
    // A buffer's pair m - 2 was last read in the second group's matrix phase m - 2, so either group may
    // store its share of pair m in the two phases after: its matrix phase m - 1, or the vector
    // phase m - 1 (m - 2 in the second group).  The stores go with the shorter phase, at hd 128 the vector
    // one, at hd 64 the matrix one (3001 tokens behind 8000, int8, 32 heads, us a call: hd 128 on 8 kv heads 976, 1331 the
    // other way; hd 64 on 4 625, 719).
    constexpr bool kStoreEarly = GR == 2 && D == 64;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int* flags = reinterpret_cast<int*>(lds + L::STAT);  // [0] a bad page
    // [4][4], by visit and block: K's powers of two, V's exponents
    float* steps = reinterpret_cast<float*>(lds + L::STAT + 64);
    int* vexps = reinterpret_cast<int*>(steps + 16);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wv / 4;
    const int col = lane & 31, hf = lane >> 5;
    const int ps = (int)c.page_size, shift = c.page_shift;
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
        u32x2 sk[L::TASKS], sv[L::TASKS];
        int ke[L::TASKS], ve[L::TASKS];  // K's chunks' blocks' exponents, and those of V there
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
        const uint8_t* kbase = c.k + ((int64_t)g << (shift + LOG_D));
        const uint8_t* vbase = c.v + ((int64_t)g << (shift + LOG_D));
        const uint32_t page_elems = (uint32_t)KVH << (shift + LOG_D);
        auto read_pages = [&](int jk, int jv) {
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i) pk[i] = pages[group_key(jk, kgroup(i)) >> shift];
            pv = pages[group_key(jv, vgroup) >> shift];
        };
        auto fetch_k = [&](int i) {
            const uint32_t at = (uint32_t)group_key(k1, kgroup(i)) & (uint32_t)(ps - 1);
            const uint64_t page = sound(pk[i]);
            sk[i] = *reinterpret_cast<const u32x2*>(kbase + (page * page_elems + (at << LOG_D)) +
                                                    (klane + (KSTEP == 8 ? i % 2 * 8 * D : 0)));
            const uint64_t block = ((page * KVH + g) << (shift - 4)) + at / kBlock;
            ke[i] = c.k_exp[block];
            ve[i] = c.v_exp[block];
        };
        auto fetch_v = [&] {
            const uint32_t at = (uint32_t)group_key(k0, vgroup) & (uint32_t)(ps - 1);
            const uint64_t page = sound(pv);
            const uint8_t* from = vbase + (page * page_elems + at);
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i) sv[i] = *reinterpret_cast<const u32x2*>(from + (32 * i << shift) + vlane);
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
                // (a chunk step of 8 rows turns bit 3 of the slot)
                const uint32_t at = (KSTEP == 8 && i % 2 ? kto ^ 128 : kto) + i * KSTEP * L::KROW;
                *reinterpret_cast<u32x4*>(buf + L::K + at) = codes_f16<C>(sk[i][0], sk[i][1]);
                if (lane == 0) {
                    steps[m % 4 * 4 + kgroup(i)] = power(ke[i]);
                    vexps[m % 4 * 4 + kgroup(i)] = counted(ve[i]) - 127;
                }
            }
            const int left = len - kstored;  // keys of V's visit and on
            if (left < U) {                  // past the sequence's end a page holds anything
                const int mine = left - 16 * vgroup - 8 * (lane & 1);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int n = min(max(mine - 4 * w, 0), 4);
                    const uint32_t keep = n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1;
#pragma unroll
                    for (int i = 0; i < L::TASKS; ++i) sv[i][w] &= keep;
                }
            }
#pragma unroll
            for (int i = 0; i < L::TASKS; ++i)
                *reinterpret_cast<u32x4*>(buf + L::V + vto + 32 * i * L::VROW) = codes_f16<C>(sv[i][0], sv[i][1]);
        };
        read_pages(k1, k0);
        fetch(0);

        u32x4 q[L::QREGS][NB];
        u32x4* ql = reinterpret_cast<u32x4*>(lds + L::QL) + wv * NB * 64 + lane;
        __syncthreads();  // (the item before is done with the LDS)
        if (tid == 0) flags[0] = 0;
        float inv = 1.0f;
        // The wave's rows of q come whole rows at a time and through its own part of the LDS: a lane's operand
        // is 32 bytes of a row, and loaded so every request would touch 32 lines (3001 tokens behind 8000, hd 128,
        // int8: 981 us, 1031 so; without the 8000 227 and 231).
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
            float up = 1.0f;
            {
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
                r[b] *= up;
                u32x4 p[2];
                parts_f16(r[b], p);
#pragma unroll
                for (int i = 0; i < L::QREGS; ++i) q[i][b] = p[i];
                if (L::kQl) ql[b * 64] = p[1];
            }
        }
        // the weights' reference; the row's largest weight times power of two, against which (as a whole power of
        // two: `rise` above the weights') the products' weights are taken
        float ref = -INFINITY, peak = -INFINITY, l = 0.0f;
        int rise = 0;
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
            u32x4 kp[2][NG], qx[2];
            auto read = [&](int b) {
#pragma unroll
                for (int u = 0; u < NG; ++u)
                    kp[b % 2][u] = *reinterpret_cast<const u32x4*>(buf + L::K + 32 * u * L::KROW + (ka ^ 32 * b));
                if (L::kQl) qx[b % 2] = ql[b * 64];
            };
            read(0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b + 1 < NB) read(b + 1);
                if (kStoreEarly && b % (NB / 4) == 0) fetch_piece(n + 2, b / (NB / 4));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 1; x >= 0; --x)
#pragma unroll
                    for (int u = 0; u < NG; ++u)
                        s[u] = mfma32<f16_t>(kp[b % 2][u], x < L::QREGS ? q[x < L::QREGS ? x : 0][b] : qx[b % 2],
                                             s[u]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (kStoreEarly) store(1);
        scores(0);
        __syncthreads();  // the first matrix phase ends
        for (int n = 0;; ++n) {
            const int j0 = vis.key(it.v0 + n);
            u32x4 p[NG][2][2];
            {
                float top = -INFINITY, high = -INFINITY, times[NG][2];
                int ve[NG][2];
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        times[u][x] = inv * steps[n % 4 * 4 + 2 * u + x];
                        ve[u][x] = vexps[n % 4 * 4 + 2 * u + x];
                    }
#pragma unroll
                for (int u = 0; u < NG; ++u) {
                    const int ju = j0 + 32 * u;
                    const bool all = ju + 31 <= wmin &&
                                     (a.window == 0 || ju > wmax - a.window || ju + 32 <= a.sinks);
                    if (!all) {
                        asm volatile("");  // (a branch: without it every visit forms its masks)
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
                    for (int x = 0; x < 2; ++x) {
                        float most = s[u][8 * x];
#pragma unroll
                        for (int e = 1; e < 8; ++e) most = fmaxf(most, s[u][8 * x + e]);
                        most *= times[u][x];  // (a power of two)
                        top = fmaxf(top, most);
                        high = fmaxf(high, most + (float)ve[u][x]);
                    }
                }
                if (__any((top > ref + kWideSlack) | (high > ref + (float)rise + kWideSlack))) {
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    high = fmaxf(high, __shfl_xor(high, 32, 64));
                    const float to = fmaxf(ref, top);
                    peak = fmaxf(peak, high);
                    const int up = to == -INFINITY ? 0 : (int)ceilf(fminf(fmaxf(peak - to, -1000.0f), 1000.0f));
                    const float f = ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - to);
                    const float fo = __builtin_amdgcn_ldexpf(f, rise - up);
                    l *= f;
                    // (held in accumulation registers: without this every visit copies all of them out, in case)
                    if constexpr (D == 256)
#pragma unroll
                        for (int i = 0; i < OT; ++i) asm volatile("" : "+a"(o[i]));
#pragma unroll
                    for (int i = 0; i < OT; ++i) o[i] *= fo;
                    ref = to;
                    rise = up;
                }
                const float from = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        // (a weight of 0 stays one: of a block that no row sees the exponent may be any)
                        const float step = __builtin_amdgcn_ldexpf(1.0f, min(ve[u][k] - rise + kWideShift, 126));
                        f32x8 w;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            w[e] = __builtin_amdgcn_exp2f(fmaf(s[u][8 * k + e], times[u][k], -from));
                            l += w[e];
                            w[e] *= step;
                        }
                        halve_weights(w, p[u][k]);
                    }
            }
            if (!kStoreEarly) store(n + 1 + grp);
            __syncthreads();  // the vector phase ends
            // (the matrix phase's wave goes first on the SIMD: 3001 tokens behind 8000, int8, at hd 128 981 us, 1004 without;
            // at hd 64 631 and 673.  At hd 256 there is one wave: 438 without, 445 so.)
            if (GR == 2) __builtin_amdgcn_s_setprio(1);
            {
                // o += p v of visit n.  Step i: dimensions 32 (i % OT) .., keys of MFMA i / OT
                const uint8_t* buf = lds + (n + 1) % GR * L::PAIR;
                uint32_t va = vat;
                asm volatile("" : "+v"(va));
                u32x4 vp[2];
                auto read = [&](int i) {
                    vp[i % 2] =
                        *reinterpret_cast<const u32x4*>(buf + L::V + 32 * (i % OT) * L::VROW + (va ^ 32 * (i / OT)));
                };
                read(0);
#pragma unroll
                for (int i = 0; i < 2 * NG * OT; ++i) {
                    if (i + 1 < 2 * NG * OT) read(i + 1);
                    // (what is stored next is requested between the first MFMAs after the stores before)
                    if (!kStoreEarly && i % (NG * OT / 2) == 0) fetch_piece(n + 2 + grp, i / (NG * OT / 2));
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int x = 1; x >= 0; --x)
                        o[i % OT] = mfma32<f16_t>(vp[i % 2], p[i / OT / 2][i / OT % 2][x], o[i % OT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (n + 1 == it.nv) {
                if (GR == 2) __builtin_amdgcn_s_setprio(0);
                break;
            }
            if (kStoreEarly) store(n + 2);
            scores(n + 1);
            if (GR == 2) __builtin_amdgcn_s_setprio(0);
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
        float chk = l * 0.0f, most = 0.0f;
        // Weights in two parts are off by up to 2^-25, and a row's sums by that times the item's keys and the
        // largest code: a row whose largest sum may have lost too much is done again (but where all values are
        // 0, or next to it, below 2^-112: their blocks' exponents are the least, and rise is -126 or little more).
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(o[i][e]));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        if (l > 0.0f && rise > -120 &&
            most * kWideLoss < C::top * ((float)min(it.nv * U, kWideLossKeys) * 0x1p-25f)) chk = 1.0f;
        // the sums against the weights' reference
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = __builtin_amdgcn_ldexpf(o[i][e], rise - kWideShift);
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
                a.ms[piece + w0 + col] = make_float2(ref, again || bad_page ? __builtin_nanf("") : l);
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

// One row and head by a wave, in plain f32: for rows whose products of parts came out non-finite (an
// infinite query, or scores past f32's range), and those of wide tiles that lost too much: an attention sink of
// value 0 may list every row of its head, and each reads all its keys for itself (2000 tokens behind 2000, 32 heads
// on 8 of 128, int8, a sink of 10 nats in each head: 13.7 ms, 0.28 without).  qf: LDS [D], the query; sc: LDS [64].  Lane el gets
// dimensions el + 64 i of out.
template <class C, int D>
__device__ void attend_row(const PagedKv8& c, const Call& a, const int* pages, int row, int h, int p,
                           float* qf, float* sc, float (&acc)[D / 64]) {
    constexpr int U = 64;
    const int el = threadIdx.x & 63, g = h / a.G, shift = c.page_shift, ps = (int)c.page_size;
    bool bad = false;
    auto head_of = [&](int j) {
        const int pg = pages[j >> shift];
        if ((unsigned)pg < (unsigned)c.n_pages) return (int64_t)pg * a.KVH + g;
        bad = true;
        return (int64_t)g;
    };
    settle_wave();
    for (int d = el; d < D; d += 64) qf[d] = a.qkv[row * a.qstride + (int64_t)h * D + d];
    settle_wave();
    float mx = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.0f;
    const Visits<U> vis(p, p, a.window, a.sinks);
    for (int v = 0; v < vis.count && !(l != l); ++v) {  // (a NaN sum stays one)
        const int j0 = vis.key(v);
        for (int i = 0; i < U / 8; ++i) {  // 8 lanes a key
            const int j = min(j0 + 8 * i + el / 8, p), off = j & (ps - 1);
            const int64_t head = head_of(j);
            const uint32_t* kr = reinterpret_cast<const uint32_t*>(c.k + ((head << shift) + off) * D + el % 8 * (D / 8));
            float dot = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 8; d += 4) {
                const f32x4 x = decode4<C>(kr[d / 4]);
#pragma unroll
                for (int e = 0; e < 4; ++e) dot = fmaf(x[e], qf[el % 8 * (D / 8) + d + e], dot);
            }
            dot += __shfl_xor(dot, 1, 64);
            dot += __shfl_xor(dot, 2, 64);
            dot += __shfl_xor(dot, 4, 64);
            dot *= power(c.k_exp[(head << shift >> 4) + off / kBlock]);
            if (el % 8 == 0) sc[8 * i + el / 8] = dot;
        }
        settle_wave();
        const int j = j0 + el;
        const bool seen = j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
        const float s = seen ? sc[el] : -INFINITY;
        const float mnew = fmaxf(mx, wave_max(s));
        const float alpha = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mnew);
        const float w = s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - mnew);
        l = l * alpha + wave_add(w);
        mx = mnew;
        settle_wave();
        sc[el] = w;
        settle_wave();
        const uint64_t mask = __ballot(seen);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) acc[i] *= alpha;
        for (int u = 0; u < U / 4; ++u) {
            if ((mask >> (4 * u) & 0xF) == 0) continue;
            const int j4 = j0 + 4 * u, off = j4 & (ps - 1);
            const int64_t head = head_of(j4);
            const float step = power(c.v_exp[(head << shift >> 4) + off / kBlock]);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const f32x4 x =
                    decode4<C>(*reinterpret_cast<const uint32_t*>(c.v + ((head * D + el + 64 * i) << shift) + off));
#pragma unroll
                for (int e = 0; e < 4; ++e)  // (a hidden key's value may be anything)
                    if (mask >> (4 * u + e) & 1) acc[i] = fmaf(sc[4 * u + e], x[e] * step, acc[i]);
            }
        }
        settle_wave();
    }
    if (__any(bad)) l = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = l != l ? l : acc[i] / l;
}

// The last kernel of a call: pieces joined, then the rows listed to be done again.
template <class C, int D>
__global__ __launch_bounds__(256) void kv8_merge_kernel(PagedKv8 c, PageTable t, Call a) {
    merge_pieces<D>(a);
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
        attend_row<C, D>(c, a, t.table + (int64_t)t.step_ids[lo] * t.max_pages, row, h, p, rows[wv],
                         rows[wv] + D, acc);
        float* o = a.out + row * a.ostride + (int64_t)h * D + (threadIdx.x & 63);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[64 * e] = acc[e];
    }
}

// ---- values read back -------------------------------------------------------------------------
constexpr int kReadRows = 64;  // rows of a workgroup, at most
struct Read {
    const int *ids, *starts, *cu;
    int B, n;
    void *k, *v;
    int64_t stride;
    int rows, heads;  // of a workgroup
};

template <class O>
struct alignas(16) Eight {  // (four, of f32)
    O v[16 / sizeof(O)];
};

// The mirror of the writes: runs of rows in one block, a wave a run of one kv head's keys and values.
// Bound by HBM: 90000 rows of 8 heads of 128, to f16, 553 MB, pages of 16 in 92 us (6.0 TB/s), of 128 in 133 (a line
// of V is eight runs', which several workgroups fetch).
template <class C, class O, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(PagedKv8 c, PageTable t, Read a) {
    constexpr int kHold = 1024;  // entries that are held, and searched, in LDS
    __shared__ Runs<kReadRows> runs;
    __shared__ uint64_t bad_rows[2];  // by row from row0 - 1 on
    __shared__ int cu[kHold], ids[kHold], starts[kHold];
    const int tid = threadIdx.x, lane = tid & 63;
    const int KVH = (int)c.n_kv_heads, groups = (KVH + a.heads - 1) / a.heads;
    const int NR = a.rows, bx = by_xcd(blockIdx.x, gridDim.x), row0 = bx / groups * NR, g0 = bx % groups * a.heads;
    const int heads = min(a.heads, KVH - g0), end = min(a.n, a.cu[a.B]);
    const bool in_lds = a.B <= kHold;
    if (in_lds)
        for (int i = tid; i < a.B; i += 256) cu[i] = a.cu[i], ids[i] = a.ids[i], starts[i] = a.starts[i];
    if (row0 >= end) return;
    __syncthreads();
    int slot = -1;
    bool bad = false;
    const int row = row0 - 1 + tid;
    if (tid < NR + 16 && row >= 0 && row < end) {
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if ((in_lds ? cu[mid] : a.cu[mid]) <= row) lo = mid;
            else hi = mid;
        }
        const int id = in_lds ? ids[lo] : a.ids[lo];
        const int64_t pos = (int64_t)(in_lds ? starts[lo] : a.starts[lo]) + row - (in_lds ? cu[lo] : a.cu[lo]);
        if (id >= 0) {
            bad = true;
            if (id < t.max_seqs && pos >= 0 && (pos >> c.page_shift) < t.max_pages) {
                const int pg = t.table[(int64_t)id * t.max_pages + (pos >> c.page_shift)];
                if (pos < t.lens[id] && (unsigned)pg < (unsigned)c.n_pages) {
                    slot = (pg << c.page_shift) + (int)(pos & (c.page_size - 1));
                    bad = false;
                }
            }
        }
    }
    if (tid < 128) {
        const uint64_t b = __ballot(bad);
        if ((tid & 63) == 0) {
            bad_rows[tid >> 6] = b;
            if (b != 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesBadRead);
        }
    }
    find_runs(runs, slot, NR);
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    O* const outs[2] = {static_cast<O*>(a.k), static_cast<O*>(a.v)};
    if ((bad_rows[0] | bad_rows[1]) != 0)
        for (int r = wv; r < NR; r += 4)
            if (bad_rows[(r + 1) / 64] >> (r + 1) % 64 & 1)
                for (int w = 0; w < 2; ++w)
                    if (outs[w])
                        for (int d = lane; d < heads * D; d += 64)
                            outs[w][(row0 + r) * a.stride + (int64_t)g0 * D + d] = (O)__builtin_nanf("");
    // a task: a run's keys and values of a head, all requested before the first is stored
    constexpr int E = 16 / sizeof(O), CH = D / E, RP = 64 / CH, KN = kBlock / RP;  // K: 16 bytes of the output a lane
    constexpr int VN = D / 128 > 0 ? D / 128 : 1;                                 // V: two dimensions a lane
    struct alignas(2 * sizeof(O)) Two {
        O v[2];
    };
    using Raw = std::conditional_t<sizeof(O) == 4, uint64_t, uint32_t>;
    for (int i = wv; i < runs.n * heads; i += 4) {
        const int g = g0 + i % heads, run = i / heads;
        const int r0 = __builtin_amdgcn_readfirstlane(runs.first[run]);
        const int n = __builtin_amdgcn_readfirstlane(runs.count[run]);
        const int sl = __builtin_amdgcn_readfirstlane(runs.slots[r0 + 1]);
        const int in_page = sl & ((int)c.page_size - 1), off = sl % kBlock;
        const int64_t head = (int64_t)(sl >> c.page_shift) * KVH + g;
        const int64_t block = (head << c.page_shift >> 4) + in_page / kBlock;
        const uint8_t* k = c.k + ((head << c.page_shift) + in_page) * D + lane % CH * E;
        const uint8_t* v = c.v + ((head * D + 2 * lane) << c.page_shift) + in_page - off;
        const float k_step = power(c.k_exp[block]), v_step = power(c.v_exp[block]);
        const int64_t at = (row0 + r0) * a.stride + (int64_t)g * D;
        uint32_t kw[KN][E / 4];
        u32x4 vw[VN][2];
#pragma unroll
        for (int x = 0; x < KN; ++x)
            if (a.k && lane / CH + x * RP < n)
#pragma unroll
                for (int e = 0; e < E / 4; ++e) kw[x][e] = once(reinterpret_cast<const uint32_t*>(k + (lane / CH + x * RP) * D) + e);
#pragma unroll
        for (int x = 0; x < VN; ++x)
            if (a.v && 2 * lane + 128 * x < D)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    vw[x][e] = *reinterpret_cast<const u32x4*>(v + ((int64_t)(128 * x + e) << c.page_shift));
#pragma unroll
        for (int x = 0; x < KN; ++x)
            if (a.k && lane / CH + x * RP < n) {
                Eight<O> y;
#pragma unroll
                for (int e = 0; e < E / 4; ++e) {
                    const f32x4 z = decode4<C>(kw[x][e]) * k_step;
#pragma unroll
                    for (int j = 0; j < 4; ++j) y.v[4 * e + j] = (O)z[j];
                }
                O* to = static_cast<O*>(a.k) + at + (lane / CH + x * RP) * a.stride + lane % CH * E;
                __builtin_nontemporal_store(__builtin_bit_cast(u32x4, y), reinterpret_cast<u32x4*>(to));
            }
#pragma unroll
        for (int x = 0; x < VN; ++x)
            if (a.v && 2 * lane + 128 * x < D)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const f32x4 p = decode4<C>(vw[x][0][w]) * v_step, q = decode4<C>(vw[x][1][w]) * v_step;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * w + e - off;
                        O* to = static_cast<O*>(a.v) + at + r * a.stride + 128 * x + 2 * lane;
                        if (r >= 0 && r < n)
                            __builtin_nontemporal_store(__builtin_bit_cast(Raw, Two{{(O)p[e], (O)q[e]}}),
                                                        reinterpret_cast<Raw*>(to));
                    }
                }
    }
}

// ---- launches ---------------------------------------------------------------------------------

// Workgroups of a kind that the device holds: wide one a CU, narrow by its registers.
int places(int kind, int64_t D) { return (kind == kWide || D == 256 ? 1 : 2) * device_info().cu_count; }
// Pieces a kind's work is dealt out in at most.
int target_pieces(int kind) { return (kind == kNarrow ? 3 : 1) * device_info().cu_count; }

int tile_rows(int kind, int64_t D) { return kind == kNarrow ? kTileRows : D < 256 ? 256 : 128; }

struct Layout {
    int64_t items[2], rows[2];
    size_t head_at[2], items_at[2], splits_at[2], q_at, ms_at, po_at, count_at, redo_at, bytes;
};

Layout layout(const PagedKv8& c, const unillm_page_table& t, int64_t n, int64_t H) {
    const int64_t KVH = c.n_kv_heads, G = H / KVH, D = c.head_dim;
    Layout l;
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += ((size_t)bytes + 255) & ~(size_t)255;
        return here;
    };
    for (int k = 0; k < 2; ++k) {
        // tiles: an entry's last may be ragged (a wide entry has more than narrow_rows).  A
        // tile of nv visits makes at most nv / C + 1 pieces, and the nv / C add up to target /
        // KVH; more than one piece, at most 2 nv / C.
        const int64_t entries = std::min<int64_t>(k == kNarrow ? n : n * G / (narrow_rows(D) + 1), t.st.max_seqs);
        const int64_t tiles = n * G / tile_rows(k, D) + entries;
        const bool some = k == kNarrow || n * G > narrow_rows(D);
        l.items[k] = some ? tiles + target_pieces(k) / KVH + 1 : 0;
        l.rows[k] = some ? 2 * (int64_t)target_pieces(k) * std::min<int64_t>(tile_rows(k, D), n * G) : 0;
        l.head_at[k] = take(2 * sizeof(int));
        l.items_at[k] = take(l.items[k] * (int64_t)sizeof(Item));
        l.splits_at[k] = take(tiles * (int64_t)sizeof(Split));
    }
    l.q_at = take(n * H * D * (int64_t)sizeof(float));
    l.ms_at = take((l.rows[0] + l.rows[1]) * (int64_t)sizeof(float2));
    l.po_at = take((l.rows[0] + l.rows[1]) * D * (int64_t)sizeof(float));
    // rows to do again: every (row, head), and again for each piece
    l.count_at = take(sizeof(int));
    l.redo_at = take((n * H + l.rows[0] + l.rows[1]) * (int64_t)sizeof(int));
    l.bytes = at;
    return l;
}

// Heads to a workgroup: one, or what leaves four workgroups a CU.
int heads_each(int64_t blocks, int64_t heads) {
    return (int)std::min<int64_t>(heads, std::max<int64_t>(1, blocks * heads / (4 * device_info().cu_count)));
}

// The writes' part of a first kernel: rows and heads to a workgroup, so that few rows and heads still make
// many workgroups (decoding requests begin a run a row, which a workgroup's waves take one after the other).
void plan_writes(const PagedKv8& c, int64_t n, Prepare& p) {
    p.rows = kWriteRows;
    while (p.rows > 2 && n * c.n_kv_heads < 1024 * p.rows) p.rows /= 2;
    const int64_t blocks = (n + p.rows - 1) / p.rows;
    p.heads = heads_each(blocks, c.n_kv_heads);
    // (a prompt's run is two tasks a head, for four waves)
    if (p.rows == kWriteRows) p.heads = (int)std::min<int64_t>(c.n_kv_heads, std::max(p.heads, 2));
    p.writes = (int)((blocks * ((c.n_kv_heads + p.heads - 1) / p.heads) + 7) / 8 * 8);
}

template <class C, int D, bool PLAN>
hipError_t launch_prepare(const PagedKv8& c, const unillm_page_table& t, const Call& a, const Prepare& p,
                          hipStream_t s) {
    constexpr int kMost = (3 * kPagesMaxSeqs + 1) * (int)sizeof(int);
    static_assert(kMost >= (2 * kBlock - 1) * 128 * (int)sizeof(double2), "31 rows of 128 pairs");
    static const bool attr = hipFuncSetAttribute((const void*)kv8_prepare_kernel<C, D, PLAN>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, kMost) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    const size_t pairs = (size_t)c.rotary_dim / 2 * sizeof(double2);
    size_t lds = std::max((size_t)(p.rows + kBlock - 1) * pairs, (size_t)p.q_rows * pairs);
    if (p.plan) lds = std::max(lds, (size_t)(3 * t.st.max_seqs + 1) * sizeof(int));  // (three ints an entry)
    const unsigned grid = (unsigned)(p.plan + p.q_groups + p.writes);
    kv8_prepare_kernel<C, D, PLAN><<<grid, 256, lds, s>>>(c, t.st, a, p);
    return hipGetLastError();
}

template <class C, int D>
hipError_t launch_typed(const PagedKv8& c, const unillm_page_table& t, const Call& a, const Prepare& p,
                        const Layout& l, hipStream_t s) {
    hipError_t e = launch_prepare<C, D, true>(c, t, a, p, s);
    if (e != hipSuccess) return e;
    using N = Narrow8Lds<D>;
    using W = Wide8Lds<D>;
    static const bool attr =
        hipFuncSetAttribute((const void*)kv8_narrow_kernel<C, D, true>, hipFuncAttributeMaxDynamicSharedMemorySize,
                            N::BYTES) == hipSuccess &&
        hipFuncSetAttribute((const void*)kv8_narrow_kernel<C, D, false>, hipFuncAttributeMaxDynamicSharedMemorySize,
                            N::BYTES) == hipSuccess &&
        hipFuncSetAttribute((const void*)kv8_wide_kernel<C, D>, hipFuncAttributeMaxDynamicSharedMemorySize,
                            W::BYTES) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    const int64_t most = 4 * device_info().cu_count;
    auto grid = [&](int64_t n, int64_t limit) { return (unsigned)std::min(n, limit); };
    if (l.items[kWide] > 0) {
        kv8_wide_kernel<C, D><<<grid(l.items[kWide] * a.KVH, 4 * most), W::NT, W::BYTES, s>>>(c, t.st, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const unsigned narrow = grid(l.items[kNarrow] * a.KVH, most);
    if (c.page_size <= 64) kv8_narrow_kernel<C, D, true><<<narrow, 256, N::BYTES, s>>>(c, t.st, a);
    else kv8_narrow_kernel<C, D, false><<<narrow, 256, N::BYTES, s>>>(c, t.st, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    kv8_merge_kernel<C, D><<<grid((l.rows[0] + l.rows[1]) / 2, most), 256, 0, s>>>(c, t.st, a);
    return hipGetLastError();
}

// f(code type, head_dim as a type) of the pool
template <class F>
hipError_t by_pool(const PagedKv8& c, F f) {
    auto by_dim = [&](auto code) {
        if (c.head_dim == 64) return f(code, std::integral_constant<int, 64>{});
        if (c.head_dim == 128) return f(code, std::integral_constant<int, 128>{});
        return f(code, std::integral_constant<int, 256>{});
    };
    return c.type == UNILLM_KV8_INT8 ? by_dim(Int8{}) : by_dim(E4m3{});
}

}  // namespace

hipError_t launch_kv8_append(const PagedKv8& c, const unillm_page_table& t, const float* kv,
                             int64_t kvstride, int64_t n, hipStream_t s) {
    Call a{};
    a.n = (int)n;
    Prepare p{nullptr, kv, kvstride, nullptr, 0, 0, 0, 1, 0, 0, 0};
    plan_writes(c, n, p);
    return by_pool(c, [&](auto code, auto dim) {
        return launch_prepare<decltype(code), decltype(dim)::value, false>(c, t, a, p, s);
    });
}

hipError_t launch_kv8_attention(const PagedKv8& c, const unillm_page_table& t, const float* qkv,
                                int64_t qstride, int64_t n, int64_t H, bool append, int64_t window,
                                int64_t sinks, float* out, int64_t ostride, hipStream_t s) {
    const Layout l = layout(c, t, n, H);
    void* ws = nullptr;
    hipError_t e = stream_workspace(s, l.bytes, &ws, kPagedSlot);
    if (e != hipSuccess) return e;
    uint8_t* w = static_cast<uint8_t*>(ws);
    // a window or sinks past any position are all of them
    const int64_t far = (int64_t)1 << 30, D = c.head_dim;
    float* q = reinterpret_cast<float*>(w + l.q_at);
    Call a{q, out, H * D, ostride, (int)n, (int)H, (int)c.n_kv_heads, (int)(H / c.n_kv_heads),
           (int)std::min(window, far), (int)std::min(sinks, far), nullptr,
           reinterpret_cast<float2*>(w + l.ms_at), reinterpret_cast<float*>(w + l.po_at),
           reinterpret_cast<int*>(w + l.count_at), reinterpret_cast<int*>(w + l.redo_at), {}};
    for (int k = 0; k < 2; ++k)
        a.kind[k] = {tile_rows(k, D), places(k, D), target_pieces(k), k == kNarrow ? 4 : 2, 5,
                     k == kNarrow ? 0 : (int)l.rows[0], reinterpret_cast<int*>(w + l.head_at[k]),
                     reinterpret_cast<Item*>(w + l.items_at[k]), reinterpret_cast<Split*>(w + l.splits_at[k])};
    Prepare p{qkv, qkv + H * D, qstride, q, 2, 0, 0, 0, 0, 1, 0};
    p.q_rows = n <= 512 ? 4 : 16;
    const int64_t blocks = (n + p.q_rows - 1) / p.q_rows;
    p.q_heads = heads_each(blocks, H);
    p.q_groups = (int)(blocks * ((H + p.q_heads - 1) / p.q_heads));
    if (append) plan_writes(c, n, p);
    return by_pool(c, [&](auto code, auto dim) {
        return launch_typed<decltype(code), decltype(dim)::value>(c, t, a, p, l, s);
    });
}

size_t kv8_workspace_bytes(const PagedKv8& c, const unillm_page_table& t, int64_t n, int64_t H) {
    return layout(c, t, n, H).bytes;
}

hipError_t launch_kv8_read(const PagedKv8& c, const unillm_page_table& t, const int* ids,
                           const int* starts, const int* cu, int64_t n_seqs, int64_t n, int type,
                           void* k_out, void* v_out, int64_t ostride, hipStream_t s) {
    // (a workgroup's tasks are its runs times its heads: of few heads it takes more rows, where they are many.
    // 171000 rows of 2 heads of 256: 16 a workgroup 174 us, so 108)
    int rows = kBlock;
    while (rows < kReadRows && rows * c.n_kv_heads < 8 * kBlock && n >= (int64_t)4096 * rows / kBlock) rows *= 2;
    const int64_t blocks = (n + rows - 1) / rows;
    Read a{ids, starts, cu, (int)n_seqs, (int)n, k_out, v_out, ostride, rows, heads_each(blocks, c.n_kv_heads)};
    const unsigned grid = (unsigned)((blocks * ((c.n_kv_heads + a.heads - 1) / a.heads) + 7) / 8 * 8);
    return by_pool(c, [&](auto code, auto dim) {
        using C = decltype(code);
        constexpr int D = decltype(dim)::value;
        if (type == UNILLM_QTYPE_F32) kv8_read_kernel<C, float, D><<<grid, 256, 0, s>>>(c, t.st, a);
        else if (type == UNILLM_QTYPE_F16) kv8_read_kernel<C, _Float16, D><<<grid, 256, 0, s>>>(c, t.st, a);
        else kv8_read_kernel<C, __bf16, D><<<grid, 256, 0, s>>>(c, t.st, a);
        return hipGetLastError();
    });
}

}  // namespace unillm
