// paged8.hip -- paged KV caches held in 8 bits: written, read back, attended.
//
// A pool's codes are int8 or e4m3, and 16 positions of a kv head share a power of two, so a code c of a
// block with byte b stands for c 2^(b - 127).  Powers of two: a block's exponent grows as further
// positions come, and its codes are rounded anew then.  Each growth at least doubles the step, so the
// roundings add up to less than one step however often it happens (with the tightest step, growing
// by little each time, to several), and rounding to half the step or rounding a code to twice
// the step is exact arithmetic: the same bits on every machine.
//
// Attention is that of paged.hip (its plan, pieces and merge are shared, paged.hpp):
//   out = sum_j w_j v_j / sum_j w_j,  w_j = e^(q k_j / sqrt(hd) - max).
// A code is exact in f16 and in bf16.  q k: codes in f16 against two f16 parts of q (22 bits), the block's
// power of two multiplied onto the scores; w v: codes in bf16 against three bf16 parts of the weight
// times its block's power of two, all 24 bits of it and of any size.
#include <hip/hip_runtime.h>

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace unillm {
namespace {

constexpr int kBlock = 16;  // positions to an exponent
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
// 2^(b - 127), of b in [1, 254] (0: 0; 255, which no block is given, as 254)
__device__ __forceinline__ float power(int b) { return __uint_as_float((uint32_t)min(b, 254) << 23); }

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

// ---- rows into their blocks -------------------------------------------------------------------
//
// Rows of consecutive slots in one block of 16 are a run: a wave writes a run of one kv head's keys, or
// values, whole, so no two waves meet in a block, and an exponent's byte is its own.
constexpr int kWriteRows = 16;  // rows of a workgroup whose runs it takes, at most

struct Runs {
    int slots[2 * kWriteRows];  // of row row0 - 1 + i, -1: none
    int first[kWriteRows], count[kWriteRows];
    int n, end;  // runs; rows from row0 on that they take in
};

// The runs that begin in rows row0 .. row0 + nr - 1 (slot: of row row0 - 1 + threadIdx.x, up to nr + 16 of
// them).  All threads of the workgroup.
__device__ __forceinline__ void find_runs(Runs& r, int slot, int nr) {
    const int tid = threadIdx.x;
    if (tid < nr + 16) r.slots[tid] = slot;
    if (tid == 0) r.end = 0;
    __syncthreads();
    if (tid < 64) {
        const int sl = tid < nr ? r.slots[tid + 1] : -1;
        const bool begins = sl >= 0 && (r.slots[tid] + 1 != sl || sl % kBlock == 0);
        const uint64_t all = __ballot(begins);
        if (begins) {
            int n = 1;
            while (sl % kBlock + n < kBlock && tid + 1 + n < nr + 16 && r.slots[tid + 1 + n] == sl + n) ++n;
            const int at = __popcll(all & ((1ull << tid) - 1));
            r.first[at] = tid;
            r.count[at] = n;
            atomicMax(&r.end, tid + n);
        }
        if (tid == 0) r.n = __popcll(all);
    }
    __syncthreads();
}

// The cosines and sines of rows row0 .. row0 + rows - 1, [rows][R / 2].  All threads of the workgroup.
__device__ __forceinline__ void turns(const PagedKv8& c, const PageTable& t, int row0, int rows, double2* turn) {
    const int pairs = c.rotary_dim / 2;
    for (int i = threadIdx.x; i < rows * pairs; i += 256) {
        double sn, cs;
        sincospi((double)t.positions[row0 + i / pairs] * c.freq[i % pairs], &sn, &cs);
        turn[i] = make_double2(cs * c.magnitude, sn * c.magnitude);
    }
    __syncthreads();
}

// Dimensions d .. d + 3 (d a multiple of 4) of the head at x, rotated.
__device__ __forceinline__ f32x4 rotated4(const PagedKv8& c, const float* x, int d, const double2* turn) {
    f32x4 v = *reinterpret_cast<const f32x4*>(x + d);
    const int R = c.rotary_dim, half = R / 2;
    if (d >= R) return v;
    if (c.layout == UNILLM_ROPE_HALF) {
        const bool lo = d < half;
        const f32x4 w = *reinterpret_cast<const f32x4*>(x + (lo ? d + half : d - half));
        const double2* z = turn + (lo ? d : d - half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double a = v[e], b = w[e];
            v[e] = (float)(lo ? a * z[e].x - b * z[e].y : b * z[e].y + a * z[e].x);
        }
    } else {
        const double2* z = turn + d / 2;
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const double a = v[e], b = v[e + 1];
            v[e] = (float)(a * z[e / 2].x - b * z[e / 2].y);
            v[e + 1] = (float)(a * z[e / 2].y + b * z[e / 2].x);
        }
    }
    return v;
}

// A value's magnitude where it is finite, else 0 (and `odd` is set).
__device__ __forceinline__ float magnitude(float v, bool& odd) {
    const float m = fabsf(v);
    if (m < INFINITY) return m;
    odd = true;
    return 0.0f;
}

// Byte of a run's block: what its values need, and what it has if it holds positions before them.
template <class C>
__device__ __forceinline__ int grow(uint8_t* exps, int64_t at, float top, bool held, int& had) {
    const int need = least_exponent<C>(wave_max(top));
    had = held ? min((int)exps[at], 254) : 0;
    const int b = max(need, had);
    if ((threadIdx.x & 63) == 0) exps[at] = (uint8_t)b;
    return b;
}

// A run's keys of kv head g: rows row .. row + n - 1 of kv (a head's keys at x), into slots sl ..
template <class C, int D>
__device__ void write_keys(const PagedKv8& c, const float* x, int64_t stride, int n, int sl, int g,
                           const double2* turn, bool& odd) {
    constexpr int CH = D / 4, RP = 64 / CH, N = kBlock / RP;  // lanes a row, rows and passes
    const int lane = threadIdx.x & 63, d = lane % CH * 4, sub = lane / CH;
    const int pairs = c.rotary_dim / 2, off = sl % kBlock;
    const int in_page = sl & ((int)c.page_size - 1);
    const int64_t head = (int64_t)(sl >> c.page_shift) * c.n_kv_heads + g;
    uint8_t* dst = c.k + ((head << c.page_shift) + in_page) * D + d;
    f32x4 v[N];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0f;
        const int r = i * RP + sub;
        if (r < n) v[i] = rotated4(c, x + r * stride, d, turn + r * pairs);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // (opaque: the keys are rows of f32 first, and rounded from there)
        asm volatile("" : "+v"(v[i]));
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, magnitude(v[i][e], odd));
    }
    int had;
    const int b = grow<C>(c.k_exp, (head << c.page_shift >> 4) + in_page / kBlock, top, off > 0, had);
    const float inv = power(254 - b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = i * RP + sub;
        if (r < n)
            *reinterpret_cast<uint32_t*>(dst + r * D) =
                encode4<C>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
    }
    if (off > 0 && b > had) {
        const float f = power(max(127 + had - b, 1));
        uint32_t* old = reinterpret_cast<uint32_t*>(dst - d - off * D);
        for (int i = lane; i < off * CH; i += 64) old[i] = again4<C>(old[i], f);
    }
}

// A run's values.
template <class C, int D>
__device__ void write_values(const PagedKv8& c, const float* x, int64_t stride, int n, int sl, int g, bool& odd) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63, off = sl % kBlock;
    const int in_page = sl & ((int)c.page_size - 1);
    const int64_t head = (int64_t)(sl >> c.page_shift) * c.n_kv_heads + g;
    uint8_t* dst = c.v + ((head * D + lane) << c.page_shift) + in_page / kBlock * kBlock;
    float v[N][kBlock], top = 0.0f;  // by position of the block
#pragma unroll
    for (int p = 0; p < kBlock; ++p) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j][p] = 0.0f;
        if (p >= off && p < off + n)
#pragma unroll
            for (int j = 0; j < N; ++j) v[j][p] = x[(p - off) * stride + 64 * j + lane];
    }
#pragma unroll
    for (int p = 0; p < kBlock; ++p)
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, magnitude(v[j][p], odd));
    int had;
    const int b = grow<C>(c.v_exp, (head << c.page_shift >> 4) + in_page / kBlock, top, off > 0, had);
    const float inv = power(254 - b), f = power(max(127 + had - b, 1));
    const bool anew = off > 0 && b > had;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        u32x4* to = reinterpret_cast<u32x4*>(dst + ((int64_t)(64 * j) << c.page_shift));
        u32x4 w = 0u;
        if (n < kBlock) w = *to;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t fresh = encode4<C>(v[j][4 * i] * inv, v[j][4 * i + 1] * inv, v[j][4 * i + 2] * inv,
                                              v[j][4 * i + 3] * inv);
            const uint32_t old = anew ? again4<C>(w[i], f) : w[i];
            uint32_t is_old = 0, is_new = 0;  // bytes of the word
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = 4 * i + e;
                if (p < off) is_old |= 0xFFu << (8 * e);
                else if (p < off + n) is_new |= 0xFFu << (8 * e);
            }
            w[i] = (fresh & is_new) | (old & is_old) | (w[i] & ~(is_new | is_old));
        }
        *to = w;
    }
}

// What a call's first kernel does: `plan` workgroups deal the work out; then q_groups take q_rows query
// rows and q_heads heads each (rotated, times log2 e / sqrt(hd), f32, into q_out); the rest write the runs
// that begin in `rows` rows, of `heads` kv heads.
struct Prepare {
    const float *q, *kv;
    int64_t stride;  // of both
    float* q_out;
    int plan, q_groups, q_rows, q_heads, rows, heads;
};

template <class C, int D>
__global__ __launch_bounds__(256) void kv8_prepare_kernel(PagedKv8 c, PageTable t, Call a, Prepare p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    double2* turn = reinterpret_cast<double2*>(lds);
    const int tid = threadIdx.x;
    if (!step_fits(t, a.n)) {
        if (p.plan == 0) {
            if (blockIdx.x == 0 && tid == 0)
                atomicCAS(&t.counts[kPagesError], 0, t.counts[kPagesStep] == 1 ? kPagesRows : kPagesNoPlan);
            return;
        }
        if (blockIdx.x < 2 && tid < 2) a.kind[blockIdx.x].head[tid] = 0;
        if (blockIdx.x == 0 && tid == 0) *a.redo_count = 0;
        fail_call(t, a, D, blockIdx.x, gridDim.x);
        return;
    }
    int bx = (int)blockIdx.x;
    if (bx < p.plan) {
        if (bx == 0 && tid == 0) *a.redo_count = 0;
        if (bx == 0) return plan<64, INT_MAX>(t, a, kNarrow, reinterpret_cast<int*>(lds));
        if (tid < 2) a.kind[kWide].head[tid] = 0;
        return;
    }
    bx -= p.plan;
    const int total = t.counts[kPagesTokens];
    if (bx < p.q_groups) {
        const int groups = (a.H + p.q_heads - 1) / p.q_heads;
        const int row0 = bx / groups * p.q_rows, h0 = bx % groups * p.q_heads;
        const int rows = min(p.q_rows, total - row0), heads = min(p.q_heads, a.H - h0);
        if (rows <= 0) return;
        turns(c, t, row0, rows, turn);
        const float scale = kLog2e / sqrtf((float)D);
        constexpr int CH = D / 4;
        for (int i = tid; i < rows * heads * CH; i += 256) {
            const int d = i % CH * 4, h = h0 + i / CH % heads, r = i / CH / heads;
            const f32x4 v = rotated4(c, p.q + (row0 + r) * p.stride + (int64_t)h * D, d, turn + r * (c.rotary_dim / 2));
            *reinterpret_cast<f32x4*>(p.q_out + ((int64_t)(row0 + r) * a.H + h) * D + d) = v * scale;
        }
        return;
    }
    bx -= p.q_groups;
    __shared__ Runs runs;
    const int KVH = (int)c.n_kv_heads, groups = (KVH + p.heads - 1) / p.heads;
    const int row0 = bx / groups * p.rows, g0 = bx % groups * p.heads, heads = min(p.heads, KVH - g0);
    if (row0 >= total) return;
    const int row = row0 - 1 + tid;
    find_runs(runs, tid < p.rows + 16 && row >= 0 && row < total ? t.slots[row] : -1, p.rows);
    if (runs.n == 0) return;
    turns(c, t, row0, runs.end, turn);
    bool odd = false;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = wv; i < runs.n * heads * 2; i += 4) {
        const int g = g0 + i / 2 % heads, run = i / 2 / heads;
        const int r = __builtin_amdgcn_readfirstlane(runs.first[run]);
        const int n = __builtin_amdgcn_readfirstlane(runs.count[run]);
        const int sl = __builtin_amdgcn_readfirstlane(runs.slots[r + 1]);
        const float* x = p.kv + (row0 + r) * p.stride + (int64_t)g * D;
        if (i % 2 == 0) write_keys<C, D>(c, x, p.stride, n, sl, g, turn + r * (c.rotary_dim / 2), odd);
        else write_values<C, D>(c, x + (int64_t)KVH * D, p.stride, n, sl, g, odd);
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
template <int D>
struct Narrow8Lds {
    static constexpr int NB = D / 32, OT = D / 16;
    static constexpr int IDS = 0;                          // page ids of 256 visits, 4 each
    static constexpr int STAT = IDS + 4096;                // row scales, maxima, sums, flags
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

template <class C, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv8_narrow_kernel(PagedKv8 c, PageTable t, Call a) {
    using L = Narrow8Lds<D>;
    constexpr int NB = L::NB, OT = L::OT, KB = D / 64, U = 64;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int* ids = reinterpret_cast<int*>(lds + L::IDS);               // [256][4]
    float* rowmax = reinterpret_cast<float*>(lds + L::STAT);       // [16]
    float* wm = rowmax + 16;                                        // [4][16]
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
        // q's parts: task (product, lane) as the B operand takes it
        constexpr int TASKS = (NB * 64 + 255) / 256;
        f32x8 qv[TASKS];
        __syncthreads();  // (the item before is done with the LDS)
        if (tid < 16) rowmax[tid] = 0.0f;
        if (tid < 2) flags[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
            const int f = i * 256 + tid, r = f % 16, b = f / 64, d = b / 2 * 64 + f / 16 % 4 * 16 + b % 2 * 8;
            qv[i] = 0.0f;
            if (f < NB * 64 && r < it.rows) {
                const int rr = it.row0 + r;
                const f32x4* x = reinterpret_cast<const f32x4*>(
                    a.qkv + (first + rr / G) * a.qstride + (int64_t)(g * G + rr % G) * D + d);
                const f32x4 lo = x[0], hi = x[1];
                float mx = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    qv[i][j] = j < 4 ? lo[j % 4] : hi[j % 4];
                    mx = fmaxf(mx, fabsf(qv[i][j]));
                }
                atomicMax(reinterpret_cast<int*>(rowmax) + r, __float_as_int(mx));  // (magnitudes order as their bits)
            }
        }
        __syncthreads();
        const float inv = row_scale(rowmax[col]).y;  // of this lane's row
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
            const int f = i * 256 + tid;
            if (f < NB * 64) {
                qv[i] *= row_scale(rowmax[f % 16]).x;
                u32x4 p[2];
                parts_f16(qv[i], p);
#pragma unroll
                for (int q = 0; q < 2; ++q) qp[q * NB * 64 + f] = p[q];
            }
        }
        const int ppos = ctx + min(it.row0 + col, it.row0 + it.rows - 1) / G;  // the lane's row's position

        float ref = -INFINITY, l = 0.0f;
        f32x4 o[OT];
#pragma unroll
        for (int i = 0; i < OT; ++i) o[i] = 0.0f;
        u32x4 q[2][NB];
        u32x4 kr[4][KB], vr[OT];
        int ke = 0, ve = 0;
        for (int seg = 0; seg < it.nv; seg += 256) {
            const int nseg = min(256, it.nv - seg);
            __syncthreads();
            for (int i = tid; i < 4 * nseg; i += 256) {  // the page of each block
                int j = vis.key(it.v0 + seg + i / 4);
                if (j + i % 4 * kBlock < len) j += i % 4 * kBlock;  // (past the sequence: the visit's first again)
                int pg = pages[j >> shift];
                if ((unsigned)pg >= (unsigned)c.n_pages) {
                    pg = 0;
                    flags[0] = 1;
                }
                ids[i] = pg;
            }
            __syncthreads();
            if (seg == 0)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int b = 0; b < NB; ++b) q[i][b] = qp[(i * NB + b) * 64 + lane];
            // block x of visit v: its page and head, and its first key's place in the page
            auto block = [&](int v, int x, int64_t& head, int& off) {
                const int j = vis.key(it.v0 + seg + v);
                head = (int64_t)ids[4 * v + x] * KVH + g;
                off = (j + (j + x * kBlock < len ? x * kBlock : 0)) & (ps - 1);
            };
            auto load_k = [&](int v) {
                int64_t head;
                int off;
                block(v, col / 4, head, off);
                const uint8_t* k = c.k + ((head << shift) + off + col % 4) * D + 16 * qd;
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int b = 0; b < KB; ++b) kr[s][b] = *reinterpret_cast<const u32x4*>(k + 4 * s * D + 64 * b);
                block(v, qd, head, off);
                ke = c.k_exp[(head << shift >> 4) + off / kBlock];
            };
            auto load_v = [&](int v) {
                int64_t head;
                int off;
                block(v, qd, head, off);
                const uint8_t* x = c.v + ((head * D + col) << shift) + off;
#pragma unroll
                for (int i = 0; i < OT; ++i) vr[i] = *reinterpret_cast<const u32x4*>(x + ((16 * i) << shift));
                ve = c.v_exp[(head << shift >> 4) + off / kBlock];
            };
            if (wv < nseg) {
                load_k(wv);
                load_v(wv);
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
                if (v + 4 < nseg) load_k(v + 4);
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
                const float step = power(ve);
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
                if (!whole) a.ms[piece] = make_float2(top, again || bad_page ? __builtin_nanf("") : sum);
            }
        }
    }
}

// One row and head by a wave, in plain f32: for rows whose products of parts came out non-finite (an
// infinite query, or scores past f32's range).  qf: LDS [D], the query; sc: LDS [64].  Lane el gets
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
struct Read {
    const int *ids, *starts, *cu;
    int B, n;
    void *k, *v;
    int64_t stride;
    int heads;  // of a workgroup
};

template <class O>
struct alignas(16) Eight {
    O v[16 / sizeof(O)];
};

// The mirror of the writes: runs of rows in one block, a wave a run of one kv head's keys or values.
template <class C, class O, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(PagedKv8 c, PageTable t, Read a) {
    constexpr int NR = kWriteRows;
    __shared__ Runs runs;
    __shared__ uint64_t bad_rows;
    const int tid = threadIdx.x, lane = tid & 63;
    const int KVH = (int)c.n_kv_heads, groups = (KVH + a.heads - 1) / a.heads;
    const int row0 = (int)(blockIdx.x / groups) * NR, g0 = (int)(blockIdx.x % groups) * a.heads;
    const int heads = min(a.heads, KVH - g0), end = min(a.n, a.cu[a.B]);
    if (row0 >= end) return;
    int slot = -1;
    bool bad = false;
    const int row = row0 - 1 + tid;
    if (tid < NR + 16 && row >= 0 && row < end) {
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.cu[mid] <= row) lo = mid;
            else hi = mid;
        }
        const int id = a.ids[lo];
        const int64_t pos = (int64_t)a.starts[lo] + row - a.cu[lo];
        if (id >= 0) {
            bad = true;
            if (id < t.max_seqs && pos >= 0 && pos < t.lens[id] && (pos >> c.page_shift) < t.max_pages) {
                const int pg = t.table[(int64_t)id * t.max_pages + (pos >> c.page_shift)];
                if ((unsigned)pg < (unsigned)c.n_pages) {
                    slot = (pg << c.page_shift) + (int)(pos & (c.page_size - 1));
                    bad = false;
                }
            }
        }
    }
    if (tid < 64) {
        const uint64_t b = __ballot(bad) >> 1;  // (bit i: row row0 + i)
        if (tid == 0) {
            bad_rows = b & ((1ull << NR) - 1);
            if (bad_rows != 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesBadRead);
        }
    }
    find_runs(runs, slot, NR);
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    O* const outs[2] = {static_cast<O*>(a.k), static_cast<O*>(a.v)};
    if (bad_rows != 0)
        for (int r = wv; r < NR; r += 4)
            if (bad_rows >> r & 1)
                for (int w = 0; w < 2; ++w)
                    if (outs[w])
                        for (int d = lane; d < heads * D; d += 64)
                            outs[w][(row0 + r) * a.stride + (int64_t)g0 * D + d] = (O)__builtin_nanf("");
    for (int i = wv; i < runs.n * heads * 2; i += 4) {
        const int g = g0 + i / 2 % heads, run = i / 2 / heads;
        O* out = outs[i % 2];
        if (!out) continue;
        const int r0 = __builtin_amdgcn_readfirstlane(runs.first[run]);
        const int n = __builtin_amdgcn_readfirstlane(runs.count[run]);
        const int sl = __builtin_amdgcn_readfirstlane(runs.slots[r0 + 1]);
        const int in_page = sl & ((int)c.page_size - 1), off = sl % kBlock;
        const int64_t head = (int64_t)(sl >> c.page_shift) * KVH + g;
        const float step = power((i % 2 ? c.v_exp : c.k_exp)[(head << c.page_shift >> 4) + in_page / kBlock]);
        out += (row0 + r0) * a.stride + (int64_t)g * D;
        if (i % 2 == 0) {
            constexpr int CH = D / 16, RP = 64 / CH;  // lanes a row, rows at a time
            const uint8_t* k = c.k + ((head << c.page_shift) + in_page) * D;
            for (int r = lane / CH; r < n; r += RP) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(k + r * D + lane % CH * 16);
                O* to = out + r * a.stride + lane % CH * 16;
                constexpr int E = 16 / sizeof(O);
#pragma unroll
                for (int x = 0; x < 16 / E; ++x) {
                    Eight<O> y;
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const f32x4 z = decode4<C>(w[(x * E + e) / 4]) * step;
#pragma unroll
                        for (int j = 0; j < 4; ++j) y.v[e + j] = (O)z[j];
                    }
                    *reinterpret_cast<Eight<O>*>(to + x * E) = y;
                }
            }
        } else {
            // two dimensions a lane
            struct alignas(2 * sizeof(O)) Two {
                O v[2];
            };
            const uint8_t* v = c.v + ((head * D) << c.page_shift) + in_page - off;
            for (int d = 2 * lane; d < D; d += 128) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(v + ((int64_t)d << c.page_shift));
                const u32x4 y = *reinterpret_cast<const u32x4*>(v + ((int64_t)(d + 1) << c.page_shift));
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const f32x4 p = decode4<C>(x[w]) * step, q = decode4<C>(y[w]) * step;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * w + e - off;
                        if (r >= 0 && r < n)
                            *reinterpret_cast<Two*>(out + r * a.stride + d) = Two{{(O)p[e], (O)q[e]}};
                    }
                }
            }
        }
    }
}

// ---- launches ---------------------------------------------------------------------------------

// Workgroups of the narrow kernel that the device holds, and pieces to deal its work out in at most.
int places(int64_t D) { return (D == 256 ? 1 : 2) * device_info().cu_count; }
int target_pieces() { return 3 * device_info().cu_count; }

struct Layout {
    int64_t items, rows;
    size_t head_at[2], items_at, splits_at, q_at, ms_at, po_at, count_at, redo_at, bytes;
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
    // tiles: an entry's last may be ragged.  A tile of nv visits makes at most nv / C + 1 pieces, and
    // the nv / C add up to target / KVH; more than one piece, at most 2 nv / C.
    const int64_t tiles = n * G / kTileRows + std::min<int64_t>(n, t.st.max_seqs);
    l.items = tiles + target_pieces() / KVH + 1;
    l.rows = 2 * (int64_t)target_pieces() * std::min<int64_t>(kTileRows, n * G);
    for (int k = 0; k < 2; ++k) l.head_at[k] = take(2 * sizeof(int));
    l.items_at = take(l.items * (int64_t)sizeof(Item));
    l.splits_at = take(tiles * (int64_t)sizeof(Split));
    l.q_at = take(n * H * D * (int64_t)sizeof(float));
    l.ms_at = take(l.rows * (int64_t)sizeof(float2));
    l.po_at = take(l.rows * D * (int64_t)sizeof(float));
    // rows to do again: every (row, head), and again for each piece
    l.count_at = take(sizeof(int));
    l.redo_at = take((n * H + l.rows) * (int64_t)sizeof(int));
    l.bytes = at;
    return l;
}

// Heads to a workgroup: one, or what leaves four workgroups a CU.
int heads_each(int64_t blocks, int64_t heads) {
    return (int)std::min<int64_t>(heads, std::max<int64_t>(1, blocks * heads / (4 * device_info().cu_count)));
}

// The writes' part of a first kernel: its workgroups.
int64_t plan_writes(const PagedKv8& c, int64_t n, Prepare& p) {
    p.rows = n <= 512 ? 4 : kWriteRows;
    const int64_t blocks = (n + p.rows - 1) / p.rows;
    p.heads = heads_each(blocks, c.n_kv_heads);
    return blocks * ((c.n_kv_heads + p.heads - 1) / p.heads);
}

template <class C, int D>
hipError_t launch_prepare(const PagedKv8& c, const unillm_page_table& t, const Call& a, const Prepare& p,
                          int64_t writes, hipStream_t s) {
    constexpr int kMost = (3 * kPagesMaxSeqs + 1) * (int)sizeof(int);
    static_assert(kMost >= (2 * kBlock - 1) * 128 * (int)sizeof(double2), "31 rows of 128 pairs");
    static const bool attr = hipFuncSetAttribute((const void*)kv8_prepare_kernel<C, D>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, kMost) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    const size_t pairs = (size_t)c.rotary_dim / 2 * sizeof(double2);
    size_t lds = std::max((size_t)(p.rows + kBlock - 1) * pairs, (size_t)p.q_rows * pairs);
    if (p.plan) lds = std::max(lds, (size_t)(3 * t.st.max_seqs + 1) * sizeof(int));  // (three ints an entry)
    const unsigned grid = (unsigned)(p.plan + p.q_groups + writes);
    kv8_prepare_kernel<C, D><<<grid, 256, lds, s>>>(c, t.st, a, p);
    return hipGetLastError();
}

template <class C, int D>
hipError_t launch_typed(const PagedKv8& c, const unillm_page_table& t, const Call& a, const Prepare& p,
                        int64_t writes, const Layout& l, hipStream_t s) {
    hipError_t e = launch_prepare<C, D>(c, t, a, p, writes, s);
    if (e != hipSuccess) return e;
    using N = Narrow8Lds<D>;
    static const bool attr = hipFuncSetAttribute((const void*)kv8_narrow_kernel<C, D>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, N::BYTES) == hipSuccess;
    if (!attr) return hipErrorInvalidValue;
    const int64_t most = 4 * device_info().cu_count;
    kv8_narrow_kernel<C, D><<<(unsigned)std::min<int64_t>(l.items * a.KVH, most), 256, N::BYTES, s>>>(c, t.st, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    kv8_merge_kernel<C, D><<<(unsigned)std::min<int64_t>(l.rows / 2, most), 256, 0, s>>>(c, t.st, a);
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
    Prepare p{nullptr, kv, kvstride, nullptr, 0, 0, 0, 1, 0, 0};
    const int64_t writes = plan_writes(c, n, p);
    return by_pool(c, [&](auto code, auto dim) {
        return launch_prepare<decltype(code), decltype(dim)::value>(c, t, a, p, writes, s);
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
    a.kind[kNarrow] = {kTileRows, places(D), target_pieces(), 4, 5, 0, reinterpret_cast<int*>(w + l.head_at[0]),
                       reinterpret_cast<Item*>(w + l.items_at), reinterpret_cast<Split*>(w + l.splits_at)};
    a.kind[kWide] = {16, 1, 1, 1, 1, 0, reinterpret_cast<int*>(w + l.head_at[1]), nullptr, nullptr};
    Prepare p{qkv, qkv + H * D, qstride, q, 2, 0, 0, 0, 0, 0};
    p.q_rows = n <= 512 ? 4 : 16;
    const int64_t blocks = (n + p.q_rows - 1) / p.q_rows;
    p.q_heads = heads_each(blocks, H);
    p.q_groups = (int)(blocks * ((H + p.q_heads - 1) / p.q_heads));
    const int64_t writes = append ? plan_writes(c, n, p) : (p.heads = 1, p.rows = 0, 0);
    return by_pool(c, [&](auto code, auto dim) {
        return launch_typed<decltype(code), decltype(dim)::value>(c, t, a, p, writes, l, s);
    });
}

size_t kv8_workspace_bytes(const PagedKv8& c, const unillm_page_table& t, int64_t n, int64_t H) {
    return layout(c, t, n, H).bytes;
}

hipError_t launch_kv8_read(const PagedKv8& c, const unillm_page_table& t, const int* ids,
                           const int* starts, const int* cu, int64_t n_seqs, int64_t n, int type,
                           void* k_out, void* v_out, int64_t ostride, hipStream_t s) {
    const int64_t blocks = (n + kWriteRows - 1) / kWriteRows;
    Read a{ids, starts, cu, (int)n_seqs, (int)n, k_out, v_out, ostride, heads_each(blocks, c.n_kv_heads)};
    const unsigned grid = (unsigned)(blocks * ((c.n_kv_heads + a.heads - 1) / a.heads));
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
