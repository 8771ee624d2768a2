// rope.hip -- rotary positions of rows of heads (unillm_hip_rope_apply).
//
// A pair (x, y) of a head, in a row at position p, becomes m (x cos a - y sin a), m (x sin a + y
// cos a) with a = p f_i, i the pair's number: dimensions i and i + R / 2 (half-split) or 2 i and
// 2 i + 1 (interleaved) of the first R; the dimensions past R stay as they are.  Angles are formed
// and reduced in f64, in half turns (at position 100000 their f32 forms are 0.003 off), and the
// products are f64 as well: a row's own type is rounded to once.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "internal.hpp"
#include "split.hpp"

namespace unillm {
namespace {

typedef _Float16 rope_f16;
struct rope_bf16 {
    uint16_t bits;
};
__device__ __forceinline__ float rope_widen(float v) { return v; }
__device__ __forceinline__ float rope_widen(rope_f16 v) { return (float)v; }
__device__ __forceinline__ float rope_widen(rope_bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
// An f64 value to a row's type, the 16-bit ones through f32, which is off by 2^-24 at most.  (Opaque between: the
// compiler would fold the two conversions into one from f64, some 30 instructions; 4096 rows of 32 heads
// of 128 took 28 us.)
template <class T>
__device__ __forceinline__ T rope_narrow(double v) {
    float f = (float)v;
    if constexpr (sizeof(T) == 4) {
        return f;
    } else {
        asm volatile("" : "+v"(f));
        if constexpr (std::is_same_v<T, rope_f16>) return (rope_f16)f;
        else return rope_bf16{(uint16_t)(pack_bf16(f, 0.0f) & 0xFFFF)};
    }
}

// V neighbouring elements; W: that many are aligned together.
template <class T, int V, int W>
struct alignas(W * sizeof(T)) Some {
    T v[V];
};

struct RopeCall {
    const void* x;
    void* out;
    const int* positions;
    const double* freq;  // half turns a position of each pair
    double magnitude;
    int64_t xstride, ostride;
    int n, heads, hd, rot, copy;
};

// A workgroup takes `rows` rows: a thread has a unit of a head, V elements (half-split: and their partners),
// of every so many of their heads, four at a time, the first four requested before the rows' cosines and
// sines are formed (in LDS).
// Bound by HBM where rows are many (20001 rows of 32 heads of 128 in f32, 655 MB in 125 us: 5.2 TB/s, a copy's
// rate), by latency for few (one row 3.3 us, 777 rows in f16 5.4).
template <class T, int V, int W, bool HALF>
__global__ __launch_bounds__(256) void rope_kernel(RopeCall a, int rows) {
    using S = Some<T, V, W>;
    constexpr int B = 4, P = HALF ? V : V / 2;  // items at a time, pairs of a unit
    constexpr bool kOdd = W < V;                // a head may end inside its last unit
    // [rows][rot / 2], pair p at p % P rot / 2 P + p / P: what lanes read together lies together
    extern __shared__ double2 turn[];
    const int tid = threadIdx.x, pairs = a.rot / 2, sets = pairs / P;
    const int64_t row0 = (int64_t)blockIdx.x * rows;
    const int n = (int)min((int64_t)rows, a.n - row0);
    // units of a head: those that turn first, then those that are copied
    const int turning = (HALF ? pairs : a.rot) / V, units = turning + (a.copy ? (a.hd - a.rot + (kOdd ? V - 1 : 0)) / V : 0);
    const int across = min(units, 256), side = tid / across, sides = 256 / across;
    const int dr = sides / a.heads, dh = sides % a.heads;
    int u = side < sides ? tid % across : units;
    // the thread's place among the rows and heads, of unit u
    int r = 0, h = 0;
    auto begin = [&] {
        r = side / a.heads;
        h = side % a.heads;
    };
    auto next = [&] {
        r += dr;
        h += dh;
        if (h >= a.heads) h -= a.heads, ++r;
    };
    S lo[B], hi[B];
    int rr[B], hh[B];
    auto load = [&] {
        const int d = u < turning ? u * V : a.rot + (u - turning) * V;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            rr[i] = r;
            hh[i] = h;
            if (u < units && r < n) {
                const T* x = static_cast<const T*>(a.x) + (row0 + r) * a.xstride + h * a.hd + d;
                if (kOdd && d + V > a.hd) lo[i].v[0] = x[0];
                else lo[i] = *reinterpret_cast<const S*>(x);
                if (HALF && u < turning) hi[i] = *reinterpret_cast<const S*>(x + pairs);
            }
            next();
        }
    };
    begin();
    load();
    for (int i = tid; i < n * pairs; i += 256) {
        double sn, cs;
        sincospi((double)a.positions[row0 + i / pairs] * a.freq[i % pairs], &sn, &cs);
        turn[i / pairs * pairs + i % pairs % P * sets + i % pairs / P] = make_double2(cs * a.magnitude, sn * a.magnitude);
    }
    __syncthreads();
    for (; u < units; u += across, begin(), load()) {
        const int d = u < turning ? u * V : a.rot + (u - turning) * V;
        for (; rr[0] < n; load())
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (rr[i] >= n) break;
                T* out = static_cast<T*>(a.out) + (row0 + rr[i]) * a.ostride + hh[i] * a.hd + d;
                if (u < turning && HALF) {
                    const double2* z = turn + rr[i] * pairs + u;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const double p = rope_widen(lo[i].v[e]), q = rope_widen(hi[i].v[e]);
                        lo[i].v[e] = rope_narrow<T>(p * z[e * sets].x - q * z[e * sets].y);
                        hi[i].v[e] = rope_narrow<T>(p * z[e * sets].y + q * z[e * sets].x);
                    }
                    *reinterpret_cast<S*>(out + pairs) = hi[i];
                } else if (u < turning) {
                    const double2* z = turn + rr[i] * pairs + u;
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        const double p = rope_widen(lo[i].v[2 * e]), q = rope_widen(lo[i].v[2 * e + 1]);
                        lo[i].v[2 * e] = rope_narrow<T>(p * z[e * sets].x - q * z[e * sets].y);
                        lo[i].v[2 * e + 1] = rope_narrow<T>(p * z[e * sets].y + q * z[e * sets].x);
                    }
                }
                if (kOdd && d + V > a.hd) out[0] = lo[i].v[0];
                else *reinterpret_cast<S*>(out) = lo[i];
            }
    }
}

template <class T, int V, int W, bool HALF>
hipError_t launch_width(const RopeCall& a, hipStream_t s) {
    // rows a workgroup: one, or what leaves 4096 workgroups; their turns in 32 KiB
    const int pairs = a.rot / 2;
    const int most = std::max(1, 2048 / pairs);
    const int rows = (int)std::min<int64_t>(most, std::max<int64_t>(1, a.n / 4096));
    const unsigned grid = (unsigned)((a.n + rows - 1) / rows);
    rope_kernel<T, V, W, HALF><<<grid, 256, (size_t)rows * pairs * sizeof(double2), s>>>(a, rows);
    return hipGetLastError();
}

template <class T, bool HALF>
hipError_t launch_type(const RopeCall& a, hipStream_t s) {
    // elements a lane moves at once: as many, up to 16 bytes, as divide everything
    auto fits = [&](int v) {
        const int64_t bytes = v * (int64_t)sizeof(T);
        return a.hd % v == 0 && (HALF ? a.rot / 2 : a.rot) % v == 0 && a.xstride % v == 0 &&
               a.ostride % v == 0 && (uintptr_t)a.x % bytes == 0 && (uintptr_t)a.out % bytes == 0;
    };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch_width<T, 8, 8, HALF>(a, s);
    if (fits(4)) return launch_width<T, 4, 4, HALF>(a, s);
    if (fits(2)) return launch_width<T, 2, 2, HALF>(a, s);
    return launch_width<T, HALF ? 1 : 2, 1, HALF>(a, s);
}

template <class T>
hipError_t launch_rope_type(bool interleaved, const RopeCall& a, hipStream_t s) {
    return interleaved ? launch_type<T, false>(a, s) : launch_type<T, true>(a, s);
}

}  // namespace

hipError_t launch_rope(const unillm_rope& r, int type, const void* x, int64_t xstride, int64_t n,
                       int64_t heads, const int* positions, void* out, int64_t ostride, hipStream_t s) {
    const RopeCall a{x, out, positions, r.freq, r.magnitude, xstride, ostride, (int)n, (int)heads,
                     (int)r.head_dim, (int)r.rotary_dim, x != out};
    const bool inter = r.layout == UNILLM_ROPE_INTERLEAVED;
    if (type == UNILLM_QTYPE_F32) return launch_rope_type<float>(inter, a, s);
    if (type == UNILLM_QTYPE_F16) return launch_rope_type<rope_f16>(inter, a, s);
    return launch_rope_type<rope_bf16>(inter, a, s);
}

}  // namespace unillm
