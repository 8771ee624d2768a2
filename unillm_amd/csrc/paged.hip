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

// What the kernels of a call share.
struct Call {
    const float* qkv;
    float* out;
    int64_t qstride, ostride;
    int n, H, KVH;
    int window, sinks;
};

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

// Keys and values of a row into its slot, a workgroup per row.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedKv c, PageTable t, Call a) {
    constexpr int HALF = D / 2;
    __shared__ double2 turn[HALF];
    const int row = blockIdx.x;
    if (!step_fits(t, a.n) || row >= t.counts[kPagesTokens]) return;
    const int slot = t.slots[row];
    if (slot < 0) return;
    if (threadIdx.x < HALF) {
        double sn, cs;
        sincospi((double)t.positions[row] * c.freq[threadIdx.x], &sn, &cs);
        turn[threadIdx.x] = make_double2(cs, sn);
    }
    __syncthreads();
    const int64_t page = slot >> c.page_shift, off = slot & (c.page_size - 1);
    const int KVH = a.KVH;
    const int64_t ps = c.page_size;
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

// One row and head by a wave, in plain f32: online softmax over 64 keys at a time.  qf: LDS
// [D], the rotated query / sqrt(D) in units of log2 e; sc: LDS [64].  Lane el gets dimensions
// el + 64 i of the unnormalized sum, with the maximum (log2) and the sum of the weights.
template <class T, int D>
__device__ void attend_row(const PagedKv& c, const int* pages, int g, int KVH, int p, int window,
                           int sinks, const float* qf, float* sc, float& mx, float& l,
                           float (&acc)[D / 64], bool& bad_page) {
    const int el = threadIdx.x & 63;
    const int64_t ps = c.page_size;
    auto settle = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto page_of = [&](int j) {
        const int pg = pages[j >> c.page_shift];
        if ((unsigned)pg < (unsigned)c.n_pages) return (int64_t)pg;
        bad_page = true;
        return (int64_t)0;
    };
    mx = -INFINITY;
    l = 0.0f;
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.0f;
    const int low = window > 0 ? max(0, p - window + 1) : 0;
    const int first = low / 64, last = p / 64;
    const int ns = window > 0 ? min((sinks + 63) / 64, first) : 0;
    for (int b = 0; b < ns + last - first + 1; ++b) {
        const int j0 = (b < ns ? b : first + b - ns) * 64;
        for (int i = 0; i < 8; ++i) {  // 8 lanes a key
            const int j = min(j0 + 8 * i + el / 8, p);
            const T* kr = static_cast<const T*>(c.k) +
                          ((page_of(j) * KVH + g) * ps + (j & (ps - 1))) * D + el % 8 * (D / 8);
            float dot = 0.0f;
            for (int d = 0; d < D / 8; ++d) dot = fmaf(widen(kr[d]), qf[el % 8 * (D / 8) + d], dot);
            dot += __shfl_xor(dot, 1, 64);
            dot += __shfl_xor(dot, 2, 64);
            dot += __shfl_xor(dot, 4, 64);
            if (el % 8 == 0) sc[8 * i + el / 8] = dot;
        }
        settle();
        const int j = j0 + el;
        const bool seen = j <= p && (j >= low || j < sinks);
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
        for (int u = 0; u < 8; ++u) {
            if ((mask >> (8 * u) & 0xFF) == 0) continue;
            const int j8 = j0 + 8 * u;
            const T* vr = static_cast<const T*>(c.v) + (page_of(j8) * KVH + g) * D * ps + (j8 & (ps - 1));
            for (int e = 0; e < 8; ++e)
                if (mask >> (8 * u + e) & 1)
                    for (int i = 0; i < D / 64; ++i)
                        acc[i] = fmaf(sc[8 * u + e], widen(vr[(el + 64 * i) * ps + e]), acc[i]);
        }
        settle();
    }
}

// A wave per (row, head).
template <class T, int D>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedKv c, PageTable t, Call a) {
    constexpr int HALF = D / 2;
    __shared__ float lds[4][D + 64];
    if (!step_fits(t, a.n)) {
        fail_call(t, a, D, blockIdx.x, gridDim.x);
        return;
    }
    const int rows = t.counts[kPagesTokens], B = t.counts[kPagesEntries];
    const int el = threadIdx.x & 63, wv = threadIdx.x >> 6;
    float* qf = lds[wv];
    const int64_t total = (int64_t)rows * a.H;
    for (int64_t i = (int64_t)blockIdx.x * 4 + wv; i < total; i += (int64_t)gridDim.x * 4) {
        const int row = (int)(i / a.H), h = (int)(i % a.H);
        int lo = 0, hi = B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (t.cu[mid] <= row) lo = mid;
            else hi = mid;
        }
        const int p = t.positions[row];
        const int* pages = t.table + (int64_t)t.step_ids[lo] * t.max_pages;
        const float* x = a.qkv + row * a.qstride + (int64_t)h * D;
        const float scale = kLog2e / sqrtf((float)D);
        for (int d = el; d < HALF; d += 64) {
            double sn, cs;
            sincospi((double)p * c.freq[d], &sn, &cs);
            const double u = x[d], v = x[d + HALF];
            qf[d] = (float)(u * cs - v * sn) * scale;
            qf[d + HALF] = (float)(u * sn + v * cs) * scale;
        }
        float mx, l, acc[D / 64];
        bool bad = false;
        attend_row<T, D>(c, pages, h / (a.H / a.KVH), a.KVH, p, a.window, a.sinks, qf, qf + D, mx, l,
                         acc, bad);
        bad = __any(bad);
        if (bad && el == 0) atomicCAS(&t.counts[kPagesError], 0, (int)kPagesBadState);
        float* o = a.out + row * a.ostride + (int64_t)h * D;
        for (int e = 0; e < D / 64; ++e) o[el + 64 * e] = bad ? __builtin_nanf("") : acc[e] / l;
    }
}

template <class T, int D>
hipError_t launch_typed(const PagedKv& c, const PageTable& t, const Call& a, hipStream_t s) {
    paged_append_kernel<T, D><<<(unsigned)a.n, 256, 0, s>>>(c, t, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t waves = (int64_t)a.n * a.H;
    paged_attention_kernel<T, D><<<(unsigned)std::min<int64_t>((waves + 3) / 4, 1 << 20), 256, 0, s>>>(
        c, t, a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_type(const PagedKv& c, const PageTable& t, const Call& a, hipStream_t s) {
    if (c.head_dim == 64) return launch_typed<T, 64>(c, t, a, s);
    if (c.head_dim == 128) return launch_typed<T, 128>(c, t, a, s);
    return launch_typed<T, 256>(c, t, a, s);
}

}  // namespace

hipError_t launch_paged_attention(const PagedKv& c, const unillm_page_table& t, const float* qkv,
                                  int64_t qstride, int64_t n, int64_t H, int64_t window,
                                  int64_t sinks, float* out, int64_t ostride, hipStream_t s) {
    // a window or sinks past any position are all of them
    const int64_t far = (int64_t)1 << 30;
    const Call a{qkv, out, qstride, ostride, (int)n, (int)H, (int)c.n_kv_heads,
                 (int)std::min(window, far), (int)std::min(sinks, far)};
    if (c.type == UNILLM_QTYPE_F32) return launch_type<float>(c, t.st, a, s);
    if (c.type == UNILLM_QTYPE_F16) return launch_type<f16_t>(c, t.st, a, s);
    return launch_type<bf16_t>(c, t.st, a, s);
}

size_t paged_workspace_bytes(const PagedKv&, const unillm_page_table&, int64_t, int64_t) { return 0; }

}  // namespace unillm
