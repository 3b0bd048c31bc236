// What the global-norm kernels (pe_gradnorm.hip) and the clipped optimizer steps (pe_optim.hip)
// share: the norm's partial results and the factor that follows from them.
#pragma once

#include "pe_common.h"
#include "pe_lanes.h"

namespace pe {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / kWave;
constexpr int kNormMaxParts = PE_NORM_MAX_SHARES / kNormWaves;   // partial results of one norm

constexpr int kNormFewShares = PE_NORM_FEW_SHARES;   // a set of so few takes one workgroup and one launch

// What turns the partial results into a factor for the gradients.
struct ClipRule {
    double grad_scale;   // applied to every gradient, part of the norm
    double max_norm;     // < 0: no clipping, the factor is grad_scale
    int kind;            // PE_NORM_L2: parts are sums of squares; PE_NORM_INF: maxima
};

// Enqueue one partial result per workgroup: over a set of spans cut into shares, and over a flat
// float32 array.  Return the number of partial results.
int launch_norm_parts(const pe_grad_span* spans, const int32_t* begin, int shares, int kind,
                      double* part, hipStream_t st);
int launch_flat_norm(const float* grad, long n, int kind, double* part, hipStream_t st);

#ifdef __HIPCC__
// Non-negative doubles (and NaN, which stays on top) order as their bits do.
__device__ __forceinline__ double norm_combine(double a, double b, int kind) {
    if (kind == PE_NORM_L2) return a + b;
    return __double_as_longlong(a) > __double_as_longlong(b) ? a : b;
}

// The wave's values as one, the same bits in every lane.
__device__ __forceinline__ double norm_wave(double v, int kind) {
    return lanes_all<64>(v, [kind](double a, double b) { return norm_combine(a, b, kind); });
}

// The workgroup's values as one, the same bits in every thread and on every call: butterfly
// inside each wave, then the waves in order.
template <int THREADS>
__device__ __forceinline__ double norm_block(double v, int kind) {
    __shared__ double wave[THREADS / kWave];
    v = norm_wave(v, kind);
    if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = wave[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) v = norm_combine(v, wave[i], kind);
    __syncthreads();
    return v;
}

// sqrt of a sum of squares, times the scale.
__device__ __forceinline__ double norm_of(double v, const ClipRule& r) {
    return (r.kind == PE_NORM_L2 ? sqrt(v) : v) * fabs(r.grad_scale);
}

// ---- a wave's share of the norm -----------------------------------------------------------
template <int KIND>
struct NormAcc {
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    uint32_t m = 0u;
    __device__ __forceinline__ void add(int k, float g) {
        if (KIND == PE_NORM_L2) {
            const double d = (double)g;
            s[k] = __builtin_fma(d, d, s[k]);
        } else {
            const uint32_t b = __float_as_uint(g) & 0x7fffffffu;   // NaN above infinity
            m = b > m ? b : m;
        }
    }
    __device__ __forceinline__ void add(const f32x4& v) {
        add(0, v.x);
        add(1, v.y);
        add(2, v.z);
        add(3, v.w);
    }
    __device__ __forceinline__ void add(const u32x4& v) {   // eight bf16
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            add(k, bf16_bits_to_float(v[k] & 0xffffu));
            add(k, __uint_as_float(v[k] & 0xffff0000u));
        }
    }
    __device__ __forceinline__ double value() const {
        return KIND == PE_NORM_L2 ? (s[0] + s[1]) + (s[2] + s[3]) : (double)__uint_as_float(m);
    }
};

template <typename T>
struct Vec16;   // 16 bytes of T
template <>
struct Vec16<float> {
    typedef f32x4 type;
    static __device__ __forceinline__ float one(float v) { return v; }
};
template <>
struct Vec16<uint16_t> {
    typedef u32x4 type;
    static __device__ __forceinline__ float one(uint16_t v) { return bf16_bits_to_float(v); }
};

// Addresses that a kernel reads from a table: known to be global memory, so that the accesses are
// global ones, not flat ones that wait for LDS as well.
template <typename T>
using Global = __attribute__((address_space(1))) T;

// Elements before the first 16-byte boundary of p, at most n.
template <typename T>
__device__ __forceinline__ int head_of(const Global<T>* p, int n) {
    const int h = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    return h < n ? h : n;
}

// One wave over n elements: eight 16-byte loads a lane under way at a time.  Past the end a lane
// reads the last vector again and counts it as 0 (a branch would make it wait for each load).
template <int KIND, typename T>
__device__ __forceinline__ void norm_span(const T* __restrict__ at, int n, int lane, NormAcc<KIND>& acc) {
    typedef typename Vec16<T>::type V;
    constexpr int PER = 16 / (int)sizeof(T), AHEAD = 8;
    const Global<T>* p = (const Global<T>*)at;
    const int h = head_of<T>(p, n);
    const int nv = (n - h) / PER;
    const int tail = h + nv * PER + lane;
    const T first = p[lane < h ? lane : 0], end = p[tail < n ? tail : 0];
    const Global<V>* q = (const Global<V>*)(p + h);
    for (int i = lane; i - lane < nv; i += 64 * AHEAD) {
        V v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u] = q[i + 64 * u < nv ? i + 64 * u : nv - 1];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (i + 64 * u >= nv) v[u] = V{0, 0, 0, 0};
            acc.add(v[u]);
        }
    }
    acc.add(0, lane < h ? Vec16<T>::one(first) : 0.0f);
    acc.add(1, tail < n ? Vec16<T>::one(end) : 0.0f);
}

// The norm from its partial results.  Every workgroup that needs it folds them for itself (8 KB
// at most, from L2), in the same order, which costs less than another launch between the two
// passes and leaves nothing to clear or to count.
__device__ __forceinline__ double norm_fold(const double* __restrict__ part, int parts,
                                            const ClipRule& r) {
    constexpr int EACH = kNormMaxParts / kNormThreads;
    double got[EACH], v = 0.0;
    if (parts > 0) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const int i = (int)threadIdx.x + u * kNormThreads;
            got[u] = part[i < parts ? i : parts - 1];
        }
#pragma unroll
        for (int u = 0; u < EACH; ++u)
            if ((int)threadIdx.x + u * kNormThreads < parts) v = norm_combine(v, got[u], r.kind);
    }
    return norm_of(norm_block<kNormThreads>(v, r.kind), r);
}

// grad_scale * min(1, max_norm / norm); NaN when the norm is not finite.
__device__ __forceinline__ double clip_factor(double norm, const ClipRule& r) {
    if (r.max_norm < 0.0) return r.grad_scale;
    if (!isfinite(norm)) return __longlong_as_double(0x7ff8000000000000ll);
    return norm > r.max_norm ? r.grad_scale * (r.max_norm / norm) : r.grad_scale;
}

// One rounding: the product of a float and a double factor.
__device__ __forceinline__ float scaled(float g, double f) { return (float)((double)g * f); }
#endif

}  // namespace pe
