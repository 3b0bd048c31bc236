// What the global-norm kernels (pe_gradnorm.hip) and the clipped optimizer steps (pe_optim.hip)
// share: the norm's partial results and the factor that follows from them.
#pragma once

#include "pe_common.h"

namespace pe {

constexpr int kNormThreads = 256;
constexpr int kNormMaxParts = PE_NORM_MAX_BLOCKS;   // partial results of one norm, at most

// What turns the partial results into a factor for the gradients.
struct ClipRule {
    double grad_scale;   // applied to every gradient, part of the norm
    double max_norm;     // < 0: no clipping, the factor is grad_scale
    int kind;            // PE_NORM_L2: parts are sums of squares; PE_NORM_INF: maxima
};

// Enqueue one partial result per workgroup: over a set of spans, and over a flat float32 array
// (*parts receives their number).
void launch_norm_parts(const pe_grad_span* spans, const int32_t* begin, int blocks, int kind,
                       double* part, hipStream_t st);
void launch_flat_norm(const float* grad, long n, int kind, double* part, int* parts, hipStream_t st);

#ifdef __HIPCC__
// Non-negative doubles (and NaN, which stays on top) order as their bits do.
__device__ __forceinline__ double norm_combine(double a, double b, int kind) {
    if (kind == PE_NORM_L2) return a + b;
    return __double_as_longlong(a) > __double_as_longlong(b) ? a : b;
}

// The workgroup's kNormThreads values as one, the same bits in every thread and on every call:
// butterfly inside each wave, then the four waves in order.
__device__ __forceinline__ double norm_block(double v, int kind) {
    __shared__ double wave[kNormThreads / kWave];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = norm_combine(v, __shfl_xor(v, off, 64), kind);
    if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = wave[0];
#pragma unroll
    for (int i = 1; i < kNormThreads / kWave; ++i) v = norm_combine(v, wave[i], kind);
    __syncthreads();
    return v;
}

// The norm from its partial results.  Every workgroup that needs it folds them for itself (8 KB
// at most, from L2), in the same order, which costs less than another launch between the two
// passes and leaves nothing to clear or to count.
__device__ __forceinline__ double norm_fold(const double* __restrict__ part, int parts,
                                            const ClipRule& r) {
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += kNormThreads) v = norm_combine(v, part[i], r.kind);
    v = norm_block(v, r.kind);
    return (r.kind == PE_NORM_L2 ? sqrt(v) : v) * fabs(r.grad_scale);
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
