// a8. Global gradient norm over many tensors, and clipping to it.
//
//   n = |a| * sqrt(sum g^2)   or   |a| * max |g|          over every element of every tensor
//   c = n > max_norm ? max_norm / n : 1;   o = round(g * (a * c))
//
// Bound: HBM bandwidth, 4 (2) bytes read per element for the norm, as much read and written for
// the clipping, which cannot start before every gradient has been read.  The tensors are cut
// into one contiguous share per workgroup (equal to a few hundred bytes whatever their lengths),
// so no workgroup waits for another and there is no search for the tensor an element is in.
// Squares are summed in float64: float32 squares overflow from 1.8e19 on and vanish below
// 1e-23, and the double-rate cost is hidden behind the loads.  The sums' order depends only on
// the lengths, so the result has the same bits on every call and every data-parallel rank.
#include <math.h>

#include "pe_common.h"
#include "pe_gradnorm.h"

namespace pe {

struct NormAcc {
    double s[4];
    uint32_t m;
    __device__ __forceinline__ NormAcc() : s{0.0, 0.0, 0.0, 0.0}, m(0u) {}
    template <int KIND>
    __device__ __forceinline__ void add(int lane, float g) {
        if (KIND == PE_NORM_L2) {
            const double d = (double)g;
            s[lane] = __builtin_fma(d, d, s[lane]);
        } else {
            const uint32_t b = __float_as_uint(g) & 0x7fffffffu;   // NaN above infinity
            m = b > m ? b : m;
        }
    }
    template <int KIND>
    __device__ __forceinline__ double value() const {
        return KIND == PE_NORM_L2 ? (s[0] + s[1]) + (s[2] + s[3]) : (double)__uint_as_float(m);
    }
};

// Elements before the first 16-byte boundary of p, at most n.
template <typename T>
__device__ __forceinline__ long head_of(const T* p, long n) {
    const long h = (long)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (long)sizeof(T);
    return h < n ? h : n;
}

template <int KIND>
__device__ __forceinline__ void norm_span(const float* __restrict__ p, long n, NormAcc& acc) {
    const long h = head_of(p, n);
    if ((long)threadIdx.x < h) acc.add<KIND>(0, p[threadIdx.x]);
    const f32x4* q = reinterpret_cast<const f32x4*>(p + h);
    const long nv = (n - h) >> 2;
    for (long i = threadIdx.x; i < nv; i += kNormThreads) {
        const f32x4 v = q[i];
        acc.add<KIND>(0, v.x);
        acc.add<KIND>(1, v.y);
        acc.add<KIND>(2, v.z);
        acc.add<KIND>(3, v.w);
    }
    const long i = h + nv * 4 + threadIdx.x;
    if (i < n) acc.add<KIND>(0, p[i]);
}

template <int KIND>
__device__ __forceinline__ void norm_span(const uint16_t* __restrict__ p, long n, NormAcc& acc) {
    const long h = head_of(p, n);
    if ((long)threadIdx.x < h) acc.add<KIND>(0, bf16_bits_to_float(p[threadIdx.x]));
    const u32x4* q = reinterpret_cast<const u32x4*>(p + h);
    const long nv = (n - h) >> 3;
    for (long i = threadIdx.x; i < nv; i += kNormThreads) {
        const u32x4 v = q[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            acc.add<KIND>(k, bf16_bits_to_float(v[k] & 0xffffu));
            acc.add<KIND>(k, __uint_as_float(v[k] & 0xffff0000u));
        }
    }
    const long i = h + nv * 8 + threadIdx.x;
    if (i < n) acc.add<KIND>(0, bf16_bits_to_float(p[i]));
}

template <int KIND>
__global__ __launch_bounds__(kNormThreads) void norm_parts_kernel(
    const pe_grad_span* __restrict__ spans, const int32_t* __restrict__ begin,
    double* __restrict__ part) {
    NormAcc acc;
    const int last = begin[blockIdx.x + 1];
    for (int k = begin[blockIdx.x]; k < last; ++k) {
        const pe_grad_span s = spans[k];
        if (s.dtype == PE_DTYPE_F32) {
            norm_span<KIND>(static_cast<const float*>(s.src), (long)s.n, acc);
        } else {
            norm_span<KIND>(static_cast<const uint16_t*>(s.src), (long)s.n, acc);
        }
    }
    const double v = norm_block(acc.value<KIND>(), KIND);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <int KIND>
__global__ __launch_bounds__(kNormThreads) void norm_flat_kernel(const float* __restrict__ g, long n,
                                                                 long share,
                                                                 double* __restrict__ part) {
    NormAcc acc;
    const long lo = (long)blockIdx.x * share;
    const long len = n - lo < share ? n - lo : share;
    norm_span<KIND>(g + lo, len, acc);
    const double v = norm_block(acc.value<KIND>(), KIND);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

__global__ __launch_bounds__(kNormThreads) void norm_final_kernel(const double* __restrict__ part,
                                                                  int parts, ClipRule r,
                                                                  float* __restrict__ norm) {
    const double n = norm_fold(part, parts, r);
    if (threadIdx.x == 0) *norm = (float)n;
}

__device__ __forceinline__ void clip_span(const float* src, float* dst, long n, double f) {
    const bool together = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
    const long h = together ? head_of(src, n) : n;
    for (long i = threadIdx.x; i < h; i += kNormThreads) dst[i] = scaled(src[i], f);
    const f32x4* q = reinterpret_cast<const f32x4*>(src + h);
    f32x4* o = reinterpret_cast<f32x4*>(dst + h);
    const long nv = (n - h) >> 2;
    for (long i = threadIdx.x; i < nv; i += kNormThreads) {
        f32x4 v = q[i];
        v.x = scaled(v.x, f);
        v.y = scaled(v.y, f);
        v.z = scaled(v.z, f);
        v.w = scaled(v.w, f);
        o[i] = v;
    }
    const long i = h + nv * 4 + threadIdx.x;
    if (i < n) dst[i] = scaled(src[i], f);
}

__device__ __forceinline__ void clip_span(const uint16_t* src, uint16_t* dst, long n, double f) {
    const bool together = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
    const long h = together ? head_of(src, n) : n;
    for (long i = threadIdx.x; i < h; i += kNormThreads)
        dst[i] = (uint16_t)float_to_bf16_bits(scaled(bf16_bits_to_float(src[i]), f));
    const u32x4* q = reinterpret_cast<const u32x4*>(src + h);
    u32x4* o = reinterpret_cast<u32x4*>(dst + h);
    const long nv = (n - h) >> 3;
    for (long i = threadIdx.x; i < nv; i += kNormThreads) {
        u32x4 v = q[i];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            v[k] = pack_bf16x2_bits(scaled(bf16_bits_to_float(v[k] & 0xffffu), f),
                                    scaled(__uint_as_float(v[k] & 0xffff0000u), f));
        o[i] = v;
    }
    const long i = h + nv * 8 + threadIdx.x;
    if (i < n) dst[i] = (uint16_t)float_to_bf16_bits(scaled(bf16_bits_to_float(src[i]), f));
}

__global__ __launch_bounds__(kNormThreads) void clip_kernel(const pe_grad_span* __restrict__ spans,
                                                            const int32_t* __restrict__ begin,
                                                            const double* __restrict__ part,
                                                            int parts, ClipRule r,
                                                            float* __restrict__ norm) {
    const double n = norm_fold(part, parts, r);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double f = clip_factor(n, r);
    const int last = begin[blockIdx.x + 1];
    for (int k = begin[blockIdx.x]; k < last; ++k) {
        const pe_grad_span s = spans[k];
        if (f == 1.0 && s.src == s.dst) continue;   // within the limit, in place: nothing changes
        if (s.dtype == PE_DTYPE_F32) {
            clip_span(static_cast<const float*>(s.src), static_cast<float*>(s.dst), (long)s.n, f);
        } else {
            clip_span(static_cast<const uint16_t*>(s.src), static_cast<uint16_t*>(s.dst), (long)s.n, f);
        }
    }
}

void launch_flat_norm(const float* grad, long n, int kind, double* part, int* parts, hipStream_t st) {
    long share = (n + kNormMaxParts - 1) / kNormMaxParts;
    if (share < 4096) share = 4096;
    share = (share + 3) & ~3l;
    const int blocks = (int)((n + share - 1) / share);
    *parts = blocks;
    if (blocks == 0) return;
    if (kind == PE_NORM_L2) {
        launch(norm_flat_kernel<PE_NORM_L2>, blocks, kNormThreads, 0, st, grad, n, share, part);
    } else {
        launch(norm_flat_kernel<PE_NORM_INF>, blocks, kNormThreads, 0, st, grad, n, share, part);
    }
}

void launch_norm_parts(const pe_grad_span* spans, const int32_t* begin, int blocks, int kind,
                       double* part, hipStream_t st) {
    if (blocks == 0) return;
    if (kind == PE_NORM_L2) {
        launch(norm_parts_kernel<PE_NORM_L2>, blocks, kNormThreads, 0, st, spans, begin, part);
    } else {
        launch(norm_parts_kernel<PE_NORM_INF>, blocks, kNormThreads, 0, st, spans, begin, part);
    }
}

// What every entry point that takes a set of gradients checks.
static int32_t check_set(const char* what, const pe_grad_span* spans, const int32_t* begin,
                         int32_t blocks, int32_t kind, float grad_scale, const float* norm,
                         const void* workspace) {
    PE_REQUIRE(blocks >= 0 && blocks <= kNormMaxParts, PE_E_INVALID, "%s: %d workgroups outside [0, %d]",
               what, blocks, kNormMaxParts);
    PE_REQUIRE(blocks == 0 || (spans && begin), PE_E_INVALID, "%s: NULL table", what);
    PE_REQUIRE(kind == PE_NORM_L2 || kind == PE_NORM_INF, PE_E_UNSUPPORTED,
               "%s: unknown norm %d", what, kind);
    PE_REQUIRE(isfinite(grad_scale), PE_E_INVALID, "%s: grad_scale must be finite", what);
    PE_REQUIRE(norm && workspace, PE_E_INVALID, "%s: NULL norm or workspace", what);
    PE_REQUIRE(aligned(workspace, 8), PE_E_INVALID, "%s: workspace must be 8-byte aligned", what);
    return PE_OK;
}

}  // namespace pe

extern "C" size_t pe_grad_norm_workspace_bytes(void) { return sizeof(double) * pe::kNormMaxParts; }

extern "C" int32_t pe_grad_norm(const pe_grad_span* spans, const int32_t* begin, int32_t blocks,
                                int32_t kind, float grad_scale, float* norm, void* workspace,
                                pe_stream_t stream) {
    using namespace pe;
    const int32_t bad = check_set("pe_grad_norm", spans, begin, blocks, kind, grad_scale, norm, workspace);
    if (bad) return bad;
    double* part = static_cast<double*>(workspace);
    launch_norm_parts(spans, begin, blocks, kind, part, as_stream(stream));
    const ClipRule r{(double)grad_scale, -1.0, kind};
    launch(norm_final_kernel, 1, kNormThreads, 0, as_stream(stream), part, blocks, r, norm);
    return check_launch("pe_grad_norm");
}

extern "C" int32_t pe_grad_clip(const pe_grad_span* spans, const int32_t* begin, int32_t blocks,
                                int32_t kind, float grad_scale, double max_norm, float* norm,
                                void* workspace, pe_stream_t stream) {
    using namespace pe;
    const int32_t bad = check_set("pe_grad_clip", spans, begin, blocks, kind, grad_scale, norm, workspace);
    if (bad) return bad;
    PE_REQUIRE(max_norm >= 0.0, PE_E_INVALID, "pe_grad_clip: max_norm must not be negative or NaN");
    double* part = static_cast<double*>(workspace);
    launch_norm_parts(spans, begin, blocks, kind, part, as_stream(stream));
    const ClipRule r{(double)grad_scale, max_norm, kind};
    if (blocks == 0) {
        launch(norm_final_kernel, 1, kNormThreads, 0, as_stream(stream), part, blocks, r, norm);
    } else {
        launch(clip_kernel, blocks, kNormThreads, 0, as_stream(stream), spans, begin, part, blocks, r, norm);
    }
    return check_launch("pe_grad_clip");
}
