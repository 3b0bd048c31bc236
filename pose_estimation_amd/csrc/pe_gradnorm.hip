// a8. Global gradient norm over many tensors, and clipping to it.
//
//   n = |a| * sqrt(sum g^2)   or   |a| * max |g|          over every element of every tensor
//   c = n > max_norm ? max_norm / n : 1;   o = round(g * (a * c))
//
// Bound: HBM bandwidth, 4 (2) bytes read per element for the norm, as much read and written for
// the clipping, which cannot start before every gradient has been read.  The tensors are cut
// into one contiguous share per WAVE, equal in weight: its bytes, and 1 KB more for each tensor
// that ends in it, so that a long list of tiny tensors is spread as well.  No wave
// waits for another, none has a long list to walk, and there is no search for the tensor an
// element is in.  Squares are summed in float64: float32 squares overflow from 1.8e19 on and
// vanish below 1e-23, and the conversion is hidden behind the loads.  The sums' order depends
// only on the tensors' lengths and 16-byte alignment, so the result has the same bits on every
// call, and on every rank with the same layout.
// Measured, 34 M float32 gradients in 170 tensors: the norm 26 us (5.2 TB/s; a share per workgroup
// of 256 threads with one load a lane under way: 27 and, out of cold caches, 41), the clipping of
// them into other tensors 47 us more, in place 46, into a tensor that lies differently to 16 bytes
// (element by element) 68; nine small tensors 4.5 us in one launch (5.5 in two).
#include <math.h>

#include "pe_common.h"
#include "pe_gradnorm.h"

namespace pe {

template <int KIND>
__device__ __forceinline__ void norm_share(const pe_grad_span* __restrict__ spans,
                                           const int32_t* __restrict__ begin, int share,
                                           NormAcc<KIND>& acc) {
    const int lane = (int)threadIdx.x & 63;
    const int last = begin[share + 1];
    for (int k = begin[share]; k < last; ++k) {
        const pe_grad_span s = spans[k];
        if (s.dtype == PE_DTYPE_F32) {
            norm_span<KIND>(static_cast<const float*>(s.src), (int)s.n, lane, acc);
        } else {
            norm_span<KIND>(static_cast<const uint16_t*>(s.src), (int)s.n, lane, acc);
        }
    }
}

// The wave's number as the scalar it is: its spans come through scalar loads.
__device__ __forceinline__ int wave_of_block() {
    return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
}

template <int KIND>
__global__ __launch_bounds__(kNormThreads) void norm_parts_kernel(
    const pe_grad_span* __restrict__ spans, const int32_t* __restrict__ begin, int shares,
    double* __restrict__ part) {
    NormAcc<KIND> acc;
    const int share = (int)blockIdx.x * kNormWaves + wave_of_block();
    if (share < shares) norm_share<KIND>(spans, begin, share, acc);
    const double v = norm_block<kNormThreads>(acc.value(), KIND);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <int KIND>
__global__ __launch_bounds__(kNormThreads) void norm_flat_kernel(const float* __restrict__ g, long n,
                                                                 int share,
                                                                 double* __restrict__ part) {
    NormAcc<KIND> acc;
    const long lo = ((long)blockIdx.x * kNormWaves + wave_of_block()) * share;
    if (lo < n)
        norm_span<KIND>(g + lo, (int)(n - lo < share ? n - lo : share), (int)threadIdx.x & 63, acc);
    const double v = norm_block<kNormThreads>(acc.value(), KIND);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

__global__ __launch_bounds__(kNormThreads) void norm_final_kernel(const double* __restrict__ part,
                                                                  int parts, ClipRule r,
                                                                  float* __restrict__ norm) {
    const double n = norm_fold(part, parts, r);
    if (threadIdx.x == 0) *norm = (float)n;
}

template <typename T>
__device__ __forceinline__ T scaled_one(T v, double f);
template <>
__device__ __forceinline__ float scaled_one<float>(float v, double f) {
    return scaled(v, f);
}
template <>
__device__ __forceinline__ uint16_t scaled_one<uint16_t>(uint16_t v, double f) {
    return (uint16_t)float_to_bf16_bits(scaled(bf16_bits_to_float(v), f));
}
__device__ __forceinline__ f32x4 scaled_vec(f32x4 v, double f) {
    return f32x4{scaled(v.x, f), scaled(v.y, f), scaled(v.z, f), scaled(v.w, f)};
}
__device__ __forceinline__ u32x4 scaled_vec(u32x4 v, double f) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        v[k] = pack_bf16x2_bits(scaled(bf16_bits_to_float(v[k] & 0xffffu), f),
                                scaled(__uint_as_float(v[k] & 0xffff0000u), f));
    return v;
}

// One wave over n elements, four loads a lane under way; from and to may be the same.  The stores
// are non-temporal: ordinary ones push out the gradients that the norm has just left in the
// caches (34 M float32 into another array: 75 us against 88, with the Adam step that reads them
// 256 against 266; in place no difference).
template <typename T>
__device__ __forceinline__ void clip_span(const T* from, T* to, int n, int lane, double f) {
    typedef typename Vec16<T>::type V;
    constexpr int PER = 16 / (int)sizeof(T), AHEAD = 4;
    const Global<T>* src = (const Global<T>*)from;
    Global<T>* dst = (Global<T>*)to;
    const bool together = (((uintptr_t)src ^ (uintptr_t)dst) & 15) == 0;
    const int h = together ? head_of<T>(src, n) : n;   // apart: element by element
    for (int i = lane; i < h; i += 64) dst[i] = scaled_one<T>(src[i], f);
    const Global<V>* q = (const Global<V>*)(src + h);
    Global<V>* o = (Global<V>*)(dst + h);
    const int nv = (n - h) / PER;
    int i = lane;
    for (; i + 64 * (AHEAD - 1) < nv; i += 64 * AHEAD) {
        V v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u] = q[i + 64 * u];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) __builtin_nontemporal_store(scaled_vec(v[u], f), o + i + 64 * u);
    }
    for (; i < nv; i += 64) o[i] = scaled_vec(q[i], f);
    const int tail = h + nv * PER + lane;
    if (tail < n) dst[tail] = scaled_one<T>(src[tail], f);
}

__device__ __forceinline__ void clip_share(const pe_grad_span* __restrict__ spans,
                                           const int32_t* __restrict__ begin, int share, double f) {
    const int lane = (int)threadIdx.x & 63;
    const int last = begin[share + 1];
    for (int k = begin[share]; k < last; ++k) {
        const pe_grad_span s = spans[k];
        if (f == 1.0 && s.src == s.dst) continue;   // within the limit, in place: nothing changes
        if (s.dtype == PE_DTYPE_F32) {
            clip_span(static_cast<const float*>(s.src), static_cast<float*>(s.dst), (int)s.n, lane, f);
        } else {
            clip_span(static_cast<const uint16_t*>(s.src), static_cast<uint16_t*>(s.dst), (int)s.n, lane, f);
        }
    }
}

__global__ __launch_bounds__(kNormThreads) void clip_kernel(const pe_grad_span* __restrict__ spans,
                                                            const int32_t* __restrict__ begin,
                                                            int shares,
                                                            const double* __restrict__ part,
                                                            int parts, ClipRule r,
                                                            float* __restrict__ norm) {
    const double n = norm_fold(part, parts, r);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const int share = (int)blockIdx.x * kNormWaves + wave_of_block();
    if (share < shares) clip_share(spans, begin, share, clip_factor(n, r));
}

// A set of few shares by one workgroup in one launch: a wave a share, the norm, and with a limit
// the clipping behind the same workgroup's barrier (so it may be in place).
template <int KIND>
__global__ __launch_bounds__(64 * kNormFewShares) void norm_few_kernel(
    const pe_grad_span* __restrict__ spans, const int32_t* __restrict__ begin, int shares, ClipRule r,
    float* __restrict__ norm) {
    NormAcc<KIND> acc;
    const int share = wave_of_block();
    if (share < shares) norm_share<KIND>(spans, begin, share, acc);
    const double n = norm_of(norm_block<64 * kNormFewShares>(acc.value(), KIND), r);
    if (threadIdx.x == 0) *norm = (float)n;
    if (r.max_norm >= 0.0 && share < shares) clip_share(spans, begin, share, clip_factor(n, r));
}

int launch_flat_norm(const float* grad, long n, int kind, double* part, hipStream_t st) {
    long share = (n + PE_NORM_MAX_SHARES - 1) / PE_NORM_MAX_SHARES;
    if (share < 1024) share = 1024;
    share = (share + 3) & ~3l;
    const int blocks = (int)((n + share * kNormWaves - 1) / (share * kNormWaves));
    if (blocks == 0) return 0;
    if (kind == PE_NORM_L2) {
        launch(norm_flat_kernel<PE_NORM_L2>, blocks, kNormThreads, 0, st, grad, n, (int)share, part);
    } else {
        launch(norm_flat_kernel<PE_NORM_INF>, blocks, kNormThreads, 0, st, grad, n, (int)share, part);
    }
    return blocks;
}

static int blocks_of(int shares) { return (shares + kNormWaves - 1) / kNormWaves; }

int launch_norm_parts(const pe_grad_span* spans, const int32_t* begin, int shares, int kind,
                      double* part, hipStream_t st) {
    const int blocks = blocks_of(shares);
    if (blocks == 0) return 0;
    if (kind == PE_NORM_L2) {
        launch(norm_parts_kernel<PE_NORM_L2>, blocks, kNormThreads, 0, st, spans, begin, shares, part);
    } else {
        launch(norm_parts_kernel<PE_NORM_INF>, blocks, kNormThreads, 0, st, spans, begin, shares, part);
    }
    return blocks;
}

static void launch_norm_few(const pe_grad_span* spans, const int32_t* begin, int shares, const ClipRule& r,
                            float* norm, hipStream_t st) {
    const unsigned threads = 64 * kNormFewShares;
    if (r.kind == PE_NORM_L2) {
        launch(norm_few_kernel<PE_NORM_L2>, 1, threads, 0, st, spans, begin, shares, r, norm);
    } else {
        launch(norm_few_kernel<PE_NORM_INF>, 1, threads, 0, st, spans, begin, shares, r, norm);
    }
}

// What every entry point that takes a set of gradients checks.
static int32_t check_set(const char* what, const pe_grad_span* spans, const int32_t* begin,
                         int32_t shares, int32_t kind, float grad_scale, const float* norm,
                         const void* workspace) {
    PE_REQUIRE(shares >= 0 && shares <= PE_NORM_MAX_SHARES, PE_E_INVALID, "%s: %d shares outside [0, %d]",
               what, shares, PE_NORM_MAX_SHARES);
    PE_REQUIRE(shares == 0 || (spans && begin), PE_E_INVALID, "%s: NULL table", what);
    PE_REQUIRE(kind == PE_NORM_L2 || kind == PE_NORM_INF, PE_E_UNSUPPORTED,
               "%s: unknown norm %d", what, kind);
    PE_REQUIRE(isfinite(grad_scale), PE_E_INVALID, "%s: grad_scale must be finite", what);
    PE_REQUIRE(norm, PE_E_INVALID, "%s: NULL norm", what);
    PE_REQUIRE(workspace || shares <= kNormFewShares, PE_E_INVALID, "%s: NULL workspace", what);
    PE_REQUIRE(aligned(workspace, 8), PE_E_INVALID, "%s: workspace must be 8-byte aligned", what);
    return PE_OK;
}

}  // namespace pe

extern "C" size_t pe_grad_norm_workspace_bytes(void) { return sizeof(double) * pe::kNormMaxParts; }

extern "C" int32_t pe_grad_norm(const pe_grad_span* spans, const int32_t* begin, int32_t shares,
                                int32_t kind, float grad_scale, float* norm, void* workspace,
                                pe_stream_t stream) {
    using namespace pe;
    const int32_t bad = check_set("pe_grad_norm", spans, begin, shares, kind, grad_scale, norm, workspace);
    if (bad) return bad;
    const ClipRule r{(double)grad_scale, -1.0, kind};
    if (shares <= kNormFewShares) {
        launch_norm_few(spans, begin, shares, r, norm, as_stream(stream));
        return check_launch("pe_grad_norm");
    }
    double* part = static_cast<double*>(workspace);
    const int parts = launch_norm_parts(spans, begin, shares, kind, part, as_stream(stream));
    launch(norm_final_kernel, 1, kNormThreads, 0, as_stream(stream), part, parts, r, norm);
    return check_launch("pe_grad_norm");
}

extern "C" int32_t pe_grad_clip(const pe_grad_span* spans, const int32_t* begin, int32_t shares,
                                int32_t kind, float grad_scale, double max_norm, float* norm,
                                void* workspace, pe_stream_t stream) {
    using namespace pe;
    const int32_t bad = check_set("pe_grad_clip", spans, begin, shares, kind, grad_scale, norm, workspace);
    if (bad) return bad;
    PE_REQUIRE(max_norm >= 0.0, PE_E_INVALID, "pe_grad_clip: max_norm must not be negative or NaN");
    const ClipRule r{(double)grad_scale, max_norm, kind};
    if (shares <= kNormFewShares) {
        launch_norm_few(spans, begin, shares, r, norm, as_stream(stream));
        return check_launch("pe_grad_clip");
    }
    double* part = static_cast<double*>(workspace);
    const int parts = launch_norm_parts(spans, begin, shares, kind, part, as_stream(stream));
    launch(clip_kernel, blocks_of(shares), kNormThreads, 0, as_stream(stream), spans, begin, shares, part,
           parts, r, norm);
    return check_launch("pe_grad_clip");
}
