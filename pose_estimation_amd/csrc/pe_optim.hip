// a6. Fused optimizer steps over a flat float32 arena (Adam, momentum SGD).
//
// Bound: HBM bandwidth.  Adam moves 16 B in (p, m, v, g) and 12 B + 2 B out (p, m, v, bf16
// copy) per parameter: 30 B.  One grid-stride kernel, 16-byte accesses, a scalar tail.
// Arithmetic is plain float32 in a fixed order with FMA contraction off (the file is built
// with -ffp-contract=off), so the result is bit-identical to the float32 NumPy restatement.
#include <math.h>

#include "pe_common.h"
#include "pe_gradnorm.h"

namespace pe {

struct AdamHyper {
    float beta1, beta2, omb1, omb2, eps, step_size, denom_scale, grad_scale;
};

__device__ __forceinline__ void adam_one(float& p, float& m, float& v, float g,
                                         const AdamHyper& h) {
    g = g * h.grad_scale;
    m = h.beta1 * m + h.omb1 * g;
    v = h.beta2 * v + (h.omb2 * g) * g;
    const float den = sqrtf(v) * h.denom_scale + h.eps;
    p = p - (h.step_size * m) / den;
}

__global__ __launch_bounds__(256) void adam_kernel(float* __restrict__ p, float* __restrict__ m,
                                                   float* __restrict__ v,
                                                   const float* __restrict__ grad,
                                                   uint16_t* __restrict__ pb, long n,
                                                   AdamHyper h) {
    const long n4 = n >> 2;
    const long tid = (long)blockIdx.x * 256 + threadIdx.x;
    const long nth = (long)gridDim.x * 256;
    float4* p4 = reinterpret_cast<float4*>(p);
    float4* m4 = reinterpret_cast<float4*>(m);
    float4* v4 = reinterpret_cast<float4*>(v);
    const f32x4* g4 = reinterpret_cast<const f32x4*>(grad);
    uint2* pb4 = reinterpret_cast<uint2*>(pb);
    for (long i = tid; i < n4; i += nth) {
        float4 pp = p4[i], mm = m4[i], vv = v4[i];
        const f32x4 gg = __builtin_nontemporal_load(g4 + i);
        adam_one(pp.x, mm.x, vv.x, gg.x, h);
        adam_one(pp.y, mm.y, vv.y, gg.y, h);
        adam_one(pp.z, mm.z, vv.z, gg.z, h);
        adam_one(pp.w, mm.w, vv.w, gg.w, h);
        p4[i] = pp;
        m4[i] = mm;
        v4[i] = vv;
        if (pb) {
            uint2 o;
            o.x = pack_bf16x2_bits(pp.x, pp.y);
            o.y = pack_bf16x2_bits(pp.z, pp.w);
            pb4[i] = o;
        }
    }
    for (long i = n4 * 4 + tid; i < n; i += nth) {
        float pp = p[i], mm = m[i], vv = v[i];
        adam_one(pp, mm, vv, grad[i], h);
        p[i] = pp;
        m[i] = mm;
        v[i] = vv;
        if (pb) pb[i] = (uint16_t)float_to_bf16_bits(pp);
    }
}

__global__ __launch_bounds__(256) void sgd_kernel(float* __restrict__ p, float* __restrict__ mom,
                                                  const float* __restrict__ grad,
                                                  uint16_t* __restrict__ pb, long n, float lr,
                                                  float momentum, float grad_scale) {
    const long n4 = n >> 2;
    const long tid = (long)blockIdx.x * 256 + threadIdx.x;
    const long nth = (long)gridDim.x * 256;
    float4* p4 = reinterpret_cast<float4*>(p);
    float4* m4 = reinterpret_cast<float4*>(mom);
    const f32x4* g4 = reinterpret_cast<const f32x4*>(grad);
    uint2* pb4 = reinterpret_cast<uint2*>(pb);
    auto one = [&](float& pp, float& mm, float g) {
        g = g * grad_scale;
        mm = momentum * mm + g;
        pp = pp - lr * mm;
    };
    for (long i = tid; i < n4; i += nth) {
        float4 pp = p4[i], mm = m4[i];
        const f32x4 gg = __builtin_nontemporal_load(g4 + i);
        one(pp.x, mm.x, gg.x);
        one(pp.y, mm.y, gg.y);
        one(pp.z, mm.z, gg.z);
        one(pp.w, mm.w, gg.w);
        p4[i] = pp;
        m4[i] = mm;
        if (pb) {
            uint2 o;
            o.x = pack_bf16x2_bits(pp.x, pp.y);
            o.y = pack_bf16x2_bits(pp.z, pp.w);
            pb4[i] = o;
        }
    }
    for (long i = n4 * 4 + tid; i < n; i += nth) {
        float pp = p[i], mm = mom[i];
        one(pp, mm, grad[i]);
        p[i] = pp;
        mom[i] = mm;
        if (pb) pb[i] = (uint16_t)float_to_bf16_bits(pp);
    }
}

// The clipped steps: the factor of the gradients comes from the partial results of a norm that the
// launch before has left in memory, so the clipped gradient is never stored and the arena is read
// once more for the norm, not twice.  Each workgroup folds the partials for itself; 2048 of them
// keep that at a hundredth of the traffic.  The factor multiplies in float64 and rounds once, so
// a step whose norm is within the limit has the bits of the plain step.  Parameters and moments
// are not read again before the next step: non-temporal accesses leave the caches to the gradients
// (34 M parameters, norm and step: 197 us against 226; stores alone change nothing).
struct ClipStep {
    const double* part;
    int parts;
    ClipRule rule;
    int skip_nonfinite;
    float* norm;
    const float* grad;   // parts < 0: no launch before, the norm is over these few_n gradients
    int few_n;
    // The gradients' factor; false: the norm is not finite and the step is to be skipped.
    __device__ __forceinline__ bool factor(double& f) const {
        const double n = parts < 0 ? few() : norm_fold(part, parts, rule);
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
        f = clip_factor(n, rule);
        return !(skip_nonfinite && !isfinite(n));
    }
    // A small arena's norm by every workgroup for itself, 64 KB at most from L2 instead of a launch
    // (16384 parameters: a call 7.8 us, one parameter more and with the launch 11.1).
    __device__ __forceinline__ double few() const {
        if (rule.kind == PE_NORM_L2) return few<PE_NORM_L2>();
        return few<PE_NORM_INF>();
    }
    template <int KIND>
    __device__ __forceinline__ double few() const {
        NormAcc<KIND> acc;
        const int share = ((few_n + kNormWaves - 1) / kNormWaves + 3) & ~3;
        const int lo = ((int)threadIdx.x >> 6) * share;
        if (lo < few_n)
            norm_span<KIND>(grad + lo, few_n - lo < share ? few_n - lo : share, (int)threadIdx.x & 63, acc);
        return norm_of(norm_block<kNormThreads>(acc.value(), KIND), rule);
    }
};

__global__ __launch_bounds__(256) void adam_clip_kernel(float* __restrict__ p, float* __restrict__ m,
                                                        float* __restrict__ v,
                                                        const float* __restrict__ grad,
                                                        uint16_t* __restrict__ pb, long n,
                                                        AdamHyper h, ClipStep c) {
    double f;
    if (!c.factor(f)) return;
    const long n4 = n >> 2;
    const long tid = (long)blockIdx.x * 256 + threadIdx.x;
    const long nth = (long)gridDim.x * 256;
    f32x4* p4 = reinterpret_cast<f32x4*>(p);
    f32x4* m4 = reinterpret_cast<f32x4*>(m);
    f32x4* v4 = reinterpret_cast<f32x4*>(v);
    const f32x4* g4 = reinterpret_cast<const f32x4*>(grad);
    uint2* pb4 = reinterpret_cast<uint2*>(pb);
    for (long i = tid; i < n4; i += nth) {
        f32x4 pp = __builtin_nontemporal_load(p4 + i);
        f32x4 mm = __builtin_nontemporal_load(m4 + i);
        f32x4 vv = __builtin_nontemporal_load(v4 + i);
        const f32x4 gg = __builtin_nontemporal_load(g4 + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float pj = pp[j], mj = mm[j], vj = vv[j];
            adam_one(pj, mj, vj, scaled(gg[j], f), h);
            pp[j] = pj;
            mm[j] = mj;
            vv[j] = vj;
        }
        __builtin_nontemporal_store(pp, p4 + i);
        __builtin_nontemporal_store(mm, m4 + i);
        __builtin_nontemporal_store(vv, v4 + i);
        if (pb) {
            uint2 o;
            o.x = pack_bf16x2_bits(pp.x, pp.y);
            o.y = pack_bf16x2_bits(pp.z, pp.w);
            pb4[i] = o;
        }
    }
    for (long i = n4 * 4 + tid; i < n; i += nth) {
        float pp = p[i], mm = m[i], vv = v[i];
        adam_one(pp, mm, vv, scaled(grad[i], f), h);
        p[i] = pp;
        m[i] = mm;
        v[i] = vv;
        if (pb) pb[i] = (uint16_t)float_to_bf16_bits(pp);
    }
}

__global__ __launch_bounds__(256) void sgd_clip_kernel(float* __restrict__ p, float* __restrict__ mom,
                                                       const float* __restrict__ grad,
                                                       uint16_t* __restrict__ pb, long n, float lr,
                                                       float momentum, ClipStep c) {
    double f;
    if (!c.factor(f)) return;
    const long n4 = n >> 2;
    const long tid = (long)blockIdx.x * 256 + threadIdx.x;
    const long nth = (long)gridDim.x * 256;
    f32x4* p4 = reinterpret_cast<f32x4*>(p);
    f32x4* m4 = reinterpret_cast<f32x4*>(mom);
    const f32x4* g4 = reinterpret_cast<const f32x4*>(grad);
    uint2* pb4 = reinterpret_cast<uint2*>(pb);
    auto one = [&](float& pp, float& mm, float g) {
        mm = momentum * mm + g;
        pp = pp - lr * mm;
    };
    for (long i = tid; i < n4; i += nth) {
        f32x4 pp = __builtin_nontemporal_load(p4 + i), mm = __builtin_nontemporal_load(m4 + i);
        const f32x4 gg = __builtin_nontemporal_load(g4 + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float pj = pp[j], mj = mm[j];
            one(pj, mj, scaled(gg[j], f));
            pp[j] = pj;
            mm[j] = mj;
        }
        __builtin_nontemporal_store(pp, p4 + i);
        __builtin_nontemporal_store(mm, m4 + i);
        if (pb) {
            uint2 o;
            o.x = pack_bf16x2_bits(pp.x, pp.y);
            o.y = pack_bf16x2_bits(pp.z, pp.w);
            pb4[i] = o;
        }
    }
    for (long i = n4 * 4 + tid; i < n; i += nth) {
        float pp = p[i], mm = mom[i];
        one(pp, mm, scaled(grad[i], f));
        p[i] = pp;
        mom[i] = mm;
        if (pb) pb[i] = (uint16_t)float_to_bf16_bits(pp);
    }
}

static unsigned clip_grid(long n) {
    long blocks = ((n >> 2) + 255) / 256;
    if (blocks < 1) blocks = 1;
    if (blocks > 2048) blocks = 2048;
    return (unsigned)blocks;
}

// Checks the clipping arguments and enqueues the norm: over the given set, or (shares < 0) over
// the step's own gradient arena.
static int32_t start_clip(const char* what, const float* grad, int64_t n, const pe_clip_desc* d,
                          float* norm, void* workspace, pe_stream_t stream, ClipStep* c) {
    PE_REQUIRE(d, PE_E_INVALID, "%s: NULL clip description", what);
    PE_REQUIRE(d->max_norm >= 0.0, PE_E_INVALID, "%s: max_norm must not be negative or NaN", what);
    PE_REQUIRE(isfinite(d->grad_scale), PE_E_INVALID, "%s: grad_scale must be finite", what);
    PE_REQUIRE(d->kind == PE_NORM_L2 || d->kind == PE_NORM_INF, PE_E_UNSUPPORTED,
               "%s: unknown norm %d", what, d->kind);
    PE_REQUIRE(d->shares <= PE_NORM_MAX_SHARES, PE_E_INVALID, "%s: %d shares, at most %d", what,
               d->shares, PE_NORM_MAX_SHARES);
    PE_REQUIRE(d->shares <= 0 || (d->spans && d->begin), PE_E_INVALID, "%s: NULL table", what);
    const bool few = d->shares < 0 && n <= PE_NORM_FEW_ELEMENTS;
    PE_REQUIRE(norm, PE_E_INVALID, "%s: NULL norm", what);
    PE_REQUIRE(workspace || few, PE_E_INVALID, "%s: NULL workspace", what);
    PE_REQUIRE(aligned(workspace, 8), PE_E_INVALID, "%s: workspace must be 8-byte aligned", what);
    double* part = static_cast<double*>(workspace);
    c->part = part;
    c->rule = ClipRule{(double)d->grad_scale, d->max_norm, d->kind};
    c->skip_nonfinite = d->skip_nonfinite;
    c->norm = norm;
    c->grad = grad;
    c->few_n = 0;
    if (d->shares >= 0) {
        c->parts = launch_norm_parts(d->spans, d->begin, d->shares, d->kind, part, as_stream(stream));
    } else if (few) {
        c->parts = -1;
        c->few_n = (int)n;
    } else {
        c->parts = launch_flat_norm(grad, (long)n, d->kind, part, as_stream(stream));
    }
    return PE_OK;
}

static unsigned optim_grid(long n) {
    long blocks = ((n >> 2) + 255) / 256;
    if (blocks < 1) blocks = 1;
    if (blocks > 256 * 128) blocks = 256 * 128;
    return (unsigned)blocks;
}

}  // namespace pe

extern "C" int32_t pe_adam_step(float* p, float* m, float* v, const float* grad, uint16_t* p_bf16,
                                int64_t n, float beta1, float beta2, float eps, float step_size,
                                float denom_scale, float grad_scale, pe_stream_t stream) {
    using namespace pe;
    PE_REQUIRE(n >= 0, PE_E_INVALID, "pe_adam_step: negative n");
    if (n == 0) return PE_OK;
    PE_REQUIRE(p && m && v && grad, PE_E_INVALID, "pe_adam_step: NULL arena pointer");
    PE_REQUIRE(aligned(p, 16) && aligned(m, 16) && aligned(v, 16) && aligned(grad, 16) &&
                   aligned(p_bf16, 8),
               PE_E_INVALID, "pe_adam_step: arenas must be 16-byte aligned (bf16 copy: 8)");
    AdamHyper h;
    h.beta1 = beta1;
    h.beta2 = beta2;
    h.omb1 = (float)(1.0 - (double)beta1);
    h.omb2 = (float)(1.0 - (double)beta2);
    h.eps = eps;
    h.step_size = step_size;
    h.denom_scale = denom_scale;
    h.grad_scale = grad_scale;
    pe::launch(adam_kernel, optim_grid(n), 256, 0, as_stream(stream), p, m, v, grad, p_bf16, (long)n, h);
    return check_launch("pe_adam_step");
}

extern "C" int32_t pe_sgd_step(float* p, float* mom, const float* grad, uint16_t* p_bf16,
                               int64_t n, float lr, float momentum, float grad_scale,
                               pe_stream_t stream) {
    using namespace pe;
    PE_REQUIRE(n >= 0, PE_E_INVALID, "pe_sgd_step: negative n");
    if (n == 0) return PE_OK;
    PE_REQUIRE(p && mom && grad, PE_E_INVALID, "pe_sgd_step: NULL arena pointer");
    PE_REQUIRE(aligned(p, 16) && aligned(mom, 16) && aligned(grad, 16) && aligned(p_bf16, 8),
               PE_E_INVALID, "pe_sgd_step: arenas must be 16-byte aligned (bf16 copy: 8)");
    pe::launch(sgd_kernel, optim_grid(n), 256, 0, as_stream(stream), p, mom, grad, p_bf16, (long)n, lr,
                                                            momentum, grad_scale);
    return check_launch("pe_sgd_step");
}

extern "C" int32_t pe_adam_clip_step(float* p, float* m, float* v, const float* grad,
                                     uint16_t* p_bf16, int64_t n, float beta1, float beta2,
                                     float eps, float step_size, float denom_scale,
                                     const pe_clip_desc* clip, float* norm, void* workspace,
                                     pe_stream_t stream) {
    using namespace pe;
    PE_REQUIRE(n >= 0, PE_E_INVALID, "pe_adam_clip_step: negative n");
    PE_REQUIRE(n == 0 || (p && m && v && grad), PE_E_INVALID, "pe_adam_clip_step: NULL arena pointer");
    PE_REQUIRE(aligned(p, 16) && aligned(m, 16) && aligned(v, 16) && aligned(grad, 16) &&
                   aligned(p_bf16, 8),
               PE_E_INVALID, "pe_adam_clip_step: arenas must be 16-byte aligned (bf16 copy: 8)");
    ClipStep c;
    const int32_t bad = start_clip("pe_adam_clip_step", grad, n, clip, norm, workspace, stream, &c);
    if (bad) return bad;
    AdamHyper h;
    h.beta1 = beta1;
    h.beta2 = beta2;
    h.omb1 = (float)(1.0 - (double)beta1);
    h.omb2 = (float)(1.0 - (double)beta2);
    h.eps = eps;
    h.step_size = step_size;
    h.denom_scale = denom_scale;
    h.grad_scale = 1.0f;   // part of the factor
    pe::launch(adam_clip_kernel, clip_grid(n), 256, 0, as_stream(stream), p, m, v, grad, p_bf16,
               (long)n, h, c);
    return check_launch("pe_adam_clip_step");
}

extern "C" int32_t pe_sgd_clip_step(float* p, float* mom, const float* grad, uint16_t* p_bf16,
                                    int64_t n, float lr, float momentum, const pe_clip_desc* clip,
                                    float* norm, void* workspace, pe_stream_t stream) {
    using namespace pe;
    PE_REQUIRE(n >= 0, PE_E_INVALID, "pe_sgd_clip_step: negative n");
    PE_REQUIRE(n == 0 || (p && mom && grad), PE_E_INVALID, "pe_sgd_clip_step: NULL arena pointer");
    PE_REQUIRE(aligned(p, 16) && aligned(mom, 16) && aligned(grad, 16) && aligned(p_bf16, 8),
               PE_E_INVALID, "pe_sgd_clip_step: arenas must be 16-byte aligned (bf16 copy: 8)");
    ClipStep c;
    const int32_t bad = start_clip("pe_sgd_clip_step", grad, n, clip, norm, workspace, stream, &c);
    if (bad) return bad;
    pe::launch(sgd_clip_kernel, clip_grid(n), 256, 0, as_stream(stream), p, mom, grad, p_bf16, (long)n,
               lr, momentum, c);
    return check_launch("pe_sgd_clip_step");
}
