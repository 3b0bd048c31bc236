// a9. Row norm after and before a residual block, with the block's gate and residual scale.
//
//   per row of C channels:  a = N(y)*gp + bp;  h = x + s*phi(gate)*a;  z = N(h)*gq + bq
//   N(v) = (v - mean(v)) * rstd (layer) or v * rstd (rms), rstd = 1/sqrt(mean((v - mean)^2) + eps)
//
// Bound: HBM bandwidth.  Forward reads y and x and writes h and z, backward reads y, x, dh and dz
// and writes dy and dx, each once: a row lives in the registers of the team of threads that owns
// it from its load to its store, so statistics, both norms and the gate cost no further pass.
// Eight channels a thread (one 16-byte load of bf16): a team is the next power of two of C/8
// threads inside one wave (8 to 64, several rows a wave side by side), or, past 512 channels, a
// workgroup of its own.  Means and variances are taken in two steps from the registers (no
// difference of large sums), all arithmetic is float32, each output is rounded once.
#include <math.h>

#include "pe_common.h"

namespace pe {

constexpr int kRnMaxC = 8192;
constexpr int kRnEl = 8;          // channels a thread holds
constexpr int kRnThreads = 256;   // of a workgroup whose rows are shorter than a wave's reach
// Items of backward (workgroups, each with a set of partial sums), about.  Two a CU: at 196608 x
// 256 bf16 the launch takes 141, 129, 133, 145, 138 us with 256, 512, 768, 1024, 2048 of them, at
// 3456 x 2048 29, 26, 28, 30, 35 us, and the fold behind it grows with their number.
constexpr int kRnItems = 512;
enum { kQ1 = 1, kQ0 = 2, kP1 = 4, kP0 = 8 };   // which sums of backward anything needs

struct RnFwd {
    const void *y, *x, *gate;
    const float *gp, *bp, *s, *gq, *bq;
    void *h, *z;
    float* stats;              // [4][rows]: mean and rstd of y, mean and rstd of h; or NULL
    long rows, gate_rows;      // rows per gate row; 0 = no gate
    long ldy, ldx, ldg, ldh, ldz;
    long rows_blk;
    float eps, inv_c;
    int C, post, pre, layer, act;
};

struct RnBwd {
    const void *dh, *dz, *y, *x, *gate;
    const float *stats, *gp, *bp, *s, *gq;
    void *dy, *dx, *dgate;
    float* part;               // [items][4][pitch]: sums of dz*hhat, dz, D*phi*yhat, D*phi
    int pitch, need;           // which of them are stored
    long rows, gate_rows;
    long lddh, lddz, ldy, ldx, ldg, lddy, lddx, lddg;
    long group, nseg, rows_blk;   // rows of a group, items of a group, rows of an item
    float inv_c;
    int C, pre, post, layer, act;
};

// ---- a thread's eight channels ------------------------------------------------------------
typedef float f32x8 __attribute__((ext_vector_type(8)));

// TEAM: the threads of a row inside a wave (8 to 64), or the most that a workgroup working on one
// row has (512, 1024: so many registers a thread can have).
__host__ __device__ constexpr bool in_wave(int team) { return team <= 64; }

template <int TEAM>
__device__ __forceinline__ int team_size() {
    return in_wave(TEAM) ? TEAM : (int)blockDim.x;
}

// VEC: channels 8t .. 8t+7 in 16-byte accesses.  Otherwise t, t + T, t + 2T, ...: any C, any
// alignment, still coalesced.
template <bool VEC>
__device__ __forceinline__ int channel(int t, int T, int j) {
    return VEC ? t * kRnEl + j : t + j * T;
}

__device__ __forceinline__ f32x8 splat(float v) { return f32x8{v, v, v, v, v, v, v, v}; }

__device__ __forceinline__ f32x8 fma8(f32x8 a, f32x8 b, f32x8 c) {
    return __builtin_elementwise_fma(a, b, c);
}

// A row's channels as they come from memory, so that the next row can be on its way in few
// registers while this one is worked on.  Channels past C read as 0.
template <typename T, bool VEC>
struct Raw {
    f32x8 f;
    __device__ __forceinline__ void load(const T* p, int t, int team, int C) {
        f = splat(0.0f);
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (t + j * team < C) {
                if (sizeof(T) == 4) {
                    f[j] = p[t + j * team];
                } else {
                    f[j] = bf16_bits_to_float(p[t + j * team]);
                }
            }
    }
    __device__ __forceinline__ f32x8 value() const { return f; }
};

template <>
struct Raw<float, true> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* p, int t, int, int C) {
        a = b = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (t * kRnEl < C) {
            a = *reinterpret_cast<const f32x4*>(p + t * kRnEl);
            b = *reinterpret_cast<const f32x4*>(p + t * kRnEl + 4);
        }
    }
    __device__ __forceinline__ f32x8 value() const {
        return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
};

template <>
struct Raw<uint16_t, true> {
    u32x4 v;
    __device__ __forceinline__ void load(const uint16_t* p, int t, int, int C) {
        v = u32x4{0, 0, 0, 0};
        if (t * kRnEl < C) v = *reinterpret_cast<const u32x4*>(p + t * kRnEl);
    }
    __device__ __forceinline__ f32x8 value() const {
        f32x8 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = bf16_bits_to_float(v[j] & 0xffffu);
            f[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
        }
        return f;
    }
};

template <bool VEC, typename T>
__device__ __forceinline__ f32x8 load8(const T* p, int t, int team, int C) {
    Raw<T, VEC> r;
    r.load(p, t, team, C);
    return r.value();
}

template <bool VEC>
__device__ __forceinline__ void store8(float* p, int t, int T, int C, f32x8 f) {
    if (VEC) {
        if (t * kRnEl < C) {
            *reinterpret_cast<f32x4*>(p + t * kRnEl) = f32x4{f[0], f[1], f[2], f[3]};
            *reinterpret_cast<f32x4*>(p + t * kRnEl + 4) = f32x4{f[4], f[5], f[6], f[7]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (t + j * T < C) p[t + j * T] = f[j];
    }
}

template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, int t, int T, int C, f32x8 f) {
    if (VEC) {
        if (t * kRnEl < C) {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = pack_bf16x2_bits(f[2 * j], f[2 * j + 1]);
            *reinterpret_cast<u32x4*>(p + t * kRnEl) = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (t + j * T < C) p[t + j * T] = (uint16_t)float_to_bf16_bits(f[j]);
    }
}

template <bool VEC>
__device__ __forceinline__ f32x8 load_param(const float* p, float absent, int t, int T, int C) {
    return p ? load8<VEC>(p, t, T, C) : splat(absent);
}

__device__ __forceinline__ float sum8(f32x8 v) {
    return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// 0 in the place of channels past C.
template <bool VEC>
__device__ __forceinline__ f32x8 inside(f32x8 v, int t, int T, int C) {
    if (VEC) {
        if (t * kRnEl >= C) v = splat(0.0f);
    } else {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (t + j * T >= C) v[j] = 0.0f;
    }
    return v;
}

// ---- sums over a row's team ---------------------------------------------------------------
// The lanes of a wave by data-parallel moves inside the vector unit, no LDS round trips: lane ^ 1
// and ^ 2 inside a quad, then mirrors of 8 and of 16 lanes (whose quads agree by then), then
// swaps of rows of 16 and of halves of the wave.  Every lane of the team ends with the same bits.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL,
                                                                     0xf, 0xf, true));
}

template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    v = dpp_add<0xB1>(v);    // quad_perm 1 0 3 2
    v = dpp_add<0x4E>(v);    // quad_perm 2 3 0 1
    v = dpp_add<0x141>(v);   // row_half_mirror
    if (W >= 16) v = dpp_add<0x140>(v);   // row_mirror
    if (W >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (W >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// A workgroup as a team: the waves' sums through LDS in order; two buffers in turn, so one
// barrier a sum is enough.
struct TeamSums {
    float2* buf;   // LDS [2][16], workgroup teams only
    int turn;
};

template <int TEAM>
__device__ __forceinline__ void team_sum2(float& a, float& b, TeamSums& ts) {
    constexpr int W = in_wave(TEAM) ? TEAM : 64;
    a = lanes_sum<W>(a);
    b = lanes_sum<W>(b);
    if (!in_wave(TEAM)) {
        float2* buf = ts.buf + 16 * ts.turn;
        ts.turn ^= 1;
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        const int waves = (int)blockDim.x >> 6;
        float2 v = buf[0];
        for (int i = 1; i < waves; ++i) {
            v.x += buf[i].x;
            v.y += buf[i].y;
        }
        a = v.x;
        b = v.y;
    }
}

// mean and rstd of the row, v replaced by the normalised row (anything past C).
template <int TEAM, bool VEC>
__device__ __forceinline__ void normalise(f32x8& v, int t, int T, int C, float inv_c, float eps,
                                          bool layer, float& mean, float& rstd, TeamSums& ts) {
    mean = 0.0f;
    float unused = 0.0f;
    if (layer) {
        float sum = sum8(v);   // channels past C hold 0
        team_sum2<TEAM>(sum, unused, ts);
        mean = sum * inv_c;
        v -= mean;
    }
    const f32x8 in = inside<VEC>(v, t, T, C);
    float sq = sum8(in * in);
    team_sum2<TEAM>(sq, unused, ts);
    rstd = 1.0f / sqrtf(sq * inv_c + eps);
    v *= rstd;
}

// ---- gate ---------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __expf(-g));
}

// phi(g) and, with a derivative, phi'(g).
__device__ __forceinline__ float gate_value(float g, int act, float& slope) {
    if (act == PE_GATE_NONE) {
        slope = 1.0f;
        return g;
    }
    const float s = sigmoid(g);
    if (act == PE_GATE_SIGMOID) {
        slope = s * (1.0f - s);
        return s;
    }
    slope = s * (1.0f + g * (1.0f - s));
    return g * s;
}

__device__ __forceinline__ void gate8(f32x8 g, int act, f32x8& phi, f32x8& slope) {
#pragma unroll
    for (int j = 0; j < kRnEl; ++j) {
        float d;
        phi[j] = gate_value(g[j], act, d);
        slope[j] = d;
    }
}

__device__ __forceinline__ long gate_row(long row, long per) {
    if (per == 1) return row;
    if (row <= 0x7fffffffl && per <= 0x7fffffffl) return (long)((unsigned)row / (unsigned)per);
    return row / per;
}

// ---- forward ------------------------------------------------------------------------------
template <typename YT, typename XT, int TEAM, bool VEC>
__global__ __launch_bounds__(in_wave(TEAM) ? kRnThreads : TEAM) void rnorm_fwd_kernel(RnFwd a) {
    __shared__ float2 lds[in_wave(TEAM) ? 1 : 32];
    TeamSums ts{lds, 0};
    const int T = team_size<TEAM>();
    const int t = in_wave(TEAM) ? (int)threadIdx.x % T : (int)threadIdx.x;
    const int teams = in_wave(TEAM) ? kRnThreads / T : 1;
    const int C = a.C;
    const f32x8 s = load_param<VEC>(a.s, 1.0f, t, T, C);
    const f32x8 A = load_param<VEC>(a.gp, 1.0f, t, T, C) * s;
    const f32x8 B = load_param<VEC>(a.bp, 0.0f, t, T, C) * s;
    const f32x8 gq = load_param<VEC>(a.gq, 1.0f, t, T, C);
    const f32x8 bq = load_param<VEC>(a.bq, 0.0f, t, T, C);
    f32x8 phi = splat(1.0f), slope;
    const long lo = (long)blockIdx.x * a.rows_blk;
    const long hi = lo + a.rows_blk < a.rows ? lo + a.rows_blk : a.rows;
    long have = -1;   // the gate row phi holds
    for (long row = lo + (in_wave(TEAM) ? (int)threadIdx.x / T : 0); row < hi; row += teams) {
        f32x8 y = load8<VEC>(static_cast<const YT*>(a.y) + row * a.ldy, t, T, C);
        f32x8 h = splat(0.0f);
        if (a.x) h = load8<VEC>(static_cast<const XT*>(a.x) + row * a.ldx, t, T, C);
        if (a.gate_rows) {
            const long g = gate_row(row, a.gate_rows);
            if (g != have) {
                gate8(load8<VEC>(static_cast<const YT*>(a.gate) + g * a.ldg, t, T, C), a.act, phi,
                      slope);
                have = g;
            }
        }
        float mean, rstd;
        if (a.post) {
            normalise<TEAM, VEC>(y, t, T, C, a.inv_c, a.eps, a.layer, mean, rstd, ts);
            if (a.stats && t == 0) {
                if (a.layer) a.stats[row] = mean;
                a.stats[a.rows + row] = rstd;
            }
        }
        h = fma8(fma8(y, A, B), phi, h);
        store8<VEC>(static_cast<XT*>(a.h) + row * a.ldh, t, T, C, h);
        if (a.pre) {
            h = inside<VEC>(h, t, T, C);
            normalise<TEAM, VEC>(h, t, T, C, a.inv_c, a.eps, a.layer, mean, rstd, ts);
            if (a.stats && t == 0) {
                if (a.layer) a.stats[2 * a.rows + row] = mean;
                a.stats[3 * a.rows + row] = rstd;
            }
            store8<VEC>(static_cast<YT*>(a.z) + row * a.ldz, t, T, C, fma8(h, gq, bq));
        }
    }
}

// ---- backward -----------------------------------------------------------------------------
// With D = dh + (norm backward of dz*gq at h), u = D*phi, yhat the normalised y:
//   dx = D;  dy = norm backward of u*s*gp at y;  dgate = phi' * sum_group D*s*(gp*yhat + bp)
//   dgq = sum dz*hhat, dbq = sum dz, dgp = s * sum u*yhat, dbp = s * sum u,
//   ds = gp * sum u*yhat + bp * sum u
// h is rebuilt in float32 from x and y, exactly as forward had it before rounding: the same bytes
// as reading the stored h, without its rounding in the gradients.  Four sums a channel stay in
// registers over an item's rows and go to the workspace once an item; a second launch folds the
// items in order in float64, so the results have the same bits on every call.  An item never
// crosses a gate row: phi is a constant of the item and is left out of its sums (the fold knows
// the item's gate), unless the gate has a row for each row, whose gradient needs no sum.
template <typename YT, typename XT, bool OWN, bool VEC>
struct RnRow {
    Raw<YT, VEC> y, dz, gate;
    Raw<XT, VEC> x, dh;
    float py, ry, ph, rh;   // mean and rstd of y and of h
    // What is absent reads as 0 (x, dh) or is not looked at (the rest).
    __device__ __forceinline__ void load(const RnBwd& a, long row, int t, int T) {
        const int C = a.C;
        y.load(static_cast<const YT*>(a.y) + row * a.ldy, t, T, C);
        x.load(static_cast<const XT*>(a.x) + row * a.ldx, t, T, a.x && a.pre ? C : 0);
        dh.load(static_cast<const XT*>(a.dh) + row * a.lddh, t, T, a.dh ? C : 0);
        py = ph = 0.0f;
        ry = rh = 1.0f;
        if (a.pre) {
            dz.load(static_cast<const YT*>(a.dz) + row * a.lddz, t, T, C);
            rh = a.stats[3 * a.rows + row];
            if (a.layer) ph = a.stats[2 * a.rows + row];
        }
        if (a.post) {
            ry = a.stats[a.rows + row];
            if (a.layer) py = a.stats[row];
        }
        if (OWN) gate.load(static_cast<const YT*>(a.gate) + row * a.ldg, t, T, C);
    }
};

// OWN: a gate row for each row.  The next row is loaded while this one is worked on, except by
// workgroups of more than 512 threads, which have no registers for it.
template <typename YT, typename XT, bool OWN, int TEAM, bool VEC>
__global__ __launch_bounds__(in_wave(TEAM) ? kRnThreads : TEAM) void rnorm_bwd_kernel(RnBwd a) {
    __shared__ float2 lds[in_wave(TEAM) ? 1 : 32];
    __shared__ float fold[in_wave(TEAM) ? kRnThreads / 64 : 1][4][in_wave(TEAM) ? TEAM * kRnEl : 1];
    TeamSums ts{lds, 0};
    const int T = team_size<TEAM>();
    const int t = in_wave(TEAM) ? (int)threadIdx.x % T : (int)threadIdx.x;
    const int teams = in_wave(TEAM) ? kRnThreads / T : 1;
    const int C = a.C;
    const f32x8 s = load_param<VEC>(a.s, 1.0f, t, T, C);
    const f32x8 A = load_param<VEC>(a.gp, 1.0f, t, T, C) * s;
    const f32x8 B = load_param<VEC>(a.bp, 0.0f, t, T, C) * s;
    const f32x8 gq = load_param<VEC>(a.gq, 1.0f, t, T, C);
    f32x8 phi = splat(1.0f), slope = splat(1.0f);
    const long g = (long)blockIdx.x / a.nseg;
    const long lo = g * a.group + ((long)blockIdx.x - g * a.nseg) * a.rows_blk;
    const long end = (g + 1) * a.group;
    const long hi = lo + a.rows_blk < end ? lo + a.rows_blk : end;
    if (!OWN && a.gate_rows)
        gate8(load8<VEC>(static_cast<const YT*>(a.gate) + g * a.ldg, t, T, C), a.act, phi, slope);
    f32x8 q1 = splat(0.0f), q0 = q1, p1 = q1, p0 = q1;
    long row = lo + (in_wave(TEAM) ? (int)threadIdx.x / T : 0);
    RnRow<YT, XT, OWN, VEC> now, next;
    constexpr bool AHEAD = TEAM != 1024;
    if (AHEAD && row < hi) now.load(a, row, t, T);
    for (; row < hi; row += teams) {
        if (!AHEAD) now.load(a, row, t, T);
        if (AHEAD && row + teams < hi) next.load(a, row + teams, t, T);
        f32x8 y = now.y.value(), d = now.dh.value();
        if (OWN) gate8(now.gate.value(), a.act, phi, slope);
        if (a.post) y = (y - now.py) * now.ry;
        if (a.pre) {
            f32x8 w = now.dz.value();
            const f32x8 hhat = (fma8(fma8(y, A, B), phi, now.x.value()) - now.ph) * now.rh;
            q0 += w;
            q1 = fma8(w, hhat, q1);
            w *= gq;
            float m1 = sum8(w), m2 = sum8(w * hhat);
            team_sum2<TEAM>(m1, m2, ts);
            m1 = a.layer ? m1 * a.inv_c : 0.0f;
            m2 *= a.inv_c;
            d = fma8(fma8(hhat, splat(-m2), w - m1), splat(now.rh), d);
        }
        if (a.dx) store8<VEC>(static_cast<XT*>(a.dx) + row * a.lddx, t, T, C, d);
        if (OWN)
            store8<VEC>(static_cast<YT*>(a.dgate) + row * a.lddg, t, T, C, d * fma8(y, A, B) * slope);
        d = inside<VEC>(d, t, T, C);
        const f32x8 u = d * phi;
        const f32x8 keep = OWN ? u : d;
        p0 += keep;
        p1 = fma8(keep, y, p1);
        f32x8 w = u * A;
        if (a.post) {
            float n1 = sum8(w), n2 = sum8(w * y);
            team_sum2<TEAM>(n1, n2, ts);
            n1 = a.layer ? n1 * a.inv_c : 0.0f;
            n2 *= a.inv_c;
            w = fma8(y, splat(-n2), w - n1) * now.ry;
        }
        store8<VEC>(static_cast<YT*>(a.dy) + row * a.lddy, t, T, C, w);
        if (AHEAD) now = next;
    }
    if (!a.need) return;
    float* out = a.part + (long)blockIdx.x * 4 * a.pitch;
    if (in_wave(TEAM)) {
        // rows side by side in the wave, then the waves in order
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const f32x8 sums = k == 0 ? q1 : k == 1 ? q0 : k == 2 ? p1 : p0;
            if (a.need & (1 << k)) {
#pragma unroll
                for (int j = 0; j < kRnEl; ++j) {
                    float v = sums[j];
#pragma unroll
                    for (int off = 32; off >= (in_wave(TEAM) ? TEAM : 64); off >>= 1)
                        v += __shfl_xor(v, off, 64);
                    if ((int)(threadIdx.x & 63) < T)
                        fold[threadIdx.x >> 6][k][channel<VEC>(t, T, j)] = v;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (a.need & (1 << k)) {
                for (int c = threadIdx.x; c < C; c += kRnThreads) {
                    float v = fold[0][k][c];
#pragma unroll
                    for (int wv = 1; wv < kRnThreads / 64; ++wv) v += fold[wv][k][c];
                    out[(long)k * a.pitch + c] = v;
                }
            }
        }
    } else {
        if (a.need & kQ1) store8<VEC>(out, t, T, C, q1);
        if (a.need & kQ0) store8<VEC>(out + a.pitch, t, T, C, q0);
        if (a.need & kP1) store8<VEC>(out + 2l * a.pitch, t, T, C, p1);
        if (a.need & kP0) store8<VEC>(out + 3l * a.pitch, t, T, C, p0);
    }
}

// ---- fold of the items --------------------------------------------------------------------
// Latency is all there is to it: a few MB that were just written.  A workgroup takes 32 channels
// (a 128-byte line of every row of sums), a thread four of them of every LANES-th item, with the
// loads of several items under way at a time; float64 sums in an order fixed by the sizes.
constexpr int kFoldCols = 32;
constexpr int kFoldMany = 32;    // items side by side
constexpr int kFoldFew = 8;      // the same where a gate row has few
typedef double f64x4 __attribute__((ext_vector_type(4)));

struct RnFold {
    float* part;
    long items, step;          // this fold's items: 0, step, 2*step, ...
    const float *gp, *bp, *s, *any;
    const void* gate;
    void* dgate;
    float *dgp, *dbp, *ds, *dgq, *dbq;
    long nseg, ldg, lddg;
    int C, act, pitch, need;
};

__device__ __forceinline__ double join64(unsigned lo, unsigned hi) {
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}

// a summed over the wave's halves in its lower half, b in its upper one.
__device__ __forceinline__ double add_halves(double a, double b) {
    const unsigned long long x = __double_as_longlong(a), y = __double_as_longlong(b);
    const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)y, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap((unsigned)(x >> 32), (unsigned)(y >> 32), false, false);
    return join64(lo[0], hi[0]) + join64(lo[1], hi[1]);
}

// a summed over pairs of rows of 16 lanes in the even rows, b in the odd ones.
__device__ __forceinline__ double add_rows(double a, double b) {
    const unsigned long long x = __double_as_longlong(a), y = __double_as_longlong(b);
    const auto lo = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)y, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((unsigned)(x >> 32), (unsigned)(y >> 32), false, false);
    return join64(lo[0], hi[0]) + join64(lo[1], hi[1]);
}

// v + v of the lane eight further in its row of 16.
__device__ __forceinline__ double add_eight(double v) {
    const unsigned long long x = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)x, 0x128, 0xf, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(x >> 32), 0x128, 0xf, 0xf, true);
    return v + join64((unsigned)lo, (unsigned)hi);
}

// sum[k] of channel c = sum over i < n of part[(first + i*step)][k][c], in the first kFoldCols
// threads, whose channel is the block's first plus their index.
template <int LANES>
__device__ __forceinline__ void fold_items(const RnFold& a, long first, long n, long step,
                                           double (&sum)[4]) {
    constexpr int QUADS = kFoldCols / 4;
    constexpr int WAVES = LANES * QUADS / 64;
    constexpr int AT_ONCE = 4;
    static_assert(QUADS == 8, "the sums over a wave's lanes");
    __shared__ double lds[WAVES][4][kFoldCols];
    const int quad = (int)threadIdx.x % QUADS, lane = (int)threadIdx.x / QUADS;
    const int c = (int)blockIdx.x * kFoldCols + quad * 4;
    f64x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = f64x4{0.0, 0.0, 0.0, 0.0};
    if (c < a.pitch) {
        // A branch around a load would make the thread wait for each in turn: items past the end
        // read the last one again and count as 0, sums that nothing needs read one that is.
        const float* p = a.part + first * 4 * a.pitch + c;
        const long jump = step * 4 * a.pitch;
        const int any = __builtin_ctz(a.need);
        long at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) at[k] = (long)((a.need & (1 << k)) ? k : any) * a.pitch;
        for (long i = lane; i < n; i += AT_ONCE * LANES) {
            f32x4 r[AT_ONCE][4];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const float* q = p + (i + u * LANES < n ? i + u * LANES : n - 1) * jump;
#pragma unroll
                for (int k = 0; k < 4; ++k) r[u][k] = *reinterpret_cast<const f32x4*>(q + at[k]);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const bool in = i + u * LANES < n;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[k][j] += (double)(in ? r[u][k][j] : 0.0f);
                }
            }
        }
    }
    // a wave's eight items into one: each step leaves half of the sums to half of the lanes
    const int l = (int)threadIdx.x & 63, k = 2 * ((l >> 4) & 1) + (l >> 5);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double u = add_eight(add_rows(add_halves(v[0][j], v[1][j]), add_halves(v[2][j], v[3][j])));
        if ((l & 15) < QUADS) lds[threadIdx.x >> 6][k][quad * 4 + j] = u;
    }
    __syncthreads();
    if (threadIdx.x < kFoldCols) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            sum[k] = lds[0][k][threadIdx.x];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum[k] += lds[w][k][threadIdx.x];
        }
    }
}

// A channel's parameters, asked for before the sums; again no branch around a load, an absent one
// reads a.any.
struct FoldParam {
    float gp, bp, s;
    __device__ __forceinline__ FoldParam(const RnFold& a, int c)
        : gp(*(a.gp ? a.gp + c : a.any)), bp(*(a.bp ? a.bp + c : a.any)), s(*(a.s ? a.s + c : a.any)) {}
    __device__ __forceinline__ void settle(const RnFold& a) {
        if (!a.gp) gp = 1.0f;
        if (!a.bp) bp = 0.0f;
        if (!a.s) s = 1.0f;
    }
};

// One gate row: its gradient, and its sums with phi in place of its first item's.
template <typename YT, int LANES>
__global__ __launch_bounds__(LANES * kFoldCols / 4) void rnorm_fold_gate_kernel(RnFold a) {
    const long g = blockIdx.y;
    const int c = (int)blockIdx.x * kFoldCols + (int)threadIdx.x;
    const bool mine = threadIdx.x < kFoldCols && c < a.C;
    FoldParam par(a, mine ? c : 0);
    const YT raw = static_cast<const YT*>(a.gate)[g * a.ldg + (mine ? c : 0)];
    double v[4];
    fold_items<LANES>(a, g * a.nseg, a.nseg, 1, v);
    if (mine) {
        par.settle(a);
        const float gv = sizeof(YT) == 4 ? (float)raw : bf16_bits_to_float((uint32_t)raw);
        float slope;
        const float phi = gate_value(gv, a.act, slope);
        const double gp = par.gp, bp = par.bp, s = par.s;
        const float dg = (float)((double)slope * s * (gp * v[2] + bp * v[3]));
        if (sizeof(YT) == 4) {
            static_cast<float*>(a.dgate)[g * a.lddg + c] = dg;
        } else {
            static_cast<uint16_t*>(a.dgate)[g * a.lddg + c] = (uint16_t)float_to_bf16_bits(dg);
        }
        float* p = a.part + g * a.nseg * 4 * a.pitch + c;
        p[0] = (float)v[0];
        p[a.pitch] = (float)v[1];
        p[2l * a.pitch] = (float)(v[2] * phi);
        p[3l * a.pitch] = (float)(v[3] * phi);
    }
}

__global__ __launch_bounds__(kFoldMany * kFoldCols / 4) void rnorm_fold_kernel(RnFold a) {
    const int c = (int)blockIdx.x * kFoldCols + (int)threadIdx.x;
    const bool mine = threadIdx.x < kFoldCols && c < a.C;
    FoldParam par(a, mine ? c : 0);
    double v[4];
    fold_items<kFoldMany>(a, 0, a.items, a.step, v);
    if (mine) {
        par.settle(a);
        const double gp = par.gp, bp = par.bp, s = par.s;
        if (a.dgq) a.dgq[c] = (float)v[0];
        if (a.dbq) a.dbq[c] = (float)v[1];
        if (a.dgp) a.dgp[c] = (float)(s * v[2]);
        if (a.dbp) a.dbp[c] = (float)(s * v[3]);
        if (a.ds) a.ds[c] = (float)(gp * v[2] + bp * v[3]);
    }
}

// ---- host ---------------------------------------------------------------------------------
static int team_of(int C) {
    const int need = (C + kRnEl - 1) / kRnEl;
    for (int t = 8; t <= 64; t *= 2)
        if (need <= t) return t;
    return need <= 512 ? 512 : 1024;
}

static unsigned block_of(int C) {   // threads of a workgroup
    return in_wave(team_of(C)) ? kRnThreads : (unsigned)(((C + kRnEl - 1) / kRnEl + 63) / 64 * 64);
}

static long rows_at_once(int C) { return in_wave(team_of(C)) ? kRnThreads / team_of(C) : 1; }

struct BwdGeom {
    long groups, group, nseg, rows_blk;
    long items() const { return groups * nseg; }
};

static int pitch_of(int C) { return (C + 3) & ~3; }   // of a row of sums: 16-byte steps

// About kRnItems items, none across a gate row, each a multiple of the rows its teams take at once.
static BwdGeom bwd_geom(const pe_rnorm_desc& d) {
    BwdGeom g;
    const bool grouped = d.gate_rows > 1;
    g.group = grouped ? d.gate_rows : d.rows;
    g.groups = grouped ? d.rows / d.gate_rows : 1;
    const long at_once = rows_at_once(d.C);
    long want = (kRnItems + g.groups - 1) / g.groups;
    long rows = (g.group + want - 1) / want;
    rows = (rows + at_once - 1) / at_once * at_once;
    if (rows < 1) rows = 1;
    g.rows_blk = rows;
    g.nseg = (g.group + rows - 1) / rows;
    return g;
}

static bool vec_ok(const void* p, long ld, int dtype) {
    return aligned(p, 16) && (ld * (dtype == PE_DTYPE_F32 ? 4 : 2)) % 16 == 0;
}

static int32_t check_desc(const char* what, const pe_rnorm_desc* d) {
    PE_REQUIRE(d, PE_E_INVALID, "%s: NULL description", what);
    PE_REQUIRE(d->rows >= 0 && d->C >= 1, PE_E_INVALID, "%s: bad sizes", what);
    PE_REQUIRE(d->C <= kRnMaxC, PE_E_UNSUPPORTED, "%s: %d channels, at most %d", what, d->C, kRnMaxC);
    PE_REQUIRE((d->y_dtype == PE_DTYPE_BF16 && (d->x_dtype == PE_DTYPE_BF16 || d->x_dtype == PE_DTYPE_F32)) ||
                   (d->y_dtype == PE_DTYPE_F32 && d->x_dtype == PE_DTYPE_F32),
               PE_E_UNSUPPORTED, "%s: types (%d, %d) of branch and residual", what, d->y_dtype,
               d->x_dtype);
    PE_REQUIRE(d->norm == PE_RNORM_LAYER || d->norm == PE_RNORM_RMS, PE_E_UNSUPPORTED,
               "%s: unknown norm %d", what, d->norm);
    PE_REQUIRE(d->eps > 0.0f && isfinite(d->eps), PE_E_INVALID, "%s: eps must be positive", what);
    PE_REQUIRE(d->gate_rows >= 0 && (d->gate_rows == 0 || d->rows % d->gate_rows == 0), PE_E_INVALID,
               "%s: %lld rows are not whole groups of %lld", what, (long long)d->rows,
               (long long)d->gate_rows);
    PE_REQUIRE(d->gate_act >= PE_GATE_NONE && d->gate_act <= PE_GATE_SILU, PE_E_UNSUPPORTED,
               "%s: unknown gate activation %d", what, d->gate_act);
    const int64_t lds[] = {d->ldy, d->ldx, d->ldgate, d->ldh, d->ldz, d->lddh, d->lddz, d->lddy, d->lddx,
                           d->lddgate};
    for (int64_t ld : lds)
        PE_REQUIRE(ld >= 0, PE_E_INVALID, "%s: negative row stride", what);
    return PE_OK;
}

// Calls F<TEAM, VEC>::go(args) for the team and layout at hand.
template <template <int, bool> class F, class... A>
static void with_team(int team, bool vec, A&&... a) {
    switch (team) {
        case 8: vec ? F<8, true>::go(a...) : F<8, false>::go(a...); break;
        case 16: vec ? F<16, true>::go(a...) : F<16, false>::go(a...); break;
        case 32: vec ? F<32, true>::go(a...) : F<32, false>::go(a...); break;
        case 64: vec ? F<64, true>::go(a...) : F<64, false>::go(a...); break;
        case 512: vec ? F<512, true>::go(a...) : F<512, false>::go(a...); break;
        default: vec ? F<1024, true>::go(a...) : F<1024, false>::go(a...);
    }
}

template <typename YT, typename XT>
struct FwdOf {
    template <int TEAM, bool VEC>
    struct F {
        static void go(const RnFwd& a, unsigned blocks, unsigned threads, hipStream_t st) {
            launch(rnorm_fwd_kernel<YT, XT, TEAM, VEC>, blocks, threads, 0, st, a);
        }
    };
};

template <typename YT, typename XT, bool OWN>
struct BwdOf {
    template <int TEAM, bool VEC>
    struct F {
        static void go(const RnBwd& a, unsigned blocks, unsigned threads, hipStream_t st) {
            launch(rnorm_bwd_kernel<YT, XT, OWN, TEAM, VEC>, blocks, threads, 0, st, a);
        }
    };
};

template <typename YT, typename XT>
static void launch_bwd(const RnBwd& a, bool vec, unsigned blocks, hipStream_t st) {
    if (a.gate_rows == 1) {
        with_team<BwdOf<YT, XT, true>::template F>(team_of(a.C), vec, a, blocks, block_of(a.C), st);
    } else {
        with_team<BwdOf<YT, XT, false>::template F>(team_of(a.C), vec, a, blocks, block_of(a.C), st);
    }
}

template <typename YT, typename XT>
static void launch_fwd(const RnFwd& a, bool vec, unsigned blocks, hipStream_t st) {
    with_team<FwdOf<YT, XT>::template F>(team_of(a.C), vec, a, blocks, block_of(a.C), st);
}

template <typename YT>
static void launch_fold_gate(const RnFold& a, bool few, dim3 grid, hipStream_t st) {
    if (few) {
        launch(rnorm_fold_gate_kernel<YT, kFoldFew>, grid, kFoldFew * kFoldCols / 4, 0, st, a);
    } else {
        launch(rnorm_fold_gate_kernel<YT, kFoldMany>, grid, kFoldMany * kFoldCols / 4, 0, st, a);
    }
}

}  // namespace pe

extern "C" int32_t pe_rnorm_fwd(const pe_rnorm_desc* d, const void* y, const void* x,
                                const float* post_gamma, const float* post_beta,
                                const float* scale, const void* gate, const float* pre_gamma,
                                const float* pre_beta, void* h, void* z, float* stats,
                                pe_stream_t stream) {
    using namespace pe;
    const int32_t bad = check_desc("pe_rnorm_fwd", d);
    if (bad) return bad;
    if (d->rows == 0) return PE_OK;
    PE_REQUIRE(y && h, PE_E_INVALID, "pe_rnorm_fwd: NULL y or h");
    PE_REQUIRE(d->rows == 1 || (d->ldh >= d->C && (!d->pre || d->ldz >= d->C)), PE_E_INVALID,
               "pe_rnorm_fwd: output rows overlap");
    PE_REQUIRE(!d->pre || z, PE_E_INVALID, "pe_rnorm_fwd: NULL z");
    PE_REQUIRE(d->gate_rows == 0 || gate, PE_E_INVALID, "pe_rnorm_fwd: NULL gate");
    PE_REQUIRE(d->post || !(post_gamma || post_beta), PE_E_INVALID,
               "pe_rnorm_fwd: parameters of a norm that is off");
    RnFwd a;
    a.y = y;
    a.x = x;
    a.gate = gate;
    a.gp = post_gamma;
    a.bp = post_beta;
    a.s = scale;
    a.gq = pre_gamma;
    a.bq = pre_beta;
    a.h = h;
    a.z = z;
    a.stats = stats;
    a.rows = d->rows;
    a.gate_rows = d->gate_rows;
    a.ldy = d->ldy;
    a.ldx = d->ldx;
    a.ldg = d->ldgate;
    a.ldh = d->ldh;
    a.ldz = d->ldz;
    a.eps = d->eps;
    a.inv_c = 1.0f / (float)d->C;
    a.C = d->C;
    a.post = d->post;
    a.pre = d->pre;
    a.layer = d->norm == PE_RNORM_LAYER;
    a.act = d->gate_act;
    const bool vec = d->C % kRnEl == 0 && vec_ok(y, d->ldy, d->y_dtype) && vec_ok(x, d->ldx, d->x_dtype) &&
                     vec_ok(gate, gate ? d->ldgate : 0, d->y_dtype) && vec_ok(h, d->ldh, d->x_dtype) &&
                     (!d->pre || vec_ok(z, d->ldz, d->y_dtype)) && aligned(post_gamma, 16) &&
                     aligned(post_beta, 16) && aligned(scale, 16) && aligned(pre_gamma, 16) &&
                     aligned(pre_beta, 16);
    const long at_once = rows_at_once(d->C);
    long rows = (d->rows + 2047) / 2048;
    rows = (rows + at_once - 1) / at_once * at_once;
    a.rows_blk = rows;
    const unsigned blocks = (unsigned)((d->rows + rows - 1) / rows);
    if (d->y_dtype == PE_DTYPE_F32) {
        launch_fwd<float, float>(a, vec, blocks, as_stream(stream));
    } else if (d->x_dtype == PE_DTYPE_F32) {
        launch_fwd<uint16_t, float>(a, vec, blocks, as_stream(stream));
    } else {
        launch_fwd<uint16_t, uint16_t>(a, vec, blocks, as_stream(stream));
    }
    return check_launch("pe_rnorm_fwd");
}

extern "C" size_t pe_rnorm_bwd_workspace_bytes(const pe_rnorm_desc* d) {
    if (pe::check_desc("pe_rnorm_bwd_workspace_bytes", d) != PE_OK) return 0;
    return sizeof(float) * 4 * (size_t)pe::pitch_of(d->C) * (size_t)(d->rows ? pe::bwd_geom(*d).items() : 0);
}

extern "C" int32_t pe_rnorm_bwd(const pe_rnorm_desc* d, const void* dh, const void* dz,
                                const void* y, const void* x, const float* stats,
                                const float* post_gamma, const float* post_beta,
                                const float* scale, const void* gate, const float* pre_gamma,
                                void* dy, void* dx, void* dgate, float* dpost_gamma,
                                float* dpost_beta, float* dscale, float* dpre_gamma,
                                float* dpre_beta, void* workspace, size_t workspace_bytes,
                                pe_stream_t stream) {
    using namespace pe;
    const int32_t bad = check_desc("pe_rnorm_bwd", d);
    if (bad) return bad;
    PE_REQUIRE(d->post || !(post_gamma || post_beta), PE_E_INVALID,
               "pe_rnorm_bwd: parameters of a norm that is off");
    PE_REQUIRE(d->post || !(dpost_gamma || dpost_beta), PE_E_INVALID,
               "pe_rnorm_bwd: gradients of a norm that is off");
    PE_REQUIRE(d->pre || !(dpre_gamma || dpre_beta || dz), PE_E_INVALID,
               "pe_rnorm_bwd: gradients of a norm that is off");
    const bool grouped = d->gate_rows > 1;
    const bool sums = dpost_gamma || dpost_beta || dscale || dpre_gamma || dpre_beta;
    const bool needs_p1 = dpost_gamma || dscale || grouped;
    const bool needs_p0 = dpost_beta || ((dscale || grouped) && post_beta);
    const int need = (dpre_gamma ? kQ1 : 0) | (dpre_beta ? kQ0 : 0) | (needs_p1 ? kP1 : 0) |
                     (needs_p0 ? kP0 : 0);
    BwdGeom g{0, 0, 0, 0};
    if (d->rows) {
        PE_REQUIRE(y && dy, PE_E_INVALID, "pe_rnorm_bwd: NULL y or dy");
        PE_REQUIRE(dh || dz, PE_E_INVALID, "pe_rnorm_bwd: neither dh nor dz");
        PE_REQUIRE(!d->pre || dz, PE_E_INVALID, "pe_rnorm_bwd: NULL dz");
        PE_REQUIRE(!(d->post || d->pre) || stats, PE_E_INVALID, "pe_rnorm_bwd: NULL stats");
        PE_REQUIRE(d->gate_rows == 0 || (gate && dgate), PE_E_INVALID, "pe_rnorm_bwd: NULL gate or dgate");
        PE_REQUIRE(d->rows == 1 || (d->lddy >= d->C && (!dx || d->lddx >= d->C)), PE_E_INVALID,
                   "pe_rnorm_bwd: output rows overlap");
        PE_REQUIRE(!dgate || d->rows == d->gate_rows || d->lddgate >= d->C, PE_E_INVALID,
                   "pe_rnorm_bwd: rows of dgate overlap");
        g = bwd_geom(*d);
        PE_REQUIRE(g.items() <= 0x7fffffffl, PE_E_UNSUPPORTED, "pe_rnorm_bwd: too many gate rows");
        if (need) {
            PE_REQUIRE(workspace && aligned(workspace, 16), PE_E_INVALID,
                       "pe_rnorm_bwd: workspace must be given, 16-byte aligned");
            PE_REQUIRE(workspace_bytes >= pe_rnorm_bwd_workspace_bytes(d), PE_E_INVALID,
                       "pe_rnorm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                       pe_rnorm_bwd_workspace_bytes(d));
        }
        RnBwd a;
        a.dh = dh;
        a.dz = dz;
        a.y = y;
        a.x = x;
        a.gate = gate;
        a.stats = stats;
        a.gp = post_gamma;
        a.bp = post_beta;
        a.s = scale;
        a.gq = pre_gamma;
        a.dy = dy;
        a.dx = dx;
        a.dgate = dgate;
        a.part = static_cast<float*>(workspace);
        a.pitch = pitch_of(d->C);
        a.need = need;
        a.rows = d->rows;
        a.gate_rows = d->gate_rows;
        a.lddh = d->lddh;
        a.lddz = d->lddz;
        a.ldy = d->ldy;
        a.ldx = d->ldx;
        a.ldg = d->ldgate;
        a.lddy = d->lddy;
        a.lddx = d->lddx;
        a.lddg = d->lddgate;
        a.group = g.group;
        a.nseg = g.nseg;
        a.rows_blk = g.rows_blk;
        a.inv_c = 1.0f / (float)d->C;
        a.C = d->C;
        a.pre = d->pre;
        a.post = d->post;
        a.layer = d->norm == PE_RNORM_LAYER;
        a.act = d->gate_act;
        const int yd = d->y_dtype, xd = d->x_dtype;
        const bool vec = d->C % kRnEl == 0 && vec_ok(y, d->ldy, yd) && vec_ok(x, x ? d->ldx : 0, xd) &&
                         vec_ok(dh, dh ? d->lddh : 0, xd) && vec_ok(dz, dz ? d->lddz : 0, yd) &&
                         vec_ok(gate, gate ? d->ldgate : 0, yd) &&
                         vec_ok(dgate, dgate ? d->lddgate : 0, yd) && vec_ok(dy, d->lddy, yd) &&
                         vec_ok(dx, dx ? d->lddx : 0, xd) && aligned(post_gamma, 16) &&
                         aligned(post_beta, 16) && aligned(scale, 16) && aligned(pre_gamma, 16);
        const unsigned items = (unsigned)g.items();
        if (yd == PE_DTYPE_F32) {
            launch_bwd<float, float>(a, vec, items, as_stream(stream));
        } else if (xd == PE_DTYPE_F32) {
            launch_bwd<uint16_t, float>(a, vec, items, as_stream(stream));
        } else {
            launch_bwd<uint16_t, uint16_t>(a, vec, items, as_stream(stream));
        }
    }
    if (!sums && !(grouped && d->rows)) return check_launch("pe_rnorm_bwd");
    RnFold f{};
    f.part = static_cast<float*>(workspace);
    f.gp = post_gamma;
    f.bp = post_beta;
    f.s = scale;
    f.gate = gate;
    f.dgate = dgate;
    f.dgp = dpost_gamma;
    f.dbp = dpost_beta;
    f.ds = dscale;
    f.dgq = dpre_gamma;
    f.dbq = dpre_beta;
    for (const float* q : {post_gamma, post_beta, scale, (const float*)f.part, (const float*)dpost_gamma,
                           (const float*)dpost_beta, (const float*)dscale, (const float*)dpre_gamma,
                           (const float*)dpre_beta})
        if (!f.any) f.any = q;
    f.nseg = g.nseg;
    f.ldg = d->ldgate;
    f.lddg = d->lddgate;
    f.C = d->C;
    f.act = d->gate_act;
    f.pitch = pitch_of(d->C);
    f.need = need;
    f.items = g.items();
    f.step = 1;
    const unsigned tiles = (unsigned)((d->C + kFoldCols - 1) / kFoldCols);
    if (grouped && d->rows) {
        for (long first = 0; first < g.groups; first += 65535) {   // a grid's y extent
            RnFold part = f;
            const long n = g.groups - first < 65535 ? g.groups - first : 65535;
            part.part += first * g.nseg * 4 * f.pitch;
            const long e = d->y_dtype == PE_DTYPE_F32 ? 4 : 2;
            part.gate = static_cast<const char*>(gate) + first * d->ldgate * e;
            part.dgate = static_cast<char*>(dgate) + first * d->lddgate * e;
            const dim3 grid(tiles, (unsigned)n);
            const bool few = g.nseg <= 4 * kFoldFew;   // one round of loads
            if (d->y_dtype == PE_DTYPE_F32) {
                launch_fold_gate<float>(part, few, grid, as_stream(stream));
            } else {
                launch_fold_gate<uint16_t>(part, few, grid, as_stream(stream));
            }
        }
        f.items = g.groups;
        f.step = g.nseg;
    }
    if (sums) launch(rnorm_fold_kernel, tiles, kFoldMany * kFoldCols / 4, 0, as_stream(stream), f);
    return check_launch("pe_rnorm_bwd");
}
