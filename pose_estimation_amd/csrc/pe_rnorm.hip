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
    float* part;               // [items][4][C]: sums of dz*hhat, dz, D*phi*yhat, D*phi
    long rows, gate_rows;
    long lddh, lddz, ldy, ldx, ldg, lddy, lddx, lddg;
    long group, nseg, rows_blk;   // rows of a group, items of a group, rows of an item
    float inv_c;
    int C, pre, post, layer, act;
};

// ---- a thread's eight channels ------------------------------------------------------------
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <int TEAM>
__device__ __forceinline__ int team_size() {
    return TEAM ? TEAM : (int)blockDim.x;
}

// VEC: channels 8t .. 8t+7 in 16-byte accesses.  Otherwise t, t + T, t + 2T, ...: any C, any
// alignment, still coalesced.
template <bool VEC>
__device__ __forceinline__ int channel(int t, int T, int j) {
    return VEC ? t * kRnEl + j : t + j * T;
}

__device__ __forceinline__ f32x8 splat(float v) { return f32x8{v, v, v, v, v, v, v, v}; }

// Channels past C read as 0.
template <bool VEC>
__device__ __forceinline__ f32x8 load8(const float* p, int t, int T, int C) {
    f32x8 f = splat(0.0f);
    if (VEC) {
        if (t * kRnEl < C) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p + t * kRnEl);
            const f32x4 b = *reinterpret_cast<const f32x4*>(p + t * kRnEl + 4);
            f = f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        }
    } else {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (t + j * T < C) f[j] = p[t + j * T];
    }
    return f;
}

template <bool VEC>
__device__ __forceinline__ f32x8 load8(const uint16_t* p, int t, int T, int C) {
    f32x8 f = splat(0.0f);
    if (VEC) {
        u32x4 v = {0, 0, 0, 0};
        if (t * kRnEl < C) v = *reinterpret_cast<const u32x4*>(p + t * kRnEl);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = bf16_bits_to_float(v[j] & 0xffffu);
            f[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (t + j * T < C) f[j] = bf16_bits_to_float(p[t + j * T]);
    }
    return f;
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
// Two values at a time.  A team inside a wave: butterfly.  A workgroup: butterfly, then the
// waves' results through LDS in order; two buffers in turn, so one barrier a sum is enough.
struct TeamSums {
    float2* buf;   // LDS [2][16], workgroup teams only
    int turn;
};

template <int TEAM>
__device__ __forceinline__ void team_sum2(float& a, float& b, TeamSums& ts) {
    constexpr int W = TEAM ? TEAM : 64;
#pragma unroll
    for (int off = W / 2; off >= 1; off >>= 1) {
        a += __shfl_xor(a, off, 64);
        b += __shfl_xor(b, off, 64);
    }
    if (TEAM == 0) {
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
__global__ __launch_bounds__(TEAM ? kRnThreads : 1024) void rnorm_fwd_kernel(RnFwd a) {
    __shared__ float2 lds[TEAM ? 1 : 32];
    TeamSums ts{lds, 0};
    const int T = team_size<TEAM>();
    const int t = TEAM ? (int)threadIdx.x % T : (int)threadIdx.x;
    const int teams = TEAM ? kRnThreads / T : 1;
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
    for (long row = lo + (TEAM ? (int)threadIdx.x / T : 0); row < hi; row += teams) {
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
        h += (y * A + B) * phi;
        store8<VEC>(static_cast<XT*>(a.h) + row * a.ldh, t, T, C, h);
        if (a.pre) {
            h = inside<VEC>(h, t, T, C);
            normalise<TEAM, VEC>(h, t, T, C, a.inv_c, a.eps, a.layer, mean, rstd, ts);
            if (a.stats && t == 0) {
                if (a.layer) a.stats[2 * a.rows + row] = mean;
                a.stats[3 * a.rows + row] = rstd;
            }
            store8<VEC>(static_cast<YT*>(a.z) + row * a.ldz, t, T, C, h * gq + bq);
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
template <typename YT, typename XT, int TEAM, bool VEC>
__global__ __launch_bounds__(TEAM ? kRnThreads : 1024) void rnorm_bwd_kernel(RnBwd a) {
    __shared__ float2 lds[TEAM ? 1 : 32];
    __shared__ float fold[TEAM ? kRnThreads / 64 : 1][4][TEAM ? TEAM * kRnEl : 1];
    TeamSums ts{lds, 0};
    const int T = team_size<TEAM>();
    const int t = TEAM ? (int)threadIdx.x % T : (int)threadIdx.x;
    const int teams = TEAM ? kRnThreads / T : 1;
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
    const bool own_gate = a.gate_rows == 1;
    if (a.gate_rows > 1)
        gate8(load8<VEC>(static_cast<const YT*>(a.gate) + g * a.ldg, t, T, C), a.act, phi, slope);
    f32x8 q1 = splat(0.0f), q0 = q1, p1 = q1, p0 = q1;
    for (long row = lo + (TEAM ? (int)threadIdx.x / T : 0); row < hi; row += teams) {
        f32x8 y = load8<VEC>(static_cast<const YT*>(a.y) + row * a.ldy, t, T, C);
        f32x8 x = splat(0.0f), d = x, w = x;
        if (a.pre && a.x) x = load8<VEC>(static_cast<const XT*>(a.x) + row * a.ldx, t, T, C);
        if (a.dh) d = load8<VEC>(static_cast<const XT*>(a.dh) + row * a.lddh, t, T, C);
        if (a.pre) w = load8<VEC>(static_cast<const YT*>(a.dz) + row * a.lddz, t, T, C);
        if (own_gate)
            gate8(load8<VEC>(static_cast<const YT*>(a.gate) + row * a.ldg, t, T, C), a.act, phi, slope);
        float rp = 1.0f;
        if (a.post) {
            rp = a.stats[a.rows + row];
            const float mean = a.layer ? a.stats[row] : 0.0f;
            y = (y - mean) * rp;
        }
        if (a.pre) {
            const float rq = a.stats[3 * a.rows + row];
            const float mean = a.layer ? a.stats[2 * a.rows + row] : 0.0f;
            const f32x8 hhat = (x + (y * A + B) * phi - mean) * rq;
            q0 += w;
            q1 += w * hhat;
            w *= gq;
            float m1 = sum8(w), m2 = sum8(w * hhat);
            team_sum2<TEAM>(m1, m2, ts);
            m1 = a.layer ? m1 * a.inv_c : 0.0f;
            m2 *= a.inv_c;
            d += (w - m1 - hhat * m2) * rq;
        }
        if (a.dx) store8<VEC>(static_cast<XT*>(a.dx) + row * a.lddx, t, T, C, d);
        if (own_gate)
            store8<VEC>(static_cast<YT*>(a.dgate) + row * a.lddg, t, T, C, d * (y * A + B) * slope);
        d = inside<VEC>(d, t, T, C);
        const f32x8 u = d * phi;
        const f32x8 keep = own_gate ? u : d;
        p0 += keep;
        p1 += keep * y;
        w = u * A;
        if (a.post) {
            float n1 = sum8(w), n2 = sum8(w * y);
            team_sum2<TEAM>(n1, n2, ts);
            n1 = a.layer ? n1 * a.inv_c : 0.0f;
            n2 *= a.inv_c;
            w = (w - n1 - y * n2) * rp;
        }
        store8<VEC>(static_cast<YT*>(a.dy) + row * a.lddy, t, T, C, w);
    }
    if (!a.part) return;
    float* out = a.part + (long)blockIdx.x * 4 * C;
    if (TEAM) {
        // rows side by side in the wave, then the waves in order
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const f32x8 sums = k == 0 ? q1 : k == 1 ? q0 : k == 2 ? p1 : p0;
#pragma unroll
            for (int j = 0; j < kRnEl; ++j) {
                float v = sums[j];
#pragma unroll
                for (int off = 32; off >= (TEAM ? TEAM : 64); off >>= 1) v += __shfl_xor(v, off, 64);
                if ((int)(threadIdx.x & 63) < T)
                    fold[threadIdx.x >> 6][k][channel<VEC>(t, T, j)] = v;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 4 * C; i += kRnThreads) {
            const int k = i / C, c = i - k * C;
            float v = fold[0][k][c];
#pragma unroll
            for (int wv = 1; wv < kRnThreads / 64; ++wv) v += fold[wv][k][c];
            out[i] = v;
        }
    } else {
        store8<VEC>(out, t, T, C, q1);
        store8<VEC>(out + C, t, T, C, q0);
        store8<VEC>(out + 2 * (long)C, t, T, C, p1);
        store8<VEC>(out + 3 * (long)C, t, T, C, p0);
    }
}

// ---- fold of the items --------------------------------------------------------------------
constexpr int kFoldLanes = 16;   // items walked side by side, for 64 channels each

struct RnFold {
    float* part;
    long items, step;          // this fold's items: 0, step, 2*step, ...
    const float *gp, *bp, *s;
    const void* gate;
    void* dgate;
    float *dgp, *dbp, *ds, *dgq, *dbq;
    long nseg, ldg, lddg;
    int C, act;
};

// Sums of part[first + k*step][0..3][c] over k < n, in threads with lane 0.
__device__ __forceinline__ void fold_items(const float* part, long first, long n, long step, int C,
                                           int c, int lane, double* v, double (*lds)[4][64]) {
    v[0] = v[1] = v[2] = v[3] = 0.0;
    if (c < C) {
        for (long i = lane; i < n; i += kFoldLanes) {
            const float* p = part + (first + i * step) * 4 * C + c;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += (double)p[(long)k * C];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) lds[lane][k][threadIdx.x & 63] = v[k];
    __syncthreads();
    if (lane == 0) {
        for (int l = 1; l < kFoldLanes; ++l) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += lds[l][k][threadIdx.x & 63];
        }
    }
}

// One gate row: its gradient, and its sums with phi in place of its first item's.
template <typename YT>
__global__ __launch_bounds__(64 * kFoldLanes) void rnorm_fold_gate_kernel(RnFold a) {
    __shared__ double lds[kFoldLanes][4][64];
    const int lane = (int)threadIdx.x >> 6;
    const int c = (int)blockIdx.x * 64 + ((int)threadIdx.x & 63);
    const long g = blockIdx.y;
    double v[4];
    fold_items(a.part, g * a.nseg, a.nseg, 1, a.C, c, lane, v, lds);
    if (lane == 0 && c < a.C) {
        float slope;
        float gv;
        if (sizeof(YT) == 4) {
            gv = static_cast<const float*>(a.gate)[g * a.ldg + c];
        } else {
            gv = bf16_bits_to_float(static_cast<const uint16_t*>(a.gate)[g * a.ldg + c]);
        }
        const float phi = gate_value(gv, a.act, slope);
        const double gp = a.gp ? a.gp[c] : 1.0, bp = a.bp ? a.bp[c] : 0.0, s = a.s ? a.s[c] : 1.0;
        const float dg = (float)((double)slope * s * (gp * v[2] + bp * v[3]));
        if (sizeof(YT) == 4) {
            static_cast<float*>(a.dgate)[g * a.lddg + c] = dg;
        } else {
            static_cast<uint16_t*>(a.dgate)[g * a.lddg + c] = (uint16_t)float_to_bf16_bits(dg);
        }
        float* p = a.part + g * a.nseg * 4 * a.C + c;
        p[0] = (float)v[0];
        p[a.C] = (float)v[1];
        p[2l * a.C] = (float)(v[2] * phi);
        p[3l * a.C] = (float)(v[3] * phi);
    }
}

__global__ __launch_bounds__(64 * kFoldLanes) void rnorm_fold_kernel(RnFold a) {
    __shared__ double lds[kFoldLanes][4][64];
    const int lane = (int)threadIdx.x >> 6;
    const int c = (int)blockIdx.x * 64 + ((int)threadIdx.x & 63);
    double v[4];
    fold_items(a.part, 0, a.items, a.step, a.C, c, lane, v, lds);
    if (lane == 0 && c < a.C) {
        const double gp = a.gp ? a.gp[c] : 1.0, bp = a.bp ? a.bp[c] : 0.0, s = a.s ? a.s[c] : 1.0;
        if (a.dgq) a.dgq[c] = (float)v[0];
        if (a.dbq) a.dbq[c] = (float)v[1];
        if (a.dgp) a.dgp[c] = (float)(s * v[2]);
        if (a.dbp) a.dbp[c] = (float)(s * v[3]);
        if (a.ds) a.ds[c] = (float)(gp * v[2] + bp * v[3]);
    }
}

// ---- host ---------------------------------------------------------------------------------
static int team_of(int C) {   // threads a row, 0: a workgroup a row
    const int need = (C + kRnEl - 1) / kRnEl;
    for (int t = 8; t <= 64; t *= 2)
        if (need <= t) return t;
    return 0;
}

static unsigned block_of(int C) {   // threads of a workgroup
    return team_of(C) ? kRnThreads : (unsigned)(((C + kRnEl - 1) / kRnEl + 63) / 64 * 64);
}

static long rows_at_once(int C) { return team_of(C) ? kRnThreads / team_of(C) : 1; }

struct BwdGeom {
    long groups, group, nseg, rows_blk;
    long items() const { return groups * nseg; }
};

// About 1024 items, none across a gate row, each a multiple of the rows its teams take at once.
static BwdGeom bwd_geom(const pe_rnorm_desc& d) {
    BwdGeom g;
    const bool grouped = d.gate_rows > 1;
    g.group = grouped ? d.gate_rows : d.rows;
    g.groups = grouped ? d.rows / d.gate_rows : 1;
    const long at_once = rows_at_once(d.C);
    long want = (1024 + g.groups - 1) / g.groups;
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

#define RN_TEAM(KERNEL, YT, XT, VEC, ...)                                                          \
    switch (team) {                                                                                \
        case 8: launch(KERNEL<YT, XT, 8, VEC>, __VA_ARGS__); break;                                \
        case 16: launch(KERNEL<YT, XT, 16, VEC>, __VA_ARGS__); break;                              \
        case 32: launch(KERNEL<YT, XT, 32, VEC>, __VA_ARGS__); break;                              \
        case 64: launch(KERNEL<YT, XT, 64, VEC>, __VA_ARGS__); break;                              \
        default: launch(KERNEL<YT, XT, 0, VEC>, __VA_ARGS__);                                      \
    }
#define RN_TYPES(KERNEL, VEC, ...)                                                                 \
    if (d->y_dtype == PE_DTYPE_F32) {                                                              \
        RN_TEAM(KERNEL, float, float, VEC, __VA_ARGS__)                                            \
    } else if (d->x_dtype == PE_DTYPE_F32) {                                                       \
        RN_TEAM(KERNEL, uint16_t, float, VEC, __VA_ARGS__)                                         \
    } else {                                                                                       \
        RN_TEAM(KERNEL, uint16_t, uint16_t, VEC, __VA_ARGS__)                                      \
    }
#define RN_LAUNCH(KERNEL, ...)                                                                     \
    if (vec) {                                                                                     \
        RN_TYPES(KERNEL, true, __VA_ARGS__)                                                        \
    } else {                                                                                       \
        RN_TYPES(KERNEL, false, __VA_ARGS__)                                                       \
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
    const int team = team_of(d->C);
    const long at_once = rows_at_once(d->C);
    long rows = (d->rows + 2047) / 2048;
    rows = (rows + at_once - 1) / at_once * at_once;
    a.rows_blk = rows;
    const unsigned blocks = (unsigned)((d->rows + rows - 1) / rows);
    RN_LAUNCH(rnorm_fwd_kernel, blocks, block_of(d->C), 0, as_stream(stream), a)
    return check_launch("pe_rnorm_fwd");
}

extern "C" size_t pe_rnorm_bwd_workspace_bytes(const pe_rnorm_desc* d) {
    if (pe::check_desc("pe_rnorm_bwd_workspace_bytes", d) != PE_OK) return 0;
    return sizeof(float) * 4 * (size_t)d->C * (size_t)(d->rows ? pe::bwd_geom(*d).items() : 0);
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
        if (sums || grouped) {
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
        a.part = sums || grouped ? static_cast<float*>(workspace) : nullptr;
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
        const int team = team_of(d->C);
        RN_LAUNCH(rnorm_bwd_kernel, (unsigned)g.items(), block_of(d->C), 0, as_stream(stream), a)
    }
    if (!sums && !(grouped && d->rows)) return check_launch("pe_rnorm_bwd");
    RnFold f;
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
    f.nseg = g.nseg;
    f.ldg = d->ldgate;
    f.lddg = d->lddgate;
    f.C = d->C;
    f.act = d->gate_act;
    f.items = g.items();
    f.step = 1;
    const unsigned tiles = (unsigned)((d->C + 63) / 64);
    if (grouped && d->rows) {
        for (long first = 0; first < g.groups; first += 65535) {   // a grid's y extent
            RnFold part = f;
            const long n = g.groups - first < 65535 ? g.groups - first : 65535;
            part.part += first * g.nseg * 4 * d->C;
            const long e = d->y_dtype == PE_DTYPE_F32 ? 4 : 2;
            part.gate = static_cast<const char*>(gate) + first * d->ldgate * e;
            part.dgate = static_cast<char*>(dgate) + first * d->lddgate * e;
            if (d->y_dtype == PE_DTYPE_F32) {
                launch(rnorm_fold_gate_kernel<float>, dim3(tiles, (unsigned)n), 64 * kFoldLanes, 0,
                       as_stream(stream), part);
            } else {
                launch(rnorm_fold_gate_kernel<uint16_t>, dim3(tiles, (unsigned)n), 64 * kFoldLanes, 0,
                       as_stream(stream), part);
            }
        }
        f.items = g.groups;
        f.step = g.nseg;
    }
    if (sums) launch(rnorm_fold_kernel, tiles, 64 * kFoldLanes, 0, as_stream(stream), f);
    return check_launch("pe_rnorm_bwd");
}
