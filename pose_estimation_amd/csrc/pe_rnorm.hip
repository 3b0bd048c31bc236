// a9. Row norm after and before a residual block, with the block's gate and residual scale.
//
//   per row of C channels:  a = N(y)*gp + bp;  h = x + s*phi(gate)*a;  z = N(h)*gq + bq
//   N(v) = (v - mean(v)) * rstd (layer) or v * rstd (rms), rstd = 1/sqrt(mean((v - mean)^2) + eps)
//
// Bound: HBM bandwidth.  Forward reads y and x and writes h and z, backward reads y, x, dh and dz
// and writes dy and dx, each once: a row lives in the registers of the team of threads that owns
// it from its load to its store, so statistics, both norms and the gate cost no further pass.
// Eight channels a thread (one 16-byte load of bf16): a team is the next power of two of C/8
// threads inside one wave (1 to 64, several rows a wave side by side), or, past 512 channels, a
// workgroup of its own.  Means and variances come from the registers in two steps, so no large sums
// cancel; all arithmetic is float32, each output is rounded once.  Wider shares of a row per thread
// would not leave a wave the registers to have the next row under way, narrower ones add lanes to
// every sum.  Where a last wave has little to do (just past 512, 1024, 2048, 4096 channels) the
// vector instructions bound it instead, about 190 for eight channels forward, 350 backward.
// Measured on the device: forward 8192 x 4096 bf16 with a float32 residual and a gate per row 88 us
// (5.3 TB/s), 196608 x 256 bf16 with a gate per image 75 us (5.4 TB/s) and backward there 129 us
// (4.7 TB/s, as a copy), 8000 x 4096 bf16 43 us (6.1 TB/s) and backward with its fold 88 us
// (4.5 TB/s), one row of 4096 3.2 us.  Where the comments below set two choices side by side, both
// were timed as calls in a row, one to three us more than the device takes.
#include <float.h>
#include <math.h>

#include <initializer_list>

#include "pe_common.h"
#include "pe_lanes.h"

namespace pe {

constexpr int kRnMaxC = 8192;
constexpr int kRnEl = 8;          // channels a thread holds
constexpr int kRnThreads = 256;   // of a workgroup whose rows are shorter than a wave's reach
// Items of backward (workgroups, each with a set of partial sums), about: as many for each compute
// unit, all of them there at once, few enough for the fold behind them.  Rows inside a wave: two
// (both launches at 60000 x 333 bf16 66 us, with 1.5, 3, 4 a unit 75, 67, 70; at 196608 x 256 135,
// 135, 139, 136).  A workgroup of 3 to 6 waves: two (10000 x 1400 45 us; 2.7, 4, 5.3 of them 49, 50, 57),
// of more: one, which is all that its registers leave room for (3000 x 4096 38 us, with two 46), of 2:
// four (60000 x 520 105 us, with three 119), or two where an item would not have eight rows
// (2000 x 1024: 22 us, with four 26).
constexpr long kRnUnits = 256;
// The sums an item leaves, as bits of what anything needs: of dz*hhat, dz, D*phi*yhat and D*phi,
// and with a gate shared by several rows also of D*yhat and D.
enum { kQ1 = 1, kQ0 = 2, kP1 = 4, kP0 = 8, kG1 = 16, kG0 = 32 };
constexpr int slots_of(long gate_rows) { return gate_rows > 1 ? 6 : 4; }

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
    float* part;               // [items][slots][pitch]; NULL: the only item writes the gradients
    float *dgp, *dbp, *ds, *dgq, *dbq;
    int pitch, need;
    long rows, gate_rows;
    long lddh, lddz, ldy, ldx, ldg, lddy, lddx, lddg;
    long group, nseg, rows_blk;   // rows of a group, items of a group, rows of an item
    long first;                   // item of the grid's first workgroup
    float inv_c;
    int C, pre, post, layer, act;
};

// ---- a thread's eight channels ------------------------------------------------------------
typedef float f32x8 __attribute__((ext_vector_type(8)));

// TEAM: the threads of a row inside a wave (1 to 64), or the most that a workgroup working on one
// row has (512, 1024: so many registers a thread can have).
__host__ __device__ constexpr bool in_wave(int team) { return team <= 64; }

template <int TEAM>
__device__ __forceinline__ int team_size() {
    return in_wave(TEAM) ? TEAM : (int)blockDim.x;
}

// How a row's channels lie over its threads.  WHOLE (C a multiple of 8): thread t has channels 8t
// to 8t+7.  TAIL: the last thread has the row's last eight, which the one before it shares: it
// computes them all and counts and stores only those from `first` on.  FEW (C < 8): one channel a
// thread.  Threads past the row read its last channels and count nothing, so that no load needs a
// branch of its own (which would make the wave wait for it).  Rows start at any element: 16-byte
// accesses need no alignment here.
enum { WHOLE, TAIL, FEW };

template <int MODE>
struct Cols {
    int c, first;
    bool on;
    __device__ __forceinline__ Cols(int t, int C) {
        constexpr int N = MODE == FEW ? 1 : kRnEl;
        on = t * N < C;
        c = t * N < C - N ? t * N : C - N;
        first = t * N - c;
    }
    // Whether the thread's j-th value is a channel of its own.
    __device__ __forceinline__ bool mine(int j) const {
        return on && (MODE == WHOLE || (MODE == TAIL && j >= first) || (MODE == FEW && j == 0));
    }
};

__device__ __forceinline__ f32x8 splat(float v) { return f32x8{v, v, v, v, v, v, v, v}; }

__device__ __forceinline__ f32x8 fma8(f32x8 a, f32x8 b, f32x8 c) {
    return __builtin_elementwise_fma(a, b, c);
}

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// A row's channels as they come from memory, so that the next row can be on its way in few
// registers while this one is worked on.
template <typename T, int MODE>
struct Raw;

template <int MODE>
struct Raw<float, MODE> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* p, const Cols<MODE>& k) {
        if (MODE == FEW) {
            a = b = f32x4{p[k.c], 0.0f, 0.0f, 0.0f};
        } else {
            a = *reinterpret_cast<const f32x4_any*>(p + k.c);
            b = *reinterpret_cast<const f32x4_any*>(p + k.c + 4);
        }
    }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(a), "+v"(b)); }
    __device__ __forceinline__ f32x8 value() const {
        return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
};

template <int MODE>
struct Raw<uint16_t, MODE> {
    u32x4 v;
    __device__ __forceinline__ void load(const uint16_t* p, const Cols<MODE>& k) {
        if (MODE == FEW) {
            v = u32x4{p[k.c], 0, 0, 0};
        } else {
            v = *reinterpret_cast<const u32x4_any*>(p + k.c);
        }
    }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(v)); }
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

template <int MODE, typename T>
__device__ __forceinline__ f32x8 load8(const T* p, const Cols<MODE>& k) {
    Raw<T, MODE> r;
    r.load(p, k);
    return r.value();
}

// ALL: also by threads whose channels are another's as well, which hold the same bits for them (and
// have read them before, inside one wave, where the output may be the input).
template <int MODE, bool ALL = false>
__device__ __forceinline__ void store8(float* p, const Cols<MODE>& k, f32x8 f) {
    if (MODE == FEW) {
        if (ALL || k.on) p[k.c] = f[0];
    } else if (ALL || (k.on && k.first == 0)) {
        *reinterpret_cast<f32x4_any*>(p + k.c) = f.lo;
        *reinterpret_cast<f32x4_any*>(p + k.c + 4) = f.hi;
    } else if (MODE == TAIL) {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (k.mine(j)) p[k.c + j] = f[j];
    }
}

template <int MODE, bool ALL = false>
__device__ __forceinline__ void store8(uint16_t* p, const Cols<MODE>& k, f32x8 f) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = pack_bf16x2_bits(f[2 * j], f[2 * j + 1]);
    if (MODE == FEW) {
        if (ALL || k.on) p[k.c] = (uint16_t)v[0];
    } else if (ALL || (k.on && k.first == 0)) {
        *reinterpret_cast<u32x4_any*>(p + k.c) = v;
    } else if (MODE == TAIL) {
#pragma unroll
        for (int j = 0; j < kRnEl; ++j)
            if (k.mine(j)) p[k.c + j] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
    }
}

// The last thread's neighbour may be in another wave of a workgroup.
constexpr bool store_all(int team, int mode) { return in_wave(team) || mode == WHOLE; }

template <int MODE>
__device__ __forceinline__ f32x8 load_param(const float* p, float absent, const Cols<MODE>& k) {
    return p ? load8<MODE>(p, k) : splat(absent);
}

// A thread's share of a sum over the row, and of a sum of products: of its own channels.
template <int MODE>
__device__ __forceinline__ f32x8 own(f32x8 v, const Cols<MODE>& k) {
    if (MODE == WHOLE) return v;
#pragma unroll
    for (int j = 0; j < kRnEl; ++j) v[j] = k.mine(j) ? v[j] : 0.0f;
    return v;
}

template <int MODE>
__device__ __forceinline__ float sum8(f32x8 own_v, const Cols<MODE>& k) {
    const f32x4 q = own_v.lo + own_v.hi;
    const float s = (q[0] + q[1]) + (q[2] + q[3]);
    return MODE != WHOLE || k.on ? s : 0.0f;
}

template <int MODE>
__device__ __forceinline__ float dot8(f32x8 own_v, f32x8 w, const Cols<MODE>& k) {
    const f32x4 q = __builtin_elementwise_fma(own_v.hi, w.hi, own_v.lo * w.lo);
    const float s = (q[0] + q[1]) + (q[2] + q[3]);
    return MODE != WHOLE || k.on ? s : 0.0f;
}

// ---- sums over a row's team ---------------------------------------------------------------
// A workgroup as a team: the waves' values through LDS, then a lane for each of the at most 16
// waves (a loop over them instead took 12 % more at 4000 x 8192 bf16); two buffers in turn, so
// one barrier a sum is enough.
struct TeamSums {
    float2* buf;    // LDS [2][16], workgroup teams only
    int wave, waves, turn;
    // 1 / this wave's channels, and the channels of the wave of the lane's index; forward only
    float per_wave, in_lane;
};

// Of a workgroup that works on one row.
__host__ __device__ constexpr int waves_of(int C) { return (C + 64 * kRnEl - 1) / (64 * kRnEl); }

__device__ __forceinline__ float2 each_wave(float2 v, TeamSums& ts) {
    float2* buf = ts.buf + 16 * ts.turn;
    ts.turn ^= 1;
    if ((threadIdx.x & 63) == 0) buf[ts.wave] = v;
    __syncthreads();
    const int w = (int)threadIdx.x & 15;
    v = buf[w];
    return w < ts.waves ? v : float2{0.0f, 0.0f};
}

template <int TEAM>
__device__ __forceinline__ void team_sum2(float& a, float& b, TeamSums& ts) {
    constexpr int W = in_wave(TEAM) ? TEAM : 64;
    a = lanes_sum<W>(a);
    b = lanes_sum<W>(b);
    if (!in_wave(TEAM)) {
        const float2 v = each_wave(float2{a, b}, ts);
        a = lanes_sum<16>(v.x);
        b = lanes_sum<16>(v.y);
    }
}

// mean and rstd of the row, v replaced by the normalised row.  In two steps, the second about the
// first's mean, so that no large sums cancel.  A workgroup would pay a barrier for each step: its
// waves take both about their own means m_w and are joined behind one,
//   sum (v - m)^2 = sum_w (sum (v - m_w)^2 + n_w (m_w - m)^2).
template <int TEAM, int MODE>
__device__ __forceinline__ void normalise(f32x8& v, const Cols<MODE>& k, float inv_c, float eps,
                                          bool layer, float& mean, float& rstd, TeamSums& ts) {
    constexpr int W = in_wave(TEAM) ? TEAM : 64;
    mean = 0.0f;
    f32x8 c = v;
    if (layer) {
        mean = lanes_sum<W>(sum8(own<MODE>(v, k), k)) * (in_wave(TEAM) ? inv_c : ts.per_wave);
        c = v - mean;
    }
    const f32x8 own_c = own<MODE>(c, k);
    float var = lanes_sum<W>(dot8(own_c, own_c, k));
    if (!in_wave(TEAM)) {
        const float2 w = each_wave(float2{mean, var}, ts);
        if (layer) {
            mean = lanes_sum<16>(w.x * ts.in_lane) * inv_c;
            const float d = w.x - mean;
            var = lanes_sum<16>(__builtin_fmaf(d * ts.in_lane, d, w.y));
            c = v - mean;
        } else {
            var = lanes_sum<16>(w.y);
        }
    }
    rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(var, inv_c, eps));   // good to 2^-23; eps is normal
    v = c * rstd;
}

// ---- gate ---------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float as_float(T v) {
    return sizeof(T) == 4 ? (float)v : bf16_bits_to_float((uint32_t)v);
}

// phi(g) and, with a derivative, phi'(g), from s = sigmoid(g) and c = 1 - s = exp(-g) s: the
// difference would lose what is left of c where s is near 1 (all of it from g = 17 on).
__device__ __forceinline__ float gate_value(float g, int act, float& slope) {
    if (act == PE_GATE_NONE) {
        slope = 1.0f;
        return g;
    }
    const float e = __expf(-g);
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    const float c = fminf(e, FLT_MAX) * s;   // 0, not NaN, where s has vanished
    if (act == PE_GATE_SIGMOID) {
        slope = s * c;
        return s;
    }
    slope = __builtin_fmaf(g * s, c, s);
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
    if (row <= 0x7fffffffl && per <= 0x7fffffffl) return (long)((unsigned)row / (unsigned)per);
    return row / per;
}

// ---- rows ---------------------------------------------------------------------------------
// Every load of a row is made, and its stores too where they can be: the compiler waits for loads
// by the number of accesses that are sure to come after them, so a branch around any of these
// would make each row wait for the next one's loads (60000 x 333 bf16, backward: 66 us, with
// branches 85).  What is absent is a row of zeros, and past its last row a team reads that one again
// (zeros instead: 5 % fewer bytes at 8192 x 4096, but 8000 x 4096 backward 97 us, not 88).
__device__ float rn_zeros[kRnMaxC];

template <typename T>
struct Rows {
    const T* p;
    long ld;
    __device__ __forceinline__ Rows(const void* at, long stride) {
        p = at ? static_cast<const T*>(at) : reinterpret_cast<const T*>(rn_zeros);
        ld = at ? stride : 0;
    }
    __device__ __forceinline__ const T* operator[](long row) const { return p + row * ld; }
};

// step(row, its data) for every teams-th row from `row` on, with load(data, row) a row ahead; two
// sets of registers in turn.
template <typename ROW, typename LOAD, typename STEP>
__device__ __forceinline__ void for_rows(long row, long hi, int teams, LOAD load, STEP step) {
    ROW one, two;
    if (row < hi) load(one, row);
    while (row < hi) {
        load(two, row + teams < hi ? row + teams : hi - 1);
        step(row, one);
        row += teams;
        if (row >= hi) break;
        load(one, row + teams < hi ? row + teams : hi - 1);
        step(row, two);
        row += teams;
    }
}

// ---- forward ------------------------------------------------------------------------------
// OWN: a gate row for each row.
template <typename YT, typename XT, bool OWN, int MODE>
struct FwdRow {
    Raw<YT, MODE> y, gate;
    Raw<XT, MODE> x;
};

template <typename YT, typename XT, bool OWN, int TEAM, int MODE>
__global__ __launch_bounds__(in_wave(TEAM) ? kRnThreads : TEAM) void rnorm_fwd_kernel(RnFwd a) {
    __shared__ float2 lds[in_wave(TEAM) ? 1 : 32];
    const int T = team_size<TEAM>();
    const int t = in_wave(TEAM) ? (int)threadIdx.x % T : (int)threadIdx.x;
    const int teams = in_wave(TEAM) ? kRnThreads / T : 1;
    const Cols<MODE> k(t, a.C);
    auto channels_of = [&](int wave) {
        const int n = a.C - wave * 64 * kRnEl;
        return (float)(n < 0 ? 0 : n < 64 * kRnEl ? n : 64 * kRnEl);
    };
    TeamSums ts{lds, (int)threadIdx.x >> 6, waves_of(a.C), 0, 0.0f, 0.0f};
    if (!in_wave(TEAM)) {
        ts.per_wave = 1.0f / channels_of((int)threadIdx.x >> 6);
        ts.in_lane = channels_of((int)threadIdx.x & 15);
    }
    const long lo = (long)blockIdx.x * a.rows_blk;
    const long hi = lo + a.rows_blk < a.rows ? lo + a.rows_blk : a.rows;
    long row = lo + (in_wave(TEAM) ? (int)threadIdx.x / T : 0);
    const Rows<YT> ys(a.y, a.ldy), gates(a.gate, a.ldg);
    const Rows<XT> xs(a.x, a.ldx);
    const f32x8 s = load_param<MODE>(a.s, 1.0f, k);
    const f32x8 A = load_param<MODE>(a.gp, 1.0f, k) * s;
    const f32x8 B = load_param<MODE>(a.bp, 0.0f, k) * s;
    const f32x8 gq = load_param<MODE>(a.gq, 1.0f, k);
    const f32x8 bq = load_param<MODE>(a.bq, 0.0f, k);
    f32x8 phi = splat(1.0f), slope;
    long until = -1;   // the row from which phi is that of another gate row
    typedef FwdRow<YT, XT, OWN, MODE> Row;
    auto load = [&](Row& r, long at) {
        r.y.load(ys[at], k);
        r.x.load(xs[at], k);
        if (OWN) r.gate.load(gates[at], k);
    };
    for_rows<Row>(row, hi, teams, load, [&](long row, const Row& now) {
        f32x8 y = now.y.value(), h = now.x.value();
        if (OWN) {
            gate8(now.gate.value(), a.act, phi, slope);
        } else if (a.gate_rows) {
            if (row >= until) {
                const long g = gate_row(row, a.gate_rows);
                gate8(load8<MODE>(gates[g], k), a.act, phi, slope);
                until = (g + 1) * a.gate_rows;
            }
        }
        float mean, rstd;
        if (a.post) {
            normalise<TEAM, MODE>(y, k, a.inv_c, a.eps, a.layer, mean, rstd, ts);
            if (a.stats && t == 0) {
                if (a.layer) a.stats[row] = mean;
                a.stats[a.rows + row] = rstd;
            }
        }
        h = fma8(fma8(y, A, B), phi, h);
        store8<MODE, store_all(TEAM, MODE)>(static_cast<XT*>(a.h) + row * a.ldh, k, h);
        if (a.pre) {
            normalise<TEAM, MODE>(h, k, a.inv_c, a.eps, a.layer, mean, rstd, ts);
            if (a.stats && t == 0) {
                if (a.layer) a.stats[2 * a.rows + row] = mean;
                a.stats[3 * a.rows + row] = rstd;
            }
            store8<MODE, store_all(TEAM, MODE)>(static_cast<YT*>(a.z) + row * a.ldz, k, fma8(h, gq, bq));
        }
    });
}

// ---- backward -----------------------------------------------------------------------------
// With D = dh + (norm backward of dz*gq at h), u = D*phi, yhat the normalised y:
//   dx = D;  dy = norm backward of u*s*gp at y;  dgate = phi' * sum_group D*s*(gp*yhat + bp)
//   dgq = sum dz*hhat, dbq = sum dz, dgp = s * sum u*yhat, dbp = s * sum u,
//   ds = gp * sum u*yhat + bp * sum u
// h is rebuilt in float32 from x and y, as forward had it before its rounding (with a gate shared by
// rows up to float32 roundings: phi is multiplied into the parameters here, once an item): the same
// bytes as reading the stored h, without its rounding in the gradients.  Four sums a channel stay in
// registers over an item's rows and go to the workspace once an item; a second launch folds the
// items in order in float64, so the results have the same bits on every call.  An item never
// crosses a gate row: phi is a constant of the item, which leaves its sums of D with phi (for the
// parameters) and without (for the gate).  A gate row for each row has its gradient in the loop.
template <typename YT, typename XT, bool OWN, int MODE>
struct BwdRow {
    Raw<YT, MODE> y, dz, gate;
    Raw<XT, MODE> x, dh;
    float py, ry, ph, rh;   // mean and rstd of y and of h
};

// Workgroups of more than 512 threads have 128 registers a thread: they keep the parameters in
// LDS, load no row ahead and leave the stores their branches (4000 x 8192 bf16 with a gate per row:
// 132 us; with all registers spilled that these cost 204).  In other workgroups the gate alone is
// taken again behind the sum, and bf16 is held to three waves a SIMD (10000 x 1400 with a gate per
// row 63 us when that was chosen, with two 72).
template <typename YT, typename XT, bool OWN, int TEAM, int MODE>
__global__ __launch_bounds__(in_wave(TEAM) ? kRnThreads : TEAM,
                             TEAM == 512 && sizeof(XT) == 2 ? 3 : 1) void rnorm_bwd_kernel(RnBwd a) {
    __shared__ float2 lds[in_wave(TEAM) ? 1 : 32];
    __shared__ float fold[in_wave(TEAM) ? kRnThreads / 64 : 1][4][in_wave(TEAM) ? TEAM * kRnEl : 1];
    constexpr bool WIDE = TEAM == 1024, ALL = !WIDE && store_all(TEAM, MODE);
    // The wave's number as the scalar it is where a register of each thread is one too many
    // (10000 x 1400 bf16 with a gate per row 60 us, with a reload in the loop 70).
    const int wave = OWN && !WIDE ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : (int)threadIdx.x >> 6;
    TeamSums ts{lds, wave, waves_of(a.C), 0, 0.0f, 0.0f};
    const int T = team_size<TEAM>();
    const int t = in_wave(TEAM) ? (int)threadIdx.x % T : (int)threadIdx.x;
    const int teams = in_wave(TEAM) ? kRnThreads / T : 1;
    const Cols<MODE> k(t, a.C);
    __shared__ f32x4 held[WIDE ? 6 : 1][WIDE ? 1024 : 1];   // each thread's own, no barrier
    const f32x8 s = load_param<MODE>(a.s, 1.0f, k);
    f32x8 A = load_param<MODE>(a.gp, 1.0f, k) * s;
    f32x8 B = load_param<MODE>(a.bp, 0.0f, k) * s;
    f32x8 gq = load_param<MODE>(a.gq, 1.0f, k);
    auto hold = [&](int i, f32x8 v) {
        held[2 * i][threadIdx.x] = v.lo;
        held[2 * i + 1][threadIdx.x] = v.hi;
    };
    auto held8 = [&](int i) {
        f32x8 v;
        v.lo = held[2 * i][threadIdx.x];
        v.hi = held[2 * i + 1][threadIdx.x];
        return v;
    };
    const long item = a.first + blockIdx.x;
    const long g = item / a.nseg;
    const long lo = g * a.group + (item - g * a.nseg) * a.rows_blk;
    const long end = (g + 1) * a.group;
    const long hi = lo + a.rows_blk < end ? lo + a.rows_blk : end;
    const bool shared = !OWN && a.gate_rows;
    const YT* item_gate = static_cast<const YT*>(a.gate) + g * a.ldg;   // of a shared gate
    f32x8 phi, slope;
    if (shared) {
        gate8(load8<MODE>(item_gate, k), a.act, phi, slope);
        A *= phi;
        B *= phi;
    }
    if (WIDE) {
        hold(0, A);
        hold(1, B);
        hold(2, gq);
    }
    f32x8 q1 = splat(0.0f), q0 = q1, p1 = q1, p0 = q1;
    long row = lo + (in_wave(TEAM) ? (int)threadIdx.x / T : 0);
    const Rows<YT> ys(a.y, a.ldy), dzs(a.pre ? a.dz : nullptr, a.lddz), gates(a.gate, a.ldg);
    const Rows<XT> xs(a.pre ? a.x : nullptr, a.ldx), dhs(a.dh, a.lddh);
    // the planes of the statistics, as rows of one element
    const Rows<float> pys(a.post && a.layer ? a.stats : nullptr, 1), rys(a.post ? a.stats + a.rows : nullptr, 1);
    const Rows<float> phs(a.pre && a.layer ? a.stats + 2 * a.rows : nullptr, 1);
    const Rows<float> rhs(a.pre ? a.stats + 3 * a.rows : nullptr, 1);
    typedef BwdRow<YT, XT, OWN, MODE> Row;
    auto load = [&](Row& r, long at) {
        r.y.load(ys[at], k);
        r.x.load(xs[at], k);
        r.dh.load(dhs[at], k);
        r.dz.load(dzs[at], k);
        if (OWN) r.gate.load(gates[at], k);
        r.py = *pys[at];
        r.ry = *rys[at];
        r.ph = *phs[at];
        r.rh = *rhs[at];
    };
    auto step = [&](long row, const Row& now) {
        f32x8 y = now.y.value(), d = now.dh.value();
        if (OWN) gate8(now.gate.value(), a.act, phi, slope);
        if (a.post) y = (y - now.py) * now.ry;
        if (a.pre) {
            if (WIDE) {
                A = held8(0);
                B = held8(1);
                gq = held8(2);
            }
            f32x8 w = now.dz.value(), h = fma8(y, A, B);
            h = OWN ? fma8(h, phi, now.x.value()) : now.x.value() + h;
            const f32x8 hhat = (h - now.ph) * now.rh;
            q0 += w;
            q1 = fma8(w, hhat, q1);
            w = w * gq;
            const f32x8 own_w = own<MODE>(w, k);
            float m1 = sum8(own_w, k), m2 = dot8(own_w, hhat, k);
            team_sum2<TEAM>(m1, m2, ts);
            m1 = a.layer ? m1 * a.inv_c : 0.0f;
            m2 *= a.inv_c;
            d = fma8(fma8(hhat, splat(-m2), w - m1), splat(now.rh), d);
        }
        if (a.dx) store8<MODE, ALL>(static_cast<XT*>(a.dx) + row * a.lddx, k, d);
        if (WIDE) A = held8(0);
        if (OWN) {
            if (WIDE) B = held8(1);
            if (!in_wave(TEAM)) {   // again, rather than kept over the sum
                Raw<YT, MODE> gate = now.gate;
                gate.forget();
                gate8(gate.value(), a.act, phi, slope);
            }
            store8<MODE, ALL>(static_cast<YT*>(a.dgate) + row * a.lddg, k, d * fma8(y, A, B) * slope);
            d *= phi;
        }
        p0 += d;
        p1 = fma8(d, y, p1);
        f32x8 w = d * A;
        if (a.post) {
            const f32x8 own_w = own<MODE>(w, k);
            float n1 = sum8(own_w, k), n2 = dot8(own_w, y, k);
            team_sum2<TEAM>(n1, n2, ts);
            n1 = a.layer ? n1 * a.inv_c * now.ry : 0.0f;
            n2 *= a.inv_c * now.ry;
            w = fma8(y, splat(-n2), fma8(w, splat(now.ry), splat(-n1)));
        }
        store8<MODE, ALL>(static_cast<YT*>(a.dy) + row * a.lddy, k, w);
    };
    if (WIDE) {
        for (; row < hi; row += teams) {
            Row now;
            load(now, row);
            step(row, now);
        }
    } else {
        for_rows<Row>(row, hi, teams, load, step);
    }
    if (!a.need) return;
    const bool direct = a.part == nullptr;
    float* out = direct ? nullptr : a.part + item * slots_of(a.gate_rows) * a.pitch;
    if (in_wave(TEAM)) {
        // rows side by side in the wave, then the waves in order
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x8 sums = i == 0 ? q1 : i == 1 ? q0 : i == 2 ? p1 : p0;
            if (a.need & ((1 << i) | (i >= 2 ? 4 << i : 0))) {
#pragma unroll
                for (int j = 0; j < kRnEl; ++j) {
                    float v = sums[j];
#pragma unroll
                    for (int off = 32; off >= (in_wave(TEAM) ? TEAM : 64); off >>= 1)
                        v += __shfl_xor(v, off, 64);
                    if ((int)(threadIdx.x & 63) < T && k.mine(j)) fold[threadIdx.x >> 6][i][k.c + j] = v;
                }
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += kRnThreads) {
            float f = 1.0f, unused;
            if (shared) f = gate_value(as_float(item_gate[c]), a.act, unused);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool weighted = a.need & (1 << i), plain = i >= 2 && (a.need & (4 << i));
                if (weighted || plain) {
                    float v = fold[0][i][c];
#pragma unroll
                    for (int wv = 1; wv < kRnThreads / 64; ++wv) v += fold[wv][i][c];
                    sum[i] = v;
                    if (weighted && !direct) out[(long)i * a.pitch + c] = i >= 2 ? v * f : v;
                    if (plain && !direct) out[(long)(i + 2) * a.pitch + c] = v;
                }
            }
            if (direct) {
                const float sc = a.s ? a.s[c] : 1.0f;
                if (a.dgq) a.dgq[c] = sum[0];
                if (a.dbq) a.dbq[c] = sum[1];
                if (a.dgp) a.dgp[c] = sc * sum[2];
                if (a.dbp) a.dbp[c] = sc * sum[3];
                if (a.ds) a.ds[c] = (a.gp ? a.gp[c] : 1.0f) * sum[2] + (a.bp ? a.bp[c] * sum[3] : 0.0f);
            }
        }
    } else if (direct) {
        if (a.dgq) store8<MODE>(a.dgq, k, q1);
        if (a.dbq) store8<MODE>(a.dbq, k, q0);
        const f32x8 sc = load_param<MODE>(a.s, 1.0f, k);
        if (a.dgp) store8<MODE>(a.dgp, k, sc * p1);
        if (a.dbp) store8<MODE>(a.dbp, k, sc * p0);
        if (a.ds) {
            f32x8 v = load_param<MODE>(a.gp, 1.0f, k) * p1;
            if (a.bp) v += load8<MODE>(a.bp, k) * p0;
            store8<MODE>(a.ds, k, v);
        }
    } else {
        f32x8 f = splat(1.0f);
        if (shared) gate8(load8<MODE>(item_gate, k), a.act, f, slope);
        if (a.need & kQ1) store8<MODE>(out, k, q1);
        if (a.need & kQ0) store8<MODE>(out + a.pitch, k, q0);
        if (a.need & kP1) store8<MODE>(out + 2l * a.pitch, k, p1 * f);
        if (a.need & kP0) store8<MODE>(out + 3l * a.pitch, k, p0 * f);
        if (a.need & kG1) store8<MODE>(out + 4l * a.pitch, k, p1);
        if (a.need & kG0) store8<MODE>(out + 5l * a.pitch, k, p0);
    }
}

// ---- fold of the items --------------------------------------------------------------------
// Latency is all there is to it: a few MB that were just written.  A workgroup takes 32 channels
// (a 128-byte line of every row of sums), a thread four of them of every 32nd item, with the
// loads of several items under way at a time; float64 sums in an order fixed by the sizes.
// Workgroups of one launch have one of two tasks: a gate row's gradient from its own items, or
// the parameters' from all of them (whose sums phi weights already).
constexpr int kFoldCols = 32;
constexpr int kFoldLanes = 32;                        // items side by side
constexpr int kFoldThreads = kFoldLanes * kFoldCols / 4;
// Items that one workgroup of the parameters folds.  Past it (a gate row for every few rows of a
// long tensor) kFoldSlices of them leave their sums behind the items for a second launch.
constexpr long kFoldItems = 4096;
constexpr int kFoldSlices = 64;
typedef double f64x4 __attribute__((ext_vector_type(4)));

struct RnFold {
    float* part;
    long items, nseg;                // items in all and of a gate row
    long first;                      // gate row of the grid's first
    int gates, slices;               // tasks of the grid: gate rows, then slices of the parameters
    const float *gp, *bp, *s, *any;
    const void* gate;
    void* dgate;
    float *dgp, *dbp, *ds, *dgq, *dbq;
    long ldg, lddg;
    int C, act, pitch, need, slots;
};

// sum[k] of channel c = sum over lo <= i < hi of part[i][slot + k][c], k < K, in the first
// kFoldCols threads, whose channel is the block's first plus their index.
template <int K>
__device__ __forceinline__ void fold_items(const RnFold& a, long lo, long hi, int slot, double (&sum)[4]) {
    constexpr int QUADS = kFoldCols / 4;
    constexpr int WAVES = kFoldThreads / 64;
    constexpr int AT_ONCE = 4;
    static_assert(QUADS == 8, "the sums over a wave's lanes");
    __shared__ double lds[WAVES][4][kFoldCols];
    const int need = a.need >> slot;
    const int quad = (int)threadIdx.x % QUADS, lane = (int)threadIdx.x / QUADS;
    const int c = (int)blockIdx.x * kFoldCols + quad * 4;
    f64x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = f64x4{0.0, 0.0, 0.0, 0.0};
    if (c < a.pitch) {
        // A branch around a load would make the thread wait for each in turn: items past the end
        // read the last one again and count as 0, sums that nothing needs read one that is.
        const long jump = (long)a.slots * a.pitch;
        const int any = __builtin_ctz(need);
        long at[K];
#pragma unroll
        for (int k = 0; k < K; ++k) at[k] = (long)(slot + ((need & (1 << k)) ? k : any)) * a.pitch + c;
        for (long i = lo + lane; i < hi; i += AT_ONCE * kFoldLanes) {
            f32x4 r[AT_ONCE][K];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const float* q = a.part + (i + u * kFoldLanes < hi ? i + u * kFoldLanes : hi - 1) * jump;
#pragma unroll
                for (int k = 0; k < K; ++k) r[u][k] = *reinterpret_cast<const f32x4*>(q + at[k]);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const bool in = i + u * kFoldLanes < hi;
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[k][j] += (double)(in ? r[u][k][j] : 0.0f);
                }
            }
        }
    }
    // a wave's eight items into one: each step leaves half of the sums to half of the lanes; the
    // last adds the lane eight further in its row of 16
    const int l = (int)threadIdx.x & 63, k = 2 * ((l >> 4) & 1) + (l >> 5);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        double x = v[0][j], x2 = v[1][j], y = v[2][j], y2 = v[3][j];
        swap_halves(x, x2);
        swap_halves(y, y2);
        x += x2;
        y += y2;
        swap_rows(x, y);
        x += y;
        const double u = x + lane_move<kEight>(x);
        if ((l & 15) < QUADS) lds[threadIdx.x >> 6][k][quad * 4 + j] = u;
    }
    __syncthreads();
    if (threadIdx.x < kFoldCols) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            sum[k] = lds[0][k][threadIdx.x];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum[k] += lds[w][k][threadIdx.x];
            if (!(need & (1 << k))) sum[k] = 0.0;
        }
    }
}

template <typename YT, bool GROUPED>
__global__ __launch_bounds__(kFoldThreads) void rnorm_fold_kernel(RnFold a) {
    const int c = (int)blockIdx.x * kFoldCols + (int)threadIdx.x;
    const bool mine = threadIdx.x < kFoldCols && c < a.C;
    const int at = mine ? c : 0;
    // the channel's parameters, asked for before the sums; an absent one reads a.any
    float gp = *(a.gp ? a.gp + at : a.any), bp = *(a.bp ? a.bp + at : a.any);
    float s = *(a.s ? a.s + at : a.any);
    double v[4];
    if (GROUPED && (int)blockIdx.y < a.gates) {
        const long g = a.first + blockIdx.y;
        const YT raw = static_cast<const YT*>(a.gate)[g * a.ldg + at];
        fold_items<2>(a, g * a.nseg, (g + 1) * a.nseg, 4, v);
        if (!mine) return;
        if (!a.gp) gp = 1.0f;
        if (!a.bp) bp = 0.0f;
        if (!a.s) s = 1.0f;
        float slope;
        gate_value(as_float(raw), a.act, slope);
        const float dg = (float)((double)slope * s * ((double)gp * v[0] + (double)bp * v[1]));
        if (sizeof(YT) == 4) {
            static_cast<float*>(a.dgate)[g * a.lddg + c] = dg;
        } else {
            static_cast<uint16_t*>(a.dgate)[g * a.lddg + c] = (uint16_t)float_to_bf16_bits(dg);
        }
        return;
    }
    const int slice = (int)blockIdx.y - a.gates;
    const long per = (a.items + a.slices - 1) / a.slices;
    const long lo = slice * per, hi = lo + per < a.items ? lo + per : a.items;
    fold_items<4>(a, lo, hi, 0, v);
    if (!mine) return;
    if (a.slices > 1) {
        float* p = a.part + a.items * a.slots * a.pitch + slice * 4l * a.pitch + c;
#pragma unroll
        for (int k = 0; k < 4; ++k) p[(long)k * a.pitch] = (float)v[k];
        return;
    }
    if (!a.gp) gp = 1.0f;
    if (!a.bp) bp = 0.0f;
    if (!a.s) s = 1.0f;
    if (a.dgq) a.dgq[c] = (float)v[0];
    if (a.dbq) a.dbq[c] = (float)v[1];
    if (a.dgp) a.dgp[c] = (float)((double)s * v[2]);
    if (a.dbp) a.dbp[c] = (float)((double)s * v[3]);
    if (a.ds) a.ds[c] = (float)((double)gp * v[2] + (double)bp * v[3]);
}

// ---- host ---------------------------------------------------------------------------------
static int team_of(int C) {
    const int need = (C + kRnEl - 1) / kRnEl;
    if (C < kRnEl) return 8;   // a channel a thread
    for (int t = 1; t <= 64; t *= 2)
        if (need <= t) return t;
    return need <= 512 ? 512 : 1024;
}

static unsigned block_of(int C) {   // threads of a workgroup
    return in_wave(team_of(C)) ? kRnThreads : 64u * waves_of(C);
}

static long rows_at_once(int C) { return in_wave(team_of(C)) ? kRnThreads / team_of(C) : 1; }

struct BwdGeom {
    long groups, group, nseg, rows_blk;
    long items() const { return groups * nseg; }
    bool direct;   // one item, which writes the parameters' gradients: no fold, no workspace
};

static int pitch_of(int C) { return (C + 3) & ~3; }   // of a row of sums: 16-byte steps

// None across a gate row, each a multiple of the rows its teams take at once.
static BwdGeom bwd_geom(const pe_rnorm_desc& d) {
    BwdGeom g;
    const bool grouped = d.gate_rows > 1;
    g.group = grouped ? d.gate_rows : d.rows;
    g.groups = grouped ? d.rows / d.gate_rows : 1;
    const long at_once = rows_at_once(d.C);
    const int waves = waves_of(d.C);   // 1: rows inside a wave
    long want = waves > 6 ? kRnUnits : 2 * kRnUnits;
    if (waves == 2 && d.rows / 8 > want) want = d.rows / 8 < 4 * kRnUnits ? d.rows / 8 : 4 * kRnUnits;
    want = (want + g.groups - 1) / g.groups;
    long rows = (g.group + want - 1) / want;
    rows = (rows + at_once - 1) / at_once * at_once;
    if (rows < 1) rows = 1;
    g.rows_blk = rows;
    // One workgroup and no fold while its rows cost less: 4 for each team inside a wave (32 x 256:
    // 7.5 us; 33 rows by items and fold 8.4, and a launch more for the host), 2 for a workgroup
    // (2 x 4096: 7.1; by items 4 rows 8.4), 1 past 4096 channels.
    const int team = team_of(d.C);
    g.direct = !grouped && d.rows <= (in_wave(team) ? 4 * at_once : team == 512 ? 2 : 1);
    if (g.direct) g.rows_blk = d.rows;
    g.nseg = (g.group + g.rows_blk - 1) / g.rows_blk;
    return g;
}

static bool element_aligned(int dtype, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (!aligned(p, dtype == PE_DTYPE_F32 ? 4 : 2)) return false;
    return true;
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
    PE_REQUIRE(d->eps >= FLT_MIN && isfinite(d->eps), PE_E_INVALID,
               "%s: eps must be positive and a normal number", what);
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

// Calls F<TEAM, MODE>::go(args) for C channels.
template <template <int, int> class F, class... A>
static void with_team(int C, A&&... a) {
    if (C < kRnEl) return F<8, FEW>::go(a...);
    const bool whole = C % kRnEl == 0;
    switch (team_of(C)) {
        case 1: return F<1, WHOLE>::go(a...);   // eight channels
        case 2: return whole ? F<2, WHOLE>::go(a...) : F<2, TAIL>::go(a...);
        case 4: return whole ? F<4, WHOLE>::go(a...) : F<4, TAIL>::go(a...);
        case 8: return whole ? F<8, WHOLE>::go(a...) : F<8, TAIL>::go(a...);
        case 16: return whole ? F<16, WHOLE>::go(a...) : F<16, TAIL>::go(a...);
        case 32: return whole ? F<32, WHOLE>::go(a...) : F<32, TAIL>::go(a...);
        case 64: return whole ? F<64, WHOLE>::go(a...) : F<64, TAIL>::go(a...);
        case 512: return whole ? F<512, WHOLE>::go(a...) : F<512, TAIL>::go(a...);
        default: return whole ? F<1024, WHOLE>::go(a...) : F<1024, TAIL>::go(a...);
    }
}

template <typename YT, typename XT, bool OWN>
struct FwdOf {
    template <int TEAM, int MODE>
    struct F {
        static void go(const RnFwd& a, unsigned blocks, hipStream_t st) {
            launch(rnorm_fwd_kernel<YT, XT, OWN, TEAM, MODE>, blocks, block_of(a.C), 0, st, a);
        }
    };
};

template <typename YT, typename XT, bool OWN>
struct BwdOf {
    template <int TEAM, int MODE>
    struct F {
        // A grid holds less than 2^32 threads: short runs of a shared gate take more than one.
        static void go(RnBwd a, long items, hipStream_t st) {
            const unsigned threads = block_of(a.C);
            const long most = 0xffffffffl / threads;
            for (a.first = 0; a.first < items; a.first += most) {
                const unsigned blocks = (unsigned)(items - a.first < most ? items - a.first : most);
                launch(rnorm_bwd_kernel<YT, XT, OWN, TEAM, MODE>, blocks, threads, 0, st, a);
            }
        }
    };
};

template <typename YT, typename XT>
static void launch_bwd(const RnBwd& a, long items, hipStream_t st) {
    if (a.gate_rows == 1) {
        with_team<BwdOf<YT, XT, true>::template F>(a.C, a, items, st);
    } else {
        with_team<BwdOf<YT, XT, false>::template F>(a.C, a, items, st);
    }
}

template <typename YT, typename XT>
static void launch_fwd(const RnFwd& a, unsigned blocks, hipStream_t st) {
    if (a.gate_rows == 1) {
        with_team<FwdOf<YT, XT, true>::template F>(a.C, a, blocks, st);
    } else {
        with_team<FwdOf<YT, XT, false>::template F>(a.C, a, blocks, st);
    }
}

// Gate rows (65535 tasks a grid at most) and the parameters in one launch where their items allow.
template <typename YT>
static void launch_fold(RnFold f, bool grouped, long groups, bool params, hipStream_t st) {
    const unsigned tiles = (unsigned)((f.C + kFoldCols - 1) / kFoldCols);
    const int slices = !params ? 0 : f.items > kFoldItems ? kFoldSlices : 1;
    f.slices = slices > 1 ? slices : 1;
    if (!grouped) {
        f.gates = 0;
        launch(rnorm_fold_kernel<YT, false>, tiles, kFoldThreads, 0, st, f);
        return;
    }
    for (f.first = 0; f.first < groups; f.first += f.gates) {
        f.gates = (int)(groups - f.first < 60000 ? groups - f.first : 60000);
        const unsigned more = f.first == 0 ? (unsigned)slices : 0;
        launch(rnorm_fold_kernel<YT, true>, dim3(tiles, (unsigned)f.gates + more), kFoldThreads, 0, st, f);
    }
    if (slices > 1) {
        f.part += f.items * f.slots * f.pitch;
        f.items = slices;
        f.slots = 4;
        f.slices = 1;
        f.gates = 0;
        launch(rnorm_fold_kernel<YT, false>, tiles, kFoldThreads, 0, st, f);
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
    PE_REQUIRE((d->post || !(post_gamma || post_beta)) && (d->pre || !(pre_gamma || pre_beta || z)),
               PE_E_INVALID, "pe_rnorm_fwd: operands of a norm that is off");
    PE_REQUIRE(element_aligned(d->y_dtype, {y, gate, z}) && element_aligned(d->x_dtype, {x, h}) &&
                   element_aligned(PE_DTYPE_F32, {post_gamma, post_beta, scale, pre_gamma, pre_beta, stats}),
               PE_E_INVALID, "pe_rnorm_fwd: a pointer between two elements");
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
    // Workgroups of equal shares, each of which loads the parameters once.  Rows inside a wave:
    // 4096 of them (196608 x 256 bf16 76 us, with 1024 82; 70000 x 512 46, 48), or 1024 where the width
    // is no multiple of eight (60000 x 333: 33 us, with 4096 38; 20000 x 333 12, 15).  A row to a
    // workgroup: whole rounds of what the chip holds at once, four (8192 x 4096 with a float32
    // residual, rms: 90 us, with two 94), or two or one where the parameters would be over half of
    // the bytes.
    const long at_once = rows_at_once(d->C);
    const long shares = d->C % kRnEl == 0 ? 4096 : 1024;
    long rows = (d->rows + shares - 1) / shares;
    if (!in_wave(team_of(d->C))) {
        const long per_cu = (d->x_dtype == PE_DTYPE_F32 ? 16 : 20) / waves_of(d->C);   // by registers
        const long round = 256 * (per_cu > 1 ? per_cu : 1);
        const long yb = d->y_dtype == PE_DTYPE_F32 ? 4 : 2, xb = d->x_dtype == PE_DTYPE_F32 ? 4 : 2;
        const long params = 4 * ((post_gamma != nullptr) + (post_beta != nullptr) + (scale != nullptr) +
                                 (pre_gamma != nullptr) + (pre_beta != nullptr));
        const long row = yb + xb + (x ? xb : 0) + (d->pre ? yb : 0) + (d->gate_rows == 1 ? yb : 0);
        long rounds = 4;
        do {
            rows = (d->rows + rounds * round - 1) / (rounds * round);
            rounds /= 2;
        } while (rounds && rows * row < 2 * params);
    }
    rows = (rows + at_once - 1) / at_once * at_once;
    a.rows_blk = rows;
    const unsigned blocks = (unsigned)((d->rows + rows - 1) / rows);
    if (d->y_dtype == PE_DTYPE_F32) {
        launch_fwd<float, float>(a, blocks, as_stream(stream));
    } else if (d->x_dtype == PE_DTYPE_F32) {
        launch_fwd<uint16_t, float>(a, blocks, as_stream(stream));
    } else {
        launch_fwd<uint16_t, uint16_t>(a, blocks, as_stream(stream));
    }
    return check_launch("pe_rnorm_fwd");
}

extern "C" size_t pe_rnorm_bwd_workspace_bytes(const pe_rnorm_desc* d) {
    if (pe::check_desc("pe_rnorm_bwd_workspace_bytes", d) != PE_OK) return 0;
    if (d->rows == 0) return 0;
    const pe::BwdGeom g = pe::bwd_geom(*d);
    if (g.direct) return 0;
    const long items = g.items();
    const long slices = items > pe::kFoldItems ? pe::kFoldSlices : 0;
    return sizeof(float) * (size_t)pe::pitch_of(d->C) *
           (size_t)(items * pe::slots_of(d->gate_rows) + 4 * slices);
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
    PE_REQUIRE((d->post || !(post_gamma || post_beta || dpost_gamma || dpost_beta)) &&
                   (d->pre || !(pre_gamma || dpre_gamma || dpre_beta || dz)),
               PE_E_INVALID, "pe_rnorm_bwd: operands of a norm that is off");
    PE_REQUIRE(element_aligned(d->y_dtype, {dz, y, gate, dy, dgate}) &&
                   element_aligned(d->x_dtype, {dh, x, dx}) &&
                   element_aligned(PE_DTYPE_F32, {stats, post_gamma, post_beta, scale, pre_gamma, dpost_gamma,
                                                  dpost_beta, dscale, dpre_gamma, dpre_beta}),
               PE_E_INVALID, "pe_rnorm_bwd: a pointer between two elements");
    const bool grouped = d->gate_rows > 1;
    const bool sums = dpost_gamma || dpost_beta || dscale || dpre_gamma || dpre_beta;
    const int need = (dpre_gamma ? kQ1 : 0) | (dpre_beta ? kQ0 : 0) | (dpost_gamma || dscale ? kP1 : 0) |
                     (dpost_beta || (dscale && post_beta) ? kP0 : 0) | (grouped ? kG1 : 0) |
                     (grouped && post_beta ? kG0 : 0);
    BwdGeom g{0, 0, 0, 0, false};
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
        if (need && !g.direct) {
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
        a.part = g.direct ? nullptr : static_cast<float*>(workspace);
        a.dgp = dpost_gamma;
        a.dbp = dpost_beta;
        a.ds = dscale;
        a.dgq = dpre_gamma;
        a.dbq = dpre_beta;
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
        const long items = g.items();
        if (yd == PE_DTYPE_F32) {
            launch_bwd<float, float>(a, items, as_stream(stream));
        } else if (xd == PE_DTYPE_F32) {
            launch_bwd<uint16_t, float>(a, items, as_stream(stream));
        } else {
            launch_bwd<uint16_t, uint16_t>(a, items, as_stream(stream));
        }
    }
    if (g.direct || (!sums && !(grouped && d->rows))) return check_launch("pe_rnorm_bwd");
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
    f.items = g.items();
    f.nseg = g.nseg;
    f.C = d->C;
    f.act = d->gate_act;
    f.pitch = pitch_of(d->C);
    f.need = need;
    f.slots = slots_of(d->gate_rows);
    f.ldg = d->ldgate;
    f.lddg = d->lddgate;
    if (d->y_dtype == PE_DTYPE_F32) {
        launch_fold<float>(f, grouped && d->rows, g.groups, sums, as_stream(stream));
    } else {
        launch_fold<uint16_t>(f, grouped && d->rows, g.groups, sums, as_stream(stream));
    }
    return check_launch("pe_rnorm_bwd");
}
