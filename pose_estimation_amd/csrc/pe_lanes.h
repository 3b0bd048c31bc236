// Sums over the lanes of a wave by data-parallel moves inside the vector unit, without the round
// trips through LDS that shuffles take (gfx950).
#pragma once

#include "pe_common.h"

#ifdef __HIPCC__
namespace pe {

// The value of another lane: lane ^ 1 and lane ^ 2 inside a quad; the mirror image inside 8 and
// inside 16 lanes (lane ^ 4 and lane ^ 8 once quads, then eights, agree); the lane eight further in
// its row of 16.
enum { kXor1 = 0xB1, kXor2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140, kEight = 0x128 };

template <int CTRL>
__device__ __forceinline__ unsigned lane_move(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return __uint_as_float(lane_move<CTRL>(__float_as_uint(v)));
}
__device__ __forceinline__ double join64(unsigned lo, unsigned hi) {
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
template <int CTRL>
__device__ __forceinline__ double lane_move(double v) {
    const unsigned long long x = __double_as_longlong(v);
    return join64(lane_move<CTRL>((unsigned)x), lane_move<CTRL>((unsigned)(x >> 32)));
}

// Exchanges the odd rows of 16 lanes of a with the even rows of b; the upper half of a with the
// lower half of b.  Afterwards the pair's combination is that of a's two parts in one place and of
// b's in the other (of a in both when a = b).
__device__ __forceinline__ void swap_rows(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap_halves(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap_rows(double& a, double& b) {
    const unsigned long long x = __double_as_longlong(a), y = __double_as_longlong(b);
    const auto lo = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)y, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((unsigned)(x >> 32), (unsigned)(y >> 32), false, false);
    a = join64(lo[0], hi[0]);
    b = join64(lo[1], hi[1]);
}
__device__ __forceinline__ void swap_halves(double& a, double& b) {
    const unsigned long long x = __double_as_longlong(a), y = __double_as_longlong(b);
    const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)y, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap((unsigned)(x >> 32), (unsigned)(y >> 32), false, false);
    a = join64(lo[0], hi[0]);
    b = join64(lo[1], hi[1]);
}

// op over each group of W lanes (1 to 64), the same bits in every lane of the group; op(a, b) has
// to give what op(b, a) gives.
template <int W, typename T, typename OP>
__device__ __forceinline__ T lanes_all(T v, OP op) {
    if (W >= 2) v = op(v, lane_move<kXor1>(v));
    if (W >= 4) v = op(v, lane_move<kXor2>(v));
    if (W >= 8) v = op(v, lane_move<kMirror8>(v));
    if (W >= 16) v = op(v, lane_move<kMirror16>(v));
    if (W >= 32) {
        T w = v;
        swap_rows(v, w);
        v = op(v, w);
    }
    if (W >= 64) {
        T w = v;
        swap_halves(v, w);
        v = op(v, w);
    }
    return v;
}

template <int W, typename T>
__device__ __forceinline__ T lanes_sum(T v) {
    return lanes_all<W>(v, [](T a, T b) { return a + b; });
}

}  // namespace pe
#endif
