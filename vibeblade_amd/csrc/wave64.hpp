// 64-bit arithmetic across a wave, and 2^x in 64 bits, for the ops whose
// results are ids: where two sums or two scores decide which of two ids comes
// first, fp32's last bits would decide it by the order of the additions.
#pragma once

#include "vb_common.hpp"

namespace vb {

// 2^x for x up to 1023, 2^-1021 for all x below, relative error below 2^-51: 2^n
// times the Chebyshev interpolation of 2^f, f = x - n in [-1/2, 1/2], at eleven
// points, whose error is 2 (ln 2 / 4)^11 / 11! = 2.2e-16.  The nearest integer n
// is what x + 3 * 2^51 is rounded to and stands in that sum's low bits, and 2^n is
// n added to the exponent.  NaN is not kept.
constexpr double EXP2_LEAST = -1021.0;
struct Exp2 {
    double c10, c9, c8, c7, c6, c5, c4, c3, c2, c1;
    // In scalar registers, and the compiler does not know them: a fma takes one of
    // them as it is, where a known constant is first moved to vector registers (five
    // instructions more a logit in the draft verification, whose 64-bit terms bound
    // it as much as memory does).
    __device__ __forceinline__ Exp2()
        : c10(0x1.e6063f7217bc7p-28), c9(0x1.b675bca4eeebbp-24), c8(0x1.62bfd47773353p-20), c7(0x1.ffcb54062e698p-17),
          c6(0x1.430913096fd9fp-13), c5(0x1.5d87fe9d7a584p-10), c4(0x1.3b2ab6fba1ddap-7), c3(0x1.c6b08d703ce49p-5),
          c2(0x1.ebfbdff82c598p-3), c1(0x1.62e42fefa3a19p-1) {
        asm("" : "+s"(c10), "+s"(c9), "+s"(c8), "+s"(c7), "+s"(c6), "+s"(c5), "+s"(c4), "+s"(c3), "+s"(c2), "+s"(c1));
    }
    __device__ __forceinline__ double normal(double x) const {
        x = fmax(x, EXP2_LEAST);
        const double shifted = x + 0x1.8p52, f = x - (shifted - 0x1.8p52);
        double p = __builtin_fma(c10, f, c9);
        p = __builtin_fma(p, f, c8);
        p = __builtin_fma(p, f, c7);
        p = __builtin_fma(p, f, c6);
        p = __builtin_fma(p, f, c5);
        p = __builtin_fma(p, f, c4);
        p = __builtin_fma(p, f, c3);
        p = __builtin_fma(p, f, c2);
        p = __builtin_fma(p, f, c1);
        p = __builtin_fma(p, f, 1.0);
        return __hiloint2double(__double2hiint(p) + (__double2loint(shifted) << 20), __double2loint(p));
    }
    // 2^x for x up to 1023, 0 below -1021.
    __device__ __forceinline__ double operator()(double x) const {
        const double p = normal(x);
        return x < EXP2_LEAST ? 0.0 : p;
    }
};

// v of the lane that CTRL names, of the rows of 16 lanes in ROWS; v itself in
// the others.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ float dpp_or_self(float v) {
    const int i = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp_or_self(double v) {
    const int lo = __double2loint(v), hi = __double2hiint(v);
    return __hiloint2double(__builtin_amdgcn_update_dpp(hi, hi, CTRL, ROWS, 0xF, false),
                            __builtin_amdgcn_update_dpp(lo, lo, CTRL, ROWS, 0xF, false));
}

__device__ __forceinline__ float lane_value(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ double lane_value(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                            __builtin_amdgcn_readlane(__double2loint(v), lane));
}

__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

// The largest value of a wave, in every lane (a NaN is passed over).
template <typename T>
__device__ __forceinline__ T wave_largest(T v) {
    v = larger(v, dpp_or_self<0xB1>(v));         // quad_perm [1,0,3,2]
    v = larger(v, dpp_or_self<0x4E>(v));         // quad_perm [2,3,0,1]
    v = larger(v, dpp_or_self<0x141>(v));        // row_half_mirror
    v = larger(v, dpp_or_self<0x140>(v));        // row_mirror
    v = larger(v, dpp_or_self<0x142, 0xA>(v));   // row_bcast:15 into rows 1, 3
    v = larger(v, dpp_or_self<0x143, 0xC>(v));   // row_bcast:31 into rows 2, 3
    return lane_value(v, 63);
}

// The sum of a wave, in every lane.
__device__ __forceinline__ double wave_sum64(double v) {
    v += dpp_or_self<0xB1>(v);
    v += dpp_or_self<0x4E>(v);
    v += dpp_or_self<0x141>(v);
    v += dpp_or_self<0x140>(v);
    // rows hold their sums in every lane: rows 0 + 1 and 2 + 3, then both
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}

}  // namespace vb
