// angles.hpp -- sine and cosine of rotary positions.
#pragma once

#include <hip/hip_runtime.h>

namespace bmo {

// Sine and cosine of a (|a| < 2^31) in double, about 1e-16 off: Cody and
// Waite's reduction by multiples of pi/2 in three parts (the first fma is
// exact: a and k pi1 are multiples of 2^-52, their difference below 1), then
// Taylor polynomials on [-pi/4, pi/4], whose first omitted terms are below
// 1e-18.  Every lane takes the same instructions: the general library
// function with its large-argument branch held RoPE's first group back by
// 0.6 us a launch at B = 1.
__device__ __forceinline__ void sincos_reduced(double a, double &sn, double &cs) {
    const double k = __builtin_rint(a * 0.6366197723675814);  // 2 / pi
    double r = __builtin_fma(-k, 1.5707963267948966, a);
    r = __builtin_fma(-k, 6.123233995736766e-17, r);
    r = __builtin_fma(k, 1.4973849048591833e-33, r);
    const double z = r * r;
    constexpr double S[8] = {-1.0 / 6.0, 1.0 / 120.0, -1.0 / 5040.0, 1.0 / 362880.0, -1.0 / 39916800.0,
                             1.0 / 6227020800.0, -1.0 / 1307674368000.0, 1.0 / 355687428096000.0};
    constexpr double C[8] = {1.0 / 24.0, -1.0 / 720.0, 1.0 / 40320.0, -1.0 / 3628800.0, 1.0 / 479001600.0,
                             -1.0 / 87178291200.0, 1.0 / 20922789888000.0, -1.0 / 6402373705728000.0};
    double ps = S[7], pc = C[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) {
        ps = __builtin_fma(ps, z, S[i]);
        pc = __builtin_fma(pc, z, C[i]);
    }
    const double s0 = __builtin_fma(r * z, ps, r);
    const double c0 = __builtin_fma(z, __builtin_fma(z, pc, -0.5), 1.0);
    const int q = (int) k;
    sn = q & 1 ? c0 : s0;
    cs = q & 1 ? s0 : c0;
    sn = q & 2 ? -sn : sn;
    cs = (q + 1) & 2 ? -cs : cs;
}

// (a, b) rotated by (c, s) = tab entry, every product and sum rounded.
__device__ __forceinline__ void rope_pair(float &a, float &b, float2 cs) {
    const float ac = a * cs.x, bs = b * cs.y, as = a * cs.y, bc = b * cs.x;
    a = ac - bs;
    b = as + bc;
}

}  // namespace bmo
