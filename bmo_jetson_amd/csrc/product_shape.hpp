// product_shape.hpp -- which kernel a product of 8-bit rows with Q4_0 weights
// takes (weights.hip).  Plain C++, so that a host test can walk the rule.
#pragma once

#include <stdint.h>

namespace bmo {

// A workgroup takes `rows` rows and `outs` outputs (gates, of a gated product);
// `waves` waves share each piece of it along the columns, a step each a unit of
// 128.  A CU runs `resident` of them at a time.  Times of a call in us: start +
// steps * (those of the fullest CU's workgroups, `resident` at a time: alone, or
// shared for each where that is more).
struct ProductShape {
    int rows, outs, waves, resident;
    double start, alone, shared;
};

// Few rows (16 x 16 matrix instructions) and many (32 x 32).  The times are
// fitted to calls with weights from HBM, 2 to 3000 rows by 512 to 32001 outputs
// of 640 to 11264 columns (gated: 2048 rows by 512 to 11264 outputs of 640 to
// 8192), and moved by up to 15% to where they choose best.  Against the fastest
// of 13 shapes (8 gated) the choice costs 1.6% in the mean over the 162 calls, 18%
// at worst (32 rows x 11264 outputs x 640: 6.4 us, 5.4 with 32 x 32); gated 0.4%
// over 80, 9% at worst.  What a shape is worth: 16 x 16 at 2 x 512 x 4096 3.5 us,
// 16 x 32 there 5.8; 16 x 64 at 64 x 4096 x 4096 8.1, 32 x 32 there 9.2; 64 x 128
// with two waves to a piece at 1500 x 11264 x 4096 203, 64 x 256 there 223, at 2048
// x 12288 x 4096 274 and 257.  Both read a unit's weights once for 64 rows; 128 x
// 128 takes 226 and 265, for its workgroups fill fewer last rounds.
constexpr ProductShape kProductShapes[] = {
    {16, 16, 8, 1, 2.45, 0.76, 0},    {16, 32, 8, 1, 2.96, 1.05, 0},    {16, 64, 8, 1, 2.61, 1.58, 0},
    {32, 32, 4, 3, 3.30, 0.80, 0.62}, {32, 64, 4, 2, 4.41, 1.21, 0.99}, {32, 128, 2, 2, 4.20, 1.13, 0.93},
    {64, 128, 2, 2, 7.01, 1.81, 1.47}, {64, 256, 1, 2, 9.10, 2.05, 1.18},
};
constexpr ProductShape kGatedShapes[] = {
    {16, 32, 8, 1, 4.23, 1.76, 0},    {32, 32, 8, 1, 5.18, 2.28, 0},     {32, 32, 4, 2, 4.33, 1.42, 1.04},
    {32, 64, 2, 2, 4.90, 1.35, 0.94}, {64, 64, 2, 2, 11.23, 1.72, 1.40}, {64, 128, 1, 2, 15.59, 1.69, 1.23},
};
constexpr int kProductKinds = sizeof(kProductShapes) / sizeof(ProductShape);
constexpr int kGatedKinds = sizeof(kGatedShapes) / sizeof(ProductShape);
// A launch has at most 65535 workgroups along the rows.
constexpr int64_t kMaxRowGroups = 65535;

constexpr double product_cost(const ProductShape &s, int64_t rows, int64_t outs, int64_t chunks) {
    const int64_t groups = ((rows + s.rows - 1) / s.rows) * ((outs + s.outs - 1) / s.outs);
    const int64_t fullest = (groups + 255) / 256, rest = fullest % s.resident;
    const double full = s.resident * s.shared, part = (double) rest * s.shared;
    const double round = (double) (fullest / s.resident) * (full > s.alone ? full : s.alone);
    const double last = rest == 0 ? 0.0 : part > s.alone ? part : s.alone;
    return s.start + (double) ((chunks + s.waves - 1) / s.waves) * (round + last);
}

// The cheapest shape's number.
constexpr int product_shape(bool gated, int64_t rows, int64_t outs, int64_t chunks) {
    const ProductShape *shapes = gated ? kGatedShapes : kProductShapes;
    const int n = gated ? kGatedKinds : kProductKinds;
    int best = n - 1;
    double cost = product_cost(shapes[best], rows, outs, chunks);
    for (int i = n - 2; i >= 0; --i) {
        if ((rows + shapes[i].rows - 1) / shapes[i].rows > kMaxRowGroups) continue;
        const double c = product_cost(shapes[i], rows, outs, chunks);
        if (c < cost) {
            best = i;
            cost = c;
        }
    }
    return best;
}

}  // namespace bmo
