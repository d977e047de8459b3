// product_shape.hpp -- which kernel a product of 8-bit rows with Q4_0 weights
// takes (weights.hip).  Plain C++, so that a host test can walk the rule.
#pragma once

#include <stdint.h>

namespace bmo {

// A workgroup takes `rows` rows and `outs` outputs (gates, of a gated product);
// `waves` waves share each piece of it along the columns, a step each a unit of
// 128.  Times of a call in us: start + steps * max(step, work * workgroups of
// the fullest CU).
struct ProductShape {
    int rows, outs, waves;
    double start, step, work;
};

// Few rows (16 x 16 matrix instructions) and many (32 x 32).  The times are
// fitted to calls with weights from HBM, 2 to 3000 rows by 512 to 32001 outputs
// of 1024 to 11264 columns (gated: 2048 rows by 512 to 5632 outputs of 1024 to
// 8192), and the product's moved by up to 15% to where they choose best.  Against
// the fastest of 10 shapes (7 gated) the choice costs 1.6% in the mean over the
// 126 calls, 15% at worst (48 rows x 4096 outputs x 5632: 10.7 us, 9.3 with 8
// waves to 32 x 32); gated 1.2% over 64, 16% at worst.  What a shape is worth:
// 16 x 16 at 2 x 512 x 4096 3.5 us, 16 x 32 there 5.8; 16 x 64 at 64 x 4096 x
// 4096 8.1, 32 x 32 there 9.2; 128 x 128 at 2048 x 12288 x 4096 267, 64 x 128
// there 303.
constexpr ProductShape kProductShapes[] = {
    {16, 16, 8, 2.34, 0.54, 0.77}, {16, 32, 8, 3.02, 0.93, 1.00},  {16, 64, 8, 3.00, 0.69, 1.49},
    {32, 32, 4, 4.17, 0.75, 0.55}, {32, 64, 4, 4.26, 1.31, 0.95},  {64, 128, 1, 6.47, 1.03, 0.74},
    {128, 128, 1, 9.82, 1.84, 1.19},
};
constexpr ProductShape kGatedShapes[] = {
    {16, 32, 8, 3.62, 1.49, 1.67},
    {32, 32, 8, 4.05, 0.12, 2.46},
    {32, 32, 4, 4.01, 1.36, 0.93},
    {128, 64, 1, 12.40, 1.96, 1.33},
};
constexpr int kProductKinds = sizeof(kProductShapes) / sizeof(ProductShape);
constexpr int kGatedKinds = sizeof(kGatedShapes) / sizeof(ProductShape);
// A launch has at most 65535 workgroups along the rows.
constexpr int64_t kMaxRowGroups = 65535;

constexpr double product_cost(const ProductShape &s, int64_t rows, int64_t outs, int64_t chunks) {
    const int64_t groups = ((rows + s.rows - 1) / s.rows) * ((outs + s.outs - 1) / s.outs);
    const double shared = s.work * (double) ((groups + 255) / 256);
    return s.start + (double) ((chunks + s.waves - 1) / s.waves) * (shared > s.step ? shared : s.step);
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
