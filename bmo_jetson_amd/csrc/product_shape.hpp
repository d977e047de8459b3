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
// 8192), to 10 to 16% in the mean.  Against the fastest of 10 shapes (7 gated)
// the choice costs 2.8% in the mean over the 126 (64) of them, 20% at worst (512
// rows x 1000 outputs x 11264: 29.8 us, 25.6 with 32 rows x 64 outputs in 16 x
// 16); one shape for all of few or many would cost up to 5 times as much.
constexpr ProductShape kProductShapes[] = {
    {16, 16, 8, 2.30, 0.45, 0.66},  {16, 32, 8, 2.83, 0.85, 0.89},   {32, 32, 4, 3.75, 0.63, 0.57},
    {32, 64, 4, 4.59, 1.11, 0.99},  {64, 128, 1, 7.19, 1.04, 0.80},  {128, 128, 1, 10.29, 1.83, 1.40},
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
