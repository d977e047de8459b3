// product_shape.hpp -- which kernel a product of 8-bit rows with Q4_0 weights
// takes (weights.hip).  Plain C++, so that a host test can walk the rule.
#pragma once

#include <stdint.h>

namespace bmo {

// A workgroup takes `rows` rows and `outs` outputs (gates, of a gated product);
// `waves` waves share each piece of it along the columns, a step each a unit of
// 128.  A CU runs `resident` of them at a time.  Times of a call in us, by the
// fullest CU's workgroups: start + each for all that is not in a step, and a
// round of `resident` at a time a step (alone, or shared for each where that is
// more).
struct ProductShape {
    int rows, outs, waves, resident;
    double start, each, alone, shared;
};

// Few rows (16 x 16 matrix instructions) and many (32 x 32).  The times are
// fitted to calls with weights from HBM, 2 to 3000 rows by 512 to 32001 outputs
// of 160 to 11264 columns (gated: 2048 rows by 512 to 11264 outputs of 128 to
// 8192), and moved by up to 15% to where they choose best.  Over these same calls
// the choice is 0.4% slower than the fastest of the shapes here in the mean of 216,
// 13% at worst (48 rows x 11264 outputs x 640: 6.6 us, 5.9 with 32 x 32); gated 0.1%
// over 112, 3% at worst.  What a shape is worth: 16 x 16 at 2 x 512 x 4096 3.5 us, 16
// x 32 there 5.8; 32 x 32 with eight waves at 48 x 4096 x 5632 8.4, with four 11.1; 32
// x 128 with one wave to a piece at 1500 x 1216 x 160 5.8, 32 x 256 at 768 x 11264 x
// 288 15.3, 64 x 256 there 20.0; 64 x 128 with two waves to a piece at 1500 x 12288 x
// 4096 200, 64 x 256 there 203, at 2048 rows 260 and 244.
constexpr ProductShape kProductShapes[] = {
    {16, 16, 8, 2, 1.47, 0.25, 0.82, 0.58},  {16, 32, 8, 2, 1.58, 0.28, 1.08, 0.84},  {16, 64, 8, 1, 1.63, 0.77, 1.44, 0},
    {32, 32, 4, 3, 2.30, 0.35, 0.63, 0.51},  {32, 32, 8, 1, 0.80, 1.82, 1.05, 0},     {32, 64, 4, 2, 2.01, 0.73, 1.31, 0.74},
    {32, 128, 1, 3, 2.14, 0.55, 0.61, 0.38}, {32, 256, 1, 3, 1.85, 0.79, 1.28, 0.70}, {64, 128, 2, 2, 3.33, 1.52, 1.56, 1.23},
    {64, 256, 1, 2, 2.12, 1.97, 2.24, 1.08},
};
constexpr ProductShape kGatedShapes[] = {
    {16, 32, 8, 1, 2.38, 0.15, 1.48, 0},     {32, 32, 8, 2, 0.66, 2.54, 1.57, 1.80}, {32, 32, 4, 2, 1.85, 0.98, 1.38, 0.80},
    {32, 64, 2, 2, 2.84, 1.19, 1.49, 0.79},  {32, 128, 1, 3, 4.12, 1.34, 1.37, 0.70}, {64, 64, 2, 2, 4.00, 2.39, 1.70, 1.18},
    {64, 128, 1, 2, 4.70, 3.38, 1.77, 1.15},
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
    return s.start + (double) fullest * s.each + (double) ((chunks + s.waves - 1) / s.waves) * (round + last);
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

// Where a workgroup works.  Workgroups go round the 8 XCDs one by one, x first,
// and each XCD has an L2 of its own: where the columns of workgroups (x: the
// outputs) are no multiple of 8 those of a column land on all of them, and each
// reads its weights.  So an XCD takes whole columns, row after row (y), and what
// rests of the columns is shared by rows (1984 rows x 12544 outputs x 4096, 49
// columns: 249 us, 267 as they come).  div_main and div_rest divide by columns / 8
// and columns % 8.
struct Place {
    uint32_t x, y;
};
template <class F, class G>
constexpr Place product_place(uint32_t x, uint32_t y, uint32_t columns, uint32_t rows, F div_main, G div_rest) {
    const uint32_t main = columns / 8, rest = columns % 8;
    if (rest == 0 || main == 0 || rows == 1) return {x, y};
    const uint32_t id = y * columns + x, turn = id / 8;
    if (turn < main * rows) {
        const uint32_t row = div_main(turn);
        return {id % 8 + 8 * (turn - row * main), row};
    }
    const uint32_t left = id - 8 * main * rows, row = div_rest(left);
    return {8 * main + left - row * rest, row};
}

}  // namespace bmo
