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
// 8192), and moved by up to 15% to where they choose best: against the fastest
// shape 0.7% in the mean over the 162 calls, 16% at worst (32 rows x 32001 outputs
// x 1024: 11.2 us, 9.7 with 32 x 64); gated 0.2% over 80, 8% at worst.  What a
// shape is worth: 16 x 16 at 2 x 512 x 4096 3.5 us, 16 x 32 there 5.7; 16 x 64 at 64 x
// 4096 x 4096 8.1, 32 x 32 there 9.0; 32 x 32 with eight waves at 48 x 4096 x 5632 9.1,
// with four 11.1; 64 x 128 with two waves to a piece at 1500 x 12288 x 4096 201, 64 x
// 256 there 213, at 2048 x 12288 x 4096 267 and 250.
constexpr ProductShape kProductShapes[] = {
    {16, 16, 8, 1, 2.50, 0.81, 0},     {16, 32, 8, 1, 3.15, 1.00, 0},    {16, 64, 8, 1, 2.90, 1.74, 0},
    {32, 32, 4, 2, 3.68, 0.75, 0.59},  {32, 32, 8, 1, 3.88, 1.32, 0},    {32, 64, 4, 2, 3.96, 1.25, 1.11},
    {32, 128, 2, 2, 4.75, 1.30, 1.01}, {64, 128, 2, 2, 6.95, 1.98, 1.29}, {64, 256, 1, 2, 9.38, 1.66, 1.12},
};
constexpr ProductShape kGatedShapes[] = {
    {16, 32, 8, 1, 3.84, 1.72, 0},    {32, 32, 8, 1, 5.06, 2.10, 0},     {32, 32, 4, 2, 4.59, 1.31, 0.94},
    {32, 64, 2, 2, 4.71, 1.34, 0.92}, {64, 64, 2, 2, 10.18, 2.07, 1.43}, {64, 128, 1, 2, 13.18, 1.52, 1.38},
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
