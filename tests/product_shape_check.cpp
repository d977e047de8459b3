// Prints the kernel of each product read from standard input, a line each: gated
// (0 or 1), rows, outputs and units of 128 columns in; the rows and outputs of
// a workgroup, and the waves that share a piece of it, out.  With an argument
// the places of a grid's workgroups: columns and rows in; out whether each place
// is taken once, and how many columns are taken by workgroups of more than one
// XCD (those that differ in their number modulo 8).  Built by tests/Makefile;
// tests/_shapes.py runs it.
#include <cinttypes>
#include <cstdio>
#include <vector>

#include "product_shape.hpp"

static void places() {
    uint32_t columns, rows;
    while (std::scanf("%" SCNu32 " %" SCNu32, &columns, &rows) == 2) {
        std::vector<int> taken((size_t) columns * rows), xcds(columns);
        for (uint32_t y = 0; y < rows; ++y)
            for (uint32_t x = 0; x < columns; ++x) {
                const bmo::Place at = bmo::product_place(
                    x, y, columns, rows, [&](uint32_t n) { return n / (columns / 8); }, [&](uint32_t n) { return n / (columns % 8); });
                if (at.x >= columns || at.y >= rows) continue;
                ++taken[(size_t) at.y * columns + at.x];
                xcds[at.x] |= 1 << (y * columns + x) % 8;
            }
        int once = 1, shared = 0;
        for (int n : taken) once &= n == 1;
        for (int n : xcds) shared += (n & (n - 1)) != 0;
        std::printf("%d %d\n", once, shared);
    }
}

int main(int argc, char **) {
    if (argc > 1) {
        places();
        return 0;
    }
    int gated;
    int64_t rows, outs, chunks;
    while (std::scanf("%d %" SCNd64 " %" SCNd64 " %" SCNd64, &gated, &rows, &outs, &chunks) == 4) {
        const int i = bmo::product_shape(gated != 0, rows, outs, chunks);
        const bmo::ProductShape s = gated ? bmo::kGatedShapes[i] : bmo::kProductShapes[i];
        std::printf("%d %d %d\n", s.rows, s.outs, s.waves);
    }
    return 0;
}
