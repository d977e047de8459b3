// Prints the kernel of each product read from standard input, a line each: gated
// (0 or 1), rows, outputs and units of 128 columns in; the rows and outputs of
// a workgroup, and the waves that share a piece of it, out.  Built by
// tests/Makefile; tests/_shapes.py runs it.
#include <cinttypes>
#include <cstdio>

#include "product_shape.hpp"

int main() {
    int gated;
    int64_t rows, outs, chunks;
    while (std::scanf("%d %" SCNd64 " %" SCNd64 " %" SCNd64, &gated, &rows, &outs, &chunks) == 4) {
        const int i = bmo::product_shape(gated != 0, rows, outs, chunks);
        const bmo::ProductShape s = gated ? bmo::kGatedShapes[i] : bmo::kProductShapes[i];
        std::printf("%d %d %d\n", s.rows, s.outs, s.waves);
    }
    return 0;
}
