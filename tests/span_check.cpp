// Prints whether two spans share bytes (1 or 0), a line for each pair read from
// standard input: address, rows, bytes of a row and stride of the one, then of
// the other.  Built by tests/Makefile; tests/test_rows_spans.py runs it.
#include <cinttypes>
#include <cstdio>

#include "spans.hpp"

int main() {
    bmo::Span s[2];
    auto read = [](bmo::Span &t) {
        uintptr_t at;
        const int n = std::scanf("%" SCNuPTR " %" SCNd64 " %" SCNd64 " %" SCNd64, &at, &t.n, &t.dense, &t.stride);
        t.p = reinterpret_cast<const void *>(at);
        return n == 4;
    };
    while (read(s[0]) && read(s[1])) std::printf("%d\n", bmo::meet(s[0], s[1]));
    return 0;
}
