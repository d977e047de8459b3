// spans.hpp -- which bytes a call reads or writes, and whether two of its
// tensors share any.  Plain C++, so that a host test can walk it.
#pragma once

#include <stdint.h>

namespace bmo {

// n rows of `dense` bytes, `stride` (at least dense) bytes apart.
struct Span {
    const void *p;
    int64_t n, dense, stride;
    bool operator==(const Span &o) const { return p == o.p && dense == o.dense && (n == 1 || stride == o.stride); }
};

typedef __int128 SpanInt;  // (2^30 rows 2^42 bytes apart)

// The least x >= 0 for which a x mod m is in [l, r] (0 <= l <= r < m), or -1.
// If no multiple of a is there itself, the first m y + [l, r] that holds one is
// sought modulo a: a step of Euclid's algorithm.
inline SpanInt first_in(SpanInt a, SpanInt m, SpanInt l, SpanInt r) {
    a %= m;
    if (l == 0) return 0;
    if (a == 0) return -1;
    if (2 * a > m) return first_in(m - a, m, m - r, m - l);
    const SpanInt x = (l + a - 1) / a;
    if (a * x <= r) return x;
    const SpanInt y = first_in(a - m % a, a, l % a, r % a);
    return y < 0 ? y : (l + m * y + a - 1) / a;
}

// Whether two spans (of at least one row and byte, or absent) share bytes.
inline bool meet(const Span &a, const Span &b) {
    if (!a.p || !b.p) return false;
    if (a.n > 1 && a.stride == a.dense) return meet({a.p, 1, a.n * a.dense, a.n * a.dense}, b);
    if (b.n > 1 && b.stride == b.dense) return meet(a, {b.p, 1, b.n * b.dense, b.n * b.dense});
    const SpanInt from = (SpanInt) reinterpret_cast<uintptr_t>(a.p) - (SpanInt) reinterpret_cast<uintptr_t>(b.p);
    const SpanInt a_step = a.stride, b_step = b.stride;
    // Rows i of a that begin at t = from + i a_step behind b's first byte, and of
    // these the ones before b's last byte that do not end before its first.
    const SpanInt low = 1 - a.dense, high = (SpanInt) (b.n - 1) * b_step + b.dense - 1;
    const SpanInt i0 = from >= low ? 0 : a.n == 1 ? 1 : (low - from + a_step - 1) / a_step;
    const SpanInt i1 = from > high ? -1 : a.n == 1 ? 0 : (high - from) / a_step < a.n - 1 ? (high - from) / a_step : a.n - 1;
    if (i0 > i1) return false;
    if (b.n == 1) return true;
    // Such a row meets one of b if less than b.dense lies between them, from t
    // back or forward: (t + a.dense - 1) mod b_step within a.dense + b.dense - 2.
    const SpanInt width = (SpanInt) a.dense + b.dense - 2;
    if (width >= b_step) return true;
    const SpanInt at = (from + i0 * a_step + a.dense - 1) % b_step;  // (from low on: not negative)
    if (at <= width) return true;
    // (at + i a_step) mod b_step in [0, width]
    const SpanInt i = first_in(a_step, b_step, b_step - at, b_step - at + width);
    return i >= 0 && i <= i1 - i0;
}

}  // namespace bmo
