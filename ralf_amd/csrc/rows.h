// Host: what the serving entries ask of [tokens][heads][dim] rows given by strides (elements; the last dim contiguous).
#pragma once
#include <stdint.h>

namespace ralf {
typedef __int128 wide;      // (sizes times strides, before anything has bounded them)
// n0 x n1 rows of `dim` elements, steps s0 and s1: every row has its own elements, one of the two axes lying within the other's steps
inline bool rows_apart(wide n0, wide s0, wide n1, wide s1, wide dim) {
    if (n0 <= 1 || n1 <= 1) return (n0 <= 1 || s0 >= dim) && (n1 <= 1 || s1 >= dim);
    return (s1 >= dim && s0 >= (n1 - 1) * s1 + dim) || (s0 >= dim && s1 >= (n0 - 1) * s0 + dim);
}

// Two such sets of n0 x n1 rows, a and b (s0, s1: their steps; `size` bytes to an element; b's rows apart): none of their elements in one place.  Exact where the steps are the
// same; otherwise by their spans, or because b's rows lie in the gaps of a's along one axis whose step they share, and other arrangements count as overlapping.
struct Rows { const void* p; int64_t s0, s1; };
inline wide floor_div(wide x, wide y) { return x / y - (x % y < 0 ? 1 : 0); }       // y > 0
inline bool rows_disjoint(const Rows& a, const Rows& b, wide n0, wide n1, wide dim, wide size) {
    const wide len_a = (n0 - 1) * a.s0 + (n1 - 1) * a.s1 + dim, len_b = (n0 - 1) * b.s0 + (n1 - 1) * b.s1 + dim, bytes = (wide)(uintptr_t)b.p - (wide)(uintptr_t)a.p;
    if (bytes >= len_a * size || -bytes >= len_b * size) return true;
    if (bytes % size) return false;
    const wide at = bytes / size;       // of b's first element, counted from a's
    if ((n0 <= 1 || a.s0 == b.s0) && (n1 <= 1 || a.s1 == b.s1)) {
        // two rows share an element where |at + i * outer + j * inner| < dim for some |i| < n, |j| < m; rows that are apart leave three values of i at most to look at
        const bool swap = n0 <= 1 || (n1 > 1 && b.s1 > b.s0);
        const wide n = swap ? n1 : n0, m = swap ? n0 : n1, outer = n > 1 ? (swap ? b.s1 : b.s0) : len_b, inner = m > 1 ? (swap ? b.s0 : b.s1) : len_b, reach = (m - 1) * inner + dim - 1;
        for (wide i = floor_div(-at - reach + outer - 1, outer); i * outer + at <= reach; ++i) {
            const wide j = floor_div(-(at + i * outer), inner), r = at + i * outer + j * inner;       // -inner < r <= 0
            if (i <= -n || i >= n) continue;
            if ((j > -m && j < m && -r < dim) || (j + 1 > -m && j + 1 < m && r + inner < dim)) return false;
        }
        return true;
    }
    auto gaps = [&](wide step, wide len_a, wide len_b) {        // both in pieces a step apart: b's between a's
        const wide r = step > 0 ? at - floor_div(at, step) * step : 0;
        return r >= len_a && r + len_b <= step;
    };
    return (n0 > 1 && a.s0 == b.s0 && gaps(a.s0, (n1 - 1) * a.s1 + dim, (n1 - 1) * b.s1 + dim)) || (n1 > 1 && a.s1 == b.s1 && gaps(a.s1, (n0 - 1) * a.s0 + dim, (n0 - 1) * b.s0 + dim));
}
}  // namespace ralf
