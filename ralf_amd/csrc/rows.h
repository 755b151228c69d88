// Host: what the serving entries ask of [tokens][heads][dim] rows given by strides (elements; the last dim contiguous).
#pragma once
#include <stdint.h>

namespace ralf {
// n0 x n1 rows of `dim` elements, steps s0 and s1: every row has its own elements, one of the two axes lying within the other's steps
inline bool rows_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t dim) {
    if (n0 <= 1 || n1 <= 1) return (n0 <= 1 || s0 >= dim) && (n1 <= 1 || s1 >= dim);
    return (s1 >= dim && s0 >= (n1 - 1) * s1 + dim) || (s0 >= dim && s1 >= (n0 - 1) * s0 + dim);
}
}  // namespace ralf
