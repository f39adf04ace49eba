// Sixteen bytes at a place near the end of a matrix, of which those from the end on are zero and not read.  Arithmetic without any HIP, so that it can be driven on a machine
// that has no GPU (tests/row_end_test.cpp).
#pragma once

namespace jitnn {

// How many bytes further down a load has to start, for a place whose sixteen bytes end `over` bytes behind the end.  64 bits: a place of the first expert is as far in front of
// the end as the matrix is large, which is more than 32 bits hold; behind it a place is by no more than a column of a row.
constexpr int bytes_behind(long long over) { return over > 0 ? (int)over : 0; }

// The two halves of what such a load gives, as the bytes that were asked for.
struct Halves {
    unsigned long long lo, hi;
};
constexpr Halves moved_down(Halves v, int behind) {
    const int by = 8 * (behind < 16 ? behind : 16);
    return {by == 0 ? v.lo : by < 64 ? v.lo >> by | v.hi << (64 - by) : by < 128 ? v.hi >> (by - 64) : 0, by < 64 ? v.hi >> by : 0};
}

}  // namespace jitnn
