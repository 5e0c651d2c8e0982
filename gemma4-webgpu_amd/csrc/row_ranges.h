// Whether operands that are rows in memory share some of it: plain functions,
// apart from the kernels so that they can be checked without a GPU.
#pragma once

#include <stdint.h>

namespace g4 {

// `rows` rows of `bytes` each, the next one `stride` bytes (at least `bytes`) on. One array: one row.
struct RowRange {
    const void* p;
    uint64_t bytes, stride, rows;
};
inline RowRange one_range(const void* p, uint64_t bytes) { return {p, bytes, bytes, 1}; }

// Rows that lie beside others in one buffer (columns of a fused projection) share nothing though their ranges overlap.
inline bool rows_meet(RowRange a, RowRange b) {
    if (!a.p || !b.p || !a.bytes || !b.bytes || !a.rows || !b.rows) return false;
    if (reinterpret_cast<uintptr_t>(a.p) > reinterpret_cast<uintptr_t>(b.p)) {
        const RowRange c = a;
        a = b;
        b = c;
    }
    const uint64_t d = reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p);
    typedef unsigned __int128 wide;
    if (d >= (wide)(a.rows - 1) * a.stride + a.bytes) return false;  // b begins behind a
    if (a.rows == 1) return true;                                    // b's first byte is among a's
    uint64_t i = d / a.stride;  // a's row at or before b's first: a row there, for d lies within the range
    if (b.rows == 1 || a.stride == b.stride) {
        // Every row of b lies alike to a's rows i and i + 1, of which the last has none after it.
        const uint64_t in = d - i * a.stride;
        return in < a.bytes || (i + 1 < a.rows && in + b.bytes > a.stride);
    }
    for (uint64_t j = 0; i < a.rows && j < b.rows;) {
        const wide x = (wide)i * a.stride, y = (wide)j * b.stride + d;
        if (x + a.bytes <= y) i++;
        else if (y + b.bytes <= x) j++;
        else return true;
    }
    return false;
}

}  // namespace g4
