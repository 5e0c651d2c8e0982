// Checks gemma4-webgpu_amd/csrc/row_ranges.h against marked bytes, over every small layout of two operands, and at the
// largest sizes, where products pass 64 bits.
#include <stdio.h>

#include <vector>

#include "../gemma4-webgpu_amd/csrc/row_ranges.h"

using g4::RowRange;

static RowRange at(uint64_t p, uint64_t bytes, uint64_t stride, uint64_t rows) {
    return {reinterpret_cast<const void*>((uintptr_t)p), bytes, stride, rows};
}
static bool by_bytes(const RowRange& a, const RowRange& b) {
    std::vector<char> mark(512, 0);
    for (uint64_t r = 0; r < a.rows; r++)
        for (uint64_t e = 0; e < a.bytes; e++) mark[(uintptr_t)a.p + r * a.stride + e] = 1;
    for (uint64_t r = 0; r < b.rows; r++)
        for (uint64_t e = 0; e < b.bytes; e++)
            if (mark[(uintptr_t)b.p + r * b.stride + e]) return true;
    return false;
}

int main() {
    long n = 0, met = 0;
    for (uint64_t ab = 1; ab <= 4; ab++)
        for (uint64_t as = ab; as <= 9; as++)
            for (uint64_t ar = 1; ar <= 4; ar++)
                for (uint64_t bb = 1; bb <= 4; bb++)
                    for (uint64_t bs = bb; bs <= 9; bs++)
                        for (uint64_t br = 1; br <= 4; br++)
                            for (uint64_t d = 1; d <= 80; d += 1) {
                                const RowRange a = at(40, ab, as, ar), b = at(d, bb, bs, br);
                                const bool want = by_bytes(a, b);
                                n++;
                                met += want;
                                if (g4::rows_meet(a, b) != want || g4::rows_meet(b, a) != want) {
                                    printf("a %lu rows of %lu, %lu apart at 40; b %lu of %lu, %lu apart at %lu: %d\n", ar, ab, as, br, bb, bs, d, want);
                                    return 1;
                                }
                            }
    // 2^22 rows 2^42 bytes apart: the range passes 64 bits.
    const uint64_t far = 1ull << 42, many = 1u << 22;
    if (!g4::rows_meet(at(4096, 64, far, many), at(4096 + 7 * far + 63, 64, far, many))) return 2;
    if (g4::rows_meet(at(4096, 64, far, many), at(4096 + 7 * far + 64, 64, far, many))) return 3;
    if (!g4::rows_meet(at(4096, 64, far, many), at(4096 + far - 1, 64, 128, 2))) return 4;
    if (g4::rows_meet(at(4096, 64, far, many), g4::one_range(nullptr, 1 << 20))) return 5;
    if (g4::rows_meet(at(4096, 64, 64, 0), g4::one_range(at(4096, 0, 0, 0).p, 64))) return 6;
    printf("%ld layouts, %ld that meet\n", n, met);
    return 0;
}
