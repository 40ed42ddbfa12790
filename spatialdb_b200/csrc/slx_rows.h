// slx_rows.h -- whether two strided arrays of rows share memory (host only).
#pragma once
#include <cstdint>

namespace slx {

// M rows of `wa` elements, `lda` apart, at `a`, and of `wb` elements, `ldb` apart, at `b`, elements of `e` bytes; widths
// at most the strides. Rows that lie between the other array's rows do not overlap it (q, k and v in one buffer).
inline bool rows_overlap(const void* a, int64_t lda, int64_t wa, const void* b, int64_t ldb, int64_t wb, int64_t M, int e) {
    if (!a || !b || M <= 0 || wa <= 0 || wb <= 0) return false;
    const __int128 pa = (__int128)(uintptr_t)a, pb = (__int128)(uintptr_t)b, sa = (__int128)lda * e, sb = (__int128)ldb * e;
    const __int128 na = (__int128)wa * e, nb = (__int128)wb * e;
    if (pa + sa * (M - 1) + na <= pb || pb + sb * (M - 1) + nb <= pa) return false;
    if (lda == ldb) {  // row j of b begins `r` bytes into row j + q of a
        const __int128 d = pb - pa;
        const __int128 q = d >= 0 ? d / sa : -((-d + sa - 1) / sa), r = d - q * sa;
        return (r < na && q > -M && q < M) || (r + nb > sa && q + 1 > -M && q + 1 < M);
    }
    for (int64_t i = 0, j = 0; i < M && j < M;) {  // both in order of their addresses
        const __int128 x = pa + sa * i, y = pb + sb * j;
        if (x + na <= y) i++;
        else if (y + nb <= x) j++;
        else return true;
    }
    return false;
}

}  // namespace slx
