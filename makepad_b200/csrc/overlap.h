// Whether an output lies over an input: host arithmetic on addresses, in front of a launch.
#pragma once
#include <stdint.h>

namespace mpq {

// [a, a + a_bytes) and any of `rows` rows of row_bytes, stride_bytes (at least row_bytes) apart from b on.  Nothing lies over a null pointer.  (128 bits: a stride is the caller's number.)
inline bool overlaps(const void* a, int64_t a_bytes, const void* b, int64_t rows, int64_t row_bytes, __int128 stride_bytes)
{
    if (!a || !b || a_bytes <= 0 || rows <= 0 || row_bytes <= 0) return false;
    const __int128 a0 = (__int128)reinterpret_cast<uintptr_t>(a), b0 = (__int128)reinterpret_cast<uintptr_t>(b);
    if (a0 + a_bytes <= b0 || b0 + (rows - 1) * stride_bytes + row_bytes <= a0) return false;          // (nearly all calls: no division)
    // the first row that ends behind a's beginning
    const __int128 i = b0 + row_bytes > a0 ? 0 : (a0 - b0 - row_bytes) / stride_bytes + 1;
    return i < rows && b0 + i * stride_bytes < a0 + a_bytes;
}
inline bool overlaps(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) { return overlaps(a, a_bytes, b, 1, b_bytes, b_bytes); }

}  // namespace mpq
