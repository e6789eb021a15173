// Shared by the attention operators: element types, division by a page size, cache rows.
#pragma once

#include <initializer_list>

#include "qxt_common.h"

namespace qxt {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T>
struct vec4_of {
    typedef T type __attribute__((ext_vector_type(4)));
};

inline bool half_type(uint32_t type) { return type == QXT_TYPE_BF16 || type == QXT_TYPE_F16; }
inline bool known_type(uint32_t type) { return type == QXT_TYPE_F32 || half_type(type); }
inline size_t type_bytes(uint32_t type) { return type == QXT_TYPE_F32 ? 4 : 2; }

inline bool all_multiples(size_t of, std::initializer_list<size_t> values) {
    for (size_t v : values)
        if (v % of) return false;
    return true;
}

// n / d and n % d for n < 2^31 and a divisor known at launch.  With s =
// ceil(log2 d) and m = floor(2^(31 + s) / d) + 1 the error of m is below
// 2^s / 2^(31 + s) relative to 1 / d, so floor(n m / 2^(31 + s)) is exact for
// every n < 2^31, and m < 2^32.  d = 1 passes n through (without a branch).
struct FastDiv {
    uint32_t divisor, magic, shift, pass;
};
inline FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0, 0xFFFFFFFFu};
    if (d <= 1) return f;
    f.pass = 0;
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    f.magic = static_cast<uint32_t>((1ull << (31 + s)) / d + 1);
    f.shift = s - 1;
    return f;
}
// (F: FastDiv, in any address space.)
template <typename F>
__host__ __device__ __forceinline__ uint32_t fast_quotient(uint32_t n, const F &f) {
    return (static_cast<uint32_t>((static_cast<uint64_t>(n) * f.magic) >> 32) + (n & f.pass)) >> f.shift;
}

// One cache (keys or values): pages of page_size slots, a row of head_dim
// elements for each slot and head.  Strides in bytes.
struct CacheView {
    char *data;
    int64_t page_stride, slot_stride, head_stride;
};

}  // namespace qxt
