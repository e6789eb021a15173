// Microscaling blocks: 32 elements of 4-bit (e2m1) or 8-bit (e4m3) floating
// point under one shared power of two, one byte E of value 2^(E - 127) (255: the
// block is NaN).  Rows of blocks: element values packed (4-bit ones two a byte,
// the lower index in the low half), scales one byte a block in a plane of their
// own.  The rule is the one of the OCP Microscaling Formats specification:
// E - 127 = floor(log2(largest magnitude)) - floor(log2(largest element)),
// elements rounded to nearest even and cut to the largest one.
#pragma once

#include "qxt_paged.h"

namespace qxt {

constexpr int kMxBlock = 32;

inline bool known_mx(uint32_t format) { return format == QXT_MX_FP4 || format == QXT_MX_FP8; }
inline size_t mx_row_bytes(uint32_t format, uint32_t columns) { return format == QXT_MX_FP4 ? columns / 2 : columns; }

// Rows in memory, `bytes` each.
struct RowSpan {
    const void *at;
    int64_t stride;
    uint64_t rows, bytes;
};
// Whether two sets of rows share memory.  (Sets of one stride may lie between each other's rows; sets of different strides
// are taken to meet where their ranges do.)
inline bool overlap(const RowSpan &x, const RowSpan &y) {
    if (x.at == nullptr || y.at == nullptr || x.rows == 0 || y.rows == 0) return false;
    const uint64_t x0 = reinterpret_cast<uintptr_t>(x.at), y0 = reinterpret_cast<uintptr_t>(y.at);
    const uint64_t x_skip = x.rows > 1 ? x.stride : y.rows > 1 ? y.stride : 0, y_skip = y.rows > 1 ? y.stride : x_skip;
    if (x0 + (x.rows - 1) * x_skip + x.bytes <= y0 || y0 + (y.rows - 1) * y_skip + y.bytes <= x0) return false;
    if (x_skip != y_skip || x_skip == 0) return true;
    const uint64_t ahead = y0 >= x0 ? (y0 - x0) % x_skip : x_skip - 1 - (x0 - y0 - 1) % x_skip;
    return ahead < x.bytes || ahead + y.bytes > x_skip;
}

// Eight neighbouring elements of a row as fp32.
struct Eight {
    float v[8];
};

typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef unsigned int u2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float bf16_bits(uint32_t high) { return __uint_as_float(high & 0xFFFF0000u); }

// From 16 bytes of half elements, or twice 16 bytes of fp32.
__device__ __forceinline__ Eight eight_of(uint32_t type, u4 a, u4 b) {
    Eight e;
    if (type == QXT_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e.v[i] = __uint_as_float(a[i]);
            e.v[4 + i] = __uint_as_float(b[i]);
        }
    } else if (type == QXT_TYPE_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e.v[2 * i] = __uint_as_float(a[i] << 16);
            e.v[2 * i + 1] = bf16_bits(a[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e.v[2 * i] = half_bits_to_float(a[i]);
            e.v[2 * i + 1] = half_bits_to_float(a[i] >> 16);
        }
    }
    return e;
}

// Two elements rounded to a half type, packed.
__device__ __forceinline__ uint32_t half_pair(uint32_t type, float x, float y) {
    if (type == QXT_TYPE_BF16) {
        typedef bf16_t pair __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, pair{static_cast<bf16_t>(x), static_cast<bf16_t>(y)});
    }
    typedef f16_t pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, pair{static_cast<f16_t>(x), static_cast<f16_t>(y)});
}

// Eight elements from / to element `index` of a row (16-byte pieces), or one by one where rows are not aligned.
template <bool VEC>
__device__ __forceinline__ Eight load_eight(uint32_t type, const char *row, uint32_t index) {
    if constexpr (VEC) {
        const char *p = row + static_cast<size_t>(index) * (type == QXT_TYPE_F32 ? 4 : 2);
        const u4 a = *reinterpret_cast<const u4 *>(p);
        u4 b = a;
        if (type == QXT_TYPE_F32) b = *reinterpret_cast<const u4 *>(p + 16);
        return eight_of(type, a, b);
    } else {
        Eight e;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (type == QXT_TYPE_F32) e.v[i] = reinterpret_cast<const float *>(row)[index + i];
            else if (type == QXT_TYPE_BF16) e.v[i] = static_cast<float>(reinterpret_cast<const bf16_t *>(row)[index + i]);
            else e.v[i] = static_cast<float>(reinterpret_cast<const f16_t *>(row)[index + i]);
        }
        return e;
    }
}

template <bool VEC>
__device__ __forceinline__ void store_eight(uint32_t type, char *row, uint32_t index, const Eight &e) {
    if constexpr (VEC) {
        char *p = row + static_cast<size_t>(index) * (type == QXT_TYPE_F32 ? 4 : 2);
        if (type == QXT_TYPE_F32) {
            *reinterpret_cast<float4 *>(p) = make_float4(e.v[0], e.v[1], e.v[2], e.v[3]);
            *reinterpret_cast<float4 *>(p + 16) = make_float4(e.v[4], e.v[5], e.v[6], e.v[7]);
        } else {
            u4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = half_pair(type, e.v[2 * i], e.v[2 * i + 1]);
            *reinterpret_cast<u4 *>(p) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (type == QXT_TYPE_F32) reinterpret_cast<float *>(row)[index + i] = e.v[i];
            else if (type == QXT_TYPE_BF16) reinterpret_cast<bf16_t *>(row)[index + i] = static_cast<bf16_t>(e.v[i]);
            else reinterpret_cast<f16_t *>(row)[index + i] = static_cast<f16_t>(e.v[i]);
        }
    }
}

// Largest magnitude's bits: as integers a NaN is above infinity is above every number, so none is lost.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The shared exponent's byte from the largest magnitude's bits.  Infinities and
// NaNs make the block NaN; zero and subnormal blocks, and those whose exponent
// would be below the byte's, take 0.
template <bool FP8>
__device__ __forceinline__ uint32_t mx_scale(uint32_t largest) {
    const int exponent = static_cast<int>(largest >> 23);
    return exponent == 255 ? 255u : static_cast<uint32_t>(max(exponent - (FP8 ? 8 : 2), 0));
}
// 2^(127 - E) for E <= 252: exact for every element that does not round to zero.
__device__ __forceinline__ float mx_inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }
// 2^(E - 127), NaN for 255.
__device__ __forceinline__ float mx_value(uint32_t scale) {
    return scale == 0 ? 0x1p-127f : scale == 255 ? __builtin_nanf("") : __uint_as_float(scale << 23);
}

typedef short s2 __attribute__((ext_vector_type(2)));

// Eight elements of a block with scale byte `scale` (255: zeros).
__device__ __forceinline__ uint32_t fp4_of(const Eight &e, uint32_t scale) {
    if (scale == 255u) return 0u;
    const float by = mx_inverse(scale);
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, e.v[0] * by, e.v[1] * by, 1.0f, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, e.v[2] * by, e.v[3] * by, 1.0f, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, e.v[4] * by, e.v[5] * by, 1.0f, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, e.v[6] * by, e.v[7] * by, 1.0f, 3);
    return word;
}
__device__ __forceinline__ u2 fp8_of(const Eight &e, uint32_t scale) {
    if (scale == 255u) return u2{0u, 0u};
    const float by = mx_inverse(scale);
    float v[8];  // the conversion does not cut at the largest element
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_fmed3f(e.v[i] * by, -448.0f, 448.0f);
    u2 word;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
        word[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
    }
    return word;
}

// The largest of four neighbouring lanes (lanes 4i to 4i + 3, all of which take part).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));  // lanes 1 0 3 2
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));  // 2 3 0 1
}

// Four neighbouring lanes hold a block, eight elements each (all four take part).  Returns its scale byte.
template <bool FP8>
__device__ __forceinline__ uint32_t block_scale(const Eight &e) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, magnitude(e.v[i]));
    return mx_scale<FP8>(quad_max(largest));
}

// Values of eight elements.
__device__ __forceinline__ Eight fp4_values(uint32_t word, float scale) {
    Eight e;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // e2m1 bits are those of an fp32 whose exponent runs from -1 (and the subnormal 0.5): 2^126 corrects the bias
        // of both (a product, exact also for the subnormal).
        const uint32_t code = word >> (4 * i);
        e.v[i] = __uint_as_float((code & 8u) << 28 | (code & 7u) << 22) * 0x1p126f * scale;
    }
    return e;
}
__device__ __forceinline__ Eight fp8_values(u2 word, float scale) {
    Eight e;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        e.v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(word[i], 0) * scale;
        e.v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(word[i], 1) * scale;
        e.v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(word[i], 2) * scale;
        e.v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(word[i], 3) * scale;
    }
    return e;
}

// Arguments of quantising and reading back (qxt_mx_quantize.hip), and their checks and launch.
struct MxRows {
    char *x;
    int64_t x_stride;
    uint32_t type;
    char *values;
    int64_t values_stride;
    uint8_t *scales;
    int64_t scales_stride;
    uint32_t scale_pad;  // bytes to clear after a row's last scale
    uint32_t pieces;     // of eight elements, of all rows
    FastDiv row;         // by the pieces of a row
};
int run_mx(bool quantize, MxRows &a, uint32_t rows, uint32_t columns, uint32_t format, void *stream);

}  // namespace qxt
