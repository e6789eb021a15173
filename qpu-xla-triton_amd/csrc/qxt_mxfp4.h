// Shared by the kernels of linears over microscaling 4-bit weights: arguments,
// the scaled matrix instruction, the gate functions and the store of results.
#pragma once

#include <type_traits>

#include "qxt_mx.h"

namespace qxt {

struct MxOperand {
    const char *values;
    int64_t stride;
    const uint8_t *scales;
    int64_t scale_stride;
};

struct MxLinearArgs {
    MxOperand a;     // activations [m, blocks]
    MxOperand w[2];  // weights [n, blocks]; the second one: up, of a gated product
    const float *bias;
    char *y;
    int64_t y_stride;
    uint8_t *y_scales;
    int64_t y_scale_stride;
    uint32_t m, n, blocks;
    uint32_t out_kind, gate;
    uint32_t vec_out;  // y's rows are aligned to 16 bytes
    uint32_t a_words;  // activations' rows of scales are words
    // Tile kernels that split K: every split's sums, fp32 [splits, weights, m, part_row].
    float *parts;
    uint32_t part_row, splits, split_steps;  // split_steps: K / 128 of a split, a multiple of four
};

typedef int i8 __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

// How activations enter the matrix instruction.  Among products of 8-bit elements it drops what lies more than 13 bits
// below the largest of eight neighbours' powers of two: up to 2^-10 of the sum of the eight magnitudes, and all of a result
// whose large products cancel.  The 8-bit elements therefore go through it in two parts, those of magnitude 2 and above and
// those below it (their bit 6 tells): within a part no product's last bit lies more than 13 bits below another's power of
// two, so nothing is dropped, at twice the matrix work.  (Products of 4-bit elements span 8 bits.)
enum Act { kAct4 = 0, kAct8 = 1 };

__device__ __forceinline__ int large_bytes(int word) {
    const uint32_t bit = (static_cast<uint32_t>(word) >> 6) & 0x01010101u;
    return static_cast<int>((bit << 8) - bit);  // 0xFF in each byte whose bit 6 is set
}

__device__ __forceinline__ i8 low_half(u4 v) {
    return i8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}
__device__ __forceinline__ i8 both_halves(u4 a, u4 b) {
    return i8{static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]),
              static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3])};
}

// Activation operands of one instruction, and acc += W A over 128 elements of K: 16 weight rows (4-bit) by 16 activation
// rows.  Lane l holds weight row l % 16 and activation row l % 16; of 4-bit rows the 32 elements of block l / 16, of 8-bit
// ones bytes 16 (l / 16) + [0, 16) and 64 + the same; and of both rows the scale of block l / 16.
// It receives weight rows 4 (l / 16) + [0, 4) of activation row l % 16.
template <int ACT>
struct ActPiece {
    i8 v, rest;
    __device__ __forceinline__ ActPiece(u4 a, u4 b) {
        if constexpr (ACT == kAct4) {
            v = low_half(a);
        } else {
            const i8 all = both_halves(a, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int large = large_bytes(all[i]);
                v[i] = all[i] & large;
                rest[i] = all[i] & ~large;
            }
        }
    }
};

template <int ACT>
__device__ __forceinline__ f4 mx_mfma(u4 w, const ActPiece<ACT> &a, f4 acc, uint32_t w_scales, uint32_t a_scales) {
    constexpr int form = ACT == kAct4 ? 4 : 0;
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(low_half(w), a.v, acc, 4, form, 0, w_scales, 0, a_scales);
    if constexpr (ACT == kAct8)
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(low_half(w), a.rest, acc, 4, form, 0, w_scales, 0, a_scales);
    return acc;
}

// SiLU from e = exp(-|g|), which cannot overflow: g / (1 + e), and g e / (1 + e) for negative g.  e comes through the
// hardware's power of two: the part of g log2(e) that its rounding loses is put back to first order, so the result is good
// to 11 units of 2^-24 for every g (without it, |g| units).  Below 2^-100 e is taken 2^64 times as large, since neither the
// power nor the product with g may fall below the normal numbers before the result does; beyond -200 it is zero.
__device__ __forceinline__ float gated(uint32_t gate, float g, float up) {
    if (gate == QXT_GATE_SILU) {
        const float a = fmaxf(-fabsf(g), -200.0f), t = a * 1.442695041f;
        const float rest = fmaf(a, 1.442695041f, -t) + a * 1.925963033e-8f;
        const bool far = t < -100.0f;
        const float e = __builtin_amdgcn_exp2f(far ? t + 64.0f : t) * (1.0f + 0.6931471806f * rest);
        const float f = (g < 0.0f ? g * e : g) * __builtin_amdgcn_rcpf(1.0f + e) * up;
        return far && g < 0.0f ? f * 0x1p-64f : f;
    }
    // (1 + erf would cancel for negative g.  What is left is the rounding of the argument, which erfc takes times g^2 + 1.)
    return 0.5f * g * erfcf(g * -0.7071067812f) * up;
}

// Source of what lies past a row's last block.
__device__ __constant__ const uint4 kZeroPiece = {};

// A value that is the same in all lanes, where the compiler cannot tell.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// 64 lanes' 16 or 4 bytes, from a wave-uniform address plus each lane's offset or from each lane's address, to LDS at `to`
// + 16 (or 4) * lane.  Inline
// assembly because the compiler waits for every such load in flight before it reads any of LDS; the waits here are the
// kernel's own.  There is no register output.
// (The compiler warns that it may not preserve m0; it has no other use for it here.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(uint64_t base, uint32_t offset, uint32_t to) {
    base = static_cast<uint64_t>(uniform(static_cast<uint32_t>(base >> 32))) << 32 | uniform(static_cast<uint32_t>(base));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(uniform(to)), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma16_from(const char *src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(uniform(to)), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma4_from(const char *src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(uniform(to)), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

// Wait until all but the wave's N youngest loads are done, and all of its LDS reads.
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void reads_done() {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void meet() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : : : "memory");
}

// How the tile kernels (qxt_mxfp4_tile.hip) take a product: the tile, and into how many parts K is split.
struct TilePlan {
    uint32_t tile, splits;
};
TilePlan plan_tiles(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, int act);
inline int act_of(uint32_t format) { return format == QXT_MX_FP4 ? kAct4 : kAct8; }
inline uint32_t part_row(uint32_t n) { return (n + 7) / 8 * 8; }
// Every row stride of values below 2^23 bytes; every row of scales aligned to four bytes and readable up to a multiple of
// four, with no NaN there; `a.parts` of the plan's size where it splits.
int mxfp4_tiles(MxLinearArgs &a, int act, bool gated, const TilePlan &plan, hipStream_t stream);

// Eight results of activation row m at columns n .. n + 7 as KIND; block kinds: four neighbouring lanes hold a whole block.
// `whole`: all eight columns lie in the row, and rows are aligned to 16 bytes.
template <int KIND>
__device__ __forceinline__ void store_results(const MxLinearArgs &a, uint32_t m, uint32_t n, bool whole, const Eight &e) {
    if constexpr (KIND == QXT_ROWS_MXFP8 || KIND == QXT_ROWS_MXFP4) {
        constexpr bool fp8 = KIND == QXT_ROWS_MXFP8;
        const uint32_t scale = block_scale<fp8>(e);
        if (m >= a.m || n >= a.n) return;  // (the row's length is a multiple of 32)
        char *row = a.y + m * a.y_stride;
        if constexpr (fp8) *reinterpret_cast<u2 *>(row + n) = fp8_of(e, scale);
        else *reinterpret_cast<uint32_t *>(row + n / 2) = fp4_of(e, scale);
        if (n % 32 == 0) a.y_scales[m * a.y_scale_stride + n / 32] = static_cast<uint8_t>(scale);
    } else {
        if (m >= a.m) return;
        char *row = a.y + m * a.y_stride;
        if (whole) {
            store_eight<true>(KIND, row, n, e);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (n + i >= a.n) return;
            if (KIND == QXT_TYPE_F32) reinterpret_cast<float *>(row)[n + i] = e.v[i];
            else if (KIND == QXT_TYPE_BF16) reinterpret_cast<bf16_t *>(row)[n + i] = static_cast<bf16_t>(e.v[i]);
            else reinterpret_cast<f16_t *>(row)[n + i] = static_cast<f16_t>(e.v[i]);
        }
    }
}

// `f` with the output's kind as a constant.
template <bool GATED, typename F>
__device__ __forceinline__ void with_kind(uint32_t kind, F &&f) {
    if (kind == QXT_TYPE_F32) return f(std::integral_constant<int, QXT_TYPE_F32>{});
    if (kind == QXT_TYPE_BF16) return f(std::integral_constant<int, QXT_TYPE_BF16>{});
    if (kind == QXT_TYPE_F16) return f(std::integral_constant<int, QXT_TYPE_F16>{});
    if constexpr (GATED) {
        if (kind == QXT_ROWS_MXFP8) return f(std::integral_constant<int, QXT_ROWS_MXFP8>{});
        f(std::integral_constant<int, QXT_ROWS_MXFP4>{});
    }
}

}  // namespace qxt
