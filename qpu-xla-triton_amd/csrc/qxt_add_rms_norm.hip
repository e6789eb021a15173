// The residual's addition and the root-mean-square norm of its rows in one pass,
// written as floats or as the quantised rows that the next linear takes.
//
//   h = round(x + residual)                      (to the residual's type; h = x without one)
//   f = round32(1 / sqrt(mean(h^2) + epsilon))   (the sum of squares and the root in 64 bits)
//   y = round32(round32(h f) weight)
// and y is rounded to a float type, or quantised: int8 rows with one scale
// (qxt_quantize_rows_int8's rule), Q8_0 blocks (qxt_quantize_q8_0's), 8-bit or
// 4-bit microscaling blocks (qxt_quantize_mx's).  A code next to a border goes by
// y's last bits, so y is defined by its roundings: the sum in 64 bits makes f,
// and with it every code, the same in any order of summation.
//
// Bound by its bytes: a workgroup holds a row in registers between the load, the
// sum over the row and the store, so every input is read once.  Measured, with a residual: 4096 rows of 4096, bf16 to
// 8-bit blocks 26.8 us (4.4 TB/s), to bf16 27.6 (4.9), to int8 rows 32 (3.7: the maximum is a second wait for all waves),
// fp32 to 4-bit blocks 46.3 (4.5); 4096 of 8192, bf16 53.6 (5.0); 777 of 11008, fp16 21.7 (3.1); one row of 2048 2.8.
// Rows of more than 8192 take four pieces a thread, and of those the last load of x and of the residual passes through
// scratch (80 bytes a thread), because the branches on the type join behind it: x, the residual and the weights are waited
// for in turn.
#include "qxt_mx.h"

namespace qxt {
namespace {

struct NormArgs {
    const char *x;
    int64_t x_stride;
    uint32_t x_type;
    const char *residual;  // nullptr: none, and no sum
    int64_t residual_stride;
    uint32_t residual_type;
    char *sum;
    int64_t sum_stride;
    const float *weight;
    double epsilon;
    char *out;
    int64_t out_stride;
    char *scales;
    int64_t scales_stride;
    uint32_t width;
};

// 1 / sqrt(mean + epsilon) from the threads' sums, over the workgroup's waves in their order.  One wave computes it for all:
// the root and two divisions in 64 bits are a hundred instructions (4096 rows of
// 4096, bf16 to 8-bit blocks: by every wave 28.1 us, by one 26.8; of 8192, bf16 to bf16 56.2, 53.6).
__device__ __forceinline__ float row_factor(double v, const NormArgs &a, double *scratch, float *factor) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x < 64) {
        v = scratch[0];
        for (uint32_t w = 1; w < blockDim.x / 64; ++w) v += scratch[w];
        if (threadIdx.x == 0) *factor = static_cast<float>(1.0 / sqrt(v / static_cast<double>(a.width) + a.epsilon));
    }
    __syncthreads();
    return *factor;
}

__device__ __forceinline__ float row_max(float v, float *scratch) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
    for (uint32_t w = 1; w < blockDim.x / 64; ++w) v = fmaxf(v, scratch[w]);
    return v;
}

__device__ __forceinline__ float round_to(uint32_t type, float v) {
    if (type == QXT_TYPE_BF16) return static_cast<float>(static_cast<bf16_t>(v));
    if (type == QXT_TYPE_F16) return static_cast<float>(static_cast<f16_t>(v));
    return v;
}

// Eight codes of an int8 row through its scale's reciprocal where that is exact (qxt_common.h).
__device__ __forceinline__ u2 int8_of(const Eight &e, float s) {
    int q[8];
    if (s >= kRecipScaleMin) {
        const float r = 1.0f / s;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = quant_recip(e.v[i], s, r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = quant_div(e.v[i], s);
    }
    return u2{pack_bytes(q[0], q[1], q[2], q[3]), pack_bytes(q[4], q[5], q[6], q[7])};
}

// Eight elements of a 34-byte block at piece `at` of a row (four neighbouring lanes hold the block).
__device__ __forceinline__ void store_q8_0(char *row, uint32_t at, const Eight &e, bool in_row) {
    float largest = fabsf(e.v[0]);  // not from zero: a block that is all NaN has a scale of NaN
#pragma unroll
    for (int i = 1; i < 8; ++i) largest = fmaxf(largest, fabsf(e.v[i]));
    largest = fmaxf(largest, __shfl_xor(largest, 1, 4));
    largest = fmaxf(largest, __shfl_xor(largest, 2, 4));
    if (!in_row) return;
    float d, inverse;
    q8_0_scale(largest, d, inverse);
    char *block = row + static_cast<size_t>(at / 4) * Q8_0_BYTES;
    if (at % 4 == 0) *reinterpret_cast<uint16_t *>(block) = static_cast<uint16_t>(float_to_half_bits(d));
    uint16_t *codes = reinterpret_cast<uint16_t *>(block + 2 + 8 * (at % 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int lo = clamp127(rintf(e.v[2 * i] * inverse)), hi = clamp127(rintf(e.v[2 * i + 1] * inverse));
        codes[i] = static_cast<uint16_t>((lo & 0xFF) | (hi & 0xFF) << 8);
    }
}

// One row a workgroup, whose threads hold CH pieces of eight elements each: width a multiple of eight (of 32 for blocks),
// rows aligned to 16 bytes.
constexpr int kMostThreads = 1024;

template <int OUT, int CH>
__global__ __launch_bounds__(kMostThreads) void add_rms_norm_kernel(NormArgs a) {
    __shared__ double sums[kMostThreads / 64];
    __shared__ float maxima[kMostThreads / 64], shared_factor;
    const uint32_t row = blockIdx.x, pieces = a.width / 8, threads = blockDim.x;
    u4 xa[CH], xb[CH], ra[CH], rb[CH];
    // With one piece a thread every load is issued before any is used; a thread past the row re-reads its last piece.  Inputs are read once: past
    // the caches (4096 rows of 4096, bf16 to 8-bit blocks: 34 -> 31 us).
    auto load_row = [&](uint32_t type, const char *from, u4 (&lo)[CH], u4 (&hi)[CH]) {
        if (type == QXT_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const u4 *p = reinterpret_cast<const u4 *>(from + static_cast<size_t>(min(threadIdx.x + i * threads, pieces - 1)) * 32);
                lo[i] = __builtin_nontemporal_load(p);
                hi[i] = __builtin_nontemporal_load(p + 1);
            }
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i)
                lo[i] = __builtin_nontemporal_load(
                    reinterpret_cast<const u4 *>(from + static_cast<size_t>(min(threadIdx.x + i * threads, pieces - 1)) * 16));
        }
    };
    load_row(a.x_type, a.x + row * a.x_stride, xa, xb);
    if (a.residual != nullptr) load_row(a.residual_type, a.residual + row * a.residual_stride, ra, rb);
    float4 w[CH][2];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const float4 *p = reinterpret_cast<const float4 *>(a.weight + min(threadIdx.x + i * threads, pieces - 1) * 8);
        w[i][0] = p[0];
        w[i][1] = p[1];
    }
    Eight h[CH];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t at = threadIdx.x + i * threads;
        h[i] = eight_of(a.x_type, xa[i], xb[i]);
        if (a.residual != nullptr) {
            const Eight r = eight_of(a.residual_type, ra[i], rb[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i].v[e] = round_to(a.residual_type, h[i].v[e] + r.v[e]);
            if (at < pieces) store_eight<true>(a.residual_type, a.sum + row * a.sum_stride, at * 8, h[i]);
        }
        if (at < pieces) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double v = static_cast<double>(h[i].v[e]);
                sum = __builtin_fma(v, v, sum);
            }
        }
    }
    const float factor = row_factor(sum, a, sums, &shared_factor);
    char *out = a.out + row * a.out_stride;
    float largest = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const float by[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[i].v[e] = h[i].v[e] * factor * by[e];
            // (Only the row's own: what a thread past it re-read may be a sum stored in place by then.)
            if (OUT == QXT_ROWS_INT8 && threadIdx.x + i * threads < pieces) largest = fmaxf(largest, fabsf(h[i].v[e]));
        }
    }
    float scale = 0.0f;
    if constexpr (OUT == QXT_ROWS_INT8) {
        scale = row_scale(row_max(largest, maxima), true);
        if (threadIdx.x == 0) reinterpret_cast<float *>(a.scales)[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t at = threadIdx.x + i * threads;
        const bool in_row = at < pieces;
        if constexpr (OUT == QXT_ROWS_INT8) {
            if (in_row) *reinterpret_cast<u2 *>(out + static_cast<size_t>(at) * 8) = int8_of(h[i], scale);
        } else if constexpr (OUT == QXT_ROWS_Q8_0) {
            store_q8_0(out, at, h[i], in_row);
        } else if constexpr (OUT == QXT_ROWS_MXFP8 || OUT == QXT_ROWS_MXFP4) {
            constexpr bool fp8 = OUT == QXT_ROWS_MXFP8;
            const uint32_t shared = block_scale<fp8>(h[i]);
            if (in_row) {
                if constexpr (fp8) *reinterpret_cast<u2 *>(out + static_cast<size_t>(at) * 8) = fp8_of(h[i], shared);
                else *reinterpret_cast<uint32_t *>(out + static_cast<size_t>(at) * 4) = fp4_of(h[i], shared);
                if (at % 4 == 0) a.scales[row * a.scales_stride + at / 4] = static_cast<char>(shared);
            }
        } else {
            if (in_row) store_eight<true>(OUT, out, at * 8, h[i]);
        }
    }
}

// Any width and alignment: a thread walks over its elements, element threadIdx.x + 256 i, three times.  What it reads
// again it wrote itself (the sum), or nobody wrote.
template <typename F>
__device__ __forceinline__ void over_row(uint32_t padded, F &&f) {
    for (uint32_t i = threadIdx.x; i < padded; i += 256) f(i);
}
__device__ __forceinline__ float element(uint32_t type, const char *row, uint32_t i) {
    if (type == QXT_TYPE_F32) return reinterpret_cast<const float *>(row)[i];
    if (type == QXT_TYPE_BF16) return static_cast<float>(reinterpret_cast<const bf16_t *>(row)[i]);
    return static_cast<float>(reinterpret_cast<const f16_t *>(row)[i]);
}
__device__ __forceinline__ void put(uint32_t type, char *row, uint32_t i, float v) {
    if (type == QXT_TYPE_F32) reinterpret_cast<float *>(row)[i] = v;
    else if (type == QXT_TYPE_BF16) reinterpret_cast<bf16_t *>(row)[i] = static_cast<bf16_t>(v);
    else reinterpret_cast<f16_t *>(row)[i] = static_cast<f16_t>(v);
}

template <int OUT>
__global__ __launch_bounds__(256) void add_rms_norm_any_kernel(NormArgs a) {
    __shared__ double sums[4];
    __shared__ float maxima[4], shared_factor;
    const uint32_t row = blockIdx.x;
    const char *x = a.x + row * a.x_stride;
    const bool adds = a.residual != nullptr;
    const char *residual = a.residual + (adds ? row * a.residual_stride : 0);
    char *total = a.sum + (adds ? row * a.sum_stride : 0);
    double sum = 0.0;
    over_row(a.width, [&](uint32_t i) {
        float h = element(a.x_type, x, i);
        if (adds) {
            h = round_to(a.residual_type, h + element(a.residual_type, residual, i));
            put(a.residual_type, total, i, h);
        }
        sum = __builtin_fma(static_cast<double>(h), static_cast<double>(h), sum);
    });
    const float factor = row_factor(sum, a, sums, &shared_factor);
    auto y_at = [&](uint32_t i) {
        const float h = adds ? element(a.residual_type, total, i) : element(a.x_type, x, i);
        return h * factor * a.weight[i];
    };
    char *out = a.out + row * a.out_stride;
    float scale = 0.0f;
    if constexpr (OUT == QXT_ROWS_INT8) {
        float largest = 0.0f;
        over_row(a.width, [&](uint32_t i) { largest = fmaxf(largest, fabsf(y_at(i))); });
        scale = row_scale(row_max(largest, maxima), true);
        if (threadIdx.x == 0) reinterpret_cast<float *>(a.scales)[row] = scale;
    }
    over_row(a.width, [&](uint32_t i) {  // blocks: the width is a multiple of 32, so halves of a wave come and go together
        const float y = y_at(i);
        if constexpr (OUT == QXT_ROWS_INT8) {
            out[i] = static_cast<char>(quant_div(y, scale));
        } else if constexpr (OUT == QXT_ROWS_Q8_0) {
            float largest = fabsf(y), d, inverse;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) largest = fmaxf(largest, __shfl_xor(largest, off, 32));
            q8_0_scale(largest, d, inverse);
            char *block = out + static_cast<size_t>(i / 32) * Q8_0_BYTES;
            if (i % 32 == 0) *reinterpret_cast<uint16_t *>(block) = static_cast<uint16_t>(float_to_half_bits(d));
            block[2 + i % 32] = static_cast<char>(clamp127(rintf(y * inverse)));
        } else if constexpr (OUT == QXT_ROWS_MXFP8 || OUT == QXT_ROWS_MXFP4) {
            constexpr bool fp8 = OUT == QXT_ROWS_MXFP8;
            uint32_t largest = magnitude(y);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1)
                largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), off, 32)));
            const uint32_t shared = mx_scale<fp8>(largest);
            Eight e{};
            e.v[0] = y;
            e.v[1] = __shfl_xor(y, 1, 32);
            if constexpr (fp8) out[i] = static_cast<char>(fp8_of(e, shared)[0]);
            else if (i % 2 == 0) out[i / 2] = static_cast<char>(fp4_of(e, shared));
            if (i % 32 == 0) a.scales[row * a.scales_stride + i / 32] = static_cast<char>(shared);
        } else {
            put(OUT, out, i, y);
        }
    });
}

template <int OUT>
int launch_norm(const NormArgs &a, uint32_t rows, bool vec, hipStream_t stream) {
    const uint32_t pieces = a.width / 8;
    auto kernel = add_rms_norm_any_kernel<OUT>;
    uint32_t threads = 256;
    const char *name = "add_rms_norm_any_kernel";
    // One piece a thread as long as a workgroup's threads reach (4096 rows of 4096, bf16 to 8-bit blocks: 31 us with two
    // pieces or eight, 28 with one), and then four (2048 rows of 14336: 64 us with two, 56 with four).
    if (vec && pieces <= 4 * kMostThreads) {
        name = "add_rms_norm_kernel";
        const uint32_t each = pieces <= kMostThreads ? 1 : 4;
        threads = ((pieces + each - 1) / each + 63) / 64 * 64;
        kernel = each == 1 ? add_rms_norm_kernel<OUT, 1> : add_rms_norm_kernel<OUT, 4>;
    }
    // A launch has fewer than 2^32 threads (the runtime takes a larger one and runs what is left of it modulo that): more rows
    // take several.
    const uint32_t most = UINT32_MAX / threads;
    NormArgs part = a;
    for (uint32_t first = 0; first < rows; first += most) {
        part.x = a.x + first * a.x_stride;
        if (a.residual != nullptr) {
            part.residual = a.residual + first * a.residual_stride;
            part.sum = a.sum + first * a.sum_stride;
        }
        part.out = a.out + first * a.out_stride;
        if (a.scales != nullptr) part.scales = a.scales + first * (OUT == QXT_ROWS_INT8 ? 4 : a.scales_stride);
        if (int rc = launch(name, kernel, dim3(min(rows - first, most)), dim3(threads), 0, stream, part)) return rc;
    }
    return QXT_OK;
}

int run_norm(NormArgs &a, uint32_t out_kind, uint32_t rows, hipStream_t stream) {
    constexpr const char *name = "add rms norm";
    const uint32_t width = a.width;
    if (!known_type(a.x_type) || (a.residual != nullptr && !known_type(a.residual_type)) || out_kind > QXT_ROWS_MXFP4)
        return fail(QXT_INVALID_ARGUMENT, "%s: unknown element type", name);
    if (width == 0 || width > INT32_MAX / 8) return fail(QXT_INVALID_ARGUMENT, "%s: columns must be in [1, 2^28)", name);
    const bool blocks = out_kind >= QXT_ROWS_Q8_0, planes = out_kind != QXT_ROWS_Q8_0 && out_kind >= QXT_ROWS_INT8;
    if (blocks && width % 32) return fail(QXT_INVALID_ARGUMENT, "%s: blocks need columns in multiples of 32", name);
    if (!(a.epsilon >= 0.0)) return fail(QXT_INVALID_ARGUMENT, "%s: epsilon must not be negative", name);
    if (rows > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "%s: more than 2^31 rows", name);
    if (rows == 0) return QXT_OK;
    if (a.x == nullptr || a.weight == nullptr || a.out == nullptr || (a.residual != nullptr && a.sum == nullptr) ||
        (planes && a.scales == nullptr))
        return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
    const size_t x_size = type_bytes(a.x_type), r_size = type_bytes(a.residual_type);
    const size_t out_align = out_kind <= QXT_TYPE_F16 ? type_bytes(out_kind) : out_kind == QXT_ROWS_Q8_0 ? 2 : 1;
    const size_t out_row = out_kind <= QXT_TYPE_F16 ? width * type_bytes(out_kind)
                           : out_kind == QXT_ROWS_Q8_0 ? static_cast<size_t>(width / 32) * Q8_0_BYTES
                           : out_kind == QXT_ROWS_MXFP4 ? width / 2 : width;
    auto strides = [&](const void *p, int64_t stride, size_t align, size_t row) {
        return aligned(p, align) && static_cast<size_t>(stride) % align == 0 && (rows == 1 || static_cast<size_t>(stride) >= row);
    };
    if (!strides(a.x, a.x_stride, x_size, width * x_size) || !strides(a.out, a.out_stride, out_align, out_row) ||
        !aligned(a.weight, 4) || (out_kind == QXT_ROWS_INT8 && !aligned(a.scales, 4)) ||
        (out_kind >= QXT_ROWS_MXFP8 && !strides(a.scales, a.scales_stride, 1, width / 32)))
        return fail(QXT_INVALID_ARGUMENT, "%s: bad strides or alignment", name);
    if (a.residual != nullptr && (!strides(a.residual, a.residual_stride, r_size, width * r_size) ||
                                  !strides(a.sum, a.sum_stride, r_size, width * r_size)))
        return fail(QXT_INVALID_ARGUMENT, "%s: bad strides or alignment", name);
    // A thread writes floats only where it has read the element of that place itself: they may lie exactly over x or the
    // residual.
    const RowSpan inputs[2] = {{a.x, a.x_stride, rows, width * x_size}, {a.residual, a.residual_stride, rows, width * r_size}};
    const RowSpan sum{a.residual != nullptr ? a.sum : nullptr, a.sum_stride, rows, width * r_size}, weight{a.weight, 0, 1, width * sizeof(float)};
    const RowSpan out{a.out, a.out_stride, rows, out_row};
    const RowSpan scales{planes ? a.scales : nullptr, out_kind == QXT_ROWS_INT8 ? 4 : a.scales_stride, rows,
                         out_kind == QXT_ROWS_INT8 ? 4 : width / 32};
    auto clash = [&](const RowSpan &to, bool may_replace) {
        for (const RowSpan &from : inputs)
            if (overlap(to, from) && !(may_replace && to.at == from.at && to.bytes == from.bytes && (rows == 1 || to.stride == from.stride)))
                return true;
        return overlap(to, weight);
    };
    if (clash(sum, true) || clash(out, out_kind <= QXT_TYPE_F16) || clash(scales, false) || overlap(sum, out) || overlap(sum, scales) ||
        overlap(out, scales))
        return fail(QXT_INVALID_ARGUMENT, "%s: an output shares memory with another operand", name);
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;
    auto sixteen = [](const void *p, int64_t stride) { return aligned(p, 16) && stride % 16 == 0; };
    const size_t store = out_kind <= QXT_TYPE_F16 ? 16 : out_kind == QXT_ROWS_Q8_0 ? 2 : out_kind == QXT_ROWS_MXFP4 ? 4 : 8;
    const bool vec = width % 8 == 0 && sixteen(a.x, a.x_stride) && aligned(a.weight, 16) && aligned(a.out, store) &&
                     static_cast<size_t>(a.out_stride) % store == 0 &&
                     (a.residual == nullptr || (sixteen(a.residual, a.residual_stride) && sixteen(a.sum, a.sum_stride)));
    switch (out_kind) {
        case QXT_TYPE_F32: return launch_norm<QXT_TYPE_F32>(a, rows, vec, stream);
        case QXT_TYPE_BF16: return launch_norm<QXT_TYPE_BF16>(a, rows, vec, stream);
        case QXT_TYPE_F16: return launch_norm<QXT_TYPE_F16>(a, rows, vec, stream);
        case QXT_ROWS_INT8: return launch_norm<QXT_ROWS_INT8>(a, rows, vec, stream);
        case QXT_ROWS_Q8_0: return launch_norm<QXT_ROWS_Q8_0>(a, rows, vec, stream);
        case QXT_ROWS_MXFP8: return launch_norm<QXT_ROWS_MXFP8>(a, rows, vec, stream);
        default: return launch_norm<QXT_ROWS_MXFP4>(a, rows, vec, stream);
    }
}

}  // namespace
}  // namespace qxt

extern "C" {

int qxt_add_rms_norm(const void *x, size_t x_row_stride, uint32_t x_type, const void *residual,
                     size_t residual_row_stride, uint32_t residual_type, void *sum, size_t sum_row_stride,
                     const float *weight, double epsilon, void *out, size_t out_row_stride, void *scales,
                     size_t scales_row_stride, uint32_t out_kind, uint32_t rows, uint32_t columns, void *stream) {
    qxt::NormArgs a{};
    a.x = static_cast<const char *>(x);
    a.x_stride = static_cast<int64_t>(x_row_stride);
    a.x_type = x_type;
    a.residual = static_cast<const char *>(residual);
    a.residual_stride = static_cast<int64_t>(residual_row_stride);
    a.residual_type = residual_type;
    a.sum = static_cast<char *>(sum);
    a.sum_stride = static_cast<int64_t>(sum_row_stride);
    a.weight = weight;
    a.epsilon = epsilon;
    a.out = static_cast<char *>(out);
    a.out_stride = static_cast<int64_t>(out_row_stride);
    a.scales = static_cast<char *>(scales);
    a.scales_stride = static_cast<int64_t>(scales_row_stride);
    a.width = columns;
    return qxt::run_norm(a, out_kind, rows, qxt::as_stream(stream));
}

}  // extern "C"
