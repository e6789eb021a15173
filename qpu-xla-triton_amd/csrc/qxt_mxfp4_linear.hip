// Linears over weights of microscaling 4-bit blocks: y = a W^T (+ bias), or the
// gated product f(a G^T) * (a U^T) of a feed-forward block, with activations in
// 8-bit or 4-bit blocks, on the scaled matrix instructions of gfx950.
//
// Every product of two elements is exact, a block's scales enter as powers of two
// and sums are fp32, so the only roundings are the sums' and the output's.
#include "qxt_mxfp4.h"

namespace qxt {
namespace {

// A workgroup owns 16 RT weight rows (of each weight) and 16 activation rows; its waves take every WAVES-th
// group of 512 elements of K, read their operands straight into registers, and add their sums through LDS.  Within a
// group lane (r, c) holds blocks 4c .. 4c + 3 of its rows, one for each of four instructions (K may be permuted as long
// as both operands agree), so that a word of scales serves all four.
template <int ACT, bool GATED, int RT, int WAVES, bool WORDS>
__global__ __launch_bounds__(64 * WAVES) void mxfp4_stream_kernel(MxLinearArgs a) {
    constexpr int W = GATED ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float sums[WAVES][W][RT][16][16];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, c = lane >> 4;
    const uint32_t column_tiles = (a.n + 16 * RT - 1) / (16 * RT);
    const uint32_t mt = blockIdx.x / column_tiles, nt = blockIdx.x - mt * column_tiles;
    const uint32_t m0 = mt * 16, n0 = nt * 16 * RT;
    const uint32_t arow = min(m0 + r, a.m - 1);  // rows past the last are computed from it and not stored
    const char *av = a.a.values + arow * a.a.stride;
    const uint8_t *as = a.a.scales + arow * a.a.scale_stride;
    const char *wv[W][RT];
    const uint8_t *ws[W][RT];
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const uint32_t row = min(n0 + 16 * t + r, a.n - 1);
            wv[w][t] = a.w[w].values + row * a.w[w].stride;
            ws[w][t] = a.w[w].scales + row * a.w[w].scale_stride;
        }
    auto piece = [](const char *p, bool in) { return in ? *reinterpret_cast<const u4 *>(p) : u4{0, 0, 0, 0}; };
    auto scale_word = [&](const uint8_t *p, uint32_t b) {
        if (WORDS) return b < a.blocks ? *reinterpret_cast<const uint32_t *>(p + b) : 0u;
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (b + j < a.blocks) word |= static_cast<uint32_t>(p[b + j]) << (8 * j);
        return word;
    };
    f4 acc[W][RT] = {};
    for (uint32_t first = 16 * wave; first < a.blocks; first += 16 * WAVES) {
        const uint32_t b0 = first + 4 * c;
        u4 wp[W][RT][4], ap[4][2];
        uint32_t wscale[W][RT];
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int t = 0; t < RT; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) wp[w][t][j] = piece(wv[w][t] + static_cast<size_t>(b0 + j) * 16, b0 + j < a.blocks);
                wscale[w][t] = scale_word(ws[w][t], b0);
            }
        const uint32_t ascale = scale_word(as, b0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (ACT != kAct4) {
                const uint32_t lo = first + 4 * (c >> 1) + j, hi = lo + 8;
                ap[j][0] = piece(av + static_cast<size_t>(lo) * 32 + 16 * (c & 1), lo < a.blocks);
                ap[j][1] = piece(av + static_cast<size_t>(hi) * 32 + 16 * (c & 1), hi < a.blocks);
            } else {
                ap[j][0] = piece(av + static_cast<size_t>(b0 + j) * 16, b0 + j < a.blocks);
                ap[j][1] = ap[j][0];
            }
        }
        auto step = [&](auto jc) {
            constexpr int j = decltype(jc)::value;
            const ActPiece<ACT> act(ap[j][0], ap[j][1]);
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    acc[w][t] = mx_mfma<ACT, j>(wp[w][t][j], act, acc[w][t], wscale[w][t], ascale);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
    }
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int t = 0; t < RT; ++t) *reinterpret_cast<f4 *>(&sums[wave][w][t][r][4 * c]) = acc[w][t];
    __syncthreads();
    // 2 RT threads an activation row, eight columns each.
    with_kind<ACT, GATED>(a.out_kind, [&](auto kind) {
        for (uint32_t i = threadIdx.x; i < 32 * RT; i += 64 * WAVES) {
            const uint32_t m = i / (2 * RT), at = i % (2 * RT), n = n0 + 8 * at;
            Eight e[W];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float *from = &sums[0][w][at / 2][m][8 * (at % 2)];
#pragma unroll
                for (int x = 0; x < 8; ++x) e[w].v[x] = from[x];
                for (int s = 1; s < WAVES; ++s) {
                    from += W * RT * 256;
#pragma unroll
                    for (int x = 0; x < 8; ++x) e[w].v[x] += from[x];
                }
            }
            if constexpr (GATED) {
#pragma unroll
                for (int x = 0; x < 8; ++x) e[0].v[x] = gated(a.gate, e[0].v[x], e[1].v[x]);
            } else if (a.bias != nullptr) {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (n + x < a.n) e[0].v[x] += a.bias[n + x];
            }
            store_results<decltype(kind)::value>(a, m0 + m, n, a.vec_out && n + 8 <= a.n, e[0]);
        }
    });
}

template <int ACT, bool GATED>
int launch_stream(const MxLinearArgs &a, bool words, hipStream_t stream) {
    constexpr int RT = 2, WAVES = 8;
    const uint64_t grid = static_cast<uint64_t>((a.m + 15) / 16) * ((a.n + 16 * RT - 1) / (16 * RT));
    if (grid > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "mxfp4 linear: too many outputs");
    return launch("mxfp4_stream_kernel",
                  words ? mxfp4_stream_kernel<ACT, GATED, RT, WAVES, true> : mxfp4_stream_kernel<ACT, GATED, RT, WAVES, false>,
                  dim3(static_cast<uint32_t>(grid)), dim3(64 * WAVES), 0, stream, a);
}

// Scales in rows of words, zeros behind the last.
__global__ __launch_bounds__(256) void pad_scales_kernel(const uint8_t *from, int64_t stride, uint32_t blocks, uint32_t *to,
                                                         uint32_t words, uint32_t total, FastDiv row) {
    const uint32_t at = blockIdx.x * 256 + threadIdx.x;
    if (at >= total) return;
    const uint32_t y = fast_quotient(at, row), x = at - y * words;
    uint32_t word = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
        if (4 * x + j < blocks) word |= static_cast<uint32_t>(from[y * stride + 4 * x + j]) << (8 * j);
    to[at] = word;
}

template <int ACT>
int launch_act(const MxLinearArgs &a, bool is_gated, bool words, hipStream_t stream) {
    return is_gated ? launch_stream<ACT, true>(a, words, stream) : launch_stream<ACT, false>(a, words, stream);
}

int check_operand(const char *name, const MxOperand &o, uint32_t format, uint32_t rows, uint32_t blocks) {
    if (o.values == nullptr || o.scales == nullptr) return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(o.values, 16) || o.stride % 16) return fail(QXT_INVALID_ARGUMENT, "%s: values must be in rows aligned to 16 bytes", name);
    if (rows > 1 && (static_cast<size_t>(o.stride) < mx_row_bytes(format, blocks * kMxBlock) ||
                     static_cast<size_t>(o.scale_stride) < blocks))
        return fail(QXT_INVALID_ARGUMENT, "%s: a row stride is below the row", name);
    return QXT_OK;
}

MxOperand operand(const qxt_mx_matrix *m) {
    return {static_cast<const char *>(m->values), static_cast<int64_t>(m->row_stride), m->scales,
            static_cast<int64_t>(m->scales_row_stride)};
}

size_t up16(size_t bytes) { return (bytes + 15) / 16 * 16; }
uint32_t padded(uint32_t blocks) { return (blocks + 3) / 4 * 4; }

// More activation rows than this go to the tile kernels.
constexpr uint32_t kStreamRows = 16;

// The workspace: quantised activations (values, scales in rows of words), and for the tile kernels room for each
// operand's scales in rows of words, and the sums of the parts of K.
struct Workspace {
    size_t scales = 0, a_scales = 0, w_scales = 0, w_each = 0, parts = 0, bytes = 0;
    Workspace(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, uint32_t format, uint32_t out_kind, bool floats) {
        const size_t pad = padded(k / kMxBlock);
        if (floats) {
            scales = up16(m * mx_row_bytes(format, k));
            bytes = scales + up16(m * pad);
        }
        if (m <= kStreamRows) return;
        a_scales = bytes;
        if (!floats) bytes += up16(m * pad);
        w_scales = bytes;
        w_each = up16(n * pad);
        bytes += weights * w_each;
        parts = bytes;
        const TilePlan plan = plan_tiles(m, n, k, weights, act_of(format, out_kind));
        if (plan.splits > 1) bytes += static_cast<size_t>(plan.splits) * weights * m * part_row(n) * sizeof(float);
    }
};

struct Floats {
    const void *x;
    size_t stride;
    uint32_t type;
};

// Checks shared by the four entry points, then the launches.  `x`: activations in floats, quantised into the workspace.
int run_linear(MxLinearArgs &a, const Floats *x, uint32_t format, bool is_gated, uint32_t k, void *workspace,
               size_t workspace_bytes, void *stream) {
    const char *name = is_gated ? "mxfp4 gated" : "mxfp4 linear";
    if (!known_mx(format)) return fail(QXT_INVALID_ARGUMENT, "%s: unknown block format", name);
    if (k == 0 || k % kMxBlock || k > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "%s: K must be a positive multiple of 32", name);
    if (a.m > INT32_MAX / 32 || a.n > INT32_MAX / 32) return fail(QXT_INVALID_ARGUMENT, "%s: too many rows or columns", name);
    const bool blocks_out = a.out_kind == QXT_ROWS_MXFP8 || a.out_kind == QXT_ROWS_MXFP4;
    if (!known_type(a.out_kind) && !(is_gated && blocks_out))
        return fail(QXT_INVALID_ARGUMENT, "%s: unknown output type", name);
    if (blocks_out && a.n % kMxBlock) return fail(QXT_INVALID_ARGUMENT, "%s: blocks need columns in multiples of 32", name);
    if (is_gated && a.gate > QXT_GATE_GELU) return fail(QXT_INVALID_ARGUMENT, "%s: unknown gate function", name);
    if (x != nullptr && !known_type(x->type)) return fail(QXT_INVALID_ARGUMENT, "%s: unknown element type", name);
    a.blocks = k / kMxBlock;
    if (a.m == 0 || a.n == 0) return QXT_OK;
    if (a.y == nullptr || (blocks_out && a.y_scales == nullptr)) return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
    const Workspace room(a.m, a.n, k, is_gated ? 2 : 1, format, a.out_kind, x != nullptr);
    if (x != nullptr) {
        const size_t element = type_bytes(x->type);
        if (x->x == nullptr) return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
        if (!aligned(x->x, element) || x->stride % element || (a.m > 1 && x->stride < k * element))
            return fail(QXT_INVALID_ARGUMENT, "%s: bad strides or alignment", name);
        a.a.values = static_cast<const char *>(workspace);
        a.a.stride = static_cast<int64_t>(mx_row_bytes(format, k));
        a.a.scales = static_cast<const uint8_t *>(workspace) + room.scales;
        a.a.scale_stride = padded(a.blocks);
    }
    if (room.bytes != 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < room.bytes))
        return fail(QXT_INVALID_ARGUMENT, "%s: workspace too small or not aligned to 16 bytes", name);
    if (int rc = check_operand(name, a.a, format, a.m, a.blocks)) return rc;
    for (int w = 0; w < (is_gated ? 2 : 1); ++w)
        if (int rc = check_operand(name, a.w[w], QXT_MX_FP4, a.n, a.blocks)) return rc;
    const size_t out_align = blocks_out ? (a.out_kind == QXT_ROWS_MXFP8 ? 8 : 4) : type_bytes(a.out_kind);
    const size_t out_row = a.out_kind == QXT_ROWS_MXFP8 ? a.n : a.out_kind == QXT_ROWS_MXFP4 ? a.n / 2 : a.n * type_bytes(a.out_kind);
    if (!aligned(a.y, out_align) || static_cast<size_t>(a.y_stride) % out_align || (a.bias != nullptr && !aligned(a.bias, 4)) ||
        (a.m > 1 && (static_cast<size_t>(a.y_stride) < out_row ||
                     (blocks_out && static_cast<size_t>(a.y_scale_stride) < a.n / kMxBlock))))
        return fail(QXT_INVALID_ARGUMENT, "%s: bad strides or alignment", name);
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;
    a.vec_out = aligned(a.y, 16) && a.y_stride % 16 == 0;
    if (x != nullptr) {
        MxRows rows{};
        rows.x = static_cast<char *>(const_cast<void *>(x->x));
        rows.x_stride = static_cast<int64_t>(x->stride);
        rows.type = x->type;
        rows.values = const_cast<char *>(a.a.values);
        rows.values_stride = a.a.stride;
        rows.scales = const_cast<uint8_t *>(a.a.scales);
        rows.scales_stride = a.a.scale_stride;
        rows.scale_pad = static_cast<uint32_t>(a.a.scale_stride) - a.blocks;
        if (int rc = run_mx(true, rows, a.m, k, format, stream)) return rc;
    }
    const hipStream_t s = as_stream(stream);
    const int act = act_of(format, a.out_kind);
    constexpr int64_t kTileStride = 1 << 23;
    const bool tiles = a.m > kStreamRows && a.a.stride < kTileStride && a.w[0].stride < kTileStride && a.w[1].stride < kTileStride;
    bool words = true;  // every row of scales in words
    for (int o = 0; o < (is_gated ? 3 : 2); ++o) {
        MxOperand &operand = o == 0 ? a.a : a.w[o - 1];
        if (o == 0 && x != nullptr) continue;  // written so
        if (a.blocks % 4 == 0 && aligned(operand.scales, 4) && operand.scale_stride % 4 == 0) continue;
        words = false;
        if (!tiles) break;
        const uint32_t rows = o == 0 ? a.m : a.n, row = padded(a.blocks) / 4;
        if (static_cast<uint64_t>(rows) * row > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "%s: too many blocks", name);
        uint8_t *to = static_cast<uint8_t *>(workspace) + (o == 0 ? room.a_scales : room.w_scales + (o - 1) * room.w_each);
        if (int rc = launch("pad_scales_kernel", pad_scales_kernel, dim3((rows * row + 255) / 256), dim3(256), 0, s, operand.scales,
                            operand.scale_stride, a.blocks, reinterpret_cast<uint32_t *>(to), row, rows * row, fast_div(row)))
            return rc;
        operand.scales = to;
        operand.scale_stride = 4 * row;
    }
    if (tiles) {
        a.parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + room.parts);
        return mxfp4_tiles(a, act, is_gated, plan_tiles(a.m, a.n, k, is_gated ? 2 : 1, act), s);
    }
    words = words && a.blocks % 4 == 0;
    switch (act) {
        case kAct4: return launch_act<kAct4>(a, is_gated, words, s);
        case kAct8: return launch_act<kAct8>(a, is_gated, words, s);
        default: return launch_act<kAct8Parts>(a, is_gated, words, s);
    }
}

MxLinearArgs linear_args(const qxt_mx_matrix *w, const qxt_mx_matrix *up, void *y, size_t ldy, uint32_t kind, uint32_t m, uint32_t n) {
    MxLinearArgs a{};
    a.w[0] = operand(w);
    if (up != nullptr) a.w[1] = operand(up);
    a.y = static_cast<char *>(y);
    a.y_stride = static_cast<int64_t>(ldy);
    a.out_kind = kind;
    a.m = m;
    a.n = n;
    return a;
}

}  // namespace
}  // namespace qxt

using namespace qxt;

extern "C" {

size_t qxt_mxfp4_linear_workspace(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, uint32_t format, uint32_t floats,
                                  uint32_t out_kind) {
    if (!known_mx(format) || k == 0 || k % kMxBlock || weights == 0 || weights > 2 || m == 0 || n == 0) return 0;
    return Workspace(m, n, k, weights, format, out_kind, floats != 0).bytes;
}

int qxt_mxfp4_gemm(const qxt_mx_matrix *a, uint32_t format, const qxt_mx_matrix *w, const float *bias, void *y, size_t ldy,
                   uint32_t y_type, uint32_t m, uint32_t n, uint32_t k, void *workspace, size_t workspace_bytes, void *stream) {
    if (a == nullptr || w == nullptr) return fail(QXT_INVALID_ARGUMENT, "mxfp4 linear: null pointer");
    MxLinearArgs args = linear_args(w, nullptr, y, ldy, y_type, m, n);
    args.a = operand(a);
    args.bias = bias;
    return run_linear(args, nullptr, format, false, k, workspace, workspace_bytes, stream);
}

int qxt_mxfp4_linear(const void *x, size_t ldx, uint32_t x_type, uint32_t format, const qxt_mx_matrix *w, const float *bias,
                     void *y, size_t ldy, uint32_t y_type, uint32_t m, uint32_t n, uint32_t k, void *workspace,
                     size_t workspace_bytes, void *stream) {
    if (w == nullptr) return fail(QXT_INVALID_ARGUMENT, "mxfp4 linear: null pointer");
    MxLinearArgs args = linear_args(w, nullptr, y, ldy, y_type, m, n);
    args.bias = bias;
    const Floats floats{x, ldx, x_type};
    return run_linear(args, &floats, format, false, k, workspace, workspace_bytes, stream);
}

int qxt_mxfp4_gated_gemm(const qxt_mx_matrix *a, uint32_t format, const qxt_mx_matrix *gate, const qxt_mx_matrix *up,
                         uint32_t gate_function, void *h, size_t ldh, uint8_t *h_scales, size_t ldhs, uint32_t h_kind,
                         uint32_t m, uint32_t n, uint32_t k, void *workspace, size_t workspace_bytes, void *stream) {
    if (a == nullptr || gate == nullptr || up == nullptr) return fail(QXT_INVALID_ARGUMENT, "mxfp4 gated: null pointer");
    MxLinearArgs args = linear_args(gate, up, h, ldh, h_kind, m, n);
    args.a = operand(a);
    args.gate = gate_function;
    args.y_scales = h_scales;
    args.y_scale_stride = static_cast<int64_t>(ldhs);
    return run_linear(args, nullptr, format, true, k, workspace, workspace_bytes, stream);
}

int qxt_mxfp4_gated_linear(const void *x, size_t ldx, uint32_t x_type, uint32_t format, const qxt_mx_matrix *gate,
                           const qxt_mx_matrix *up, uint32_t gate_function, void *h, size_t ldh, uint8_t *h_scales,
                           size_t ldhs, uint32_t h_kind, uint32_t m, uint32_t n, uint32_t k, void *workspace,
                           size_t workspace_bytes, void *stream) {
    if (gate == nullptr || up == nullptr) return fail(QXT_INVALID_ARGUMENT, "mxfp4 gated: null pointer");
    MxLinearArgs args = linear_args(gate, up, h, ldh, h_kind, m, n);
    args.gate = gate_function;
    args.y_scales = h_scales;
    args.y_scale_stride = static_cast<int64_t>(ldhs);
    const Floats floats{x, ldx, x_type};
    return run_linear(args, &floats, format, true, k, workspace, workspace_bytes, stream);
}

}  // extern "C"
