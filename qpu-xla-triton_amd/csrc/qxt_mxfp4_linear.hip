// Linears over weights of microscaling 4-bit blocks: y = a W^T (+ bias), or the
// gated product f(a G^T) * (a U^T) of a feed-forward block, with activations in
// 8-bit or 4-bit blocks, on the scaled matrix instructions of gfx950.
//
// Every product of two elements is exact, a block's scales enter as powers of two
// and sums are fp32, so the only roundings are the sums' and the output's.
#include "qxt_mxfp4.h"

namespace qxt {
namespace {

// Few activation rows: bound by the weights' bytes.  A workgroup owns 16 RT rows of each weight and all of the (at most 16)
// activation rows, which lie in LDS for the whole of K, and its waves take every WAVES-th unit of 256 elements of K: 128
// bytes of each weight row, a cache line, fetched by DMA into the wave's own LDS buffer, where it lies so that the reads of
// a piece (16 bytes) over 16 rows touch all banks.  A wave requests its next unit once it has read one into registers, and
// waits for nothing but its own loads until the sums of all are added up: what is in flight meanwhile are the other waves'
// units (two buffers a wave leave room for fewer workgroups: one row, K = 14336, N = 4096 8.6 -> 8.9 us, gated K = 4096,
// N = 14336 14.1 -> 14.7 us).  Float activations come into LDS as they are and are quantised there, by every
// workgroup for itself: less than a launch where they are few (one row of bf16, K = N = 4096 5.3 us, from blocks 4.8; a
// launch takes 2.9).  Activations too are fetched by DMA, ahead of the first
// weights: waiting for a load into registers would wait for every weight requested after it.
// Measured: one row, gated, K = 4096, N = 14336 14.1 us (4.4 TB/s); one weight, the same sizes 8.4 (3.7), eight rows 9.7; K
// = 2048, N = 5632 4.3.  What the short ones take beyond their bytes is a launch, two waits for memory and the waves' sums.
struct Floats {
    const char *x;
    int64_t stride;
    uint32_t type;
};

// LDS of the activations: rows of whole units and 16 bytes more (so that rows start in different banks), then their scales.
struct ActRows {
    uint32_t row, scale_row, scales, bytes;
};
template <int ACT>
__host__ __device__ inline ActRows act_rows(uint32_t m, uint32_t blocks) {
    const uint32_t units = (blocks + 7) / 8;
    ActRows r;
    r.row = units * (ACT == kAct4 ? 128 : 256) + 16;
    r.scale_row = units * 8 + 4;
    r.scales = m * r.row;
    r.bytes = (r.scales + m * r.scale_row + 15) / 16 * 16;
    return r;
}

// Bytes of a float row in LDS.
__host__ __device__ inline uint32_t float_row(uint32_t type, uint32_t blocks) { return blocks * (type == QXT_TYPE_F32 ? 128 : 64); }

template <int ACT, bool GATED, bool FLOATS, bool WORDS, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mxfp4_stream_kernel(MxLinearArgs a, Floats f) {
    constexpr int W = GATED ? 2 : 1, TILES = W * RT, THREADS = 64 * WAVES;
    constexpr int DATA = 2 * TILES, SCALES = WORDS ? (TILES + 1) / 2 : 0, LOADS = DATA + SCALES;  // loads of a unit
    constexpr uint32_t kSlot = TILES * 2048 + (TILES + 1) / 2 * 256;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x * 16 * RT, blocks = a.blocks, units = (blocks + 7) / 8;
    const ActRows rows = act_rows<ACT>(a.m, blocks);
    const uint32_t slot = rows.bytes + wave * kSlot;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)));

    // Rows of `bytes` (a multiple of 16) to LDS, `pitch` apart: the waves take 1024 bytes in turn.
    auto fetch_rows = [&](const char *src, int64_t stride, uint32_t bytes, uint32_t to, uint32_t pitch) {
        const uint32_t loads = (bytes + 1023) / 1024;
        uint32_t row = 0, at = wave;
        while (at >= loads && row < a.m) at -= loads, ++row;
        while (row < a.m) {
            const uint32_t byte = at * 1024 + lane * 16;
            if (byte < bytes) dma16_from(src + row * stride + byte, lds0 + to + row * pitch + at * 1024);
            at += WAVES;
            while (at >= loads && row < a.m) at -= loads, ++row;
        }
    };
    const uint32_t raw = rows.bytes + WAVES * kSlot, raw_row = FLOATS ? float_row(f.type, blocks) : 0;
    if constexpr (FLOATS) {
        fetch_rows(f.x, f.stride, raw_row, raw, raw_row);
    } else {
        if (a.a_words) {
            for (uint32_t row = 0; row < a.m; ++row)
                for (uint32_t at = wave * 64; at < blocks / 4; at += THREADS)
                    if (at + lane < blocks / 4)
                        dma4_from(reinterpret_cast<const char *>(a.a.scales + row * a.a.scale_stride + (at + lane) * 4),
                                  lds0 + rows.scales + row * rows.scale_row + at * 4);
        } else {  // through registers: nothing else is in flight yet
            for (uint32_t i = threadIdx.x; i < a.m * blocks; i += THREADS) {
                const uint32_t row = i / blocks, at = i - row * blocks;
                lds[rows.scales + row * rows.scale_row + at] = static_cast<char>(a.a.scales[row * a.a.scale_stride + at]);
            }
        }
        fetch_rows(a.a.values, a.a.stride, blocks * (ACT == kAct4 ? 16 : 32), 0, rows.row);
    }

    // A unit's weights: a load is eight rows of 128 bytes; its scales: a load is 32 rows of eight bytes.
    const uint32_t wrow = lane / 8, wpiece = (lane % 8) ^ wrow;
    const char *w_from[TILES][2];
    const uint8_t *s_from[(TILES + 1) / 2];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const MxOperand &o = a.w[t % W];
            w_from[t][h] = o.values + min(n0 + t / W * 16 + h * 8 + wrow, a.n - 1) * o.stride + wpiece * 16;
        }
#pragma unroll
    for (int i = 0; i < (TILES + 1) / 2; ++i) {
        const uint32_t row = min(i * 32 + lane / 2, TILES * 16 - 1u), t = row / 16;
        const uint32_t at = min(n0 + t / W * 16 + row % 16, a.n - 1);
        s_from[i] = a.w[0].scales + at * a.w[0].scale_stride;
        if (W == 2 && t % 2 == 1) s_from[i] = a.w[1].scales + at * a.w[1].scale_stride;
    }
    auto fetch = [&](uint32_t unit) {
        const bool whole = 8 * unit + 8 <= blocks;
        const char *zero = reinterpret_cast<const char *>(&kZeroPiece);
#pragma unroll
        for (int i = 0; i < (TILES + 1) / 2; ++i) {
            const uint32_t block = 8 * unit + lane % 2 * 4, at = slot + TILES * 2048 + i * 256;
            if constexpr (WORDS) {
                const char *src = reinterpret_cast<const char *>(s_from[i] + block);
                dma4_from(block < blocks ? src : zero, lds0 + at);
            } else {
                uint32_t word = 0;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (block + j < blocks) word |= static_cast<uint32_t>(s_from[i][block + j]) << (8 * j);
                *reinterpret_cast<uint32_t *>(lds + at + lane * 4) = word;
            }
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char *src = w_from[t][h] + unit * 128ull;
                dma16_from(whole || 8 * unit + wpiece < blocks ? src : zero, lds0 + slot + t * 2048 + h * 1024);
            }
    };
    if (wave < units) {
        fetch(wave);
        landed<LOADS>();  // the activations: only the weights are left in flight
    } else {
        landed<0>();
    }
    if constexpr (FLOATS) {
        meet();
        for (uint32_t row = 0; row < a.m; ++row) {
            const char *from = lds + raw + row * raw_row;
            char *to = lds + row * rows.row;
            for (uint32_t at = threadIdx.x; at < blocks * 4; at += THREADS) {  // four neighbouring threads a block
                const Eight e = load_eight<true>(f.type, from, at * 8);
                const uint32_t scale = block_scale<ACT != kAct4>(e);
                if constexpr (ACT == kAct4) *reinterpret_cast<uint32_t *>(to + at * 4) = fp4_of(e, scale);
                else *reinterpret_cast<u2 *>(to + at * 8) = fp8_of(e, scale);
                if (at % 4 == 0) lds[rows.scales + row * rows.scale_row + at / 4] = static_cast<char>(scale);
            }
        }
    }
    // Zeros from the last block to the end of its unit.
    const uint32_t pad = units * 8 - blocks, block_bytes = ACT == kAct4 ? 16 : 32;
    if (threadIdx.x < a.m * 8 && threadIdx.x % 8 < pad) {
        const uint32_t row = threadIdx.x / 8, block = blocks + threadIdx.x % 8;
        char *to = lds + row * rows.row + block * block_bytes;
        *reinterpret_cast<u4 *>(to) = u4{0, 0, 0, 0};
        if (ACT != kAct4) *reinterpret_cast<u4 *>(to + 16) = u4{0, 0, 0, 0};
        lds[rows.scales + row * rows.scale_row + block] = 0;
    }
    __builtin_amdgcn_sched_barrier(0);
    reads_done();
    meet();

    const uint32_t arow = min(r, a.m - 1);  // rows past the last are computed from it and not stored
    const char *a_at = lds + arow * rows.row + c * 16;
    const char *as_at = lds + rows.scales + arow * rows.scale_row + c;
    f4 acc[TILES] = {};
    for (uint32_t unit = wave; unit < units; unit += WAVES) {
        landed<0>();
        const char *from = lds + slot;
        u4 w[TILES][2], lo[2], hi[2];
        uint32_t wscale[TILES][2], ascale[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t step = 2 * unit + u;
            lo[u] = *reinterpret_cast<const u4 *>(a_at + step * (ACT == kAct4 ? 64 : 128));
            hi[u] = ACT == kAct4 ? lo[u] : *reinterpret_cast<const u4 *>(a_at + step * 128 + 64);
            ascale[u] = *reinterpret_cast<const uint8_t *>(as_at + step * 4);
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                w[t][u] = *reinterpret_cast<const u4 *>(from + t * 2048 + r * 128 + ((4 * u + c) ^ (r % 8)) * 16);
                wscale[t][u] = *reinterpret_cast<const uint8_t *>(from + TILES * 2048 + t * 128 + r * 8 + 4 * u + c);
            }
        }
        reads_done();
        if (unit + WAVES < units) fetch(unit + WAVES);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const ActPiece<ACT> act(lo[u], hi[u]);
#pragma unroll
            for (int t = 0; t < TILES; ++t) acc[t] = mx_mfma<ACT>(w[t][u], act, acc[t], wscale[t][u], ascale[u]);
        }
    }

    // The waves' sums lie where the units were.
    __syncthreads();
    float *sums = reinterpret_cast<float *>(lds + rows.bytes);  // [WAVES][TILES][16 rows][16 columns]
#pragma unroll
    for (int t = 0; t < TILES; ++t) *reinterpret_cast<f4 *>(sums + ((wave * TILES + t) * 16 + r) * 16 + 4 * c) = acc[t];
    __syncthreads();
    // 2 RT threads an activation row, eight columns each.
    with_kind<GATED>(a.out_kind, [&](auto kind) {
        for (uint32_t i = threadIdx.x; i < a.m * 2 * RT; i += THREADS) {
            const uint32_t m = i / (2 * RT), at = i % (2 * RT), n = n0 + 8 * at;
            Eight e[W];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float *from = sums + ((at / 2 * W + w) * 16 + m) * 16 + 8 * (at % 2);
                f4 x = {}, y = {};
#pragma unroll
                for (int s = 0; s < WAVES; ++s) {
                    x += *reinterpret_cast<const f4 *>(from + s * TILES * 256);
                    y += *reinterpret_cast<const f4 *>(from + s * TILES * 256 + 4);
                }
                e[w] = Eight{{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}};
            }
            if constexpr (GATED) {
#pragma unroll
                for (int x = 0; x < 8; ++x) e[0].v[x] = gated(a.gate, e[0].v[x], e[1].v[x]);
            } else if (a.bias != nullptr) {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (n + x < a.n) e[0].v[x] += a.bias[n + x];
            }
            store_results<decltype(kind)::value>(a, m, n, a.vec_out && n + 8 <= a.n, e[0]);
        }
    });
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

template <int ACT, bool GATED, int RT, int WAVES>
constexpr size_t stream_lds(const MxLinearArgs &a, const Floats *f) {
    constexpr uint32_t tiles = RT * (GATED ? 2 : 1), slot = tiles * 2048 + (tiles + 1) / 2 * 256;
    static_assert(slot >= tiles * 1024, "the sums lie where the units were");
    return act_rows<ACT>(a.m, a.blocks).bytes + WAVES * slot + (f != nullptr ? a.m * float_row(f->type, a.blocks) : 0);
}

template <int ACT, bool GATED, int RT, int WAVES>
int launch_stream(const MxLinearArgs &a, const Floats *f, bool words, hipStream_t stream) {
    auto kernel = f != nullptr ? (words ? mxfp4_stream_kernel<ACT, GATED, true, true, RT, WAVES>
                                        : mxfp4_stream_kernel<ACT, GATED, true, false, RT, WAVES>)
                               : (words ? mxfp4_stream_kernel<ACT, GATED, false, true, RT, WAVES>
                                        : mxfp4_stream_kernel<ACT, GATED, false, false, RT, WAVES>);
    return launch("mxfp4_stream_kernel", kernel, dim3((a.n + 16 * RT - 1) / (16 * RT)), dim3(64 * WAVES),
                  stream_lds<ACT, GATED, RT, WAVES>(a, f), stream, a, f != nullptr ? *f : Floats{});
}

// Which rows and waves.  Gated products hold 32 rows of each weight, for whole blocks of results.  A single weight of many
// columns, or of a short K, in 32 rows by four waves (one row, K = 4096, N = 14336 8.4 us, with 16 rows by eight waves 9.8;
// K = 2048, N = 5632 4.3, 4.6), else in 16 rows by eight waves (K = 14336, N = 4096 8.5 us, with 32 rows by four 11.6; K =
// 4096 4.8, 5.8).
template <int ACT>
int launch_act(const MxLinearArgs &a, const Floats *f, bool is_gated, bool words, hipStream_t stream) {
    if (is_gated) return launch_stream<ACT, true, 2, 4>(a, f, words, stream);
    if (a.n >= 12288 || a.blocks <= 64) return launch_stream<ACT, false, 2, 4>(a, f, words, stream);
    return launch_stream<ACT, false, 1, 8>(a, f, words, stream);
}

constexpr uint32_t kMostK = 1u << 22;

int check_operand(const char *name, const MxOperand &o, uint32_t format, uint32_t rows, uint32_t blocks) {
    if (o.values == nullptr || o.scales == nullptr) return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!aligned(o.values, 16) || o.stride % 16) return fail(QXT_INVALID_ARGUMENT, "%s: values must be in rows aligned to 16 bytes", name);
    if (rows > 1 && static_cast<size_t>(o.stride) >= 1u << 23) return fail(QXT_INVALID_ARGUMENT, "%s: rows of values must lie less than 8 MiB apart", name);
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

// Activation rows that the streaming kernel takes: up to 16 of 48 KB, so that two workgroups of a single weight share a CU
// (of a gated product, whose weights take 34 KB, up to 46 KB), or as many as leave room for the weights of one where there
// are no more workgroups than CUs (a single weight in 16 rows a workgroup).  Four rows, K = 14336, N =
// 4096: 9.2 us, on tiles 13.2; eight 10.2, 13.2; sixteen of K = 4096 7.3, 8.2.  (With more workgroups than CUs, or few
// columns that parts of K spread over the CUs, tiles are faster: 16 rows, K = 4096, N = 14336 12.3 us, 16.3 here; K = 8192,
// N = 1024 8.1, 8.6.)
constexpr size_t kStreamBytes = 48 * 1024, kAloneBytes = 136 * 1024;
bool alone(uint32_t n, uint32_t weights) { return weights == 1 && n > 64 * 16 && n <= 256 * 16; }
// Bytes of float activations that every workgroup of it quantises for itself (in LDS, beside their blocks).  With a launch
// before it instead, K = 4096, N = 14336, bf16: one row 7.9 us, 9.8 with the launch, gated 13.6, 15.9; three rows 9.4, 10.1,
// gated 14.4, 16.0; four rows, at the limit, 10.5, 10.2, gated 21.3, 16.1 (one workgroup a CU); K = 2048, N = 5632, four
// rows 5.7, 6.5, eight 7.4, 7.1.
constexpr size_t kFusedBytes = 32 * 1024;
bool streams(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, uint32_t format) {
    const uint32_t blocks = k / kMxBlock;
    return m <= 16 && (format == QXT_MX_FP4 ? act_rows<kAct4>(m, blocks) : act_rows<kAct8>(m, blocks)).bytes <=
                          (alone(n, weights) ? kAloneBytes : kStreamBytes);
}
// x_kind: 0 for blocks, else 1 + the floats' type, with QXT_ROWS_ALIGNED where rows start at multiples of 16 bytes.
uint32_t kind_of(const Floats *x, uint32_t m) {
    if (x == nullptr) return 0;
    return 1 + x->type + (aligned(x->x, 16) && (m == 1 || x->stride % 16 == 0) ? QXT_ROWS_ALIGNED : 0);
}
bool fuses(uint32_t x_kind, uint32_t m, uint32_t n, uint32_t k, uint32_t weights, uint32_t format) {
    return (x_kind & QXT_ROWS_ALIGNED) != 0 && streams(m, n, k, weights, format) &&
           m * static_cast<size_t>(float_row((x_kind & ~QXT_ROWS_ALIGNED) - 1, k / kMxBlock)) <= kFusedBytes;
}

// The workspace: quantised activations (values, scales in rows of words), and for the tile kernels room for each
// operand's scales in rows of words, and the sums of the parts of K.
struct Workspace {
    size_t scales = 0, a_scales = 0, w_scales = 0, w_each = 0, parts = 0, bytes = 0;
    Workspace(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, uint32_t format, uint32_t x_kind) {
        const size_t pad = padded(k / kMxBlock);
        const bool floats = x_kind != 0;
        if (floats && !fuses(x_kind, m, n, k, weights, format)) {
            scales = up16(m * mx_row_bytes(format, k));
            bytes = scales + up16(m * pad);
        }
        if (streams(m, n, k, weights, format)) return;
        a_scales = bytes;
        if (!floats) bytes += up16(m * pad);
        w_scales = bytes;
        w_each = up16(n * pad);
        bytes += weights * w_each;
        parts = bytes;
        const TilePlan plan = plan_tiles(m, n, k, weights, act_of(format));
        if (plan.splits > 1) bytes += static_cast<size_t>(plan.splits) * weights * m * part_row(n) * sizeof(float);
    }
};

// Checks shared by the four entry points, then the launches.  `x`: activations in floats, quantised into the workspace.
int run_linear(MxLinearArgs &a, const Floats *x, uint32_t format, bool is_gated, uint32_t k, void *workspace,
               size_t workspace_bytes, void *stream) {
    const char *name = is_gated ? "mxfp4 gated" : "mxfp4 linear";
    if (!known_mx(format)) return fail(QXT_INVALID_ARGUMENT, "%s: unknown block format", name);
    if (k == 0 || k % kMxBlock || k >= kMostK) return fail(QXT_INVALID_ARGUMENT, "%s: K must be a positive multiple of 32 below 2^22", name);
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
    const uint32_t x_kind = kind_of(x, a.m), weights = is_gated ? 2 : 1;
    const Workspace room(a.m, a.n, k, weights, format, x_kind);
    if (x != nullptr) {
        const size_t element = type_bytes(x->type);
        if (x->x == nullptr) return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
        if (!aligned(x->x, element) || static_cast<size_t>(x->stride) % element ||
            (a.m > 1 && static_cast<size_t>(x->stride) < k * element))
            return fail(QXT_INVALID_ARGUMENT, "%s: bad strides or alignment", name);
    }
    const bool fused = fuses(x_kind, a.m, a.n, k, weights, format);
    if (x != nullptr && !fused) {
        a.a.values = static_cast<const char *>(workspace);
        a.a.stride = static_cast<int64_t>(mx_row_bytes(format, k));
        a.a.scales = static_cast<const uint8_t *>(workspace) + room.scales;
        a.a.scale_stride = padded(a.blocks);
    }
    if (room.bytes != 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < room.bytes))
        return fail(QXT_INVALID_ARGUMENT, "%s: workspace too small or not aligned to 16 bytes", name);
    if (!fused)
        if (int rc = check_operand(name, a.a, format, a.m, a.blocks)) return rc;
    for (uint32_t w = 0; w < weights; ++w)
        if (int rc = check_operand(name, a.w[w], QXT_MX_FP4, a.n, a.blocks)) return rc;
    const size_t out_align = blocks_out ? (a.out_kind == QXT_ROWS_MXFP8 ? 8 : 4) : type_bytes(a.out_kind);
    const size_t out_row = a.out_kind == QXT_ROWS_MXFP8 ? a.n : a.out_kind == QXT_ROWS_MXFP4 ? a.n / 2 : a.n * type_bytes(a.out_kind);
    if (!aligned(a.y, out_align) || static_cast<size_t>(a.y_stride) % out_align || (a.bias != nullptr && !aligned(a.bias, 4)) ||
        (a.m > 1 && (static_cast<size_t>(a.y_stride) < out_row ||
                     (blocks_out && static_cast<size_t>(a.y_scale_stride) < a.n / kMxBlock))))
        return fail(QXT_INVALID_ARGUMENT, "%s: bad strides or alignment", name);
    const RowSpan y{a.y, a.y_stride, a.m, out_row}, y_scales{blocks_out ? a.y_scales : nullptr, a.y_scale_stride, a.m, a.n / kMxBlock};
    auto clash = [&](const RowSpan &from) { return overlap(y, from) || overlap(y_scales, from); };
    auto clashes = [&](const MxOperand &o, uint32_t kind, uint32_t rows) {
        return clash({o.values, o.stride, rows, mx_row_bytes(kind, k)}) || clash({o.scales, o.scale_stride, rows, a.blocks});
    };
    if (overlap(y, y_scales) || clash({a.bias, 0, 1, a.n * sizeof(float)}) || clashes(a.w[0], QXT_MX_FP4, a.n) ||
        (is_gated && clashes(a.w[1], QXT_MX_FP4, a.n)) ||
        (x != nullptr ? clash({x->x, x->stride, a.m, k * type_bytes(x->type)}) : clashes(a.a, format, a.m)))
        return fail(QXT_INVALID_ARGUMENT, "%s: an output shares memory with another operand", name);
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;
    a.vec_out = aligned(a.y, 16) && a.y_stride % 16 == 0;
    if (x != nullptr && !fused) {
        MxRows rows{};
        rows.x = const_cast<char *>(x->x);
        rows.x_stride = x->stride;
        rows.type = x->type;
        rows.values = const_cast<char *>(a.a.values);
        rows.values_stride = a.a.stride;
        rows.scales = const_cast<uint8_t *>(a.a.scales);
        rows.scales_stride = a.a.scale_stride;
        rows.scale_pad = static_cast<uint32_t>(a.a.scale_stride) - a.blocks;
        if (int rc = run_mx(true, rows, a.m, k, format, stream)) return rc;
    }
    const hipStream_t s = as_stream(stream);
    const bool tiles = !streams(a.m, a.n, k, weights, format);
    bool words = true;  // the weights' rows of scales are in words
    for (uint32_t o = 0; o <= weights; ++o) {
        MxOperand &operand = o == 0 ? a.a : a.w[o - 1];
        if (o == 0 && (x != nullptr || !tiles)) continue;  // written so, or read byte by byte
        if (a.blocks % 4 == 0 && aligned(operand.scales, 4) && operand.scale_stride % 4 == 0) continue;
        words = false;
        if (!tiles) continue;
        const uint32_t rows = o == 0 ? a.m : a.n, row = padded(a.blocks) / 4;
        if (static_cast<uint64_t>(rows) * row > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "%s: too many blocks", name);
        uint8_t *to = static_cast<uint8_t *>(workspace) + (o == 0 ? room.a_scales : room.w_scales + (o - 1) * room.w_each);
        if (int rc = launch("pad_scales_kernel", pad_scales_kernel, dim3((rows * row + 255) / 256), dim3(256), 0, s, operand.scales,
                            operand.scale_stride, a.blocks, reinterpret_cast<uint32_t *>(to), row, rows * row, fast_div(row)))
            return rc;
        operand.scales = to;
        operand.scale_stride = 4 * row;
    }
    a.a_words = a.blocks % 4 == 0 && aligned(a.a.scales, 4) && a.a.scale_stride % 4 == 0;
    if (tiles) {
        a.parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + room.parts);
        const int act = act_of(format);
        return mxfp4_tiles(a, act, is_gated, plan_tiles(a.m, a.n, k, weights, act), s);
    }
    Floats f{};
    if (fused) f = *x;
    if (format == QXT_MX_FP4) return launch_act<kAct4>(a, fused ? &f : nullptr, is_gated, words, s);
    return launch_act<kAct8>(a, fused ? &f : nullptr, is_gated, words, s);
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

size_t qxt_mxfp4_linear_workspace(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, uint32_t format, uint32_t x_kind,
                                  uint32_t /* out_kind: every one takes the same */) {
    if (!known_mx(format) || k == 0 || k % kMxBlock || k >= kMostK || weights == 0 || weights > 2 || m == 0 || n == 0 ||
        (x_kind & ~QXT_ROWS_ALIGNED) > 1 + QXT_TYPE_F16)
        return 0;
    return Workspace(m, n, k, weights, format, x_kind).bytes;
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
    const Floats floats{static_cast<const char *>(x), static_cast<int64_t>(ldx), x_type};
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
    const Floats floats{static_cast<const char *>(x), static_cast<int64_t>(ldx), x_type};
    return run_linear(args, &floats, format, true, k, workspace, workspace_bytes, stream);
}

}  // extern "C"
