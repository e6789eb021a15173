// Linears over microscaling 4-bit weights for many rows: tiles of the result
// whose operands pass through LDS once for all the waves that share them.
//
// A workgroup of WN x WM waves owns 16 TW WN weight rows by 16 TA WM activation
// rows, each wave 16 TW by 16 TA of them as 16 x 16 x 128 products.  K advances
// 128 elements a stage through a ring of LDS buffers filled by DMA: a wave's
// 16-byte pieces land in lane order, so which piece a lane fetches decides the
// layout.  Rows of 64 bytes (4-bit) or 128 (8-bit) are fetched whole by
// neighbouring lanes, and piece p of row r lies at p ^ (r / 2 % 4) or p ^ (r % 8),
// so that the reads of one piece over 16 rows spread over the banks (0.9 conflicts
// are counted for each LDS instruction, of which about half read one byte of scales).
// A gated product takes the tiles of gate and up in turn, so that a wave holds both
// sums of a result.
//
// Measured: 4096 x 4096 x 14336 with 4-bit activations 166 us (2.9 PFLOP/s; matrix
// units 38 % busy), gated with 8-bit ones 627 us (1.5 PFLOP/s, each product in two
// parts; matrix units 62 % busy, vector units, which part them, 47 %).  With the rest taken out, at 8192 x 8192 x 8192 in 4 bits, the
// products alone take 59 % of the time and the fetches alone 52 % (33 clocks a KB on
// each CU); the two overlap in part only, since a fetch's writes and the waves' reads
// share LDS.
// 77 x 11008 x 4096: 12.4 us and 4.1 for joining four parts of K, against 4.8 for
// its bytes: two workgroups a CU of eleven stages each, which more parts, larger
// tiles or deeper rings do not make faster (16.3 to 17.5 us together).
#include "qxt_mxfp4.h"

namespace qxt {
namespace {

// Output tile (ty, tx) of a workgroup.  Workgroups go to the eight XCDs in turn, each with its own L2: every XCD takes a
// contiguous run of a grouped order (`gm` tile rows at a time, column by column), so that what it runs together shares
// panels.
__device__ __forceinline__ void xcd_tile(uint32_t id, uint32_t tm, uint32_t tn, uint32_t gm, uint32_t &ty, uint32_t &tx) {
    const uint32_t total = tm * tn, per = total / 8, more = total % 8, xcd = id % 8, local = id / 8;
    const uint32_t at = xcd < more ? xcd * (per + 1) + local : more * (per + 1) + (xcd - more) * per + local;
    const uint32_t group = at / (gm * tn), first = group * gm, rows = min(gm, tm - first), in = at - group * gm * tn;
    ty = first + in % rows;
    tx = in / rows;
}

template <int ACT, bool GATED, int TW, int TA, int WN, int WM, int SUB, int RING>
struct Tiles {
    static constexpr bool FP8 = ACT != kAct4;
    static constexpr int WAVES = WN * WM, THREADS = 64 * WAVES;
    static constexpr int BN = 16 * TW * WN, BM = 16 * TA * WM;  // weight rows (of both weights), activation rows
    static constexpr int W_ROW = 64 * SUB, A_ROW = (FP8 ? 128 : 64) * SUB;  // bytes of a row a stage
    static constexpr int W_BYTES = BN * W_ROW, A_BYTES = BM * A_ROW, STAGE = W_BYTES + A_BYTES;
    static constexpr int W_LOADS = W_BYTES / 1024, A_LOADS = A_BYTES / 1024, S_LOADS = (BN + BM + 63) / 64;
    static constexpr int W_EACH = W_LOADS / WAVES, A_EACH = A_LOADS / WAVES, S_EACH = (S_LOADS + WAVES - 1) / WAVES;
    static constexpr int LOADS = W_EACH + A_EACH;           // of each wave a stage, but for scales
    static constexpr int GROUP = 4 / SUB;                   // stages that share a row's 16 bytes of scales
    static constexpr int SCALES = S_LOADS * 1024;          // bytes of a group
    static constexpr int OUT = 16 * TW / (GATED ? 2 : 1);   // result columns of a wave
    static constexpr int OUT_ROW = OUT + 4;                 // floats, in LDS
    static constexpr int OPERANDS = RING * STAGE + 2 * SCALES, RESULTS = WAVES * 16 * OUT_ROW * 4;
    static constexpr int LDS = OPERANDS > RESULTS ? OPERANDS : RESULTS;
    static_assert(W_LOADS % WAVES == 0 && A_LOADS % WAVES == 0 && LDS <= 160 * 1024, "tile shape");
    static_assert(OUT % 32 == 0 && OUT <= 128, "a wave's results hold whole blocks, and 64 lanes at most 16 rows of them");
    static_assert(RING >= 2 && RING <= 3 && RING <= GROUP, "a group's scales are fetched with the last stage of the group before");
};

// Where piece p (16 bytes) of row r of a stage lies, in pieces from the row's start.
template <int ROW>
__device__ __forceinline__ uint32_t turned(uint32_t p, uint32_t r) {
    static_assert(ROW == 64 || ROW == 128, "");
    return ROW == 64 ? p ^ (r / 2 % 4) : p ^ (r % 8);
}

template <int ACT, bool GATED, int TW, int TA, int WN, int WM, int SUB, int RING>
__global__ __launch_bounds__(64 * WN * WM) void mxfp4_tile_kernel(MxLinearArgs a) {
    typedef Tiles<ACT, GATED, TW, TA, WN, WM, SUB, RING> T;
    __shared__ __attribute__((aligned(16))) char lds[T::LDS];
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
    constexpr uint32_t kColumns = T::BN / (GATED ? 2 : 1);  // result columns of the workgroup
    uint32_t ty, tx;
    const uint32_t tiles = gridDim.x / a.splits, split = blockIdx.x / tiles;
    xcd_tile(blockIdx.x - split * tiles, (a.m + T::BM - 1) / T::BM, (a.n + kColumns - 1) / kColumns, 4, ty, tx);
    const uint32_t m0 = ty * T::BM, n0 = tx * kColumns;
    const uint32_t first_block = split * a.split_steps * 4, blocks = min(a.blocks - first_block, a.split_steps * 4);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)));

    // What this wave fetches: loads wave * W_EACH + i of the weights, wave * A_EACH + i of the activations, each of whole
    // rows, and 16 bytes of the scales of 64 rows.  Rows past the last are the last one again: their results are not stored.
    constexpr uint32_t kWPieces = T::W_ROW / 16, kWRows = 64 / kWPieces, kAPieces = T::A_ROW / 16, kARows = 64 / kAPieces;
    const uint32_t wrow = lane / kWPieces, arow = lane / kAPieces;
    const uint32_t wpiece = turned<T::W_ROW>(lane % kWPieces, wrow);
    const uint32_t apiece = turned<T::A_ROW>(lane % kAPieces, arow);
    static_assert(kWRows >= 8 && (kARows >= 8), "a load's rows turn alike");
    uint64_t w_base[T::W_EACH];
    uint32_t w_off[T::W_EACH];
#pragma unroll
    for (int i = 0; i < T::W_EACH; ++i) {
        const uint32_t row = (wave * T::W_EACH + i) * kWRows, t = row / 16, which = GATED ? t & 1 : 0;
        const uint32_t first = min(n0 + (GATED ? t / 2 * 16 + row % 16 : row), a.n - 1);
        const int64_t stride = which ? a.w[1].stride : a.w[0].stride;
        w_base[i] = reinterpret_cast<uint64_t>((which ? a.w[1].values : a.w[0].values) + first * stride + first_block * 16ull);
        w_off[i] = min(wrow, a.n - 1 - first) * static_cast<uint32_t>(stride) + wpiece * 16;
    }
    const uint64_t a_base = reinterpret_cast<uint64_t>(a.a.values + m0 * a.a.stride + first_block * (T::FP8 ? 32ull : 16ull));
    uint32_t a_off[T::A_EACH];
#pragma unroll
    for (int i = 0; i < T::A_EACH; ++i)
        a_off[i] = min((wave * T::A_EACH + i) * kARows + arow, a.m - 1 - m0) * static_cast<uint32_t>(a.a.stride) + apiece * 16;
    const uint8_t *scales[T::S_EACH];
#pragma unroll
    for (int i = 0; i < T::S_EACH; ++i) {
        const uint32_t row = min(wave * T::S_EACH + i, T::S_LOADS - 1u) * 64 + lane;  // weight rows, then activation rows
        const uint32_t t = row / 16;
        const uint32_t at = row >= T::BN ? min(m0 + row - T::BN, a.m - 1) : min(n0 + (GATED ? t / 2 * 16 + row % 16 : row), a.n - 1);
        const MxOperand &o = row >= T::BN ? a.a : a.w[0];
        scales[i] = o.scales + at * o.scale_stride;
        if (GATED && row < T::BN && t % 2 == 1) scales[i] = a.w[1].scales + at * a.w[1].scale_stride;
        scales[i] += first_block;
    }
    const uint32_t steps = (blocks + 3) / 4, stages = (steps + SUB - 1) / SUB;
    // Scales of blocks 16 g to 16 g + 15.  (Waves past the last load fetch that one again, to the same place with the same
    // bytes.)
    auto fetch_scales = [&](uint32_t g) {
        const uint32_t at = RING * T::STAGE + g % 2 * T::SCALES;
#pragma unroll
        for (int i = 0; i < T::S_EACH; ++i) {
            const uint32_t to = at + min(wave * T::S_EACH + i, T::S_LOADS - 1u) * 1024;
            if (16 * g + 16 <= blocks) {
                dma16_from(reinterpret_cast<const char *>(scales[i] + g * 16ull), lds0 + to);
            } else {  // the last words of a row, and nothing behind them
                u4 v;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    v[j] = 16 * g + 4 * j < blocks ? *reinterpret_cast<const uint32_t *>(scales[i] + g * 16ull + 4 * j) : 0u;
                *reinterpret_cast<u4 *>(lds + to + lane * 16) = v;
            }
        }
    };
    auto fetch = [&](uint32_t s, uint32_t buffer) {
        if (s % T::GROUP == T::GROUP - 1 && (s + 1) * SUB < steps) fetch_scales((s + 1) / T::GROUP);
        const uint32_t to = lds0 + buffer * T::STAGE;
        const uint32_t w_to = to + wave * T::W_EACH * 1024, a_to = to + T::W_BYTES + wave * T::A_EACH * 1024;
        const uint64_t w_skip = s * static_cast<uint64_t>(T::W_ROW), a_from = a_base + s * static_cast<uint64_t>(T::A_ROW);
        if (4 * SUB * (s + 1) <= blocks) {
#pragma unroll
            for (int i = 0; i < T::W_EACH; ++i) dma16(w_base[i] + w_skip, w_off[i], w_to + i * 1024);
#pragma unroll
            for (int i = 0; i < T::A_EACH; ++i) dma16(a_from, a_off[i], a_to + i * 1024);
        } else {  // the last stage of a K that does not fill it: zeros past the rows' ends
            const char *zero = reinterpret_cast<const char *>(&kZeroPiece);
#pragma unroll
            for (int i = 0; i < T::W_EACH; ++i)
                dma16_from(4 * SUB * s + wpiece < blocks ? reinterpret_cast<const char *>(w_base[i] + w_skip + w_off[i]) : zero,
                           w_to + i * 1024);
            const bool in = 4 * SUB * s + (T::FP8 ? apiece / 2 : apiece) < blocks;
#pragma unroll
            for (int i = 0; i < T::A_EACH; ++i)
                dma16_from(in ? reinterpret_cast<const char *>(a_from + a_off[i]) : zero, a_to + i * 1024);
        }
    };

    f4 acc[TW][TA];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TA; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

    // Where this lane's operands of a stage's first step lie, and its scales of a group's.  (The pieces of the second step
    // lie where bit 6 of the address is turned.)
    const uint32_t w_row = wn * TW * 16 + r, a_row = wm * TA * 16 + r;
    const uint32_t w_at = w_row * T::W_ROW + turned<T::W_ROW>(c, r) * 16;
    const uint32_t a_lo = T::W_BYTES + a_row * T::A_ROW + turned<T::A_ROW>(c, r) * 16;
    const uint32_t a_hi = T::W_BYTES + a_row * T::A_ROW + turned<T::A_ROW>(4 + c, r) * 16;
    const uint32_t ws_at = RING * T::STAGE + w_row * 16 + c, as_at = RING * T::STAGE + (T::BN + a_row) * 16 + c;
    uint32_t wscale[TW], ascale[TA];
    u4 w[TW], lo[TA], hi[TA];
    auto read = [&](uint32_t step, uint32_t buffer) {
        const char *from = lds + buffer * T::STAGE;
        const char *from_scales = lds + step / 4 % 2 * T::SCALES + step % 4 * 4;
        const uint32_t turn = step % SUB * 64;
#pragma unroll
        for (int j = 0; j < TA; ++j) {
            lo[j] = *reinterpret_cast<const u4 *>(from + (a_lo ^ turn) + j * 16 * T::A_ROW);
            hi[j] = T::FP8 ? *reinterpret_cast<const u4 *>(from + a_hi + j * 16 * T::A_ROW) : lo[j];
            ascale[j] = *reinterpret_cast<const uint8_t *>(from_scales + as_at + j * 256);
        }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            w[i] = *reinterpret_cast<const u4 *>(from + (w_at ^ turn) + i * 16 * T::W_ROW);
            wscale[i] = *reinterpret_cast<const uint8_t *>(from_scales + ws_at + i * 256);
        }
    };
    auto multiply = [&]() {
#pragma unroll
        for (int j = 0; j < TA; ++j) {
            const ActPiece<ACT> act(lo[j], hi[j]);
#pragma unroll
            for (int i = 0; i < TW; ++i) acc[i][j] = mx_mfma<ACT>(w[i], act, acc[i][j], wscale[i], ascale[j]);
        }
    };
    // All but the youngest `younger` stages in flight have landed.  (A group's scales are fetched before a stage's rows,
    // so they have landed with them, or before.)
    auto landed_but = [&](uint32_t younger) {
        if (RING > 2 && younger == 1) landed<T::LOADS>();
        else landed<0>();
    };

    fetch_scales(0);
#pragma unroll
    for (int s = 0; s < RING - 1; ++s)
        if (s < static_cast<int>(stages)) fetch(s, s);
    uint32_t buffer = 0;
    if constexpr (T::WAVES == 8) {
        // The waves of a SIMD take turns: waves 0 - 3 read a step's operands while waves 4 - 7 multiply those of the one
        // before, and the other way round.  A buffer is free once waves 4 - 7 have read it; the next stage has to be there
        // when waves 0 - 3 begin to read it, so they wait after their products, waves 4 - 7 (a phase behind) after their
        // reads.
        const bool second = wave >= 4;
        landed_but(min(stages - 1, static_cast<uint32_t>(RING - 2)));
        meet();
        if (second) meet();
        uint32_t s = 0;
        for (uint32_t step = 0; step < stages * SUB; ++step) {
            // In flight behind stage s + 1 once the next fetch is issued.
            const uint32_t younger = s + 2 < stages ? min(stages - 2 - s, static_cast<uint32_t>(RING - 2)) : 0u;
            const bool last = SUB == 1 || step % SUB == SUB - 1;  // of its stage
            if ((SUB == 1 || step % SUB == 0) && s + RING - 1 < stages) fetch(s + RING - 1, buffer == 0 ? RING - 1 : buffer - 1);
            read(step, buffer);
            if (second && last) landed_but(younger);
            else landed<63>();
            meet();
            __builtin_amdgcn_s_setprio(1);
            multiply();
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (!second && last) landed_but(younger);
            meet();
            if (last) {
                ++s;
                buffer = buffer + 1 == RING ? 0 : buffer + 1;
            }
        }
        if (!second) meet();
    } else {
        for (uint32_t s = 0; s < stages; ++s) {
            landed_but(min(stages - 1 - s, static_cast<uint32_t>(RING - 2)));
            meet();  // all of stage s, from every wave; and every wave has read stage s - 1, whose buffer the fetch fills
            if (s + RING - 1 < stages) fetch(s + RING - 1, buffer == 0 ? RING - 1 : buffer - 1);
            for (uint32_t u = 0; u < SUB; ++u) {
                read(s * SUB + u, buffer);
                multiply();
            }
            buffer = buffer + 1 == RING ? 0 : buffer + 1;
        }
    }

    if (a.splits > 1) {  // sums of a part of K, joined by another kernel: four columns a lane
        const uint64_t plane = static_cast<uint64_t>(a.m) * a.part_row;
        float *to = a.parts + split * (GATED ? 2 : 1) * plane;
#pragma unroll
        for (int j = 0; j < TA; ++j) {
            const uint32_t m = m0 + (wm * TA + j) * 16 + r;
            if (m >= a.m) continue;
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                const uint32_t n = n0 + wn * T::OUT + (GATED ? i / 2 : i) * 16 + 4 * c;
                if (n < a.part_row)
                    *reinterpret_cast<f4 *>(to + (GATED && i % 2 ? plane : 0) + static_cast<uint64_t>(m) * a.part_row + n) = acc[i][j];
            }
        }
        return;
    }

    // Results by 16 rows through LDS, so that a lane stores eight neighbouring columns.
    __syncthreads();
    float *mine = reinterpret_cast<float *>(lds) + wave * 16 * T::OUT_ROW;
    constexpr uint32_t kEights = T::OUT / 8, kRows = 64 / kEights;  // lanes a row, rows a step
    const uint32_t out_n = n0 + wn * T::OUT + lane % kEights * 8;
    float bias[8];
    if constexpr (!GATED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = a.bias != nullptr && out_n + e < a.n ? a.bias[out_n + e] : 0.0f;
    }
    const bool whole = a.vec_out && out_n + 8 <= a.n;
    with_kind<GATED>(a.out_kind, [&](auto kind) {
#pragma unroll
        for (int j = 0; j < TA; ++j) {
#pragma unroll
            for (int i = 0; i < TW / (GATED ? 2 : 1); ++i) {
                f4 v;
                if constexpr (GATED) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = gated(a.gate, acc[2 * i][j][e], acc[2 * i + 1][j][e]);
                } else {
                    v = acc[i][j];
                }
                *reinterpret_cast<f4 *>(mine + r * T::OUT_ROW + 16 * i + 4 * c) = v;
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" : : : "memory");
#pragma unroll
            for (uint32_t step = 0; step < 16; step += kRows) {
                const uint32_t row = step + lane / kEights;
                const float *from = mine + row * T::OUT_ROW + lane % kEights * 8;
                const f4 x = *reinterpret_cast<const f4 *>(from), y = *reinterpret_cast<const f4 *>(from + 4);
                Eight e{{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}};
                if constexpr (!GATED) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) e.v[q] += bias[q];
                }
                store_results<decltype(kind)::value>(a, m0 + wm * TA * 16 + j * 16 + row, out_n, whole, e);
            }
            asm volatile("" : : : "memory");
            __builtin_amdgcn_wave_barrier();
        }
    });
}

// Joins the parts of K: a thread adds up eight columns of a row, in the order of the parts, whose loads it issues several
// parts at a time (77 x 4096 results of eight parts: 4.1 us, one part at a time 5.1).
template <bool GATED>
__global__ __launch_bounds__(256) void mxfp4_join_kernel(MxLinearArgs a, FastDiv row) {
    const uint32_t at = blockIdx.x * 256 + threadIdx.x, m = fast_quotient(at, row), n = (at - m * row.divisor) * 8;
    if (m >= a.m) return;  // (rows of four lanes leave together where blocks are stored)
    const uint64_t plane = static_cast<uint64_t>(a.m) * a.part_row;
    const float *from = a.parts + static_cast<uint64_t>(m) * a.part_row + n;
    f4 sum[GATED ? 2 : 1][2] = {};
    constexpr uint32_t kWeights = GATED ? 2 : 1, kParts = 8 / kWeights;
    for (uint32_t first = 0; first < a.splits; first += kParts) {
        f4 part[kParts][kWeights][2];
#pragma unroll
        for (uint32_t s = 0; s < kParts; ++s)
#pragma unroll
            for (uint32_t w = 0; w < kWeights; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    part[s][w][h] = *reinterpret_cast<const f4 *>(from + (min(first + s, a.splits - 1) * kWeights + w) * plane + 4 * h);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t s = 0; s < kParts; ++s) {
            if (first + s >= a.splits) break;
#pragma unroll
            for (uint32_t w = 0; w < kWeights; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) sum[w][h] += part[s][w][h];
        }
    }
    Eight e;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        e.v[i] = sum[0][i / 4][i % 4];
        if constexpr (GATED) e.v[i] = gated(a.gate, e.v[i], sum[1][i / 4][i % 4]);
        else if (a.bias != nullptr && n + i < a.n) e.v[i] += a.bias[n + i];
    }
    with_kind<GATED>(a.out_kind, [&](auto kind) {
        store_results<decltype(kind)::value>(a, m, n, a.vec_out && n + 8 <= a.n, e);
    });
}

template <int ACT, bool GATED, int TW, int TA, int WN, int WM, int SUB, int RING>
int launch_tile(MxLinearArgs &a, const char *name, uint32_t splits, hipStream_t stream) {
    typedef Tiles<ACT, GATED, TW, TA, WN, WM, SUB, RING> T;
    constexpr uint32_t columns = T::BN / (GATED ? 2 : 1);
    const uint32_t groups = (a.blocks + 15) / 16;
    a.split_steps = (groups + splits - 1) / splits * 4;
    a.splits = (groups + a.split_steps / 4 - 1) / (a.split_steps / 4);  // none is empty
    a.part_row = part_row(a.n);
    const uint64_t grid = static_cast<uint64_t>((a.m + T::BM - 1) / T::BM) * ((a.n + columns - 1) / columns) * a.splits;
    const uint32_t row = a.part_row / 8;
    const uint64_t joins = (static_cast<uint64_t>(a.m) * row + 255) / 256;
    if (grid > INT32_MAX || (a.splits > 1 && joins * 256 > INT32_MAX)) return fail(QXT_INVALID_ARGUMENT, "mxfp4 linear: too many outputs");
    const int rc = launch(name, mxfp4_tile_kernel<ACT, GATED, TW, TA, WN, WM, SUB, RING>,
                          dim3(static_cast<uint32_t>(grid)), dim3(T::THREADS), 0, stream, a);
    if (rc != QXT_OK || a.splits == 1) return rc;
    return launch("mxfp4_join_kernel", mxfp4_join_kernel<GATED>, dim3(static_cast<uint32_t>(joins)), dim3(256), 0, stream, a,
                  fast_div(row));
}

// The tiles of a plan, weight rows by activation rows.  The first has eight waves, which take turns, the others four, and
// two to four workgroups a CU.
constexpr uint32_t kTiles = 5;
constexpr uint32_t kTileRows[kTiles][2] = {{256, 256}, {128, 128}, {128, 64}, {64, 64}, {128, 32}};
constexpr const char *kTileNames[kTiles] = {"mxfp4_tile_kernel 256x256", "mxfp4_tile_kernel 128x128", "mxfp4_tile_kernel 128x64",
                                            "mxfp4_tile_kernel 64x64", "mxfp4_tile_kernel 128x32"};

template <int ACT, bool GATED>
int launch_tiles(MxLinearArgs &a, const TilePlan &plan, hipStream_t stream) {
    // 4-bit rows take two steps of K a stage, for whole cache lines.  Eight waves alone on a CU take the stages that fit.
    // Where several workgroups share a CU two stages are better than three, or as good (8-bit, 333 x 4096 x 14336 56.3 ->
    // 48.1 us).
    constexpr int SUB = ACT == kAct4 ? 2 : 1, RING = ACT == kAct4 ? 2 : 3;
    const char *name = kTileNames[plan.tile];
    switch (plan.tile) {
        case 0: return launch_tile<ACT, GATED, 8, 4, 2, 4, SUB, RING>(a, name, plan.splits, stream);
        case 1: return launch_tile<ACT, GATED, 4, 4, 2, 2, SUB, 2>(a, name, plan.splits, stream);
        case 2: return launch_tile<ACT, GATED, 4, 2, 2, 2, SUB, 2>(a, name, plan.splits, stream);
        case 3: return launch_tile<ACT, GATED, 4, 1, 1, 4, SUB, 2>(a, name, plan.splits, stream);
        default: return launch_tile<ACT, GATED, 4, 1, 2, 2, SUB, 2>(a, name, plan.splits, stream);
    }
}

// Estimated microseconds of a launch: a step of 128 elements of K takes `least`, or `base` plus `share` for each workgroup
// a CU; `edge`: filling the ring and storing the results, for each workgroup a CU.  (Workgroups a CU: a third of their mean
// over 256 CUs and two thirds of the fullest CU's.)  Fitted to 3459 measured calls (198 products of 24 to 4096 rows, 8-bit
// ones to 1024, K 512 to 14336, 1024 to 14336 columns, every tile and number of parts below; rms error 9 % and 6 %); the
// least estimate is on average 1 % slower than the fastest of them, in one product more than 10 % (10.8 %).
struct TileCost {
    float least, base, share, edge;
};
constexpr TileCost kCosts[2][kTiles] = {
    // kAct4
    {{0.96f, 0.03f, 0.90f, 7.3f}, {0.41f, 0.03f, 0.26f, 2.4f}, {0.30f, 0.01f, 0.20f, 1.6f}, {0.25f, 0.08f, 0.11f, 0.6f}, {0.30f, 0.07f, 0.15f, 1.2f}},
    // kAct8
    {{0.21f, 1.39f, 1.36f, 8.4f}, {0.95f, 0.64f, 0.42f, 3.7f}, {0.00f, 0.44f, 0.18f, 2.1f}, {0.47f, 0.12f, 0.22f, 1.1f}, {0.48f, 0.10f, 0.25f, 1.3f}},
};
// The second kernel that parts of K need, and a megabyte of their sums, written and read.
constexpr float kJoin = 2.3f, kJoinMegabyte = 0.175f;
// Numbers of parts, and the most workgroups that K is split for.
constexpr uint32_t kParts[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr float kMostSplitTiles = 600.0f;

}  // namespace

TilePlan plan_tiles(uint32_t m, uint32_t n, uint32_t k, uint32_t weights, int act) {
    TilePlan best{0, 1};
    float least = 0.0f;
    const uint32_t steps = (k + 127) / 128, groups = (steps + 3) / 4;
    const float sums = static_cast<float>(weights) * static_cast<float>(m) * static_cast<float>(n) * 4e-6f;
    for (uint32_t t = 0; t < kTiles; ++t) {
        const float tiles = static_cast<float>((m + kTileRows[t][1] - 1) / kTileRows[t][1]) *
                            static_cast<float>((static_cast<uint64_t>(n) * weights + kTileRows[t][0] - 1) / kTileRows[t][0]);
        for (const uint32_t wanted : kParts) {
            if (wanted > groups || (wanted > 1 && tiles * static_cast<float>(wanted) > kMostSplitTiles)) break;
            const uint32_t each = (groups + wanted - 1) / wanted, splits = (groups + each - 1) / each;
            if (splits < wanted) continue;  // the same as fewer
            const TileCost &c = kCosts[act][t];
            const float mean = tiles * static_cast<float>(splits) / 256.0f, load = (mean + 2.0f * ceilf(mean)) / 3.0f;
            const float depth = static_cast<float>(min(4 * each, steps));
            float cost = depth * fmaxf(c.least, c.base + c.share * load) + c.edge * load;
            if (splits > 1) cost += kJoin + kJoinMegabyte * 2.0f * static_cast<float>(splits) * sums;
            if (least == 0.0f || cost < least) {
                least = cost;
                best = {t, splits};
            }
        }
    }
    return best;
}

int mxfp4_tiles(MxLinearArgs &a, int act, bool gated, const TilePlan &plan, hipStream_t stream) {
    switch (act) {
        case kAct4: return gated ? launch_tiles<kAct4, true>(a, plan, stream) : launch_tiles<kAct4, false>(a, plan, stream);
        default: return gated ? launch_tiles<kAct8, true>(a, plan, stream) : launch_tiles<kAct8, false>(a, plan, stream);
    }
}

}  // namespace qxt
