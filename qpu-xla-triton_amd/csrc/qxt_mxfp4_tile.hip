// Linears over microscaling 4-bit weights for many rows: tiles of the result
// whose operands pass through LDS once for all the waves that share them.
//
// A workgroup of WN x WM waves owns 16 TW WN weight rows by 16 TA WM activation
// rows, each wave 16 TW by 16 TA of them as 16 x 16 x 128 products.  K advances
// 128 elements a stage through a ring of LDS buffers filled by DMA: a wave's
// 16-byte pieces land in lane order, so which piece a lane fetches decides the
// layout.  Rows of 64 bytes (4-bit) or 128 (8-bit) are fetched whole by
// neighbouring lanes, and piece p of row r lies at p ^ (r / 2 % 4) or p ^ (r % 8),
// so that the reads of one piece over 16 rows touch all banks.  A gated product
// takes the tiles of gate and up in turn, so that a wave holds both sums of a
// result.
#include "qxt_mxfp4.h"

namespace qxt {
namespace {

// Source of what lies past a row's last block.
__device__ __constant__ const uint4 kZeroPiece = {};

// 64 lanes' 16 or 4 bytes, from a wave-uniform address plus each lane's offset or from each lane's address, to LDS at `to`
// + 16 (or 4) * lane.  Inline
// assembly because the compiler waits for every such load in flight before it reads any of LDS; the waits here are the
// kernel's own.  There is no register output.
// (The compiler warns that it may not preserve m0; it has no other use for it here.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(uint64_t base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma16_from(const char *src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma4_from(const uint8_t *src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

// Wait until all but the wave's N youngest loads are done, and all of its LDS reads.
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void meet() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

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

template <int ACT, bool GATED, int TW, int TA, int WN, int WM, int RING>
struct Tiles {
    static constexpr bool FP8 = ACT != kAct4;
    static constexpr int WAVES = WN * WM, THREADS = 64 * WAVES;
    static constexpr int BN = 16 * TW * WN, BM = 16 * TA * WM;  // weight rows (of both weights), activation rows
    static constexpr int ROW = FP8 ? 128 : 64;                 // bytes of an activation row a stage
    static constexpr int W_BYTES = BN * 64, A_BYTES = BM * ROW, S_BYTES = (BN + BM) * 4;
    static constexpr int STAGE = W_BYTES + A_BYTES + S_BYTES;
    static constexpr int W_LOADS = W_BYTES / 1024, A_LOADS = A_BYTES / 1024, S_LOADS = (BN + BM) / 64;
    static constexpr int W_EACH = W_LOADS / WAVES, A_EACH = A_LOADS / WAVES, S_EACH = (S_LOADS + WAVES - 1) / WAVES;
    static constexpr int LOADS = W_EACH + A_EACH + S_EACH;  // of each wave a stage
    static constexpr int OUT = 16 * TW / (GATED ? 2 : 1);   // result columns of a wave
    static constexpr int OUT_ROW = OUT + 4;                 // floats, in LDS
    static constexpr int LDS = RING * STAGE > WAVES * 16 * OUT_ROW * 4 ? RING * STAGE : WAVES * 16 * OUT_ROW * 4;
    static_assert(W_LOADS % WAVES == 0 && A_LOADS % WAVES == 0 && LDS <= 160 * 1024, "tile shape");
};

template <int ACT, bool GATED, int TW, int TA, int WN, int WM, int RING>
__global__ __launch_bounds__(64 * WN * WM) void mxfp4_tile_kernel(MxLinearArgs a) {
    typedef Tiles<ACT, GATED, TW, TA, WN, WM, RING> T;
    __shared__ __attribute__((aligned(16))) char lds[T::LDS];
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
    constexpr uint32_t kColumns = T::BN / (GATED ? 2 : 1);  // result columns of the workgroup
    uint32_t ty, tx;
    xcd_tile(blockIdx.x, (a.m + T::BM - 1) / T::BM, (a.n + kColumns - 1) / kColumns, 4, ty, tx);
    const uint32_t m0 = ty * T::BM, n0 = tx * kColumns;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)));

    // What this wave fetches: weight row tiles wave * W_EACH + i, activation pieces wave * A_EACH + i, scales of 64 rows.
    // Rows past the last are the last one again: their results are not stored.
    const uint32_t wrow = lane / 4, wpiece = (lane % 4) ^ (wrow / 2 % 4);
    uint64_t w_base[T::W_EACH];
    uint32_t w_off[T::W_EACH];
#pragma unroll
    for (int i = 0; i < T::W_EACH; ++i) {
        const uint32_t t = wave * T::W_EACH + i, which = GATED ? t & 1 : 0, first = n0 + 16 * (GATED ? t / 2 : t);
        const MxOperand &w = a.w[0], &u = a.w[1];
        const int64_t stride = which ? u.stride : w.stride;
        const uint32_t base = min(first, a.n - 1);
        w_base[i] = reinterpret_cast<uint64_t>((which ? u.values : w.values) + base * stride);
        w_off[i] = min(wrow, a.n - 1 - base) * static_cast<uint32_t>(stride) + wpiece * 16;
    }
    constexpr uint32_t kPieces = T::ROW / 16, kRowsPerLoad = 64 / kPieces;
    const uint32_t arow = lane / kPieces, apiece = (lane % kPieces) ^ (T::FP8 ? arow % 8 : arow / 2 % 4);
    uint64_t a_base = reinterpret_cast<uint64_t>(a.a.values + m0 * a.a.stride);
    uint32_t a_off[T::A_EACH];
#pragma unroll
    for (int i = 0; i < T::A_EACH; ++i) {
        const uint32_t row = (wave * T::A_EACH + i) * kRowsPerLoad + arow;
        a_off[i] = min(row, a.m - 1 - m0) * static_cast<uint32_t>(a.a.stride) + apiece * 16;
    }
    const uint8_t *scales[T::S_EACH];
#pragma unroll
    for (int i = 0; i < T::S_EACH; ++i) {
        const uint32_t row = min(wave * T::S_EACH + i, T::S_LOADS - 1u) * 64 + lane;  // weight rows, then activation rows
        const uint32_t t = row / 16;
        const uint32_t at = row >= T::BN ? min(m0 + row - T::BN, a.m - 1) : min(n0 + (GATED ? t / 2 * 16 + row % 16 : row), a.n - 1);
        const MxOperand &o = row >= T::BN ? a.a : a.w[0];
        scales[i] = o.scales + at * o.scale_stride;
        if (GATED && row < T::BN && t % 2 == 1) scales[i] = a.w[1].scales + at * a.w[1].scale_stride;
    }
    const uint32_t stages = (a.blocks + 3) / 4, blocks = a.blocks;
    auto fetch = [&](uint32_t s, uint32_t buffer) {
        const uint32_t to = lds0 + buffer * T::STAGE;
        const bool whole = 4 * s + 4 <= blocks;
#pragma unroll
        for (int i = 0; i < T::W_EACH; ++i) {
            const uint32_t at = to + (wave * T::W_EACH + i) * 1024;
            if (whole) {
                dma16(w_base[i] + s * 64ull, w_off[i], at);
            } else {
                const char *src = reinterpret_cast<const char *>(w_base[i] + s * 64ull + w_off[i]);
                dma16_from(4 * s + wpiece < blocks ? src : reinterpret_cast<const char *>(&kZeroPiece), at);
            }
        }
#pragma unroll
        for (int i = 0; i < T::A_EACH; ++i) {
            const uint32_t at = to + T::W_BYTES + (wave * T::A_EACH + i) * 1024;
            if (whole) {
                dma16(a_base + s * static_cast<uint64_t>(T::ROW), a_off[i], at);
            } else {
                const char *src = reinterpret_cast<const char *>(a_base + s * static_cast<uint64_t>(T::ROW) + a_off[i]);
                const uint32_t block = 4 * s + (T::FP8 ? apiece / 2 : apiece);
                dma16_from(block < blocks ? src : reinterpret_cast<const char *>(&kZeroPiece), at);
            }
        }
#pragma unroll
        for (int i = 0; i < T::S_EACH; ++i) {
            // (Waves past the last load fetch that one again, to the same place with the same bytes.)
            const uint32_t at = to + T::W_BYTES + T::A_BYTES + min(wave * T::S_EACH + i, T::S_LOADS - 1u) * 256;
            dma4_from(scales[i] + s * 4ull, at);
        }
    };

    f4 acc[TW][TA];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TA; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

    // Where this lane's operands lie in a stage.
    const uint32_t w_at = (wn * TW * 16 + r) * 64 + (c ^ (r / 2 % 4)) * 16;
    const uint32_t a_row = wm * TA * 16 + r;
    const uint32_t a_lo = T::W_BYTES + a_row * T::ROW + (T::FP8 ? c ^ (r % 8) : c ^ (r / 2 % 4)) * 16;
    const uint32_t a_hi = T::FP8 ? T::W_BYTES + a_row * T::ROW + ((4 + c) ^ (r % 8)) * 16 : a_lo;
    const uint32_t ws_at = T::W_BYTES + T::A_BYTES + (wn * TW * 16 + r) * 4 + c;
    const uint32_t as_at = T::W_BYTES + T::A_BYTES + (T::BN + a_row) * 4 + c;

#pragma unroll
    for (int s = 0; s < RING - 1; ++s)
        if (s < static_cast<int>(stages)) fetch(s, s);
    uint32_t buffer = 0;
    for (uint32_t s = 0; s < stages; ++s) {
        // Stage s has landed when at most the younger ones that are in flight are left.
        const uint32_t younger = min(stages - 1 - s, static_cast<uint32_t>(RING - 2));
        if (RING > 3 && younger == 2) landed<2 * T::LOADS>();
        else if (younger == 1) landed<T::LOADS>();
        else landed<0>();
        meet();  // all of it, from every wave; and every wave has read stage s - 1, whose buffer the next fetch fills
        if (s + RING - 1 < stages) fetch(s + RING - 1, buffer == 0 ? RING - 1 : buffer - 1);
        const char *from = lds + buffer * T::STAGE;
        uint32_t wscale[TW], ascale[TA];
        u4 w[TW], lo[TA], hi[TA];
#pragma unroll
        for (int j = 0; j < TA; ++j) {
            lo[j] = *reinterpret_cast<const u4 *>(from + a_lo + j * 16 * T::ROW);
            hi[j] = T::FP8 ? *reinterpret_cast<const u4 *>(from + a_hi + j * 16 * T::ROW) : lo[j];
            ascale[j] = *reinterpret_cast<const uint8_t *>(from + as_at + j * 64);
        }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            w[i] = *reinterpret_cast<const u4 *>(from + w_at + i * 1024);
            wscale[i] = *reinterpret_cast<const uint8_t *>(from + ws_at + i * 64);
        }
#pragma unroll
        for (int j = 0; j < TA; ++j) {
            const ActPiece<ACT> act(lo[j], hi[j]);
#pragma unroll
            for (int i = 0; i < TW; ++i) acc[i][j] = mx_mfma<ACT, 0>(w[i], act, acc[i][j], wscale[i], ascale[j]);
        }
        buffer = buffer + 1 == RING ? 0 : buffer + 1;
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
                if (a.bias != nullptr) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) e.v[q] += bias[q];
                }
            }
            store_results(a, m0 + wm * TA * 16 + j * 16 + row, out_n, e);
        }
        asm volatile("" : : : "memory");
        __builtin_amdgcn_wave_barrier();
    }
}

template <int ACT, bool GATED, int TW, int TA, int WN, int WM, int RING>
int launch_tile(const MxLinearArgs &a, hipStream_t stream) {
    typedef Tiles<ACT, GATED, TW, TA, WN, WM, RING> T;
    constexpr uint32_t columns = T::BN / (GATED ? 2 : 1);
    const uint64_t grid = static_cast<uint64_t>((a.m + T::BM - 1) / T::BM) * ((a.n + columns - 1) / columns);
    if (grid > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "mxfp4 linear: too many outputs");
    return launch("mxfp4_tile_kernel", mxfp4_tile_kernel<ACT, GATED, TW, TA, WN, WM, RING>, dim3(static_cast<uint32_t>(grid)),
                  dim3(T::THREADS), 0, stream, a);
}

template <int ACT, bool GATED>
int launch_tiles(const MxLinearArgs &a, hipStream_t stream) {
    return launch_tile<ACT, GATED, 8, 4, 2, 4, 3>(a, stream);
}

}  // namespace

int mxfp4_tiles(const MxLinearArgs &a, int act, bool gated, hipStream_t stream) {
    switch (act) {
        case kAct4: return gated ? launch_tiles<kAct4, true>(a, stream) : launch_tiles<kAct4, false>(a, stream);
        case kAct8: return gated ? launch_tiles<kAct8, true>(a, stream) : launch_tiles<kAct8, false>(a, stream);
        default: return gated ? launch_tiles<kAct8Parts, true>(a, stream) : launch_tiles<kAct8Parts, false>(a, stream);
    }
}

}  // namespace qxt
