// The attention weight that each cached slot received from new tokens:
//   scores[b, head, j] = previous + sum over the sequence's tokens t and the
//   query heads h of the group of exp(scale q.k_j - lse[t, h]),
// with the log-sums of the attention over the same slots.
//
// Slots are independent, so a wave keeps its keys in registers as the second
// operand of S = Q K^T (32x32x16 MFMAs) and each lane adds up the weights of its
// own key: no atomics, one order of the sum.
//
// Many rows (tokens times heads of a group): a workgroup's 256 keys stay, the
// rows pass by in LDS in steps of 64.  Where key tiles, heads and sequences alone
// are too few workgroups, the steps are dealt out over splits, whose sums a
// second launch adds in order.  Bound by the matrix and vector units together:
// 32 MFMAs and 64 exponentials with three more operations each a wave and step.
// Measured: a 4k prompt, 32 heads of 128 over 8 key heads, causal, 156 us for
// 68.7 GFLOP; the vector units are busy 54 % of the time, the matrix units 28 %.
//
// Every score of the table's width is read and written, in place too, so tables
// wider than the contexts cost: one token each of 16 sequences of 6k slots, 8 key
// heads, 42 us with a table of 6k slots, 67 with 32k, 147 with 128k.
//
// Up to 32 rows (one token a sequence, or a few): the rows stay in registers and
// the keys pass by, each wave streaming its own run of slots with the next 32
// keys and the page numbers after those under way; bound by the keys' bytes.
#include <algorithm>

#include "qxt_paged_attention.h"

namespace qxt {
namespace {

struct ScoreArgs {
    PagedArgs paged;  // its lse is read here
    const float *previous;
    int64_t previous_sequence, previous_head;
    float *out;
    int64_t out_sequence, out_head;
    float *parts;  // [splits, sequences, kv_heads, slots], splits > 1
};

constexpr int kScoreWaves = 4, kScoreKeys = 64, kScoreTile = kScoreWaves * kScoreKeys, kScoreRows = 64;
constexpr float kLog2e = 1.44269504f;

__device__ __forceinline__ float previous_score(Kernarg<ScoreArgs> &sa, uint32_t b, uint32_t head, int32_t slot) {
    return sa.previous != nullptr ? sa.previous[b * sa.previous_sequence + head * sa.previous_head + slot] : 0.0f;
}
__device__ __forceinline__ void store_score(Kernarg<ScoreArgs> &sa, uint32_t b, uint32_t head, int32_t slot, int32_t length,
                                            float total) {
    const float was = previous_score(sa, b, head, slot);
    // (was itself, not was + 0, where nothing was added: unused slots keep their bits.)
    sa.out[b * sa.out_sequence + head * sa.out_head + slot] = slot < length ? was + total : was;
}

template <typename T, int DP>
__global__ __launch_bounds__(64 * kScoreWaves, DP <= 128 ? 2 : 1) void paged_scores_kernel(ScoreArgs) {
    using TL = Tile<DP>;
    using M = Mfma<T>;
    typedef typename M::frag frag;
    constexpr int kTileBytes = kScoreRows * DP * 2, kOwn = kScoreRows / kScoreWaves, kLoads = kOwn / TL::kRowsPerLoad;
    __shared__ __align__(16) char rows_lds[2][kTileBytes];
    __shared__ __align__(16) float row_lse[2][kScoreRows];
    __shared__ __align__(16) int32_t row_low[2][kScoreRows], row_high[2][kScoreRows];
    __shared__ int32_t odd_rows[2];  // the step has rows that count for nothing

    Kernarg<ScoreArgs> &sa = *kernargs<ScoreArgs>();
    Kernarg<PagedArgs> &a = sa.paged;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int col = lane % 32, half = lane / 32;
    uint32_t id = blockIdx.x;
    const uint32_t head = id % a.kv_heads;
    id /= a.kv_heads;
    const uint32_t first_tile = id % a.tiles;
    id /= a.tiles;
    const uint32_t split = id % a.splits, b = id / a.splits;
    const Sequence seq = sequence_of(a, b);
    FastDiv by_group{a.group.divisor, a.group.magic, a.group.shift, a.group.pass};
    const int32_t group = by_group.divisor, rows = seq.tokens * group;
    uint64_t query = reinterpret_cast<uint64_t>(a.query + seq.start * a.query_token + static_cast<int64_t>(head) * group * a.query_head);
    const float *lses = a.lse + seq.start * a.lse_token + static_cast<int64_t>(head) * group;
    uint64_t query_token = a.query_token, query_head = a.query_head, lse_token = a.lse_token;
    int32_t splits = a.splits, head_dim = a.head_dim;
    float scale = a.scale;
    keep(by_group.magic);
    keep(by_group.shift);
    keep(by_group.pass);
    keep(query);
    keep(lses);
    keep(query_token);
    keep(query_head);
    keep(lse_token);
    keep(splits);
    keep(head_dim);
    keep(scale);
    const int row_at = col * TL::kRowBytes + ((half ^ TL::key_turn(col)) * 16);
    const uint32_t my_rows = lds_offset(rows_lds[0]) + wave * kOwn * TL::kRowBytes;

    for (int64_t tile0 = static_cast<int64_t>(first_tile) * kScoreTile; tile0 < a.slots;
         tile0 += static_cast<int64_t>(a.tiles) * kScoreTile) {
        const int32_t key0 = static_cast<int32_t>(tile0), key_end = min(key0 + kScoreTile, seq.length);
        float total[2] = {0.0f, 0.0f};
        const int32_t mine0 = key0 + wave * kScoreKeys;
        // Tokens that see any slot of the tile.
        int32_t first = 0, last = seq.tokens;
        const int32_t before = seq.length - seq.tokens;
        if (a.causal) first = max(0, key0 - before);
        if (a.window > 0)
            last = static_cast<int32_t>(max<int64_t>(0, min<int64_t>(last, static_cast<int64_t>(key_end) - 1 + a.window - before)));
        const int32_t row_first = first * group, row_last = last * group;
        if (key0 < key_end && row_first < row_last) {
            frag k[2][DP / 16];
            const int32_t *table = a.table + b * a.table_stride;
            const char *keys = a.keys.data + head * a.keys.head_stride;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int32_t slot = mine0 + 32 * kb + col;
                const char *row = nullptr;
                if (slot < key_end) {
                    const uint32_t page = fast_quotient(static_cast<uint32_t>(slot), a.page);
                    const uint32_t in_page = static_cast<uint32_t>(slot) - page * a.page.divisor;
                    const int32_t page_id = table[page];
                    if (static_cast<uint32_t>(page_id) < a.pages)
                        row = keys + static_cast<int64_t>(page_id) * a.keys.page_stride +
                              static_cast<int64_t>(in_page) * a.keys.slot_stride;
                }
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    k[kb][c] = frag{};
                    if (row != nullptr && 16 * c + 8 * half < head_dim)
                        k[kb][c] = *reinterpret_cast<const frag *>(row + (16 * c + 8 * half) * 2);
                }
            }
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) asm volatile("" : "+v"(k[0][c]), "+v"(k[1][c]));  // arrived
            const int32_t step0 = row_first / kScoreRows, steps = (row_last + kScoreRows - 1) / kScoreRows;
            // Rows 64 t .. 64 t + 63 into LDS, a quarter by each wave; wave 0 also fetches what they see and their log-sums.
            float lse = 0.0f;
            Range sees{0, 0};
            auto stage = [&](int32_t t, int buffer) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = wave * kOwn + i * TL::kRowsPerLoad + lane / TL::kChunks;
                    const int32_t row = min(kScoreRows * t + r, rows - 1);
                    const int32_t token = fast_quotient(static_cast<uint32_t>(row), by_group), h = row - token * group;
                    const int chunk = (lane % TL::kChunks) ^ TL::key_turn(r);
                    const uint64_t src = query + token * query_token + h * query_head + chunk * 16;
                    dma16(reinterpret_cast<const char *>(chunk * 8 < head_dim ? src : reinterpret_cast<uint64_t>(kZeroRow)),
                          my_rows + buffer * kTileBytes + i * 1024);
                }
                if (wave == 0) {
                    const int32_t row = kScoreRows * t + lane;
                    sees = Range{0, 0};
                    lse = 0.0f;
                    if (row < rows) {
                        const int32_t token = fast_quotient(static_cast<uint32_t>(row), by_group), h = row - token * group;
                        sees = seen_by(a, seq, token);
                        lse = lses[token * lse_token + h];
                    }
                }
            };
            int buffer = 0;
            int32_t t = step0 + split;
            if (t < steps) stage(t, 0);
            for (; t < steps; t += splits, buffer ^= 1) {
                landed<0>();
                if (wave == 0) {
                    if (lse == -__builtin_inff()) {  // a row without weights
                        sees = Range{0, 0};
                        lse = 0.0f;
                    }
                    row_lse[buffer][lane] = lse;
                    row_low[buffer][lane] = sees.low;
                    row_high[buffer][lane] = sees.high;
                    const bool odd = __any(sees.high == 0);
                    if (lane == 0) odd_rows[buffer] = odd;
                    reads_done();  // (and writes)
                }
                meet();  // step t is staged, and step t - 1 has been read
                if (t + splits < steps) stage(t + splits, buffer ^ 1);
                // Rows see contiguous ranges that only move up: all see all of the wave's slots if the first and last do.
                const bool partial = __builtin_amdgcn_readfirstlane(odd_rows[buffer]) != 0 ||
                                     __builtin_amdgcn_readfirstlane(row_high[buffer][0]) < mine0 + kScoreKeys ||
                                     __builtin_amdgcn_readfirstlane(row_low[buffer][kScoreRows - 1]) > mine0;
#pragma unroll
                for (int rb = 0; rb < kScoreRows / 32; ++rb) {
                    const char *q_tile = rows_lds[buffer] + rb * 32 * TL::kRowBytes;
                    f32x16 s[2] = {f32x16{}, f32x16{}};
                    constexpr int kAhead = 4, kProducts = DP / 16;
                    frag q[kAhead];
#pragma unroll
                    for (int i = 0; i < kProducts + kAhead; ++i) {  // reads go ahead of their products in the source's order
                        if (i >= kAhead) {
                            s[0] = M::run(q[(i - kAhead) % kAhead], k[0][i - kAhead], s[0]);
                            s[1] = M::run(q[(i - kAhead) % kAhead], k[1][i - kAhead], s[1]);
                        }
                        if (i < kProducts) q[i % kAhead] = *reinterpret_cast<const frag *>(q_tile + (row_at ^ (32 * i)));
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 32 * rb + 8 * i + 4 * half;
                        float4 l = *reinterpret_cast<const float4 *>(&row_lse[buffer][at]);
                        float *ls = &l.x;
                        if (partial) {
                            // (A NaN log-sum goes into the logits of what its row sees: -inf minus NaN would not hide the rest.)
                            const int4 lo = *reinterpret_cast<const int4 *>(&row_low[buffer][at]);
                            const int4 hi = *reinterpret_cast<const int4 *>(&row_high[buffer][at]);
                            const int32_t *los = &lo.x, *his = &hi.x;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const bool none = ls[e] != ls[e];
#pragma unroll
                                for (int kb = 0; kb < 2; ++kb) {
                                    const int32_t slot = mine0 + 32 * kb + col;
                                    const float logit = none ? ls[e] : s[kb][4 * i + e];
                                    s[kb][4 * i + e] = slot < los[e] || slot >= his[e] ? -__builtin_inff() : logit;
                                }
                                ls[e] = none ? 0.0f : ls[e];
                            }
                        }
#pragma unroll
                        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                // The difference first: its rounding, not the log-sum's, bounds the weight's error.
                                total[kb] += __builtin_amdgcn_exp2f(fmaf(s[kb][4 * i + e], scale, -ls[e]) * kLog2e);
                    }
                }
            }
            __syncthreads();  // before the next tile's staging
        }
        Kernarg<ScoreArgs> &z = *late(&sa);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            total[kb] = add_halves(total[kb]);
            const int32_t slot = mine0 + 32 * kb + col;
            if (half != 0 || slot >= z.paged.slots) continue;
            if (splits > 1)
                z.parts[((static_cast<int64_t>(split) * z.paged.sequences + b) * z.paged.kv_heads + head) * z.paged.slots + slot] = total[kb];
            else
                store_score(z, b, head, slot, seq.length, total[kb]);
        }
    }
}

// Up to 32 rows a sequence and key head (more in further rounds): waves of their
// own, `run` slots each (at most kRun).  Keys go through a ring of tiles in LDS:
// a lane that fetched its own key's row straight into registers would touch
// every cache line four times, and more lines are in flight than L1 holds (92 us
// over 215 MB of keys, this way 57).  Totals wait in LDS until the run is done, so
// that no wait for a score to add to drains the ring.
constexpr int kRun = 1024;
template <int DP>
struct Few {
    static constexpr int kTileBytes = 32 * DP * 2, kRing = DP <= 128 ? 4 : 2, kWaveBytes = kRing * kTileBytes + kRun * 4;
    static constexpr int kLds = kScoreWaves * kWaveBytes;
};

template <typename T, int DP>
__global__ __launch_bounds__(64 * kScoreWaves, 1) void paged_scores_few_kernel(ScoreArgs, int32_t run) {
    using M = Mfma<T>;
    using F = Few<DP>;
    using TL = Tile<DP>;
    using St = Stager<DP, 32>;
    typedef typename M::frag frag;
    constexpr int kSteps = DP / 16;
    extern __shared__ __align__(16) char lds[];
    Kernarg<ScoreArgs> &sa = *kernargs<ScoreArgs>();
    Kernarg<PagedArgs> &a = sa.paged;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int col = lane % 32, half = lane / 32;
    uint32_t id = blockIdx.x;
    const uint32_t head = id % a.kv_heads;
    id /= a.kv_heads;
    const int32_t first = (id % a.tiles) * kScoreWaves + wave, b = id / a.tiles;
    const Sequence seq = sequence_of(a, b);
    const int32_t group = a.group.divisor, rows = seq.tokens * group, slots = a.slots, head_dim = a.head_dim;
    const int64_t stride = static_cast<int64_t>(a.tiles) * kScoreWaves * run;
    float scale = a.scale;
    keep(scale);
    char *const ring = lds + wave * F::kWaveBytes;
    float *const totals = reinterpret_cast<float *>(ring + F::kRing * F::kTileBytes);
    const uint32_t to_ring = lds_offset(ring);
    const int key_at = col * TL::kRowBytes + ((half ^ TL::key_turn(col)) * 16);
    St stager;
    stager.start(a, b, head, 0);

    for (int32_t row0 = 0; row0 == 0 || row0 < rows; row0 += 32) {
        // This lane's row as the first operand; log-sums of the rows that its products land in, and which of them count.
        const int32_t row = min(row0 + col, rows - 1);
        frag q[kSteps];
#pragma unroll
        for (int c = 0; c < kSteps; ++c) q[c] = frag{};
        if (row >= 0) {
            const int32_t token = fast_quotient(static_cast<uint32_t>(row), a.group), in_group = row - token * group;
            const char *query = a.query + (seq.start + token) * a.query_token +
                                (static_cast<int64_t>(head) * group + in_group) * a.query_head;
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
                if (16 * c + 8 * half < head_dim) q[c] = *reinterpret_cast<const frag *>(query + (16 * c + 8 * half) * 2);
        }
        float lse[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // all asked for at once, before any is looked at
            lse[i] = 0.0f;
            if (rows > 0) {
                const int32_t r = min(row0 + 8 * (i / 4) + 4 * half + i % 4, rows - 1);
                const int32_t t = fast_quotient(static_cast<uint32_t>(r), a.group);
                lse[i] = a.lse[(seq.start + t) * a.lse_token + static_cast<int64_t>(head) * group + (r - t * group)];
            }
        }
        uint32_t counts = 0;
        int32_t all_low = 0, all_high = INT32_MAX;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int32_t r = row0 + 8 * (i / 4) + 4 * half + i % 4;
            const Range sees = seen_by(a, seq, fast_quotient(static_cast<uint32_t>(min(r, max(rows - 1, 0))), a.group));
            const bool one = r < rows && lse[i] != -__builtin_inff() && sees.high > 0;
            counts |= one ? 1u << i : 0u;
            all_low = max(all_low, one ? sees.low : 0);
            all_high = min(all_high, one ? sees.high : INT32_MAX);
        }
        all_low = __builtin_amdgcn_readfirstlane(max(all_low, __shfl_xor(all_low, 32, 64)));
        all_high = __builtin_amdgcn_readfirstlane(min(all_high, __shfl_xor(all_high, 32, 64)));
        const bool any = __any(counts != 0);
#pragma unroll
        for (int c = 0; c < kSteps; ++c) asm volatile("" : "+v"(q[c]));  // arrived (not waited for at every tile)
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(lse[i]));

        for (int64_t run0 = static_cast<int64_t>(first) * run; run0 < slots; run0 += stride) {
            const int32_t from = static_cast<int32_t>(run0), to = static_cast<int32_t>(min<int64_t>(run0 + run, slots));
            const int32_t used = any ? min(to, seq.length) : 0, tiles = used > from ? (used - from + 31) / 32 : 0;
            auto stage = [&](int32_t t) {
                const typename St::Rows keys = stager.locate(from + 32 * t, seq.length);
                stager.load_keys(keys, to_ring + (t % F::kRing) * F::kTileBytes, 0);
            };
            for (int32_t t = 0; t < F::kRing && t < tiles; ++t) stage(t);
            for (int32_t t = 0; t < tiles; ++t) {
                if (t + F::kRing <= tiles)
                    landed<(F::kRing - 1) * St::kLoads>();
                else
                    landed<0>();
                const char *tile = ring + (t % F::kRing) * F::kTileBytes;
                const int32_t base = from + 32 * t, slot = base + col;
                f32x16 s = f32x16{};
                frag k[kSteps];
#pragma unroll
                for (int c = 0; c < kSteps; ++c) k[c] = *reinterpret_cast<const frag *>(tile + (key_at ^ (32 * c)));
#pragma unroll
                for (int c = 0; c < kSteps; ++c) s = M::run(q[c], k[c], s);
                if (t + F::kRing < tiles) {
                    reads_done();
                    stage(t + F::kRing);
                }
                uint32_t enter = counts;  // rows whose weights enter (left out is the weight: the log-sum may be NaN)
                if (base < all_low || base + 32 > all_high) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int32_t r = min(row0 + 8 * (i / 4) + 4 * half + i % 4, rows - 1);
                        const Range sees = seen_by(a, seq, fast_quotient(static_cast<uint32_t>(r), a.group));
                        if (slot < sees.low || slot >= sees.high) enter &= ~(1u << i);
                    }
                }
                float total = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    // The difference first: its rounding, not the log-sum's, bounds the weight's error.
                    const float w = __builtin_amdgcn_exp2f(fmaf(s[i], scale, -lse[i]) * kLog2e);
                    total += enter >> i & 1 ? w : 0.0f;
                }
                total = add_halves(total);
                if (half == 0) totals[32 * t + col] = total;
            }
            reads_done();  // (and writes: the totals are this wave's own)
            for (int32_t slot = from + lane; slot < to; slot += 64) {
                const float total = slot < used ? totals[slot - from] : 0.0f;
                if (row0 == 0)
                    store_score(sa, b, head, slot, used, total);
                else if (slot < used)
                    sa.out[b * sa.out_sequence + head * sa.out_head + slot] += total;
            }
            reads_done();  // before the next run's totals
        }
    }
}

__global__ __launch_bounds__(256) void paged_scores_join_kernel(ScoreArgs) {
    Kernarg<ScoreArgs> &sa = *kernargs<ScoreArgs>();
    Kernarg<PagedArgs> &a = sa.paged;
    const uint32_t b = blockIdx.z, head = blockIdx.y;
    const int32_t length = sequence_of(a, b).length;
    for (int32_t slot = blockIdx.x * 256 + threadIdx.x; slot < a.slots; slot += gridDim.x * 256) {
        const float was = sa.previous != nullptr ? sa.previous[b * sa.previous_sequence + head * sa.previous_head + slot] : 0.0f;
        float sum = 0.0f;
        if (slot < length)
            for (uint32_t s = 0; s < a.splits; ++s)
                sum += sa.parts[((static_cast<int64_t>(s) * a.sequences + b) * a.kv_heads + head) * a.slots + slot];
        sa.out[b * sa.out_sequence + head * sa.out_head + slot] = slot < length ? was + sum : was;
    }
}

struct ScorePlan {
    uint32_t tiles, splits;
    int32_t run;  // slots of a wave of the kernel for up to 32 rows; 0: the other
};

ScorePlan score_plan(uint32_t group, uint32_t kv_heads, uint32_t sequences, uint32_t tokens, uint32_t max_query,
                     uint32_t max_context) {
    ScorePlan p{};
    const uint64_t rows = static_cast<uint64_t>(std::min(max_query, tokens)) * group, cus = compute_units();
    p.splits = 1;
    if (rows <= 32) {
        // One workgroup a CU where sequences are alike, waves of 64 slots at least (16 sequences of 4k to 8k slots:
        // 56 us, with two 61, with four 68).
        const uint64_t all = static_cast<uint64_t>(std::max(1u, max_context)) * kv_heads * sequences;
        p.run = static_cast<int32_t>(std::min<uint64_t>(kRun, std::max<uint64_t>(64, (all / (4 * cus) + 63) / 64 * 64)));
        p.tiles = std::max<uint32_t>(1, static_cast<uint32_t>((max_context + static_cast<uint64_t>(p.run) * kScoreWaves - 1) /
                                                              (static_cast<uint64_t>(p.run) * kScoreWaves)));
        return p;
    }
    p.tiles = std::max(1u, static_cast<uint32_t>((static_cast<uint64_t>(max_context) + kScoreTile - 1) / kScoreTile));
    const uint64_t base = static_cast<uint64_t>(p.tiles) * kv_heads * sequences, wanted = 4 * cus;
    const uint64_t steps = (rows + kScoreRows - 1) / kScoreRows;
    p.splits = static_cast<uint32_t>(std::min<uint64_t>({(wanted + base - 1) / base, std::max<uint64_t>(1, steps / 8), 64}));
    return p;
}

size_t score_workspace(const ScorePlan &p, uint64_t sequences, uint64_t kv_heads, uint64_t slots) {
    return p.splits <= 1 ? 0 : p.splits * sequences * kv_heads * slots * 4;
}

template <typename T, int DP>
int launch_scores_dim(const ScoreArgs &sa, int32_t run, uint32_t grid, hipStream_t stream) {
    if (run > 0)
        return launch("paged_scores_few_kernel", paged_scores_few_kernel<T, DP>, dim3(grid), dim3(64 * kScoreWaves), Few<DP>::kLds,
                      stream, sa, run);
    return launch("paged_scores_kernel", paged_scores_kernel<T, DP>, dim3(grid), dim3(64 * kScoreWaves), 0, stream, sa);
}

template <typename T>
int launch_scores(const ScoreArgs &sa, int32_t run, uint32_t grid, hipStream_t stream) {
    const uint32_t d = sa.paged.head_dim;
    if (d <= 64) return launch_scores_dim<T, 64>(sa, run, grid, stream);
    if (d <= 128) return launch_scores_dim<T, 128>(sa, run, grid, stream);
    return launch_scores_dim<T, 256>(sa, run, grid, stream);
}

}  // namespace
}  // namespace qxt

extern "C" {

size_t qxt_paged_attention_scores_workspace(uint32_t query_heads, uint32_t kv_heads, uint32_t sequences, uint32_t tokens,
                                            uint32_t slots, uint32_t max_query, uint32_t max_context) {
    if (kv_heads == 0 || query_heads == 0 || query_heads % kv_heads || sequences == 0) return 0;
    auto bytes = [&](uint32_t longest) {
        return qxt::score_workspace(
            qxt::score_plan(query_heads / kv_heads, kv_heads, sequences, tokens, longest, std::min(max_context, slots)), sequences,
            kv_heads, slots);
    };
    return tokens == sequences ? std::max(bytes(max_query), bytes(1)) : bytes(max_query);  // a call without starts plans for 1
}

int qxt_paged_attention_scores(const void *query, size_t query_token_stride, size_t query_head_stride,
                               const qxt_paged_cache *cache, const int32_t *query_starts, const float *lse,
                               size_t lse_token_stride, const float *previous, size_t previous_sequence_stride,
                               size_t previous_head_stride, float *scores, size_t scores_sequence_stride,
                               size_t scores_head_stride, uint32_t tokens, uint32_t query_heads, float scale,
                               uint32_t causal, uint32_t window, uint32_t max_query, uint32_t max_context,
                               void *workspace, size_t workspace_bytes, void *stream) {
    using namespace qxt;
    if (int rc = check_paged_cache("paged attention scores", cache, false)) return rc;
    if (cache->sequences == 0) return QXT_OK;
    if (scores == nullptr || (tokens > 0 && (query == nullptr || lse == nullptr)))
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: null pointer");
    if (query_heads == 0 || query_heads % cache->heads)
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: query heads must be a multiple of the cache's");
    if (!(scale > 0.0f) || scale > 3e38f)
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: scale must be positive and finite");
    if (causal > 1 || window > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "paged attention scores: bad causal or window");
    if (query_starts == nullptr && tokens != cache->sequences)
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: without query starts every sequence has one token");
    if (static_cast<uint64_t>(tokens) * query_heads > INT32_MAX / 2)
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: 2^30 rows or more");
    if (!aligned(query, 16) || !all_multiples(16, {query_token_stride, query_head_stride}))
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: query rows must be 16-byte aligned");
    if (!aligned(lse, 4) || !aligned(previous, 4) || !aligned(scores, 4) ||
        !all_multiples(4, {lse_token_stride, previous_sequence_stride, previous_head_stride, scores_sequence_stride, scores_head_stride}))
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: misaligned scores or log-sums");
    if (cache->heads > 65535 || cache->sequences > 65535)
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: more than 65535 heads or sequences");
    if (query_starts == nullptr) max_query = 1;
    const uint32_t slots = cache->page_size * cache->table_width, group = query_heads / cache->heads;
    const ScorePlan p = score_plan(group, cache->heads, cache->sequences, tokens, max_query, std::min(max_context, slots));
    const size_t needed = score_workspace(p, cache->sequences, cache->heads, slots);
    if (needed > 0 && (workspace == nullptr || workspace_bytes < needed || !aligned(workspace, 4)))
        return fail(QXT_INVALID_ARGUMENT, "paged attention scores: workspace of %zu bytes needed", needed);
    const uint64_t grid = static_cast<uint64_t>(p.tiles) * p.splits * cache->heads * cache->sequences;
    if (grid > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "paged attention scores: too many slot tiles");
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;

    ScoreArgs sa{};
    PagedArgs &a = sa.paged;
    a.query = static_cast<const char *>(query);
    a.query_token = query_token_stride;
    a.query_head = query_head_stride;
    a.keys = {static_cast<char *>(cache->keys), static_cast<int64_t>(cache->key_page_stride),
              static_cast<int64_t>(cache->key_slot_stride), static_cast<int64_t>(cache->key_head_stride)};
    a.table = cache->block_table;
    a.table_stride = cache->block_table_stride / 4;
    a.pages = cache->pages;
    a.page = fast_div(cache->page_size);
    a.slots = static_cast<int32_t>(slots);
    a.lens = cache->context_lens;
    a.starts = query_starts;
    a.sequences = cache->sequences;
    a.tokens = tokens;
    a.kv_heads = cache->heads;
    a.head_dim = cache->head_dim;
    a.group = fast_div(group);
    a.scale = scale;
    a.causal = causal;
    a.window = window_of(window);
    const uint32_t dim = cache->head_dim <= 64 ? 64 : cache->head_dim <= 128 ? 128 : 256;
    a.even = cache->page_size % 8 == 0 && cache->head_dim == dim && cache->key_slot_stride < (1u << 28) &&
             static_cast<uint64_t>(cache->page_size) * (cache->key_slot_stride / 16) <= UINT32_MAX;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.lse = const_cast<float *>(lse);
    a.lse_token = lse_token_stride / 4;
    sa.previous = previous;
    sa.previous_sequence = previous_sequence_stride / 4;
    sa.previous_head = previous_head_stride / 4;
    sa.out = scores;
    sa.out_sequence = scores_sequence_stride / 4;
    sa.out_head = scores_head_stride / 4;
    sa.parts = static_cast<float *>(workspace);
    const int rc = cache->type == QXT_TYPE_BF16 ? launch_scores<bf16_t>(sa, p.run, static_cast<uint32_t>(grid), as_stream(stream))
                                                : launch_scores<f16_t>(sa, p.run, static_cast<uint32_t>(grid), as_stream(stream));
    if (rc != QXT_OK || p.splits == 1) return rc;
    return launch("paged_scores_join_kernel", paged_scores_join_kernel,
                  dim3(std::min(1024u, (slots + 255) / 256), cache->heads, cache->sequences), dim3(256), 0, as_stream(stream), sa);
}

}  // extern "C"
