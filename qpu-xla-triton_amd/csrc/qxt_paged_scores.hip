// The attention weight that each cached slot received from new tokens:
//   scores[b, head, j] = previous + sum over the sequence's tokens t and the
//   query heads h of the group of exp(scale q.k_j - lse[t, h]),
// with the log-sums of the attention over the same slots.
//
// Slots are independent, so a wave keeps its keys (two blocks of 32) in
// registers as the second operand of S = Q K^T (32x32x16 MFMAs), the rows of the
// chunk pass by in LDS, and each lane adds up the weights of its own key: no
// atomics, one order of the sum.  With one new token a sequence there is one
// step and the operator is bound by the bytes of the keys; over a prompt it is
// half the matrix work of the attention.  Where key tiles, heads and sequences
// alone are too few workgroups, the rows are dealt out over splits, whose sums a
// second launch adds in order.
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

constexpr int kScoreWaves = 4, kScoreKeys = 64, kScoreTile = kScoreWaves * kScoreKeys;

template <typename T, int DP>
__global__ __launch_bounds__(64 * kScoreWaves, DP <= 128 ? 2 : 1) void paged_scores_kernel(ScoreArgs sa) {
    using TL = Tile<DP>;
    using M = Mfma<T>;
    typedef typename M::frag frag;
    const PagedArgs &a = sa.paged;
    constexpr int kTileBytes = 32 * DP * 2, kOwn = 32 / kScoreWaves, kLoads = kOwn / TL::kRowsPerLoad;
    static_assert(kOwn % TL::kRowsPerLoad == 0, "a wave stages whole loads");
    __shared__ __align__(16) char rows_lds[2][kTileBytes];
    __shared__ __align__(16) float row_lse[2][32];
    __shared__ __align__(16) int32_t row_low[2][32], row_high[2][32];
    __shared__ int32_t odd_rows[2];  // the step has rows that count for nothing

    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int col = lane % 32, half = lane / 32;
    uint32_t id = blockIdx.x;
    const uint32_t head = id % a.kv_heads;
    id /= a.kv_heads;
    const uint32_t first_tile = id % a.tiles;
    id /= a.tiles;
    const uint32_t split = id % a.splits, b = id / a.splits;
    const Sequence seq = sequence_of(a, b);
    const int32_t group = a.group.divisor, rows = seq.tokens * group;
    const int32_t *table = a.table + b * a.table_stride;
    const char *keys = a.keys.data + head * a.keys.head_stride;
    const int row_at = col * TL::kRowBytes + ((half ^ TL::key_turn(col)) * 16);

    for (int64_t tile0 = static_cast<int64_t>(first_tile) * kScoreTile; tile0 < a.slots;
         tile0 += static_cast<int64_t>(a.tiles) * kScoreTile) {
        const int32_t key0 = static_cast<int32_t>(tile0), key_end = min(key0 + kScoreTile, seq.length);
        float total[2] = {0.0f, 0.0f};
        const int32_t mine0 = key0 + wave * kScoreKeys;
        // Tokens that see any slot of the tile.
        int32_t first = 0, last = seq.tokens;
        const int32_t before = seq.length - seq.tokens;
        if (a.causal) first = max(0, key0 - before);
        if (a.window > 0) last = static_cast<int32_t>(min<int64_t>(last, static_cast<int64_t>(key_end) - 1 + a.window - before));
        const int32_t row_first = first * group, row_last = last * group;
        if (key0 < key_end && row_first < row_last) {
            frag k[2][DP / 16];
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
                    if (row != nullptr && 16 * c + 8 * half < static_cast<int>(a.head_dim))
                        k[kb][c] = *reinterpret_cast<const frag *>(row + (16 * c + 8 * half) * 2);
                }
            }
            const int32_t step0 = row_first / 32, steps = (row_last + 31) / 32;
            // Rows 32 t + 8 wave .. + 7 of step t into LDS; wave 0 also fetches what the rows see and their log-sums.
            float lse = 0.0f;
            Range sees{0, 0};
            auto stage = [&](int32_t t, int buffer) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = wave * kOwn + i * TL::kRowsPerLoad + lane / TL::kChunks;
                    const int32_t row = min(32 * t + r, rows - 1);
                    const int32_t token = fast_quotient(row, a.group), h = row - token * group;
                    const int chunk = (lane % TL::kChunks) ^ TL::key_turn(r);
                    const char *src = a.query + (seq.start + token) * a.query_token +
                                      static_cast<int64_t>(head * group + h) * a.query_head + chunk * 16;
                    if (chunk * 8 >= static_cast<int>(a.head_dim)) src = reinterpret_cast<const char *>(kZeroRow);
                    __builtin_amdgcn_global_load_lds(
                        (const __attribute__((address_space(1))) void *)src,
                        (__attribute__((address_space(3))) void *)(rows_lds[buffer] + wave * kOwn * TL::kRowBytes + i * 1024),
                        16, 0, 0);
                }
                if (wave == 0) {
                    const int32_t row = 32 * t + col;
                    sees = Range{0, 0};
                    lse = 0.0f;
                    if (row < rows) {
                        const int32_t token = fast_quotient(row, a.group), h = row - token * group;
                        sees = seen_by(a, seq, token);
                        lse = a.lse[(seq.start + token) * a.lse_token + static_cast<int64_t>(head) * group + h];
                    }
                }
            };
            int buffer = 0;
            int32_t t = step0 + split;
            if (t < steps) stage(t, 0);
            for (; t < steps; t += a.splits, buffer ^= 1) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                if (wave == 0) {
                    if (lse == -__builtin_inff()) sees = Range{0, 0};  // a row without weights
                    if (half == 0) {
                        row_lse[buffer][col] = lse;
                        row_low[buffer][col] = sees.low;
                        row_high[buffer][col] = sees.high;
                    }
                    const bool odd = __any(sees.high == 0);
                    if (lane == 0) odd_rows[buffer] = odd;
                }
                __syncthreads();  // step t is staged, and step t - 1 has been read
                if (t + static_cast<int32_t>(a.splits) < steps) stage(t + a.splits, buffer ^ 1);
                f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    const frag q = *reinterpret_cast<const frag *>(rows_lds[buffer] + (row_at ^ (32 * c)));
                    s[0] = M::run(q, k[0][c], s[0]);
                    s[1] = M::run(q, k[1][c], s[1]);
                }
                // Rows see contiguous ranges that only move up: all see all of the wave's slots if the first and last do.
                const bool partial = __builtin_amdgcn_readfirstlane(odd_rows[buffer]) != 0 ||
                                     __builtin_amdgcn_readfirstlane(row_high[buffer][0]) < mine0 + kScoreKeys ||
                                     __builtin_amdgcn_readfirstlane(row_low[buffer][31]) > mine0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 l = *reinterpret_cast<const float4 *>(&row_lse[buffer][8 * i + 4 * half]);
                    const float *ls = &l.x;
                    int4 lo = make_int4(0, 0, 0, 0), hi = lo;
                    if (partial) {
                        lo = *reinterpret_cast<const int4 *>(&row_low[buffer][8 * i + 4 * half]);
                        hi = *reinterpret_cast<const int4 *>(&row_high[buffer][8 * i + 4 * half]);
                    }
                    const int32_t *los = &lo.x, *his = &hi.x;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // The difference first: its rounding, not the log-sum's, bounds the weight's error.
                            float w = __builtin_amdgcn_exp2f(fmaf(s[kb][4 * i + e], a.scale, -ls[e]) * 1.44269504f);
                            const int32_t slot = mine0 + 32 * kb + col;
                            if (partial && (slot < los[e] || slot >= his[e])) w = 0.0f;
                            total[kb] += w;
                        }
                }
            }
            __syncthreads();  // before the next tile's staging
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            total[kb] = add_halves(total[kb]);
            const int32_t slot = mine0 + 32 * kb + col;
            if (half != 0 || slot >= a.slots) continue;
            if (a.splits > 1) {
                sa.parts[((static_cast<int64_t>(split) * a.sequences + b) * a.kv_heads + head) * a.slots + slot] = total[kb];
                continue;
            }
            const float was = sa.previous != nullptr ? sa.previous[b * sa.previous_sequence + head * sa.previous_head + slot] : 0.0f;
            // (was itself, not was + 0, where nothing was added: unused slots keep their bits.)
            sa.out[b * sa.out_sequence + head * sa.out_head + slot] = slot < seq.length ? was + total[kb] : was;
        }
    }
}

__global__ __launch_bounds__(256) void paged_scores_join_kernel(ScoreArgs sa) {
    const PagedArgs &a = sa.paged;
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
};

ScorePlan score_plan(uint32_t group, uint32_t kv_heads, uint32_t sequences, uint32_t tokens, uint32_t max_query,
                     uint32_t max_context) {
    ScorePlan p;
    p.tiles = std::max(1u, (max_context + kScoreTile - 1) / kScoreTile);
    const uint64_t base = static_cast<uint64_t>(p.tiles) * kv_heads * sequences, wanted = 4ull * compute_units();
    const uint64_t steps = (static_cast<uint64_t>(std::min(max_query, tokens)) * group + 31) / 32;
    p.splits = static_cast<uint32_t>(std::min<uint64_t>({(wanted + base - 1) / base, std::max<uint64_t>(1, steps / 8), 64}));
    return p;
}

size_t score_workspace(const ScorePlan &p, uint64_t sequences, uint64_t kv_heads, uint64_t slots) {
    return p.splits <= 1 ? 0 : p.splits * sequences * kv_heads * slots * 4;
}

template <typename T>
int launch_scores(const ScoreArgs &sa, uint32_t grid, hipStream_t stream) {
    const uint32_t threads = 64 * kScoreWaves, d = sa.paged.head_dim;
    if (d <= 64) return launch("paged_scores_kernel", paged_scores_kernel<T, 64>, dim3(grid), dim3(threads), 0, stream, sa);
    if (d <= 128) return launch("paged_scores_kernel", paged_scores_kernel<T, 128>, dim3(grid), dim3(threads), 0, stream, sa);
    return launch("paged_scores_kernel", paged_scores_kernel<T, 256>, dim3(grid), dim3(threads), 0, stream, sa);
}

}  // namespace
}  // namespace qxt

extern "C" {

size_t qxt_paged_attention_scores_workspace(uint32_t query_heads, uint32_t kv_heads, uint32_t sequences, uint32_t tokens,
                                            uint32_t slots, uint32_t max_query, uint32_t max_context) {
    if (kv_heads == 0 || query_heads == 0 || query_heads % kv_heads || sequences == 0) return 0;
    return qxt::score_workspace(
        qxt::score_plan(query_heads / kv_heads, kv_heads, sequences, tokens, max_query, max_context), sequences, kv_heads, slots);
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
    a.window = static_cast<int32_t>(window);
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
    const int rc = cache->type == QXT_TYPE_BF16 ? launch_scores<bf16_t>(sa, static_cast<uint32_t>(grid), as_stream(stream))
                                                : launch_scores<f16_t>(sa, static_cast<uint32_t>(grid), as_stream(stream));
    if (rc != QXT_OK || p.splits == 1) return rc;
    return launch("paged_scores_join_kernel", paged_scores_join_kernel,
                  dim3(std::min(1024u, (slots + 255) / 256), cache->heads, cache->sequences), dim3(256), 0, as_stream(stream), sa);
}

}  // extern "C"
