// Eviction from a paged cache by accumulated attention weight.
//
// A sequence of more than `budget` slots keeps, for each head, the `budget`
// slots that come first by (recent or not, score, lower slot).  Kept slots below
// `budget` stay where they are; the i-th slot there that is given up takes the
// i-th kept slot at or above `budget`, so every read lies at or above it and
// every write below: rows move in place, in any order, once, and only those that
// have to.  (Attention does not ask for an order of slots whose keys are rotated
// already; positions travel with them.)
//
// Selection is by radix: the recent slots and the scores give 32-bit keys of the
// same order, and three passes over 11, 11 and 10 bits of them find the
// budget-th largest; ties at it go to the lowest slots by a scan in slot order.
// One workgroup does that for a (sequence, head); a second launch over all of
// them moves the rows.
// Measured: 32k slots to 4k for 32 (sequence, head) pairs 55 us to select
// (32 of 256 CUs work, their vector units 52 % busy with the passes over the
// keys), and 20 to move, near the rate of a copy; one slot over for 256 pairs 8 us.
#include <algorithm>
#include <utility>

#include "qxt_paged.h"

namespace qxt {
int check_paged_cache(const char *name, const qxt_paged_cache *cache, bool needs_values);

namespace {

struct EvictArgs {
    CacheView keys, values;
    const int32_t *table;
    int64_t table_stride;
    uint32_t pages;
    FastDiv page;
    int32_t slots;
    const int32_t *lens;
    int32_t *lens_out;
    uint32_t heads, row_chunks;  // 16-byte chunks of a row
    int32_t budget, recent;
    const float *scores;
    float *scores_out;
    const int32_t *positions;
    int32_t *positions_out;
    int64_t score_sequence, score_head, position_sequence, position_head;          // elements
    int64_t score_out_sequence, score_out_head, position_out_sequence, position_out_head;
    int32_t *moves;  // per (sequence, head): count, then `most` pairs (to, from)
    int32_t most;
};

// Unsigned keys in the order of the scores; NaN is the least, -0 equals 0.
__device__ __forceinline__ uint32_t ordered(float score) {
    if (score != score) return 0;
    const uint32_t u = __float_as_uint(score + 0.0f);
    return u ^ (static_cast<int32_t>(u) < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
constexpr uint32_t kRecentKey = 0xFFFFFFFFu;  // above +inf's

__device__ __forceinline__ int wave_sum(int x) {
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    return x;
}

// Rows of the moved slots of one (sequence, head): a row is row_chunks lanes.
__device__ __forceinline__ void move_rows(const EvictArgs &a, uint32_t b, uint32_t head, const int32_t *moves,
                                          int32_t count, uint32_t first, uint32_t step) {
    const int32_t *table = a.table + b * a.table_stride;
    const uint64_t work = static_cast<uint64_t>(count) * a.row_chunks;
    for (uint64_t i = first; i < work; i += step) {
        const uint32_t move = static_cast<uint32_t>(i / a.row_chunks), chunk = static_cast<uint32_t>(i - static_cast<uint64_t>(move) * a.row_chunks);
        const int2 m = make_int2(moves[2 * move], moves[2 * move + 1]);
        const uint32_t to_page = fast_quotient(m.x, a.page), from_page = fast_quotient(m.y, a.page);
        const int64_t to_id = table[to_page], from_id = table[from_page];
        if (to_id < 0 || to_id >= a.pages) continue;
        const int64_t to_in = m.x - to_page * a.page.divisor, from_in = m.y - from_page * a.page.divisor;
        uint4 key = {0, 0, 0, 0}, value = key;  // a slot without a page counts as a zero row
        if (from_id >= 0 && from_id < a.pages) {
            key = *reinterpret_cast<const uint4 *>(a.keys.data + from_id * a.keys.page_stride + from_in * a.keys.slot_stride +
                                                   head * a.keys.head_stride + chunk * 16);
            value = *reinterpret_cast<const uint4 *>(a.values.data + from_id * a.values.page_stride +
                                                     from_in * a.values.slot_stride + head * a.values.head_stride + chunk * 16);
        }
        *reinterpret_cast<uint4 *>(a.keys.data + to_id * a.keys.page_stride + to_in * a.keys.slot_stride +
                                   head * a.keys.head_stride + chunk * 16) = key;
        *reinterpret_cast<uint4 *>(a.values.data + to_id * a.values.page_stride + to_in * a.values.slot_stride +
                                   head * a.values.head_stride + chunk * 16) = value;
    }
}

constexpr int kBins = 2048;
constexpr int kFew = 4;
constexpr int kBatch = 8;         // loads under way in passes over memory (one at a time took most of the kernel's time)
constexpr int kHeldKeys = 32768;  // keys that LDS holds (128 KB); longer sequences read their scores again

template <int THREADS, bool MOVE>
__global__ __launch_bounds__(THREADS) void paged_evict_plan_kernel(EvictArgs a) {
    constexpr int kWaves = THREADS / 64;
    extern __shared__ uint32_t held[];
    __shared__ uint32_t bins[kBins];
    __shared__ int32_t parts[3][kWaves];
    __shared__ uint32_t chosen_digit, still_wanted;
    __shared__ uint64_t ranks[kWaves];
    __shared__ int32_t dropped[kFew], few_moves[2 * kFew], few_count;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const uint32_t head = blockIdx.x, b = blockIdx.y;
    const int32_t length = min(max(a.lens[b], 0), a.slots);
    const float *scores = a.scores + b * a.score_sequence + head * a.score_head;
    const int32_t *positions = a.positions + b * a.position_sequence + head * a.position_head;
    float *scores_out = a.scores_out + b * a.score_out_sequence + head * a.score_out_head;
    int32_t *positions_out = a.positions_out + b * a.position_out_sequence + head * a.position_out_head;
    int32_t *moves = a.moves + (static_cast<int64_t>(b) * a.heads + head) * (2 * static_cast<int64_t>(a.most) + 2);
    const int32_t budget = a.budget, kept_length = min(length, budget);
    if (head == 0 && tid == 0) a.lens_out[b] = kept_length;

    // Slots from `begin` to `end` that stay as they are (nothing to do in place).
    auto copy = [&](int32_t begin, int32_t end) {
        if (scores_out == scores && positions_out == positions) return;
        for (int32_t s0 = begin + tid; s0 < end; s0 += kBatch * THREADS) {
            float score[kBatch];
            int32_t position[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                score[u] = scores[min(s0 + u * THREADS, end - 1)];
                position[u] = positions[min(s0 + u * THREADS, end - 1)];
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int32_t s = s0 + u * THREADS;
                if (s >= end) break;
                if (scores_out != scores) scores_out[s] = score[u];
                if (positions_out != positions) positions_out[s] = position[u];
            }
        }
    };
    if (MOVE) copy(length, a.slots);
    if (length <= budget) {
        copy(0, length);
        if (tid == 0) moves[0] = 0;
        return;
    }

    // One pass over scores and positions: keys by score alone, the newest position, what stays below the budget.
    const bool holds = length <= kHeldKeys;
    int32_t newest = INT32_MIN;
    for (int32_t s0 = tid; s0 < length; s0 += kBatch * THREADS) {
        float score[kBatch];
        int32_t position[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            score[u] = scores[min(s0 + u * THREADS, length - 1)];
            position[u] = positions[min(s0 + u * THREADS, length - 1)];
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int32_t s = s0 + u * THREADS;
            if (s >= length) break;
            newest = max(newest, position[u]);
            if (holds) held[s] = min(ordered(score[u]), kRecentKey - 1);
            if (s < budget && scores_out != scores) scores_out[s] = score[u];
            if (s < budget && positions_out != positions) positions_out[s] = position[u];
        }
    }
    for (int off = 32; off > 0; off >>= 1) newest = max(newest, __shfl_xor(newest, off, 64));
    if (lane == 0) parts[0][wave] = newest;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) newest = max(newest, parts[0][w]);
    const int64_t recent_after = static_cast<int64_t>(newest) - a.recent;

    auto key_from_memory = [&](int32_t s) {
        return positions[s] > recent_after ? kRecentKey : min(ordered(scores[s]), kRecentKey - 1);
    };
    if (holds && a.recent > 0)  // the recent slots' keys, from positions that are in cache now
        for (int32_t s0 = tid; s0 < length; s0 += kBatch * THREADS) {
            int32_t position[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) position[u] = positions[min(s0 + u * THREADS, length - 1)];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (s0 + u * THREADS < length && position[u] > recent_after) held[s0 + u * THREADS] = kRecentKey;
        }
    auto key_of = [&](int32_t s) { return holds ? held[s] : key_from_memory(s); };

    // The moves' effect on scores and positions, and (MOVE) on the rows.
    auto apply = [&](const int32_t *pairs, int32_t count) {
        for (int i = tid; i < count; i += THREADS) {
            const int32_t to = pairs[2 * i], from = pairs[2 * i + 1];
            scores_out[to] = scores[from];
            positions_out[to] = positions[from];
        }
        if (!MOVE) return;  // the second launch does the rest
        move_rows(a, b, head, pairs, count, tid, THREADS);
        __syncthreads();  // in place, the freed slots have been read
        for (int32_t s = budget + tid; s < length; s += THREADS) {
            scores_out[s] = 0.0f;
            positions_out[s] = -1;
        }
    };

    // A slot or a few over the budget, as at every decode step: the last slots in order are found one after another
    // (one of 2049: 18.5 us by radix, 8.0 this way).
    if (MOVE && holds && length - budget <= kFew) {
        const int32_t over = length - budget;
        uint64_t last = 0;  // key and reversed slot, plus one, of the slot found before
        __syncthreads();    // the keys are in place
        for (int32_t r = 0; r < over; ++r) {
            uint64_t least = UINT64_MAX;
            for (int32_t s = tid; s < length; s += THREADS) {
                const uint64_t rank = (static_cast<uint64_t>(held[s]) << 32) | (0x7FFFFFFFu - static_cast<uint32_t>(s));
                if (rank >= last && rank < least) least = rank;
            }
            for (int off = 32; off > 0; off >>= 1) {
                const uint64_t other = __shfl_xor(static_cast<unsigned long long>(least), off, 64);
                least = other < least ? other : least;
            }
            if (lane == 0) ranks[wave] = least;
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) least = ranks[w] < least ? ranks[w] : least;
            if (tid == 0) dropped[r] = 0x7FFFFFFF - static_cast<int32_t>(least & 0xFFFFFFFFu);
            last = least + 1;
            __syncthreads();
        }
        int32_t count = 0;
        if (tid == 0) {
            // Dropped slots below the budget in rising order, with the slots above it that were not dropped.
            int32_t from = budget;
            for (int32_t done = -1;;) {
                int32_t to = budget;
                for (int32_t r = 0; r < over; ++r)
                    if (dropped[r] > done && dropped[r] < to) to = dropped[r];
                if (to == budget) break;
                for (bool gone = true; gone; ++from) {
                    gone = false;
                    for (int32_t r = 0; r < over; ++r) gone = gone || dropped[r] == from;
                }
                few_moves[2 * count] = to;
                few_moves[2 * count + 1] = from - 1;
                ++count;
                done = to;
            }
            few_count = count;
        }
        __syncthreads();
        apply(few_moves, few_count);
        return;
    }

    // The budget-th largest key, most significant digit first.
    uint32_t prefix = 0, wanted = budget;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kBins; i += THREADS) bins[i] = 0;
        __syncthreads();
        for (int32_t s = tid; s < length; s += THREADS) {
            const uint32_t key = key_of(s);
            if (pass == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&bins[(key >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // The bin where the count from the top passes what is wanted: each thread sums a run of bins, a scan
        // over threads gives what lies above the run.
        constexpr int kRun = kBins / THREADS > 0 ? kBins / THREADS : 1;
        int mine = 0;
        for (int i = 0; i < kRun; ++i) mine += bins[(THREADS - 1 - tid) * kRun + i];  // high bins first
        int scan = mine;
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(scan, off, 64);
            if (lane >= off) scan += up;
        }
        if (lane == 63) parts[1][wave] = scan;
        __syncthreads();
        int above = scan - mine;
        for (int w = 0; w < wave; ++w) above += parts[1][w];
        if (above < static_cast<int>(wanted) && above + mine >= static_cast<int>(wanted)) {
            for (int i = kRun - 1; i >= 0; --i) {
                const int bin = (THREADS - 1 - tid) * kRun + i, count = bins[bin];
                if (above + count >= static_cast<int>(wanted)) {
                    chosen_digit = bin;
                    still_wanted = wanted - above;
                    break;
                }
                above += count;
            }
        }
        __syncthreads();
        prefix = pass == 0 ? chosen_digit : (prefix << bits) | chosen_digit;
        wanted = still_wanted;
    }
    const uint32_t threshold = prefix;  // keys above it stay, and the first `wanted` slots that have it

    // Waves own runs of slots (whole multiples of 64) and count in slot order with ballots.
    const int32_t run = ((length + 64 * kWaves - 1) / (64 * kWaves)) * 64, run0 = min(wave * run, length), run1 = min(run0 + run, length);
    int ties = 0;
    for (int32_t s0 = run0; s0 < run1; s0 += 64) {
        const int32_t s = s0 + lane;
        ties += __popcll(__ballot(s < run1 && key_of(s) == threshold));
    }
    if (lane == 0) parts[0][wave] = ties;
    __syncthreads();
    int ties_before = 0;
    for (int w = 0; w < wave; ++w) ties_before += parts[0][w];
    const uint64_t below = (1ull << lane) - 1;
    auto kept_at = [&](int32_t s, int &seen_ties) {  // wave-wide; s in slot order over calls
        const bool in = s < run1;
        const uint32_t key = in ? key_of(s) : 0;
        const uint64_t tie = __ballot(in && key == threshold);
        const bool keep = in && (key > threshold || (key == threshold && seen_ties + __popcll(tie & below) < static_cast<int>(wanted)));
        seen_ties += __popcll(tie);
        return keep;
    };
    int holes = 0, movers = 0, running = ties_before;
    for (int32_t s0 = run0; s0 < run1; s0 += 64) {
        const int32_t s = s0 + lane;
        const bool keep = kept_at(s, running);
        holes += __popcll(__ballot(s < run1 && !keep && s < budget));
        movers += __popcll(__ballot(keep && s >= budget));
    }
    if (lane == 0) {
        parts[1][wave] = holes;
        parts[2][wave] = movers;
    }
    __syncthreads();
    int hole_at = 0, mover_at = 0, count = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) {
            hole_at += parts[1][w];
            mover_at += parts[2][w];
        }
        count += parts[1][w];
    }
    running = ties_before;
    for (int32_t s0 = run0; s0 < run1; s0 += 64) {
        const int32_t s = s0 + lane;
        const bool keep = kept_at(s, running);
        const bool hole = s < run1 && !keep && s < budget, mover = keep && s >= budget;
        const uint64_t hole_mask = __ballot(hole), mover_mask = __ballot(mover);
        if (hole) moves[2 + 2 * (hole_at + __popcll(hole_mask & below))] = s;
        if (mover) moves[2 + 2 * (mover_at + __popcll(mover_mask & below)) + 1] = s;
        hole_at += __popcll(hole_mask);
        mover_at += __popcll(mover_mask);
    }
    if (tid == 0) moves[0] = count;
    __threadfence_block();
    __syncthreads();
    apply(moves + 2, count);
}

// Over the whole chip: the rows of the moves that the first launch left, zeros in the freed slots, and what lies past
// the sequences.
__global__ __launch_bounds__(256) void paged_evict_move_kernel(EvictArgs a) {
    const uint32_t head = blockIdx.y, b = blockIdx.z, first = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
    const int32_t *moves = a.moves + (static_cast<int64_t>(b) * a.heads + head) * (2 * static_cast<int64_t>(a.most) + 2);
    move_rows(a, b, head, moves + 2, moves[0], first, step);
    const int32_t length = min(max(a.lens[b], 0), a.slots);
    const float *scores = a.scores + b * a.score_sequence + head * a.score_head;
    const int32_t *positions = a.positions + b * a.position_sequence + head * a.position_head;
    float *scores_out = a.scores_out + b * a.score_out_sequence + head * a.score_out_head;
    int32_t *positions_out = a.positions_out + b * a.position_out_sequence + head * a.position_out_head;
    for (int64_t s = static_cast<int64_t>(a.budget) + first; s < length; s += step) {
        scores_out[s] = 0.0f;
        positions_out[s] = -1;
    }
    for (int64_t s = static_cast<int64_t>(length) + first; s < a.slots; s += step) {
        if (scores_out != scores) scores_out[s] = scores[s];
        if (positions_out != positions) positions_out[s] = positions[s];
    }
}

int32_t most_moves(uint64_t slots, uint32_t budget) {
    return slots <= budget ? 0 : static_cast<int32_t>(std::min<uint64_t>(budget, slots - budget));
}

// One row of `bytes` for each (sequence, head).
struct RowSet {
    const void *data;
    size_t sequence, head;  // strides in bytes
};

// Whether rows of x and y share memory, those at one place in both (in place) aside.  A workgroup whose scores others
// write meanwhile would count them differently from pass to pass, and follow moves of which one end was never written.
bool rows_overlap(RowSet x, RowSet y, uint32_t sequences, uint32_t heads, size_t bytes) {
    if (sequences == 1) x.sequence = y.sequence = 0;
    if (heads == 1) x.head = y.head = 0;
    const int64_t apart = static_cast<int64_t>(reinterpret_cast<uintptr_t>(y.data) - reinterpret_cast<uintptr_t>(x.data));
    auto span = [&](const RowSet &r) { return static_cast<int64_t>((sequences - 1) * r.sequence + (heads - 1) * r.head + bytes); };
    if (apart >= span(x) || -apart >= span(y)) return false;
    if (x.sequence != y.sequence || x.head != y.head) return true;  // interleaved in two ways: not worth telling apart
    if (apart == 0) {
        // The usual orders: whole sequences one after another, or whole heads.
        const bool by_head = heads > 1 && (sequences == 1 || x.head < x.sequence);
        const size_t inner = by_head ? x.head : x.sequence, outer = by_head ? x.sequence : x.head;
        const uint32_t inner_rows = by_head ? heads : sequences, outer_rows = by_head ? sequences : heads;
        if ((inner_rows == 1 || inner >= bytes) && (outer_rows == 1 || outer >= (inner_rows - 1) * inner + bytes)) return false;
    }
    const int64_t row = static_cast<int64_t>(bytes);
    for (int64_t i = 1 - static_cast<int64_t>(sequences); i < static_cast<int64_t>(sequences); ++i)
        for (int64_t j = 1 - static_cast<int64_t>(heads); j < static_cast<int64_t>(heads); ++j) {
            if (apart == 0 && i == 0 && j == 0) continue;
            const int64_t between = apart + i * static_cast<int64_t>(x.sequence) + j * static_cast<int64_t>(x.head);
            if (between < row && -between < row) return true;
        }
    return false;
}

template <int THREADS, bool MOVE>
int launch_plan(const EvictArgs &a, uint32_t sequences, size_t lds, hipStream_t stream) {
    return launch("paged_evict_plan_kernel", paged_evict_plan_kernel<THREADS, MOVE>, dim3(a.heads, sequences), dim3(THREADS),
                  lds, stream, a);
}

}  // namespace
}  // namespace qxt

extern "C" {

size_t qxt_paged_cache_evict_workspace(uint32_t heads, uint32_t sequences, uint32_t slots, uint32_t budget) {
    return static_cast<size_t>(heads) * sequences * (2 * static_cast<size_t>(qxt::most_moves(slots, budget)) + 2) * 4;
}

int qxt_paged_cache_evict(const qxt_paged_cache *cache, const float *scores, size_t scores_sequence_stride,
                          size_t scores_head_stride, float *scores_out, size_t scores_out_sequence_stride,
                          size_t scores_out_head_stride, const int32_t *positions, size_t positions_sequence_stride,
                          size_t positions_head_stride, int32_t *positions_out, size_t positions_out_sequence_stride,
                          size_t positions_out_head_stride, int32_t *lens_out, uint32_t budget, uint32_t recent,
                          uint32_t max_context, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace qxt;
    if (int rc = check_paged_cache("paged cache evict", cache, true)) return rc;
    if (cache->sequences == 0) return QXT_OK;
    if (scores == nullptr || scores_out == nullptr || positions == nullptr || positions_out == nullptr || lens_out == nullptr)
        return fail(QXT_INVALID_ARGUMENT, "paged cache evict: null pointer");
    if (lens_out < cache->context_lens + cache->sequences && cache->context_lens < lens_out + cache->sequences)
        // (other workgroups still read the old ones)
        return fail(QXT_INVALID_ARGUMENT, "paged cache evict: new lengths must not replace the old ones in place");
    if (budget == 0 || budget > INT32_MAX / 2 || recent > budget)
        return fail(QXT_INVALID_ARGUMENT, "paged cache evict: budget must be positive and recent at most the budget");
    if (!all_multiples(4, {scores_sequence_stride, scores_head_stride, scores_out_sequence_stride, scores_out_head_stride,
                           positions_sequence_stride, positions_head_stride, positions_out_sequence_stride,
                           positions_out_head_stride}) ||
        !aligned(scores, 4) || !aligned(scores_out, 4) || !aligned(positions, 4) || !aligned(positions_out, 4) || !aligned(lens_out, 4))
        return fail(QXT_INVALID_ARGUMENT, "paged cache evict: misaligned scores, positions or lengths");
    if (cache->heads > 65535 || cache->sequences > 65535)
        return fail(QXT_INVALID_ARGUMENT, "paged cache evict: more than 65535 heads or sequences");
    const uint32_t slots = cache->page_size * cache->table_width;
    for (const auto &[in, out] : {std::pair<RowSet, RowSet>{{scores, scores_sequence_stride, scores_head_stride},
                                                            {scores_out, scores_out_sequence_stride, scores_out_head_stride}},
                                  {{positions, positions_sequence_stride, positions_head_stride},
                                   {positions_out, positions_out_sequence_stride, positions_out_head_stride}}})
        if (rows_overlap(out, out, cache->sequences, cache->heads, 4 * static_cast<size_t>(slots)) ||
            rows_overlap(in, out, cache->sequences, cache->heads, 4 * static_cast<size_t>(slots)))
            return fail(QXT_INVALID_ARGUMENT, "paged cache evict: output rows share memory with other rows");
    const size_t needed = qxt_paged_cache_evict_workspace(cache->heads, cache->sequences, slots, budget);
    if (workspace == nullptr || workspace_bytes < needed || !aligned(workspace, 8))
        return fail(QXT_INVALID_ARGUMENT, "paged cache evict: workspace of %zu bytes needed", needed);
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;

    EvictArgs a{};
    a.keys = {static_cast<char *>(cache->keys), static_cast<int64_t>(cache->key_page_stride),
              static_cast<int64_t>(cache->key_slot_stride), static_cast<int64_t>(cache->key_head_stride)};
    a.values = {static_cast<char *>(cache->values), static_cast<int64_t>(cache->value_page_stride),
                static_cast<int64_t>(cache->value_slot_stride), static_cast<int64_t>(cache->value_head_stride)};
    a.table = cache->block_table;
    a.table_stride = cache->block_table_stride / 4;
    a.pages = cache->pages;
    a.page = fast_div(cache->page_size);
    a.slots = static_cast<int32_t>(slots);
    a.lens = cache->context_lens;
    a.lens_out = lens_out;
    a.heads = cache->heads;
    a.row_chunks = cache->head_dim / 8;
    a.budget = static_cast<int32_t>(budget);
    a.recent = static_cast<int32_t>(recent);
    a.scores = scores;
    a.scores_out = scores_out;
    a.positions = positions;
    a.positions_out = positions_out;
    a.score_sequence = scores_sequence_stride / 4;
    a.score_head = scores_head_stride / 4;
    a.position_sequence = positions_sequence_stride / 4;
    a.position_head = positions_head_stride / 4;
    a.score_out_sequence = scores_out_sequence_stride / 4;
    a.score_out_head = scores_out_head_stride / 4;
    a.position_out_sequence = positions_out_sequence_stride / 4;
    a.position_out_head = positions_out_head_stride / 4;
    a.moves = static_cast<int32_t *>(workspace);
    a.most = most_moves(slots, budget);
    // Bounds from the host's longest context size the launches; longer ones on the device still move in full.
    const uint32_t longest = std::min(max_context, slots);
    const int32_t moved = most_moves(longest, budget);
    const size_t lds = static_cast<size_t>(std::min<uint32_t>(slots, kHeldKeys)) * 4;
    const bool few = moved <= 32;  // one launch: the planning workgroup moves them itself
    const hipStream_t on = as_stream(stream);
    int rc;
    if (longest > 8192)
        rc = few ? launch_plan<1024, true>(a, cache->sequences, lds, on) : launch_plan<1024, false>(a, cache->sequences, lds, on);
    else
        rc = few ? launch_plan<256, true>(a, cache->sequences, lds, on) : launch_plan<256, false>(a, cache->sequences, lds, on);
    if (rc != QXT_OK || few) return rc;
    const uint64_t chunks = static_cast<uint64_t>(moved) * a.row_chunks;
    const uint32_t blocks = static_cast<uint32_t>(std::min<uint64_t>((std::max<uint64_t>(chunks, slots) + 1023) / 1024, 256));
    return launch("paged_evict_move_kernel", paged_evict_move_kernel, dim3(blocks, cache->heads, cache->sequences), dim3(256), 0, on, a);
}

}  // extern "C"
