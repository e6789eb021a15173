// Attention of new tokens over a paged cache: one pass over the visible slots
// with the running maximum and sum of a softmax.
//
// For token t and query head h of a sequence of length L with n new tokens,
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)
// over the slots j that the token sees, m the largest logit so far.  The rows
// of a workgroup are the (token, head) pairs that share one key head (token
// major), so a key and value row that was fetched serves the whole group of
// heads; with one new token a sequence the rows are the group alone.
//
// WQ x WK waves: wave (wq, wk) computes rows 32 wq .. 32 wq + 31 against the
// wk-th part of every step's keys.  Logits are taken transposed, S^T = K Q^T
// (32x32x16 MFMAs): a lane then holds 16 keys of one row, the row's maximum
// and sum need one exchange between half-waves, and the rounded weights are
// already the second operand of O^T = V^T P^T: the sum over keys may run in any
// order, so V^T is read (transposed, from LDS) in the order the lanes hold.
//
// The matrix units take weights in the cache's type, and so they are rounded for
// the product with the values, also where the output is fp32; the sum that
// divides keeps them in 32 bits.  Relative error of outputs against 64 bits, one
// token over 3000 slots, heads of 128: bf16 cache 2.3e-3 in bf16 (the output's
// own rounding is 1.7e-3), 1.5e-3 in fp32; fp16 cache 2.8e-4 in fp16, 1.9e-4 in
// fp32.  In fp16 weights below 2^-25 of the largest add to the sum alone.
#include <algorithm>

#include "qxt_paged_attention.h"

namespace qxt {
namespace {

constexpr float kNone = -__builtin_inff();
// The running maximum moves only when a logit exceeds it by this much (in log2
// units): weights stay up to 2^8, in range of fp16, and the rescaling of the
// outputs is rare.
constexpr float kSlack = 8.0f;

template <typename TO>
__device__ __forceinline__ void put4(char *p, float a, float b, float c, float d) {
    typename vec4_of<TO>::type v;
    v[0] = static_cast<TO>(a);
    v[1] = static_cast<TO>(b);
    v[2] = static_cast<TO>(c);
    v[3] = static_cast<TO>(d);
    *reinterpret_cast<typename vec4_of<TO>::type *>(p) = v;
}

__device__ __forceinline__ void put4_as(uint32_t type, char *row, int d, float a, float b, float c, float e) {
    if (type == QXT_TYPE_BF16)
        put4<bf16_t>(row + 2 * d, a, b, c, e);
    else if (type == QXT_TYPE_F16)
        put4<f16_t>(row + 2 * d, a, b, c, e);
    else
        put4<float>(row + 4 * d, a, b, c, e);
}

// Natural-log sum of a row's exponentials from its maximum (log2 units) and sum.
__device__ __forceinline__ float lse_of(float top2, float sum) {
    return sum == 0.0f ? kNone : (top2 + __log2f(sum)) * 0.69314718055994531f;
}

// One row without matrix instructions, a slot at a time: only the slots that it
// sees enter.  For the rare waves whose rows see different slots of a step that
// holds infinite or NaN values.  Lane l gets elements l + 64 k; the slots are
// [from, to) in parts of `part` every `step`.
// Right, and slow: keys are read element by element, the rows one after another,
// and the call waits for its slowest wave.  One such value three slots from the
// end: 8k prompt of 32 heads of 128 0.64 -> 201 ms, 512 tokens over 32k slots
// 0.31 -> 166 ms, 9 tokens over 1k slots 14 us -> 1.1 ms.
template <typename T, int DP, typename A>
__device__ __forceinline__ float2 attend_alone(const A &a, const T *query, const Range &mine, int32_t from,
                                               int32_t to, int32_t step, int32_t part, const int32_t *table,
                                               const char *keys, const char *values, float (&out)[DP / 64]) {
    const int lane = threadIdx.x % 64;
    float top = kNone, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < DP / 64; ++k) out[k] = 0.0f;
    for (int32_t base = from; base < to; base += step) {
        const int32_t slot = base + lane;
        const bool seen = lane < part && slot >= mine.low && slot < mine.high;
        float logit = kNone;
        int64_t value_at = -1;
        if (seen) {
            const uint32_t page = fast_quotient(static_cast<uint32_t>(slot), a.page);
            const int64_t in_page = static_cast<uint32_t>(slot) - page * a.page.divisor, id = table[page];
            logit = 0.0f;
            if (id >= 0 && id < a.pages) {
                const T *key = reinterpret_cast<const T *>(keys + id * a.keys.page_stride + in_page * a.keys.slot_stride);
                value_at = id * a.values.page_stride + in_page * a.values.slot_stride;
                for (uint32_t e = 0; e < a.head_dim; ++e)
                    logit = fmaf(static_cast<float>(query[e]), static_cast<float>(key[e]), logit);
            }
        }
        float most = logit;
        for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
        const float next = fmaxf(top, most);
        const float factor = next == kNone ? 1.0f : __builtin_amdgcn_exp2f((top - next) * a.scale2);
        top = next;
        const float weight = seen ? __builtin_amdgcn_exp2f(fmaf(logit, a.scale2, top == kNone ? 0.0f : -top * a.scale2)) : 0.0f;
        float part_sum = weight;
        for (int off = 32; off > 0; off >>= 1) part_sum += __shfl_xor(part_sum, off, 64);
        sum = sum * factor + part_sum;
#pragma unroll
        for (int k = 0; k < DP / 64; ++k) out[k] *= factor;
        for (int j = 0; j < part; ++j) {
            if (!__shfl(static_cast<int>(seen), j, 64)) continue;
            const float w = __shfl(weight, j, 64);
            const int64_t at = __shfl(static_cast<long long>(value_at), j, 64);
            if (at < 0) continue;  // a slot without a page: zero values
#pragma unroll
            for (int k = 0; k < DP / 64; ++k) {
                const uint32_t e = lane + 64 * k;
                if (e < a.head_dim) out[k] = fmaf(w, static_cast<float>(reinterpret_cast<const T *>(values + at)[e]), out[k]);
            }
        }
    }
    return make_float2(top == kNone ? kNone : top * a.scale2, sum);
}

__device__ __forceinline__ void put_as(uint32_t type, char *row, int d, float x) {
    if (type == QXT_TYPE_BF16)
        reinterpret_cast<bf16_t *>(row)[d] = static_cast<bf16_t>(x);
    else if (type == QXT_TYPE_F16)
        reinterpret_cast<f16_t *>(row)[d] = static_cast<f16_t>(x);
    else
        reinterpret_cast<float *>(row)[d] = x;
}

// What one wave does with KB x 32 staged keys and its 32 rows.
template <typename T, int DP, int KB>
struct Core {
    using TL = Tile<DP>;
    using M = Mfma<T>;
    typedef typename M::frag frag;
    static constexpr int kCols = DP / 32, kSteps = DP / 16;

    int32_t key_at, value_at;  // operand addresses within a tile (bytes), without the block's own offset
    frag q[kSteps];
    f32x16 acc[kCols];
    float top, sum;  // running maximum (unscaled logits) of the row, sum over this lane's keys
    bool special;    // unseen values that are no numbers reached acc

    __device__ __forceinline__ void place(int lane) {
        const int col = lane % 32, half = lane / 32, vr = 4 * half + (lane % 16) / 4;
        key_at = col * TL::kRowBytes + ((half ^ TL::key_turn(col)) * 16);
        const int value_chunk = (2 * ((lane / 16) % 2) + (lane % 4) / 2) ^ TL::value_turn(vr);
        value_at = vr * TL::kRowBytes + value_chunk * 16 + (lane % 2) * 8;
    }

    __device__ __forceinline__ void begin(const char *query_row, int half, int head_dim) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = frag{};
            if (16 * s + 8 * half < head_dim) q[s] = *reinterpret_cast<const frag *>(query_row + (16 * s + 8 * half) * 2);
        }
#pragma unroll
        for (int d = 0; d < kCols; ++d) acc[d] = f32x16{};
        top = kNone;
        sum = 0.0f;
        special = false;
    }

    // Operands are read a few products before their use: in this order in the source, since where scalar registers are
    // short the compiler keeps the source's order, and by `ahead` where it reorders.
    static constexpr int kKeysAhead = 6, kValuesAhead = 4;
    // The surrounding block's LDS reads (READS a product) go AHEAD products before their use.
    template <int PRODUCTS, int READS, int AHEAD>
    __device__ __forceinline__ static void ahead() {
        __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 0);  // LDS reads
#pragma unroll
        for (int i = 0; i < PRODUCTS - AHEAD; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instructions
            __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
    }

    // s[kb][i]: logit of this lane's row with key 32 kb + 8 (i / 4) + 4 half + i % 4 of the tile.
    __device__ __forceinline__ void logits(const char *keys, f32x16 (&s)[KB]) const {
        constexpr int kProducts = KB * kSteps, kAhead = kKeysAhead < kProducts ? kKeysAhead : kProducts;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
        frag k[kAhead];
#pragma unroll
        for (int i = 0; i < kProducts + kAhead; ++i) {
            if (i >= kAhead) {
                const int j = i - kAhead, kb = j % KB, c = j / KB;
                s[kb] = M::run(k[j % kAhead], q[c], s[kb]);
            }
            if (i < kProducts)
                k[i % kAhead] = *reinterpret_cast<const frag *>(keys + (i % KB) * 32 * TL::kRowBytes + (key_at ^ (32 * (i / KB))));
        }
        ahead<kProducts, 1, kAhead>();
    }

    __device__ __forceinline__ static void hide(f32x16 (&s)[KB], int32_t base, int half, const Range &mine) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int32_t slot = base + 32 * kb + 8 * (i / 4) + 4 * half + i % 4;
                if (slot < mine.low || slot >= mine.high) s[kb][i] = kNone;
            }
    }

    // Weights of the logits, rounded; the running maximum and sum move on.
    __device__ __forceinline__ void weigh(const f32x16 (&s)[KB], float scale2, frag (&p)[KB][2]) {
        float most = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, s[kb][i]);
        most = max_halves(most);
        // A row without a maximum yet takes any; others wait for the slack.
        if (__any(most * scale2 > top * scale2 + kSlack)) {
            const float next = fmaxf(top, most);
            const float factor = next == kNone ? 1.0f : __builtin_amdgcn_exp2f((top - next) * scale2);
            top = next;
            sum *= factor;
#pragma unroll
            for (int d = 0; d < kCols; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= factor;
        }
        const float shift = top == kNone ? 0.0f : top * scale2;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[kb][i], scale2, -shift));
                part += w;
                p[kb][i / 8][i % 8] = static_cast<T>(w);
            }
            sum += part;
        }
    }

    // Sixteen values of columns 32 d + col, in the order of p[kb][h].
    __device__ __forceinline__ uint4 value_frag(const char *values, int kb, int h, int d) const {
        const char *at = values + (32 * kb + 16 * h) * TL::kRowBytes + (value_at ^ (64 * d));
        const uint2 v0 = read_transposed(at), v1 = read_transposed(at + 8 * TL::kRowBytes);
        return uint4{v0.x, v0.y, v1.x, v1.y};
    }

    // A weight of 0 times an infinite or NaN value is NaN: where this wave's rows see different slots, such values
    // may belong to slots that a row does not see, and the wave's rows are taken one by one in the end.
    __device__ __forceinline__ void inspect(const char *values) {
        uint32_t found = 0;
#pragma unroll 1
        for (int x = 0; x < 2 * KB; ++x)
#pragma unroll
            for (int d = 0; d < kCols; ++d) {
                const uint4 v = value_frag(values, x / 2, x % 2, d);
                found |= M::special(v.x) | M::special(v.y) | M::special(v.z) | M::special(v.w);
            }
        special = special || __any(found & 0x80008000u);
    }

    __device__ __forceinline__ void add_values(const char *values, const frag (&p)[KB][2]) {
        constexpr int kProducts = KB * 2 * kCols, kAhead = kValuesAhead < kProducts ? kValuesAhead : kProducts;
        uint4 v[kAhead];
#pragma unroll
        for (int i = 0; i < kProducts + kAhead; ++i) {
            if (i >= kAhead) {
                const int j = i - kAhead, d = j % kCols, x = j / kCols;
                acc[d] = M::run(__builtin_bit_cast(frag, v[j % kAhead]), p[x / 2][x % 2], acc[d]);
            }
            if (i < kProducts) v[i % kAhead] = value_frag(values, i / kCols / 2, i / kCols % 2, i % kCols);
        }
        ahead<kProducts, 2, kAhead>();
    }

    // Have the queries arrive here: left to their first use, the compiler waits for all loads in flight at every step.
    __device__ __forceinline__ void hold_queries() {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q[s]));
    }
};

// The rows of a workgroup's tile and what they see.
struct RowTile {
    int32_t row, token, in_group;           // this lane's row (its last one repeated past the end)
    Range mine;
    int32_t low, high;                      // any row of the workgroup's (low rounded down)
    int32_t any_low, all_low, all_high, any_high;  // this wave's rows, any of them or all
    int32_t from, to;                       // steps of this split
    int32_t tile;                           // its number, below 0: none

    template <typename A>
    __device__ __forceinline__ RowTile(const A &a, const Sequence &seq, int32_t tile, int tile_rows, int wave_row,
                                       int32_t rows, uint32_t split, int step)
        : tile(tile) {
        row = tile * tile_rows + wave_row + threadIdx.x % 32;
        token = fast_quotient(min(row, rows - 1), a.group);
        in_group = min(row, rows - 1) - token * a.group.divisor;
        mine = seen_by(a, seq, token);
        low = seen_by(a, seq, fast_quotient(tile * tile_rows, a.group)).low & ~7;  // whole units
        high = seen_by(a, seq, fast_quotient(min(rows, (tile + 1) * tile_rows) - 1, a.group)).high;
        any_low = __builtin_amdgcn_readlane(mine.low, 0);
        all_low = __builtin_amdgcn_readlane(mine.low, 31);
        all_high = __builtin_amdgcn_readlane(mine.high, 0);
        any_high = __builtin_amdgcn_readlane(mine.high, 31);
        const int32_t steps = (high - low + step - 1) / step, share = (steps + a.splits - 1) / a.splits;
        from = min<int32_t>(split * share, steps);
        to = min<int32_t>(from + share, steps);
    }

    // A step from slot `base` on may hold real slots that some row of the wave does not see.
    __device__ __forceinline__ bool mixed(int32_t base) const {
        return any_low != all_low || any_high != all_high || base < all_low || any_high != high;
    }
};

// Where the results of row (token, head) go.
struct RowOut {
    int64_t index, head, part;

    template <typename A>
    __device__ __forceinline__ RowOut(const A &a, const Sequence &seq, uint32_t kv_head, int32_t token, int32_t in_group,
                                      uint32_t split) {
        index = seq.start + token;
        head = static_cast<int64_t>(kv_head) * a.group.divisor + in_group;
        part = (static_cast<int64_t>(split) * a.tokens + index) * (a.kv_heads * a.group.divisor) + head;
    }
    template <typename A>
    __device__ __forceinline__ void put_sums(const A &a, float top2, float total) const {
        if (a.splits > 1)
            a.part_sum[part] = make_float2(top2, total);
        else if (a.lse != nullptr)
            a.lse[index * a.lse_token + head] = lse_of(top2, total);
    }
    template <typename A>
    __device__ __forceinline__ char *row(const A &a) const {
        return a.splits > 1 ? reinterpret_cast<char *>(a.part_out + part * a.head_dim)
                            : a.out + index * a.out_token + head * a.out_head;
    }
};

// acc times `by` to a row: elements 32 d + 8 i + 4 half .. + 3 are acc[d][4 i .. 4 i + 3].
template <typename TO, int COLS>
__device__ __forceinline__ void put_row(char *row, const f32x16 (&acc)[COLS], float by, int half, int head_dim) {
#pragma unroll
    for (int d = 0; d < COLS; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 32 * d + 8 * i + 4 * half;
            if (e < head_dim)
                put4<TO>(row + e * sizeof(TO), acc[d][4 * i] * by, acc[d][4 * i + 1] * by, acc[d][4 * i + 2] * by,
                         acc[d][4 * i + 3] * by);
        }
}

// attend_alone for each of a wave's rows from `first` on; `put` takes (row of the wave, its place, its sums, its elements).
template <typename T, int DP, typename A, typename Put>
__device__ __forceinline__ void rows_alone(const A &a, const Sequence &seq, uint32_t b, uint32_t kv_head, uint32_t split,
                                           int32_t first, int32_t rows, int32_t from, int32_t to, int32_t step, int32_t part,
                                           Put put) {
    for (int r = 0; r < 32 && first + r < rows; ++r) {
        const int32_t t = fast_quotient(first + r, a.group);
        const RowOut place(a, seq, kv_head, t, first + r - t * a.group.divisor, split);
        const T *query = reinterpret_cast<const T *>(a.query + place.index * a.query_token + place.head * a.query_head);
        float o[DP / 64];
        const float2 sums = attend_alone<T, DP>(a, query, seen_by(a, seq, t), from, to, step, part, a.table + b * a.table_stride,
                                                a.keys.data + kv_head * a.keys.head_stride,
                                                a.values.data + kv_head * a.values.head_stride, o);
        put(r, place, sums, o);
    }
}

// A wave's 32 rows to memory.
template <typename T, int DP, int KB, typename A>
__device__ __forceinline__ void put_rows(const A &a, const Sequence &seq, uint32_t b, uint32_t kv_head, uint32_t split,
                                         const RowTile &tile, int32_t rows, int32_t step, const Core<T, DP, KB> &core) {
    int lane = threadIdx.x % 64;
    asm volatile("" : "+v"(lane));  // keeps the elements' offsets out of the main loop's registers
    const int half = lane / 32, head_dim = a.head_dim;
    if (core.special) {
        rows_alone<T, DP>(a, seq, b, kv_head, split, tile.row - threadIdx.x % 32, rows, tile.low + tile.from * step,
                          tile.low + tile.to * step, step, step,
                          [&](int, const RowOut &place, const float2 &sums, const float (&o)[DP / 64]) {
                              if (lane == 0) place.put_sums(a, sums.x, sums.y);
                              const float by = a.splits > 1 ? 1.0f : (sums.y == 0.0f ? 0.0f : 1.0f / sums.y);
                              for (int k = 0; k < DP / 64; ++k)
                                  if (lane + 64 * k < head_dim)
                                      put_as(a.splits > 1 ? QXT_TYPE_F32 : a.out_type, place.row(a), lane + 64 * k, o[k] * by);
                          });
        return;
    }
    const float total = add_halves(core.sum);
    if (tile.row >= rows) return;
    const RowOut place(a, seq, kv_head, tile.token, tile.in_group, split);
    if (half == 0) place.put_sums(a, core.top == kNone ? kNone : core.top * a.scale2, total);
    char *out = place.row(a);
    if (a.splits > 1) {
        if (total != 0.0f) put_row<float>(out, core.acc, 1.0f, half, head_dim);
        return;
    }
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    if (a.out_type == QXT_TYPE_BF16)
        put_row<bf16_t>(out, core.acc, by, half, head_dim);
    else if (a.out_type == QXT_TYPE_F16)
        put_row<f16_t>(out, core.acc, by, half, head_dim);
    else
        put_row<float>(out, core.acc, by, half, head_dim);
}

// kv_heads x tiles x splits x sequences, kv_heads fastest.
struct Place {
    uint32_t head, tile, split, b;
    template <typename A>
    __device__ __forceinline__ explicit Place(const A &a) {
        uint32_t id = blockIdx.x;
        head = id % a.kv_heads;
        id /= a.kv_heads;
        tile = id % a.tiles;
        id /= a.tiles;
        split = id % a.splits;
        b = id / a.splits;
    }
};

template <int DP, int WQ, int WK>
struct Shape {
    static constexpr int kKeys = DP <= 128 && WQ >= 4 ? 64 : 32;  // keys of one step and key part
    static constexpr int kStep = kKeys * WK;                      // keys of one step
    static constexpr int kRows = kKeys / WQ;                      // rows that a wave stages
    static constexpr int kTileBytes = kKeys * DP * 2;
    static constexpr int kStageBytes = 2 * kTileBytes * WK;
    static constexpr int kLds = 2 * kStageBytes;
    static constexpr int kThreads = 64 * WQ * WK;
};

// Two waves a SIMD (256 registers each) up to 128 elements of head size, one above.
// Measured: one token for each of 64 sequences of 3k to 16k slots (2.6 GB of keys
// and values, heads of 128) 464 us, 5.5 TB/s: bound by memory.  Seven chunks of 1
// to 300 tokens with a window, heads of 256: 62 us for 17.5 GFLOP, matrix units
// 23 % busy, vector units 25 %: with one wave a SIMD nothing covers its waits.
template <typename T, int DP, int WQ, int WK>
__global__ __launch_bounds__(64 * WQ * WK, DP <= 128 ? 2 : 1) void paged_attention_kernel(PagedArgs) {
    Kernarg<PagedArgs> *const args = kernargs<PagedArgs>();
    Kernarg<PagedArgs> &a = *args;
    using S = Shape<DP, WQ, WK>;
    using C = Core<T, DP, S::kKeys / 32>;
    typedef typename C::frag frag;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wq = wave % WQ, wk = wave / WQ, col = lane % 32, half = lane / 32;
    const Place at(a);
    const Sequence seq = sequence_of(a, at.b);
    const int32_t rows = seq.tokens * a.group.divisor, tiles = (rows + 32 * WQ - 1) / (32 * WQ);
    Stager<DP, S::kRows> stager;
    stager.start(a, at.b, at.head, wq * S::kRows);
    float scale2 = a.scale2;
    keep(scale2);
    C core;
    core.place(lane);
    const char *const my_keys = lds + 2 * S::kTileBytes * wk;  // this key part's tiles of stage 0
    const uint32_t my_rows = lds_offset(my_keys) + wq * S::kRows * Tile<DP>::kRowBytes;

    for (int32_t turn = at.tile; turn < tiles; turn += a.tiles) {
        const int32_t tile = tiles - 1 - turn;  // the longest rows first: the last tiles of a causal sequence
        Kernarg<PagedArgs> &y = *late(args);
        const RowTile rt(y, seq, tile, 32 * WQ, 32 * wq, rows, at.split, S::kStep);
        core.begin(y.query + (seq.start + rt.token) * y.query_token +
                       static_cast<int64_t>(at.head * y.group.divisor + rt.in_group) * y.query_head,
                   half, y.head_dim);
        auto stage = [&](int32_t t) {
            const uint32_t to = my_rows + (t & 1) * S::kStageBytes;
            const auto staged = stager.locate(rt.low + t * S::kStep + wk * S::kKeys + wq * S::kRows, rt.high);
            stager.load_keys(staged, to, wq * S::kRows);
            stager.load_values(staged, to + S::kTileBytes);
        };
        auto compute = [&](int32_t t) {
            const int32_t base = rt.low + t * S::kStep + wk * S::kKeys;
            if (base >= rt.any_high || base + S::kKeys <= rt.any_low) return;
            const char *kt = my_keys + (t & 1) * S::kStageBytes, *vt = kt + S::kTileBytes;
            f32x16 s[S::kKeys / 32];
            frag p[S::kKeys / 32][2];
            core.logits(kt, s);
            const bool partial = base < rt.all_low || base + S::kKeys > rt.all_high;
            if (partial) C::hide(s, base, half, rt.mine);
            core.weigh(s, scale2, p);
            if (partial && rt.mixed(base)) core.inspect(vt);
            core.add_values(vt, p);
        };
        if constexpr (WQ == 1) {
            // The wave reads only what it staged itself: two steps are in flight, and no one is waited for.
            if (rt.from < rt.to) stage(rt.from);
            if (rt.from + 1 < rt.to) stage(rt.from + 1);
            core.hold_queries();
            for (int32_t t = rt.from; t < rt.to; ++t) {
                if (t + 1 < rt.to)
                    landed<2 * Stager<DP, S::kRows>::kLoads>();
                else
                    landed<0>();
                compute(t);
                if (t + 2 < rt.to) {
                    reads_done();
                    stage(t + 2);
                }
            }
        } else {
            if (rt.from < rt.to) stage(rt.from);
            core.hold_queries();
            for (int32_t t = rt.from; t < rt.to; ++t) {
                landed<0>();  // this wave's rows of step t
                meet();       // everyone's, and step t - 1 has been read
                if (t + 1 < rt.to) stage(t + 1);
                compute(t);
            }
        }
        Kernarg<PagedArgs> &z = *late(args);
        if constexpr (WK == 1) {
            put_rows<T, DP>(z, seq, at.b, at.head, at.split, rt, rows, S::kStep, core);
            if (WQ > 1) __syncthreads();  // before the next tile's staging
        } else {
            // Join the key parts: every wave puts its outputs in LDS, then the threads add up and store shares of the elements.
            constexpr int kPitch = DP + 4;  // floats a row
            float *joined = reinterpret_cast<float *>(lds);                              // [WK][32 WQ][kPitch]
            float2 *sums = reinterpret_cast<float2 *>(joined + WK * 32 * WQ * kPitch);   // [WK][32 WQ]
            __syncthreads();                                                             // staged tiles have been read
            const int part_at = wk * 32 * WQ + 32 * wq;                                  // this wave's rows
            if (core.special) {
                rows_alone<T, DP>(z, seq, at.b, at.head, at.split, tile * 32 * WQ + 32 * wq, rows,
                                  rt.low + rt.from * S::kStep + wk * S::kKeys, rt.low + rt.to * S::kStep, S::kStep, S::kKeys,
                                  [&](int r, const RowOut &, const float2 &one, const float (&o)[DP / 64]) {
                                      if (lane == 0) sums[part_at + r] = one;
                                      for (int k = 0; k < DP / 64; ++k) joined[(part_at + r) * kPitch + lane + 64 * k] = o[k];
                                  });
            } else {
                const float total = add_halves(core.sum);
                if (half == 0) sums[part_at + col] = make_float2(core.top == kNone ? kNone : core.top * z.scale2, total);
                put_row<float>(reinterpret_cast<char *>(joined + (part_at + col) * kPitch), core.acc, 1.0f, half, DP);
            }
            __syncthreads();
            constexpr int kLanes = DP / 4;  // threads a row, four elements each
            for (int r = threadIdx.x / kLanes; r < 32 * WQ; r += S::kThreads / kLanes) {
                const int32_t out_row = tile * 32 * WQ + r;
                if (out_row >= rows) break;
                const int e = 4 * (threadIdx.x % kLanes);
                float most = kNone, total = 0.0f;
                float2 ms[WK];
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    ms[w] = sums[w * 32 * WQ + r];
                    most = fmaxf(most, ms[w].x);
                }
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    if (ms[w].y == 0.0f) continue;  // saw nothing
                    const float f = ms[w].x == kNone ? 1.0f : __builtin_amdgcn_exp2f(ms[w].x - most);
                    const float4 y = *reinterpret_cast<const float4 *>(joined + (w * 32 * WQ + r) * kPitch + e);
                    total += ms[w].y * f;
                    x.x += y.x * f;
                    x.y += y.y * f;
                    x.z += y.z * f;
                    x.w += y.w * f;
                }
                const int32_t t = fast_quotient(out_row, z.group);
                const RowOut place(z, seq, at.head, t, out_row - t * z.group.divisor, at.split);
                if (e == 0) place.put_sums(z, most, total);
                if (e < static_cast<int>(z.head_dim)) {
                    const float by = z.splits > 1 ? 1.0f : (total == 0.0f ? 0.0f : 1.0f / total);
                    put4_as(z.splits > 1 ? QXT_TYPE_F32 : z.out_type, place.row(z), e, x.x * by, x.y * by, x.z * by, x.w * by);
                }
            }
            __syncthreads();
        }
    }
}

// Many rows (heads of up to 128 elements): eight waves of 32 rows over steps of
// 64 keys, two waves on each SIMD in opposite phases.  While waves 0-3 feed the
// matrix cores (logits of step t, outputs of step t - 1), waves 4-7, on the same
// SIMDs, turn their logits into weights on the vector unit, and at the next
// barrier they change places; in step, both units idle in turns.
// Three buffers each of keys and values, staged in the vector phases: in that of
// step t the first four waves ask for keys t + 2 and values t + 1, the others,
// whose vector phase t comes one phase later, for keys t + 3 and values t + 2;
// all of these buffers were last read a phase or more before.  Each wave waits
// for its share two phases on, before the barrier after which the first wave
// reads it, with the loads of its next vector phase already under way.
// Measured: 8192 new tokens, 32 heads of 128, 32 key heads, causal, 570 us
// (0.96 PFLOP/s; a library product of two 8192 x 8192 matrices 1.37).  When this
// took 600 us, all waves in step took 651; at 620, the DMA issued in the matrix
// phases instead 653.  Bound by the vector phases, about 2000 cycles a step
// against 1350 of matrix work: half of them the softmax, the rest page look-ups,
// addresses and DMA issue of the staging.
template <typename T, int DP>
__global__ __launch_bounds__(512, 2) void paged_attention_long_kernel(PagedArgs) {
    constexpr int kKeys = 64, kWaveRows = kKeys / 8, kTileBytes = kKeys * DP * 2, kRing = 3;
    using C = Core<T, DP, kKeys / 32>;
    using St = Stager<DP, kWaveRows>;
    typedef typename C::frag frag;
    extern __shared__ __align__(16) char lds[];  // kRing tiles of keys, kRing of values
    Kernarg<PagedArgs> *const args = kernargs<PagedArgs>();
    Kernarg<PagedArgs> &a = *args;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), half = lane / 32;
    const bool second = wave >= 4;
    St stager;
    {
        const Place at(a);
        stager.start(a, at.b, at.head, wave * kWaveRows);
    }
    float scale2 = a.scale2;
    keep(scale2);
    C core;
    core.place(lane);
    const uint32_t my_rows = lds_offset(lds) + wave * kWaveRows * Tile<DP>::kRowBytes;

    for (int32_t round = 0;; ++round) {
        // (Where the workgroup stands is worked out anew before and after the main loop.)
        Kernarg<PagedArgs> &y = *late(args);
        const RowTile rt = [&] {
            const Place at(y);
            const Sequence seq = sequence_of(y, at.b);
            const int32_t rows = seq.tokens * y.group.divisor, tiles = (rows + 255) / 256;
            const int32_t tile = tiles - 1 - static_cast<int32_t>(at.tile) - round * static_cast<int32_t>(y.tiles);
            RowTile r(y, seq, tile, 256, 32 * wave, rows, at.split, kKeys);
            if (tile >= 0)
                core.begin(y.query + (seq.start + r.token) * y.query_token +
                               static_cast<int64_t>(at.head * y.group.divisor + r.in_group) * y.query_head,
                           half, y.head_dim);
            return r;
        }();
        if (rt.tile < 0) break;
        const int32_t end = min(rt.high, rt.low + rt.to * kKeys);  // steps past the last stage rows of zeros
        stager.forget();  // (with a window a later tile's share of the slots may end above an earlier one's)
        auto locate = [&](int32_t t) { return stager.locate(rt.low + t * kKeys + wave * kWaveRows, end); };
        auto load_keys = [&](const typename St::Rows &r, int place) {
            stager.load_keys(r, my_rows + place * kTileBytes, wave * kWaveRows);
        };
        auto load_values = [&](const typename St::Rows &r, int place) {
            stager.load_values(r, my_rows + (kRing + place) * kTileBytes);
        };
        auto shown = [&](int32_t t) {  // some row of this wave sees some slot of step t
            const int32_t base = rt.low + t * kKeys;
            return t >= rt.from && t < rt.to && base < rt.any_high && base + kKeys > rt.any_low;
        };
        typename St::Rows next = locate(rt.from);
        load_keys(next, 0);
        load_values(next, 0);
        next = locate(rt.from + 1);
        load_keys(next, 1);
        if (second) {
            load_values(next, 1);
            next = locate(rt.from + 2);
            load_keys(next, 2);
        }
        core.hold_queries();
        landed<0>();
        meet();
        if (second) meet();

        f32x16 s[kKeys / 32];
        frag p[kKeys / 32][2];
        int place = 0, before = kRing - 1;  // buffers of steps t and t - 1
        int32_t pending = 0, ragged = 0;  // step t - 1 has weights; its rows see different slots
        for (int32_t t = rt.from; t < rt.to; ++t) {
            // Matrix phase.
            const int after = place == kRing - 1 ? 0 : place + 1;
            const int32_t base = rt.low + t * kKeys;
            const bool live = shown(t);
            if (live) core.logits(lds + place * kTileBytes, s);
            if (pending) {
                const char *vt = lds + (kRing + before) * kTileBytes;
                if (ragged) core.inspect(vt);
                core.add_values(vt, p);
            }
            if (second) landed<2 * St::kLoads>();
            meet();
            // Vector phase.  Keys two (three) steps on take the buffer of keys t - 1 (t), values one less that of t - 2 (t - 1).
            const typename St::Rows later = locate(t + (second ? 3 : 2));
            load_keys(later, second ? place : before);
            load_values(next, second ? before : after);
            next = later;
            if (live) {
                const bool partial = base < rt.all_low || base + kKeys > rt.all_high;
                if (partial) C::hide(s, base, half, rt.mine);
                core.weigh(s, scale2, p);
                ragged = partial && rt.mixed(base) ? 1 : 0;
            }
            pending = live ? 1 : 0;
            before = place;
            place = after;
            if (!second) landed<2 * St::kLoads>();
            meet();
        }
        if (pending) {
            const char *vt = lds + (kRing + before) * kTileBytes;
            if (ragged) core.inspect(vt);
            core.add_values(vt, p);
        }
        if (!second) meet();
        landed<0>();
        Kernarg<PagedArgs> &z = *late(args);
        const Place at(z);
        const Sequence seq = sequence_of(z, at.b);
        put_rows<T, DP>(z, seq, at.b, at.head, at.split, rt, seq.tokens * z.group.divisor, kKeys, core);
        __syncthreads();  // before the next tile's staging
    }
}

// Join the parts of rows whose slots were split over workgroups.  LANES lanes a
// row, four elements each; the row's sums are read at once, the parts with four
// in flight (read one after another, eight parts took 7 us at any size).
template <int LANES>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(PagedArgs a) {
    const uint32_t heads = a.kv_heads * a.group.divisor;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * heads;
    if (row >= rows) return;  // whole groups of LANES leave together
    const int64_t token = row / heads, head = row - token * heads;
    if (a.starts != nullptr && (token < a.starts[0] || token >= a.starts[a.sequences])) return;  // nobody's row
    const uint32_t lane = threadIdx.x % LANES;
    const int e = 4 * lane;
    float top = kNone, total = 0.0f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t s0 = 0; s0 < a.splits; s0 += LANES) {
        // This round's parts: their sums in the lanes, their common maximum.
        const uint32_t count = min<uint32_t>(LANES, a.splits - s0);
        float2 mine = make_float2(kNone, 0.0f);
        if (lane < count) mine = a.part_sum[(s0 + lane) * rows + row];
        float most = mine.x;
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, LANES));
        const float next = fmaxf(top, most), back = top == kNone ? 0.0f : __builtin_amdgcn_exp2f(top - next);
        if (s0 > 0) {
            const float old = next == kNone ? 1.0f : back;
            total *= old;
            x.x *= old;
            x.y *= old;
            x.z *= old;
            x.w *= old;
        }
        top = next;
        // A part without a maximum is empty (sum 0, no outputs written), or NaN throughout.
        const float factor = mine.y == 0.0f ? 0.0f : mine.x == kNone ? 1.0f : __builtin_amdgcn_exp2f(mine.x - top);
        for (uint32_t s1 = 0; s1 < count; s1 += 4) {
            float4 y[4];
            float f[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t s = min(s1 + k, count - 1);
                const float sum = __shfl(mine.y, s, LANES);
                f[k] = s1 + k < count ? __shfl(factor, s, LANES) : 0.0f;
                total += s1 + k < count && sum != 0.0f ? sum * f[k] : 0.0f;
                y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (s1 + k < count && sum != 0.0f && e < static_cast<int>(a.head_dim))
                    y[k] = *reinterpret_cast<const float4 *>(a.part_out + ((s0 + s) * rows + row) * a.head_dim + e);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x.x += y[k].x * f[k];
                x.y += y[k].y * f[k];
                x.z += y[k].z * f[k];
                x.w += y[k].w * f[k];
            }
        }
    }
    if (lane == 0 && a.lse != nullptr) a.lse[token * a.lse_token + head] = lse_of(top, total);
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    if (e < static_cast<int>(a.head_dim))
        put4_as(a.out_type, a.out + token * a.out_token + head * a.out_head, e, x.x * by, x.y * by, x.z * by, x.w * by);
}

// ------------------------------------------------------------------ host side

struct Plan {
    uint32_t wq, wk, tiles, splits;
};

// Waves by the rows that share a key head (new tokens of the longest chunk
// times heads of a group).  A CU holds one workgroup of most shapes, so the slots
// of each row tile are split while tiles, heads and sequences alone leave CUs
// idle, up to one workgroup a CU, each with two steps at least (four of the long
// shapes).  Measured, main kernel and join: a 512-token chunk over 32k slots (64
// workgroups) 848 us whole, 455 in two, 281 in four, 301 in eight; one TinyLlama
// token over 1900 slots (4) 16.7 us whole, 11.6 in four, 10.1 in eight.  Of few
// rows, whose contexts differ most, eight workgroups a CU even out: 64 sequences
// of 3k to 16k slots (512 workgroups) 506 us whole, 463 in four, 481 in eight.
Plan plan_of(uint32_t head_dim, uint32_t group, uint32_t kv_heads, uint32_t sequences, uint32_t tokens,
             uint32_t max_query, uint32_t max_context) {
    const uint64_t rows = static_cast<uint64_t>(std::max(1u, std::min(max_query, tokens))) * group;
    Plan p;
    const bool wide = head_dim > 128;
    p.wq = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 || wide ? 4 : 8;
    p.wk = p.wq == 1 ? (wide ? 2 : 4) : p.wq == 2 ? (wide ? 1 : 2) : 1;
    p.tiles = static_cast<uint32_t>((rows + 32 * p.wq - 1) / (32 * p.wq));
    const uint64_t base = static_cast<uint64_t>(p.tiles) * kv_heads * sequences, cus = compute_units();
    const uint32_t step = (p.wq >= 4 && !wide ? 64 : 32) * p.wk;
    uint64_t splits = 1;
    if (2 * base <= cus)
        splits = cus / base;
    else if (p.wq <= 2)
        splits = std::min<uint64_t>((8 * cus + base - 1) / base, 8);
    else if (base < 2 * cus)
        for (uint64_t s = 2; s <= 4; ++s)  // rounds of workgroups per part
            if ((base * s + cus - 1) / cus * splits < (base * splits + cus - 1) / cus * s) splits = s;
    const uint64_t most = std::max<uint64_t>(1, max_context / ((p.wq <= 2 ? 2 : 4) * step));
    p.splits = static_cast<uint32_t>(std::min<uint64_t>({splits, most, 64}));
    return p;
}

size_t workspace_of(const Plan &p, uint64_t tokens, uint64_t heads, uint64_t head_dim) {
    return p.splits <= 1 ? 0 : p.splits * tokens * heads * (head_dim * 4 + 8);
}

template <typename T, int DP, int WQ, int WK>
int launch_attention(const PagedArgs &a, uint32_t grid, hipStream_t stream) {
    using S = Shape<DP, WQ, WK>;
    constexpr size_t join = WK > 1 ? WK * 32 * WQ * (DP + 4) * 4 + WK * 32 * WQ * 8 : 0;
    constexpr size_t lds = join > S::kLds ? join : S::kLds;
    static_assert(lds <= 160 * 1024, "LDS");
    return launch("paged_attention_kernel", paged_attention_kernel<T, DP, WQ, WK>, dim3(grid), dim3(S::kThreads), lds,
                  stream, a);
}

template <typename T, int DP>
int launch_attention_shape(const PagedArgs &a, const Plan &p, uint32_t grid, hipStream_t stream) {
    constexpr bool wide = DP > 128;
    if (p.wq == 1) return launch_attention<T, DP, 1, wide ? 2 : 4>(a, grid, stream);
    if (p.wq == 2) return launch_attention<T, DP, 2, wide ? 1 : 2>(a, grid, stream);
    if (p.wq == 4) return launch_attention<T, DP, 4, 1>(a, grid, stream);
    if constexpr (!wide)
        return launch("paged_attention_long_kernel", paged_attention_long_kernel<T, DP>, dim3(grid), dim3(512), 6 * 64 * DP * 2,
                      stream, a);
    return fail(QXT_INTERNAL_ERROR, "paged attention: no launch for %u waves", p.wq);
}

template <typename T>
int launch_attention_dim(const PagedArgs &a, const Plan &p, uint32_t grid, hipStream_t stream) {
    if (a.head_dim <= 64) return launch_attention_shape<T, 64>(a, p, grid, stream);
    if (a.head_dim <= 128) return launch_attention_shape<T, 128>(a, p, grid, stream);
    return launch_attention_shape<T, 256>(a, p, grid, stream);
}

}  // namespace

int check_paged_cache(const char *name, const qxt_paged_cache *c, bool needs_values) {
    if (c == nullptr || c->keys == nullptr || (needs_values && c->values == nullptr) || c->block_table == nullptr ||
        c->context_lens == nullptr)
        return fail(QXT_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!half_type(c->type)) return fail(QXT_INVALID_ARGUMENT, "%s: the cache must be bf16 or fp16", name);
    if (c->page_size == 0 || c->heads == 0 || c->table_width == 0)
        return fail(QXT_INVALID_ARGUMENT, "%s: page size, heads and table width must be positive", name);
    if (c->head_dim == 0 || c->head_dim % 8 || c->head_dim > 256)
        return fail(QXT_INVALID_ARGUMENT, "%s: head size must be a multiple of 8 up to 256", name);
    if (static_cast<uint64_t>(c->page_size) * c->table_width > INT32_MAX / 2)
        return fail(QXT_INVALID_ARGUMENT, "%s: a sequence has 2^30 slots or more", name);
    if (!aligned(c->keys, 16) || !all_multiples(16, {c->key_page_stride, c->key_slot_stride, c->key_head_stride}) ||
        (needs_values &&
         (!aligned(c->values, 16) || !all_multiples(16, {c->value_page_stride, c->value_slot_stride, c->value_head_stride}))))
        return fail(QXT_INVALID_ARGUMENT, "%s: cache rows must be 16-byte aligned", name);
    if ((c->key_page_stride | c->value_page_stride | c->key_slot_stride | c->value_slot_stride) >> 36)
        return fail(QXT_INVALID_ARGUMENT, "%s: page or slot strides of 64 GiB or more", name);
    if (c->block_table_stride % 4 || !aligned(c->block_table, 4) || !aligned(c->context_lens, 4))
        return fail(QXT_INVALID_ARGUMENT, "%s: misaligned block table or lengths", name);
    return QXT_OK;
}

}  // namespace qxt

extern "C" {

size_t qxt_paged_attention_workspace(uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t sequences,
                                     uint32_t tokens, uint32_t max_query, uint32_t max_context) {
    if (kv_heads == 0 || query_heads % kv_heads || query_heads == 0 || sequences == 0 || tokens == 0) return 0;
    auto bytes = [&](uint32_t longest) {
        return qxt::workspace_of(
            qxt::plan_of(head_dim, query_heads / kv_heads, kv_heads, sequences, tokens, longest, max_context), tokens, query_heads,
            head_dim);
    };
    return tokens == sequences ? std::max(bytes(max_query), bytes(1)) : bytes(max_query);  // a call without starts plans for 1
}

int qxt_paged_attention(const void *query, size_t query_token_stride, size_t query_head_stride,
                        const qxt_paged_cache *cache, const int32_t *query_starts, void *out, size_t out_token_stride,
                        size_t out_head_stride, uint32_t out_type, float *lse, size_t lse_token_stride, uint32_t tokens,
                        uint32_t query_heads, float scale, uint32_t causal, uint32_t window, uint32_t max_query,
                        uint32_t max_context, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace qxt;
    if (int rc = check_paged_cache("paged attention", cache, true)) return rc;
    if (tokens == 0 || cache->sequences == 0) return QXT_OK;
    if (query == nullptr || out == nullptr) return fail(QXT_INVALID_ARGUMENT, "paged attention: null pointer");
    if (query_heads == 0 || query_heads % cache->heads)
        return fail(QXT_INVALID_ARGUMENT, "paged attention: query heads must be a multiple of the cache's");
    if (!known_type(out_type)) return fail(QXT_INVALID_ARGUMENT, "paged attention: unknown element type");
    if (!(scale > 0.0f) || scale > 3e38f) return fail(QXT_INVALID_ARGUMENT, "paged attention: scale must be positive and finite");
    if (causal > 1 || window > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "paged attention: bad causal or window");
    if (query_starts == nullptr && tokens != cache->sequences)
        return fail(QXT_INVALID_ARGUMENT, "paged attention: without query starts every sequence has one token");
    const uint32_t group = query_heads / cache->heads;
    if (static_cast<uint64_t>(tokens) * query_heads > INT32_MAX / 2)
        return fail(QXT_INVALID_ARGUMENT, "paged attention: 2^30 rows or more");
    if (!aligned(query, 16) || !all_multiples(16, {query_token_stride, query_head_stride}))
        return fail(QXT_INVALID_ARGUMENT, "paged attention: query rows must be 16-byte aligned");
    const size_t quad = 4 * type_bytes(out_type);
    if (!aligned(out, quad) || !all_multiples(quad, {out_token_stride, out_head_stride}) || !aligned(lse, 4) || lse_token_stride % 4)
        return fail(QXT_INVALID_ARGUMENT, "paged attention: misaligned output");
    if (query_starts == nullptr) max_query = 1;
    const Plan p = plan_of(cache->head_dim, group, cache->heads, cache->sequences, tokens, max_query, max_context);
    const size_t needed = workspace_of(p, tokens, query_heads, cache->head_dim);
    if (needed > 0 && (workspace == nullptr || workspace_bytes < needed || !aligned(workspace, 16)))
        return fail(QXT_INVALID_ARGUMENT, "paged attention: workspace of %zu bytes needed", needed);
    const uint64_t grid = static_cast<uint64_t>(p.tiles) * p.splits * cache->heads * cache->sequences;
    if (grid > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "paged attention: too many row tiles");
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;

    PagedArgs a{};
    a.query = static_cast<const char *>(query);
    a.query_token = query_token_stride;
    a.query_head = query_head_stride;
    a.keys = {static_cast<char *>(cache->keys), static_cast<int64_t>(cache->key_page_stride),
              static_cast<int64_t>(cache->key_slot_stride), static_cast<int64_t>(cache->key_head_stride)};
    a.values = {static_cast<char *>(cache->values), static_cast<int64_t>(cache->value_page_stride),
                static_cast<int64_t>(cache->value_slot_stride), static_cast<int64_t>(cache->value_head_stride)};
    a.table = cache->block_table;
    a.table_stride = cache->block_table_stride / 4;
    a.pages = cache->pages;
    a.page = fast_div(cache->page_size);
    a.slots = static_cast<int32_t>(cache->page_size * cache->table_width);
    a.lens = cache->context_lens;
    a.starts = query_starts;
    a.sequences = cache->sequences;
    a.tokens = tokens;
    a.kv_heads = cache->heads;
    a.head_dim = cache->head_dim;
    a.group = fast_div(group);
    a.scale = scale;
    a.scale2 = static_cast<float>(scale * 1.4426950408889634);
    a.causal = causal;
    a.window = window_of(window);
    // Pages in whole units; one layout of keys and values, whose places in a page 32 bits (of 16 bytes) hold; head
    // sizes without padding.
    const uint32_t dim = cache->head_dim <= 64 ? 64 : cache->head_dim <= 128 ? 128 : 256;
    a.even = cache->page_size % 8 == 0 && cache->head_dim == dim && cache->key_page_stride == cache->value_page_stride &&
             cache->key_slot_stride == cache->value_slot_stride && cache->key_slot_stride < (1u << 28) &&
             static_cast<uint64_t>(cache->page_size) * (cache->key_slot_stride / 16) <= UINT32_MAX;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.out = static_cast<char *>(out);
    a.out_token = out_token_stride;
    a.out_head = out_head_stride;
    a.out_type = out_type;
    a.lse = lse;
    a.lse_token = lse_token_stride / 4;
    if (p.splits > 1) {
        a.part_out = static_cast<float *>(workspace);
        a.part_sum = reinterpret_cast<float2 *>(a.part_out + static_cast<size_t>(p.splits) * tokens * query_heads * cache->head_dim);
    }
    const int rc = cache->type == QXT_TYPE_BF16
                       ? launch_attention_dim<bf16_t>(a, p, static_cast<uint32_t>(grid), as_stream(stream))
                       : launch_attention_dim<f16_t>(a, p, static_cast<uint32_t>(grid), as_stream(stream));
    if (rc != QXT_OK || p.splits == 1) return rc;
    const uint64_t rows = static_cast<uint64_t>(tokens) * query_heads;
    auto join = [&](auto kernel, uint32_t lanes) {
        return launch("paged_attention_join_kernel", kernel, dim3(static_cast<uint32_t>((rows * lanes + 255) / 256)), dim3(256), 0,
                      as_stream(stream), a);
    };
    if (cache->head_dim <= 64) return join(paged_attention_join_kernel<16>, 16);
    if (cache->head_dim <= 128) return join(paged_attention_join_kernel<32>, 32);
    return join(paged_attention_join_kernel<64>, 64);
}

}  // extern "C"
