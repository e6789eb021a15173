// Device pieces shared by the kernels that multiply queries with the keys of a
// paged cache: which slots a token sees, and staging of cache rows into LDS.
#pragma once

#include "qxt_paged.h"

namespace qxt {

struct PagedArgs {
    const char *query;
    int64_t query_token, query_head;
    CacheView keys, values;
    const int32_t *table;
    int64_t table_stride;  // elements
    uint32_t pages;
    FastDiv page;
    int32_t slots;  // a sequence's most: table columns times page size
    const int32_t *lens, *starts;
    uint32_t sequences, tokens, kv_heads, head_dim;
    FastDiv group;  // query heads per key head
    float scale, scale2;  // scale2 = scale * log2(e)
    int32_t causal, window;
    uint32_t tiles, splits;  // grid: kv_heads x tiles x splits x sequences, kv_heads fastest
    char *out;
    int64_t out_token, out_head;
    uint32_t out_type;
    float *lse;
    int64_t lse_token;
    float *part_out;   // [splits, tokens, heads, head_dim], unnormalised
    float2 *part_sum;  // [splits, tokens, heads]: (maximum in log2 units, sum)
};

// The tokens and cache length of one sequence; lengths from the device are
// clamped to what the tensors hold, so no index leaves them.
struct Sequence {
    int32_t start, tokens, length;
};

__device__ __forceinline__ Sequence sequence_of(const PagedArgs &a, uint32_t b) {
    Sequence s;
    const int32_t most = static_cast<int32_t>(a.tokens);
    int32_t first = b, last = b + 1;
    if (a.starts != nullptr) {
        first = a.starts[b];
        last = a.starts[b + 1];
    }
    first = min(max(first, 0), most);
    last = min(max(last, first), most);
    s.start = first;
    s.tokens = last - first;
    s.length = min(max(a.lens[b], 0), a.slots);
    return s;
}

// Slots [low, high) that the sequence's new token number `token` sees.
struct Range {
    int32_t low, high;
};
__device__ __forceinline__ Range seen_by(const PagedArgs &a, const Sequence &s, int32_t token) {
    const int32_t at = s.length - s.tokens + token;  // its own slot
    Range r;
    r.high = a.causal ? min(s.length, max(at + 1, 0)) : s.length;
    r.low = a.window > 0 ? max(0, at - a.window + 1) : 0;
    r.low = min(r.low, r.high);
    return r;
}

// LDS layout of a staged tile: rows of DP elements (the head size rounded up),
// in 16-byte chunks.  Chunk c of row r lies at c ^ turn(r): a wave's reads of
// one chunk column over 16 rows (keys), or of a pair of chunks over four rows
// (values, transposed), then touch different banks.  The DMA writes LDS in
// lane order, so the exchange is made by which chunk each lane fetches.
template <int DP>
struct Tile {
    static constexpr int kChunks = DP / 8;               // 16-byte chunks a row
    static constexpr int kRowBytes = DP * 2;
    static constexpr int kRowsPerLoad = 64 / kChunks;    // rows of one wave-wide 16-byte DMA
    static __device__ __forceinline__ int key_turn(int row) { return row & (kChunks < 16 ? kChunks - 1 : 15); }
    static __device__ __forceinline__ int value_turn(int row) { return 2 * (row & (kChunks < 16 ? 3 : 7)); }
};

// Source of rows that are not in the cache: slots past a sequence's end, pages
// that its table does not name, and the columns from head_dim up to DP.
__device__ __constant__ const uint4 kZeroRow = {0, 0, 0, 0};

// One wave's share of staging: rows [0, ROWS) of its part of a tile, one row
// per lane for the address work (lanes past ROWS repeat).
template <int DP, int ROWS>
struct Stager {
    const int32_t *table;
    int32_t page_id;  // of this lane's row of the next tile to stage

    // Fetch the page of slot `slot` (one tile ahead of its use).
    __device__ __forceinline__ void look_up(const PagedArgs &a, int32_t slot, int32_t high) {
        page_id = -1;
        if (slot < high) page_id = table[fast_quotient(static_cast<uint32_t>(slot), a.page)];
    }

    // Byte offset of this lane's row in a cache, or -1.
    __device__ __forceinline__ int64_t offset_in(const PagedArgs &a, const CacheView &c, int32_t slot) const {
        const uint32_t page = fast_quotient(static_cast<uint32_t>(slot), a.page);
        const uint32_t in_page = static_cast<uint32_t>(slot) - page * a.page.divisor;
        return static_cast<uint32_t>(page_id) < a.pages
                   ? static_cast<int64_t>(page_id) * c.page_stride + static_cast<int64_t>(in_page) * c.slot_stride
                   : -1;
    }

    // DMA this wave's ROWS rows into LDS at `to` (wave-uniform), KEYS choosing the chunk exchange.
    template <bool KEYS>
    __device__ __forceinline__ void load(const char *base, int64_t offset, char *to, int lane, int row0,
                                         uint32_t head_dim) const {
        using TL = Tile<DP>;
        const int lo = static_cast<int>(offset), hi = static_cast<int>(offset >> 32);
#pragma unroll
        for (int i = 0; i < ROWS / TL::kRowsPerLoad; ++i) {
            const int r = i * TL::kRowsPerLoad + lane / TL::kChunks;
            const int64_t off = (static_cast<int64_t>(__shfl(hi, r, 64)) << 32) | static_cast<uint32_t>(__shfl(lo, r, 64));
            const int turn = KEYS ? TL::key_turn(row0 + r) : TL::value_turn(row0 + r);
            const int chunk = (lane % TL::kChunks) ^ turn;
            const char *src = base + off + chunk * 16;
            if (off < 0 || chunk * 8 >= static_cast<int>(head_dim)) src = reinterpret_cast<const char *>(&kZeroRow);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                             (__attribute__((address_space(3))) void *)(to + i * 1024), 16, 0, 0);
        }
    }
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct Mfma;
template <>
struct Mfma<bf16_t> {
    typedef bf16_t frag __attribute__((ext_vector_type(8)));
    static constexpr uint32_t kMantissa = 0x7F;
    // Bits 15 and 31 are set where the element in bits 0-15 or 16-31 is infinite or NaN.
    static __device__ __forceinline__ uint32_t special(uint32_t two) { return (two & 0x7F807F80u) + 0x00800080u; }
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mfma<f16_t> {
    typedef f16_t frag __attribute__((ext_vector_type(8)));
    static constexpr uint32_t kMantissa = 0x3FF;
    static __device__ __forceinline__ uint32_t special(uint32_t two) { return (two & 0x7C007C00u) + 0x04000400u; }
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// Four rows of one column from LDS (ds_read_b64_tr_b16): lanes 4r + q of a group
// of 16 give the address of columns 4q .. 4q+3 of row r; lane i gets column i.
typedef short tr_quad __attribute__((__vector_size__(8)));
__device__ __forceinline__ uint2 read_transposed(const char *p) {
    const tr_quad q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr_quad *)p);
    return __builtin_bit_cast(uint2, q);
}

// The other half-wave's value (lane ^ 32), as a pair {low lanes', high lanes'}.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Checks of a cache description that every operator over it shares (qxt_paged_attention.hip).
int check_paged_cache(const char *name, const qxt_paged_cache *cache, bool needs_values);

}  // namespace qxt
