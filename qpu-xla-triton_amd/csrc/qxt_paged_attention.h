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
    uint32_t even;   // units of eight slots lie in one page, in rows of DP elements; keys and values at one distance
    uint32_t tiles, splits;  // grid: kv_heads x tiles x splits x sequences, kv_heads fastest
    char *out;
    int64_t out_token, out_head;
    uint32_t out_type;
    float *lse;
    int64_t lse_token;
    float *part_out;   // [splits, tokens, heads, head_dim], unnormalised
    float2 *part_sum;  // [splits, tokens, heads]: (maximum in log2 units, sum)
};

// A kernel's arguments in the kernarg segment, where they are the first.  The
// kernels read them there instead of from the parameter: what is only needed
// before or after the main loop is then loaded there (`late` hides that it is
// the same memory) and holds no scalar registers over it.  With all arguments
// live the loop needs more than there are, and the compiler gives up ordering it.
template <typename A>
using Kernarg = const __attribute__((address_space(4))) A;
template <typename A>
__device__ __forceinline__ Kernarg<A> *kernargs() {
    return (Kernarg<A> *)__builtin_amdgcn_kernarg_segment_ptr();
}
template <typename A>
__device__ __forceinline__ A *late(A *args) {
    asm volatile("" : "+s"(args));
    return args;
}

// A wave-uniform value that stays in a register from here on.
template <typename V>
__device__ __forceinline__ void keep(V &value) {
    asm volatile("" : "+s"(value));
}

// (A: PagedArgs, in any address space.)
// The tokens and cache length of one sequence; lengths from the device are
// clamped to what the tensors hold, so no index leaves them.
struct Sequence {
    int32_t start, tokens, length;
};

template <typename A>
__device__ __forceinline__ Sequence sequence_of(const A &a, uint32_t b) {
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
// A window as seen_by takes it: at - window + 1 stays in 32 bits (at > -2^30), and 2^30 covers every slot.
inline int32_t window_of(uint32_t window) { return static_cast<int32_t>(window < (1u << 30) ? window : 1u << 30); }

template <typename A>
__device__ __forceinline__ Range seen_by(const A &a, const Sequence &s, int32_t token) {
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
    static __device__ __forceinline__ int key_turn(int row) { return row & (kChunks < 16 ? 7 : 15); }
    static __device__ __forceinline__ int value_turn(int row) { return kChunks < 16 ? 2 * (row & 3) : 4 * (row & 3); }
};

// Source of rows that are not in the cache: slots past a sequence's end, pages
// that its table does not name, and the columns from head_dim up to DP.
__device__ __constant__ const uint4 kZeroRow[32] = {};

// 64 lanes' 16 bytes from `src` (each lane its own) to LDS at `to` + 16 * lane.
// Inline assembly because the compiler, which cannot tell the buffers of a
// ring apart, waits for every such load in flight before it reads any of LDS;
// here the waits are the kernels' own (landed<N>).  There is no register output.
// (The compiler warns that it may not preserve m0; it has no other use for it in these kernels.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const char *src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(src) : "memory", "m0");
}
// The same from a wave-uniform address plus each lane's offset.
__device__ __forceinline__ void dma16_at(uint64_t base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// Wait until all but the wave's N youngest loads are done.
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// All of the wave's LDS reads have returned.
__device__ __forceinline__ void reads_done() {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// A workgroup barrier that, unlike __syncthreads, waits for no load in flight.
__device__ __forceinline__ void meet() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ uint32_t lds_offset(const char *p) {
    return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char *)p)));
}

// One wave's share of staging: ROWS consecutive slots of a tile.  Rows go in
// units of eight.  Where pages hold whole units (`even`), a unit's address is
// the same for the wave and the lanes' offsets in it never change: scalar
// arithmetic and one instruction a load.  Otherwise, and for the units at a
// sequence's end, each lane works out a row's address and the lanes that load
// it fetch it from there.  Each lane holds the page id of one of 64 consecutive
// table entries, refetched when the slots leave them, so that a tile's
// addresses wait for no load.
template <int DP, int ROWS>
struct Stager {
    using TL = Tile<DP>;
    static constexpr int kLoads = ROWS / TL::kRowsPerLoad;  // of keys, and as many of values
    static constexpr int kUnit = 8, kUnits = ROWS / kUnit, kUnitLoads = kUnit / TL::kRowsPerLoad;
    // Arguments that the main loops need, in registers: left in the kernarg segment they are loaded, and
    // waited for, at every use.
    const int32_t *table;
    uint64_t keys, values;  // of this head
    FastDiv page;
    uint32_t pages, even, head_dim;
    uint32_t key_page, key_slot, value_page, value_slot;  // strides in 16 bytes
    int32_t held, page0;        // page id of entry page0 + lane
    int32_t holes;              // some of them name no page
    // Of this lane's 16 bytes within a unit; keys of even and odd units (of a wave's single unit: its own).
    static constexpr int kKinds = kUnits > 1 ? 2 : 1;
    uint32_t key_offset[kKinds][kUnitLoads], value_offset[kUnitLoads];

    template <typename A>
    __device__ __forceinline__ void start(const A &a, uint32_t b, uint32_t head, int first_row) {
        table = a.table + b * a.table_stride;
        keys = reinterpret_cast<uint64_t>(a.keys.data + head * a.keys.head_stride);
        values = reinterpret_cast<uint64_t>(a.values.data + head * a.values.head_stride);
        page = FastDiv{a.page.divisor, a.page.magic, a.page.shift, a.page.pass};
        pages = a.pages;
        even = a.even;
        head_dim = a.head_dim;
        key_page = static_cast<uint32_t>(a.keys.page_stride / 16);
        key_slot = static_cast<uint32_t>(a.keys.slot_stride / 16);
        value_page = static_cast<uint32_t>(a.values.page_stride / 16);
        value_slot = static_cast<uint32_t>(a.values.slot_stride / 16);
        keep(table);
        keep(keys);
        keep(values);
        keep(page.divisor);
        keep(page.magic);
        keep(page.shift);
        keep(page.pass);
        keep(pages);
        keep(even);
        keep(head_dim);
        keep(key_page);
        keep(key_slot);
        keep(value_page);
        keep(value_slot);
        held = -1;
        page0 = -64;
        holes = 0;
        const int lane = threadIdx.x % 64;
#pragma unroll
        for (int i = 0; i < kUnitLoads; ++i) {
            const int r = i * TL::kRowsPerLoad + lane / TL::kChunks, chunk = lane % TL::kChunks;
#pragma unroll
            for (int k = 0; k < kKinds; ++k)
                key_offset[k][i] = r * static_cast<uint32_t>(a.keys.slot_stride) + (chunk ^ TL::key_turn(first_row + 8 * k + r)) * 16;
            value_offset[i] = r * static_cast<uint32_t>(a.values.slot_stride) + (chunk ^ TL::value_turn(r)) * 16;
        }
    }

    // The rows of slots slot0 .. slot0 + ROWS - 1 (those from `high` on are zeros).
    struct Rows {
        int32_t whole;                           // wave-uniform: units by the addresses below
        uint64_t at[kUnits];                     // (of keys; values lie at one distance from them)
        int32_t id;                              // else page id (or -1) and place in the page of this lane's row
        uint32_t in_page;
    };

    // Before a tile whose `high` may be larger than the one before: what is held repeats the last entry below the old one.
    __device__ __forceinline__ void forget() { page0 = -64; }

    // Page ids of the entries from `first` on (the last one below `high` repeated: right while `high` does not grow).
    __device__ __forceinline__ void fetch(int32_t first, int32_t high) {
        page0 = first;
        held = table[min(first + static_cast<int32_t>(threadIdx.x % 64), static_cast<int32_t>(fast_quotient(high - 1, page)))];
        holes = __any(static_cast<uint32_t>(held) >= pages) ? 1 : 0;
        asm volatile("" : "+v"(held));  // waited for here, not (with every DMA in flight) at each use
    }
    __device__ __forceinline__ static uint64_t address(uint64_t base, uint32_t page_stride, uint32_t slot_stride, uint32_t id,
                                                       uint32_t in_page) {
        return base + ((static_cast<uint64_t>(id) * page_stride + static_cast<uint64_t>(in_page) * slot_stride) << 4);
    }

    __device__ __forceinline__ Rows locate(int32_t slot0, int32_t high) {
        Rows r;
        r.id = -1;
        r.in_page = 0;
        r.whole = 0;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) r.at[u] = 0;
        if (even != 0 && slot0 + ROWS <= high) {
            const int32_t last = fast_quotient(slot0 + ROWS - kUnit, page);
            const int32_t first = kUnits > 1 ? static_cast<int32_t>(fast_quotient(slot0, page)) : last;
            if (first < page0 || last >= page0 + 64) fetch(first, high);
            if (holes == 0) {
                r.whole = 1;
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
                    const uint32_t slot = slot0 + u * kUnit, entry = fast_quotient(slot, page), in_page = slot - entry * page.divisor;
                    const uint32_t id = __builtin_amdgcn_readlane(held, entry - page0);
                    r.at[u] = keys + ((static_cast<uint64_t>(id) * key_page + in_page * key_slot) << 4);
                }
                return r;
            }
        }
        // At the last rows, in other pages and among entries without a page the lanes work on their own.
        if (slot0 < high) {
            const int32_t first = fast_quotient(slot0, page), last = fast_quotient(min(slot0 + ROWS, high) - 1, page);
            if (first < page0 || last >= page0 + 64) fetch(first, high);
        }
        const int32_t slot = slot0 + static_cast<int32_t>(threadIdx.x % 64) % ROWS;
        const uint32_t entry = fast_quotient(static_cast<uint32_t>(slot), page);
        r.in_page = static_cast<uint32_t>(slot) - entry * page.divisor;
        const int32_t id = __shfl(held, static_cast<int>(entry) - page0, 64);
        r.id = slot < high && static_cast<uint32_t>(id) < pages ? id : -1;
        return r;
    }

    template <bool KEYS>
    __device__ __forceinline__ void load(const Rows &rows, uint32_t to, int first_row) const {
        if (rows.whole) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
#pragma unroll
                for (int i = 0; i < kUnitLoads; ++i)
                    dma16_at(KEYS ? rows.at[u] : rows.at[u] + (values - keys), KEYS ? key_offset[u % kKinds][i] : value_offset[i],
                             to + (u * kUnitLoads + i) * 1024);
            return;
        }
        const int lane = threadIdx.x % 64;
        const uint64_t row = rows.id < 0 ? reinterpret_cast<uint64_t>(kZeroRow)
                             : KEYS      ? address(keys, key_page, key_slot, rows.id, rows.in_page)
                                         : address(values, value_page, value_slot, rows.id, rows.in_page);
        const int lo = static_cast<int>(row), hi = static_cast<int>(row >> 32);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = i * TL::kRowsPerLoad + lane / TL::kChunks;
            const uint64_t at = (static_cast<uint64_t>(static_cast<uint32_t>(__shfl(hi, r, 64))) << 32) |
                                static_cast<uint32_t>(__shfl(lo, r, 64));
            const int chunk = (lane % TL::kChunks) ^ (KEYS ? TL::key_turn(first_row + r) : TL::value_turn(r));
            const uint64_t src = chunk * 8 < static_cast<int>(head_dim) ? at + chunk * 16 : reinterpret_cast<uint64_t>(kZeroRow);
            dma16(reinterpret_cast<const char *>(src), to + i * 1024);
        }
    }
    __device__ __forceinline__ void load_keys(const Rows &rows, uint32_t to, int first_row) const {
        load<true>(rows, to, first_row);
    }
    __device__ __forceinline__ void load_values(const Rows &rows, uint32_t to) const { load<false>(rows, to, 0); }
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct Mfma;
template <>
struct Mfma<bf16_t> {
    typedef bf16_t frag __attribute__((ext_vector_type(8)));
    // Bits 15 and 31 are set where the element in bits 0-15 or 16-31 is infinite or NaN.
    static __device__ __forceinline__ uint32_t special(uint32_t two) { return (two & 0x7F807F80u) + 0x00800080u; }
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mfma<f16_t> {
    typedef f16_t frag __attribute__((ext_vector_type(8)));
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
