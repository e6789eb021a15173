// Norms of queries and keys per head and the position rotation in one pass,
// optionally storing keys and values into a paged cache.
//
// For a row x of head_dim elements with weight w:
//   y = x * rsqrt(mean(x^2) + epsilon) * w        (y = x without a weight)
// and for each i < rotary_dim / 2 the pair (a, b) = (y[i], y[i + rotary_dim/2]),
// or (y[2i], y[2i+1]) when interleaved, becomes
//   (a cos - b sin, b cos + a sin),  cos/sin at [position, i].
// Everything is fp32 until the one rounding of the store.
//
// The operator is bound by the bytes of its rows.  A row is held by
// ceil(head_dim / 8) neighbouring lanes (a power of two of them reduce the sum
// of squares with shuffles), and a lane holds two runs of four elements that
// contain both members of its pairs, so no element is read twice and the
// rotation needs no exchange: runs i and i + rotary_dim/8 for the split pairs,
// 2i and 2i + 1 for the interleaved ones and past the rotated part.
// Measured: 4096 tokens of 32 + 8 + 8 heads of 128 (153 MB read and written)
// 28.7 us, 5.3 TB/s, where a 2 GiB copy reaches 4.9; one token 3.9 us, a launch.
#include "qxt_paged.h"

namespace qxt {
namespace {

struct RopeArgs {
    const char *in[3];  // query, key, value
    int64_t in_token[3], in_head[3];
    const float *weight[2];
    const float *cos, *sin;
    int64_t table_stride;
    uint32_t table_rows;
    const int32_t *positions;
    char *query_out;
    int64_t query_out_token, query_out_head;
    CacheView out[2];  // key, value: cache views, or rows by token (page_size 1)
    const int64_t *slots;
    int64_t slot_count;
    uint32_t page_size;
    FastDiv page;  // by page_size, for caches of fewer than 2^31 slots
    uint32_t tokens, query_heads, key_heads, rows;  // rows = tokens * all heads
    FastDiv heads;                                  // all heads of a token
    uint32_t head_dim, rotary_dim;
    float epsilon;
};

// Where row (token, head) comes from and goes to; out == nullptr: not stored.
struct RowPlace {
    const char *in;
    char *out;
    const float *weight;
    bool turns;  // a query or a key
    uint32_t token;
};

// (Selections between values, not an index into the argument arrays or a choice between their elements: an
// address that the compiler does not know sends the whole argument block through scratch memory.)
__device__ __forceinline__ RowPlace place_row(const RopeArgs &a, uint32_t row) {
    RowPlace p;
    p.token = fast_quotient(row, a.heads);
    uint32_t head = row - p.token * a.heads.divisor;
    const bool query = head < a.query_heads;
    head -= query ? 0 : a.query_heads;
    const bool key = !query && head < a.key_heads;
    head -= query || key ? 0 : a.key_heads;
    p.turns = query || key;
    const float *const weight0 = a.weight[0], *const weight1 = a.weight[1];
    p.weight = query ? weight0 : key ? weight1 : nullptr;
    const char *const in0 = a.in[0], *const in1 = a.in[1], *const in2 = a.in[2];
    const int64_t token0 = a.in_token[0], token1 = a.in_token[1], token2 = a.in_token[2];
    const int64_t head0 = a.in_head[0], head1 = a.in_head[1], head2 = a.in_head[2];
    p.in = (query ? in0 : key ? in1 : in2) + p.token * (query ? token0 : key ? token1 : token2) +
           head * (query ? head0 : key ? head1 : head2);
    p.out = a.query_out + p.token * a.query_out_token + head * a.query_out_head;
    if (!query) {
        const int64_t slot = a.slots != nullptr ? a.slots[p.token] : p.token;
        int64_t page = slot, offset = 0;
        if (a.page_size > 1) {
            page = a.slot_count <= INT32_MAX ? fast_quotient(static_cast<uint32_t>(slot), a.page) : slot / a.page_size;
            offset = slot - page * a.page_size;
        }
        const CacheView keys = a.out[0], values = a.out[1];
        p.out = (key ? keys.data : values.data) + page * (key ? keys.page_stride : values.page_stride) +
                offset * (key ? keys.slot_stride : values.slot_stride) + head * (key ? keys.head_stride : values.head_stride);
        if (slot < 0 || slot >= a.slot_count) p.out = nullptr;  // padding tokens, and nothing outside the cache
    }
    return p;
}

template <typename T>
__device__ __forceinline__ float4 load4(const T *p) {
    typedef typename vec4_of<T>::type v4;
    const v4 v = *reinterpret_cast<const v4 *>(p);
    return make_float4(static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]),
                       static_cast<float>(v[3]));
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const float4 &x) {
    typedef typename vec4_of<T>::type v4;
    v4 v;
    v[0] = static_cast<T>(x.x);
    v[1] = static_cast<T>(x.y);
    v[2] = static_cast<T>(x.z);
    v[3] = static_cast<T>(x.w);
    *reinterpret_cast<v4 *>(p) = v;
}

__device__ __forceinline__ float squares(const float4 &v) { return v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w; }

__device__ __forceinline__ float4 scaled(const float4 &v, float s, const float4 &w) {
    return make_float4(v.x * s * w.x, v.y * s * w.y, v.z * s * w.z, v.w * s * w.w);
}

__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}

// LANES lanes (a power of two) a row of at most 8 LANES elements.  head_dim and
// rotary_dim / 2 (split) or rotary_dim (interleaved) are multiples of four,
// every row and table row is aligned to four elements.
template <typename TI, typename TO, int LANES, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
    const uint32_t lane = threadIdx.x % LANES;
    const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= a.rows) return;  // whole groups of LANES leave together
    const RowPlace p = place_row(a, row);
    const TI *in = reinterpret_cast<const TI *>(p.in);
    TO *out = reinterpret_cast<TO *>(p.out);
    const uint32_t runs = a.head_dim / 4, turned = a.rotary_dim / 8;  // runs of four, lanes with split pairs
    uint32_t r0 = 2 * lane, r1 = 2 * lane + 1;
    if (!INTERLEAVED && lane < turned) {
        r0 = lane;
        r1 = lane + turned;
    }
    const bool has0 = r0 < runs, has1 = r1 < runs;
    float4 x0 = make_float4(0.f, 0.f, 0.f, 0.f), x1 = x0;
    if (has0) x0 = load4(in + 4 * r0);
    if (has1) x1 = load4(in + 4 * r1);
    if (p.turns) {
        const int32_t position = a.positions[p.token];
        const float *weight = p.weight;
        if (weight != nullptr) {
            float sum = squares(x0) + squares(x1);
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, LANES);
            const float s = rsqrtf(sum / static_cast<float>(a.head_dim) + a.epsilon);
            if (has0) x0 = scaled(x0, s, *reinterpret_cast<const float4 *>(weight + 4 * r0));
            if (has1) x1 = scaled(x1, s, *reinterpret_cast<const float4 *>(weight + 4 * r1));
        }
        if (static_cast<uint32_t>(position) < a.table_rows) {
            const float *cos = a.cos + position * a.table_stride, *sin = a.sin + position * a.table_stride;
            if (INTERLEAVED) {
                if (4 * r0 < a.rotary_dim) {
                    const float2 c = *reinterpret_cast<const float2 *>(cos + 2 * r0);
                    const float2 s = *reinterpret_cast<const float2 *>(sin + 2 * r0);
                    turn(x0.x, x0.y, c.x, s.x);
                    turn(x0.z, x0.w, c.y, s.y);
                }
                if (4 * r1 < a.rotary_dim) {
                    const float2 c = *reinterpret_cast<const float2 *>(cos + 2 * r1);
                    const float2 s = *reinterpret_cast<const float2 *>(sin + 2 * r1);
                    turn(x1.x, x1.y, c.x, s.x);
                    turn(x1.z, x1.w, c.y, s.y);
                }
            } else if (lane < turned) {
                const float4 c = *reinterpret_cast<const float4 *>(cos + 4 * lane);
                const float4 s = *reinterpret_cast<const float4 *>(sin + 4 * lane);
                turn(x0.x, x1.x, c.x, s.x);
                turn(x0.y, x1.y, c.y, s.y);
                turn(x0.z, x1.z, c.z, s.z);
                turn(x0.w, x1.w, c.w, s.w);
            }
        } else {
            // A position outside the table has no angle: the rotated part is NaN, not a wrong angle's.
            const float nan = __builtin_nanf("");
            if (4 * r0 < a.rotary_dim) x0 = make_float4(nan, nan, nan, nan);
            if (4 * r1 < a.rotary_dim) x1 = make_float4(nan, nan, nan, nan);
        }
    }
    if (out == nullptr) return;
    if (has0) store4(out + 4 * r0, x0);
    if (has1) store4(out + 4 * r1, x1);
}

// Any head_dim, even rotary_dim and element alignment: one wave a row, pair by
// pair (past the rotated part "pairs" are neighbours that stay as they are).
template <typename TI, typename TO, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_norm_rope_any_kernel(RopeArgs a) {
    const uint32_t lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64;
    if (row >= a.rows) return;
    const RowPlace p = place_row(a, row);
    const TI *in = reinterpret_cast<const TI *>(p.in);
    TO *out = reinterpret_cast<TO *>(p.out);
    const float *weight = p.weight;
    float scale = 1.0f;
    if (weight != nullptr) {
        float sum = 0.0f;
        for (uint32_t i = lane; i < a.head_dim; i += 64) {
            const float v = static_cast<float>(in[i]);
            sum += v * v;
        }
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        scale = rsqrtf(sum / static_cast<float>(a.head_dim) + a.epsilon);
    }
    if (out == nullptr) return;
    const int32_t position = p.turns ? a.positions[p.token] : 0;
    const bool known = static_cast<uint32_t>(position) < a.table_rows;
    const uint32_t half = p.turns ? a.rotary_dim / 2 : 0, rotated = 2 * half;
    for (uint32_t i = lane; i < half + (a.head_dim - rotated + 1) / 2; i += 64) {
        const bool turns = i < half;
        const uint32_t e0 = turns && !INTERLEAVED ? i : 2 * i, e1 = turns && !INTERLEAVED ? i + half : 2 * i + 1;
        float v0 = static_cast<float>(in[e0]), v1 = e1 < a.head_dim ? static_cast<float>(in[e1]) : 0.0f;
        if (weight != nullptr) {
            v0 = v0 * scale * weight[e0];
            if (e1 < a.head_dim) v1 = v1 * scale * weight[e1];
        }
        if (turns) {
            if (known)
                turn(v0, v1, a.cos[position * a.table_stride + i], a.sin[position * a.table_stride + i]);
            else
                v0 = v1 = __builtin_nanf("");
        }
        out[e0] = static_cast<TO>(v0);
        if (e1 < a.head_dim) out[e1] = static_cast<TO>(v1);
    }
}

template <typename TI, typename TO, bool INTERLEAVED>
int launch_rope(const RopeArgs &a, bool runs_of_four, hipStream_t stream) {
    const uint32_t lanes = (a.head_dim + 7) / 8;
    if (!runs_of_four || lanes > 64)
        return launch("qk_norm_rope_any_kernel", qk_norm_rope_any_kernel<TI, TO, INTERLEAVED>, dim3((a.rows + 3) / 4),
                      dim3(256), 0, stream, a);
#define QXT_ROPE(L)                                                                                                 \
    if (lanes <= L)                                                                                                 \
    return launch("qk_norm_rope_kernel", qk_norm_rope_kernel<TI, TO, L, INTERLEAVED>,                               \
                  dim3((a.rows + 256 / L - 1) / (256 / L)), dim3(256), 0, stream, a)
    QXT_ROPE(8);
    QXT_ROPE(16);
    QXT_ROPE(32);
    QXT_ROPE(64);
#undef QXT_ROPE
    return fail(QXT_INTERNAL_ERROR, "qk norm rope: no launch for %u lanes", lanes);
}

template <typename TI, typename TO>
int launch_rope_form(const RopeArgs &a, bool interleaved, bool runs_of_four, hipStream_t stream) {
    return interleaved ? launch_rope<TI, TO, true>(a, runs_of_four, stream)
                       : launch_rope<TI, TO, false>(a, runs_of_four, stream);
}

template <typename TI>
int launch_rope_out(const RopeArgs &a, uint32_t output_type, bool interleaved, bool runs, hipStream_t stream) {
    switch (output_type) {
        case QXT_TYPE_BF16: return launch_rope_form<TI, bf16_t>(a, interleaved, runs, stream);
        case QXT_TYPE_F16: return launch_rope_form<TI, f16_t>(a, interleaved, runs, stream);
        default: return launch_rope_form<TI, float>(a, interleaved, runs, stream);
    }
}

// Checks shared by both entry points, then the launch.  `a` is complete but for rows and heads.
int run_rope(RopeArgs &a, bool cached, uint32_t input_type, uint32_t output_type, uint32_t flags, hipStream_t stream) {
    if (!known_type(input_type) || !known_type(output_type))
        return fail(QXT_INVALID_ARGUMENT, "qk norm rope: unknown element type");
    if (flags & ~QXT_ROPE_INTERLEAVED) return fail(QXT_INVALID_ARGUMENT, "qk norm rope: unknown flags");
    if (a.head_dim == 0 || a.query_heads + a.key_heads == 0)
        return fail(QXT_INVALID_ARGUMENT, "qk norm rope: head size and heads must be positive");
    if (a.rotary_dim % 2 || a.rotary_dim > a.head_dim)
        return fail(QXT_INVALID_ARGUMENT, "qk norm rope: rotary size must be even and at most the head size");
    const uint64_t heads = static_cast<uint64_t>(a.query_heads) + static_cast<uint64_t>(a.key_heads) * (cached ? 2 : 1);
    if (heads * a.tokens > INT32_MAX) return fail(QXT_INVALID_ARGUMENT, "qk norm rope: more than 2^31 rows");
    if (a.tokens == 0) return QXT_OK;
    if ((a.query_heads && (a.in[0] == nullptr || a.query_out == nullptr)) ||
        (a.key_heads && (a.in[1] == nullptr || a.out[0].data == nullptr)) ||
        (cached && a.key_heads && (a.in[2] == nullptr || a.out[1].data == nullptr || a.slots == nullptr)) ||
        a.positions == nullptr || (a.rotary_dim && (a.cos == nullptr || a.sin == nullptr)))
        return fail(QXT_INVALID_ARGUMENT, "qk norm rope: null pointer");
    if (a.rotary_dim == 0) a.table_rows = UINT32_MAX;  // nothing is looked up
    const size_t ti = type_bytes(input_type), to = type_bytes(output_type);
    for (int i = 0; i < 3; ++i)
        if (!aligned(a.in[i], ti) || !all_multiples(ti, {static_cast<size_t>(a.in_token[i]), static_cast<size_t>(a.in_head[i])}))
            return fail(QXT_INVALID_ARGUMENT, "qk norm rope: misaligned input");
    bool in_runs = true, out_runs = true;
    for (int i = 0; i < 3; ++i)
        in_runs = in_runs && aligned(a.in[i], 4 * ti) &&
                  all_multiples(4 * ti, {static_cast<size_t>(a.in_token[i]), static_cast<size_t>(a.in_head[i])});
    auto output_ok = [&](size_t by) {
        bool ok = aligned(a.query_out, by) && all_multiples(by, {static_cast<size_t>(a.query_out_token), static_cast<size_t>(a.query_out_head)});
        for (int i = 0; i < (cached ? 2 : 1); ++i)
            ok = ok && aligned(a.out[i].data, by) &&
                 all_multiples(by, {static_cast<size_t>(a.out[i].page_stride), static_cast<size_t>(a.out[i].slot_stride),
                                    static_cast<size_t>(a.out[i].head_stride)});
        return ok;
    };
    if (!output_ok(to)) return fail(QXT_INVALID_ARGUMENT, "qk norm rope: misaligned output");
    out_runs = output_ok(4 * to);
    if (!aligned(a.cos, 4) || !aligned(a.sin, 4) || !aligned(a.positions, 4) || !aligned(a.slots, 8) ||
        !aligned(a.weight[0], 4) || !aligned(a.weight[1], 4))
        return fail(QXT_INVALID_ARGUMENT, "qk norm rope: misaligned table, weight or index");
    if (int rc = injected(QXT_FAIL_SUBMISSION)) return rc;
    const bool interleaved = flags & QXT_ROPE_INTERLEAVED;
    const size_t table = interleaved ? 8 : 16;
    const bool runs = in_runs && out_runs && a.head_dim % 4 == 0 && a.rotary_dim % (interleaved ? 4 : 8) == 0 &&
                      aligned(a.cos, table) && aligned(a.sin, table) && (a.table_stride * 4) % table == 0 &&
                      aligned(a.weight[0], 16) && aligned(a.weight[1], 16);
    a.page = fast_div(a.page_size);
    a.heads = fast_div(static_cast<uint32_t>(heads));
    a.rows = static_cast<uint32_t>(heads * a.tokens);
    switch (input_type) {
        case QXT_TYPE_BF16: return launch_rope_out<bf16_t>(a, output_type, interleaved, runs, stream);
        case QXT_TYPE_F16: return launch_rope_out<f16_t>(a, output_type, interleaved, runs, stream);
        default: return launch_rope_out<float>(a, output_type, interleaved, runs, stream);
    }
}

}  // namespace
}  // namespace qxt

extern "C" {

int qxt_qk_norm_rope(const void *query, size_t query_token_stride, size_t query_head_stride, const void *key,
                     size_t key_token_stride, size_t key_head_stride, const float *query_weight,
                     const float *key_weight, float epsilon, const float *cos, const float *sin,
                     size_t table_row_stride, uint32_t table_rows, const int32_t *positions, void *query_out,
                     size_t query_out_token_stride, size_t query_out_head_stride, void *key_out,
                     size_t key_out_token_stride, size_t key_out_head_stride, uint32_t tokens, uint32_t query_heads,
                     uint32_t key_heads, uint32_t head_dim, uint32_t rotary_dim, uint32_t input_type,
                     uint32_t output_type, uint32_t flags, void *stream) {
    if (table_row_stride % 4) return qxt::fail(QXT_INVALID_ARGUMENT, "qk norm rope: misaligned table, weight or index");
    qxt::RopeArgs a{};
    a.in[0] = static_cast<const char *>(query);
    a.in[1] = static_cast<const char *>(key);
    a.in_token[0] = query_token_stride;
    a.in_token[1] = key_token_stride;
    a.in_head[0] = query_head_stride;
    a.in_head[1] = key_head_stride;
    a.weight[0] = query_weight;
    a.weight[1] = key_weight;
    a.cos = cos;
    a.sin = sin;
    a.table_stride = table_row_stride / 4;
    a.table_rows = table_rows;
    a.positions = positions;
    a.query_out = static_cast<char *>(query_out);
    a.query_out_token = query_out_token_stride;
    a.query_out_head = query_out_head_stride;
    a.out[0] = {static_cast<char *>(key_out), static_cast<int64_t>(key_out_token_stride), 0,
                static_cast<int64_t>(key_out_head_stride)};
    a.slot_count = tokens;
    a.page_size = 1;
    a.tokens = tokens;
    a.query_heads = query_heads;
    a.key_heads = key_heads;
    a.head_dim = head_dim;
    a.rotary_dim = rotary_dim;
    a.epsilon = epsilon;
    return qxt::run_rope(a, false, input_type, output_type, flags, qxt::as_stream(stream));
}

int qxt_qk_norm_rope_cache(const void *query, size_t query_token_stride, size_t query_head_stride, const void *key,
                           size_t key_token_stride, size_t key_head_stride, const void *value,
                           size_t value_token_stride, size_t value_head_stride, const float *query_weight,
                           const float *key_weight, float epsilon, const float *cos, const float *sin,
                           size_t table_row_stride, uint32_t table_rows, const int32_t *positions,
                           const int64_t *slots, void *query_out, size_t query_out_token_stride,
                           size_t query_out_head_stride, const qxt_paged_cache *cache, uint32_t tokens,
                           uint32_t query_heads, uint32_t rotary_dim, uint32_t input_type, uint32_t flags,
                           void *stream) {
    if (cache == nullptr) return qxt::fail(QXT_INVALID_ARGUMENT, "qk norm rope: null pointer");
    if (table_row_stride % 4) return qxt::fail(QXT_INVALID_ARGUMENT, "qk norm rope: misaligned table, weight or index");
    if (!qxt::half_type(cache->type)) return qxt::fail(QXT_INVALID_ARGUMENT, "qk norm rope: the cache must be bf16 or fp16");
    if (cache->page_size == 0) return qxt::fail(QXT_INVALID_ARGUMENT, "qk norm rope: page size must be positive");
    qxt::RopeArgs a{};
    a.in[0] = static_cast<const char *>(query);
    a.in[1] = static_cast<const char *>(key);
    a.in[2] = static_cast<const char *>(value);
    a.in_token[0] = query_token_stride;
    a.in_token[1] = key_token_stride;
    a.in_token[2] = value_token_stride;
    a.in_head[0] = query_head_stride;
    a.in_head[1] = key_head_stride;
    a.in_head[2] = value_head_stride;
    a.weight[0] = query_weight;
    a.weight[1] = key_weight;
    a.cos = cos;
    a.sin = sin;
    a.table_stride = table_row_stride / 4;
    a.table_rows = table_rows;
    a.positions = positions;
    a.query_out = static_cast<char *>(query_out);
    a.query_out_token = query_out_token_stride;
    a.query_out_head = query_out_head_stride;
    a.out[0] = {static_cast<char *>(cache->keys), static_cast<int64_t>(cache->key_page_stride),
                static_cast<int64_t>(cache->key_slot_stride), static_cast<int64_t>(cache->key_head_stride)};
    a.out[1] = {static_cast<char *>(cache->values), static_cast<int64_t>(cache->value_page_stride),
                static_cast<int64_t>(cache->value_slot_stride), static_cast<int64_t>(cache->value_head_stride)};
    a.slots = slots;
    a.slot_count = static_cast<int64_t>(cache->pages) * cache->page_size;
    a.page_size = cache->page_size;
    a.tokens = tokens;
    a.query_heads = query_heads;
    a.key_heads = cache->heads;
    a.head_dim = cache->head_dim;
    a.rotary_dim = rotary_dim;
    a.epsilon = epsilon;
    return qxt::run_rope(a, true, input_type, cache->type, flags, qxt::as_stream(stream));
}

}  // extern "C"
