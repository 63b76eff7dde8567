// The KV cache held in 4 bits: where its rows lie, the view that kernels take, and the checks
// that its entry points share.
#pragma once

#include <algorithm>

#include "internal.hpp"
#include "route.hpp"

namespace swq {

constexpr int kQ4Group = 64;      // dims of one scale and bias
constexpr int kQ4Block = 8;       // rows of one v word
constexpr int kQ4MaxRows = 1 << 27;  // of a sequence: a head's parameters of one kind stay below 4 GiB
constexpr int kQ4RowPad = 32;     // rows are allocated in multiples of this: a reader's tile
constexpr int kQ4MaxHeadGroup = 16;  // query heads per kv head

enum { kQ4KScale = 0, kQ4KBias = 1, kQ4VScale = 2, kQ4VBias = 3 };

// Device view of a swq_q4_cache.  All offsets are 64-bit: a cache passes 4 GiB.
struct Q4View {
    uint32_t *k;      // [B][KVH][R][hd / 8]
    uint32_t *v;      // [B][KVH][R / 8][hd]
    _Float16 *par;    // [B][KVH][4][hd / 64][R]
    int32_t B, KVH, hd, maxp, R;

    __host__ __device__ __forceinline__ int64_t head(int b, int h) const { return static_cast<int64_t>(b) * KVH + h; }
    __device__ __forceinline__ uint32_t *k_head(int b, int h) const { return k + head(b, h) * R * (hd / 8); }
    __device__ __forceinline__ uint32_t *v_head(int b, int h) const { return v + head(b, h) * (R / 8) * hd; }
    __device__ __forceinline__ _Float16 *par_head(int b, int h) const { return par + head(b, h) * 4 * (hd / kQ4Group) * R; }
};

// Rows r0 .. r1 - 1 of the cache, which a sequence's tokens n0, n0 + 1, .. go into.
struct Q4Rows {
    int32_t n0, r0, r1;

    // Blocks with such rows.  None where there are no rows: then n0 may be no token of the call, and nothing is loaded.
    __host__ __device__ __forceinline__ int block0() const { return r0 / kQ4Block; }
    __host__ __device__ __forceinline__ int block_end() const { return r0 < r1 ? (r1 - 1) / kQ4Block + 1 : block0(); }
    __host__ __device__ __forceinline__ bool has(int row) const { return row >= r0 && row < r1; }
    // The token whose k and v a lane loads for a row of these blocks (the first for rows that are not its sequence's new ones).
    __host__ __device__ __forceinline__ int token(int row) const { return n0 + (has(row) ? row - r0 : 0); }
};

// Device view of a swq_q4_batch.  What comes from device memory is clamped where it is read, so
// that no value of it leads out of a buffer.
struct Q4Batch {
    int32_t B, N, max_tokens, rope_positions, rot;
    const int32_t *starts, *rows, *positions;
    const float2 *rope;

    __host__ __device__ __forceinline__ int first(int b) const { return starts ? min(max(starts[b], 0), N) : b * max_tokens; }
    __host__ __device__ __forceinline__ int count(int b) const { return starts ? max(min(starts[b + 1], N) - first(b), 0) : max_tokens; }
    __host__ __device__ __forceinline__ int row0(int b, int maxp) const { return min(max(rows[b], 0), maxp); }
    __host__ __device__ __forceinline__ Q4Rows written(int b, int maxp) const {
        const int r0 = row0(b, maxp);
        return {first(b), r0, static_cast<int32_t>(min(static_cast<int64_t>(r0) + count(b), static_cast<int64_t>(maxp)))};
    }
    __device__ __forceinline__ int position(int b, int i) const {
        const int64_t p = static_cast<int64_t>(positions ? positions[b] : rows[b]) + i;
        return static_cast<int>(min(max(p, static_cast<int64_t>(0)), static_cast<int64_t>(rope_positions - 1)));
    }
};

inline size_t q4_align(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

inline int64_t q4_rows(int maxp) { return (static_cast<int64_t>(maxp) + kQ4RowPad - 1) / kQ4RowPad * kQ4RowPad; }

struct Q4Layout {
    size_t codes, params, total;  // bytes of either code part and of the parameters, padded
};

inline Q4Layout q4_layout(int64_t B, int64_t kvh, int64_t hd, int maxp) {
    const int64_t n = B * kvh * q4_rows(maxp);
    Q4Layout l{};
    l.codes = q4_align(static_cast<size_t>(n * hd / 2));
    l.params = q4_align(static_cast<size_t>(n * 4 * (hd / kQ4Group) * 2));
    l.total = 2 * l.codes + l.params;
    return l;
}

inline bool q4_head_dim(int hd) { return hd == 64 || hd == 128 || hd == 256; }

inline int check_q4_shape(int sequences, int kvh, int hd, int maxp) {
    if (sequences <= 0 || kvh <= 0 || maxp <= 0 || hd <= 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (!q4_head_dim(hd) || maxp > kQ4MaxRows || static_cast<int64_t>(sequences) * kvh > 65535) return SWQ_ERR_LIMIT;
    return SWQ_OK;
}

inline int check_q4_cache(const swq_q4_cache *c) {
    if (!c) return SWQ_ERR_INVALID_ARGUMENT;
    const int st = check_q4_shape(c->sequences, c->num_kv_heads, c->head_dim, c->max_positions);
    if (st != SWQ_OK) return st;
    if (!c->data) return SWQ_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(c->data) % 256 != 0) return SWQ_ERR_MISALIGNED;
    if (c->bytes < q4_layout(c->sequences, c->num_kv_heads, c->head_dim, c->max_positions).total) return SWQ_ERR_WORKSPACE;
    return SWQ_OK;
}

inline Q4View q4_view(const swq_q4_cache *c) {
    const Q4Layout l = q4_layout(c->sequences, c->num_kv_heads, c->head_dim, c->max_positions);
    Q4View v{};
    uint8_t *p = static_cast<uint8_t *>(c->data);
    v.k = reinterpret_cast<uint32_t *>(p);
    v.v = reinterpret_cast<uint32_t *>(p + l.codes);
    v.par = reinterpret_cast<_Float16 *>(p + 2 * l.codes);
    v.B = c->sequences;
    v.KVH = c->num_kv_heads;
    v.hd = c->head_dim;
    v.maxp = c->max_positions;
    v.R = static_cast<int32_t>(q4_rows(c->max_positions));
    return v;
}

// swq_attention_layer as the 4-bit cache's calls take it (max_positions is the cache's).
inline int check_q4_layer(const swq_attention_layer *l) {
    if (!l || l->reserved != 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (l->num_heads <= 0 || l->num_kv_heads <= 0 || l->num_heads % l->num_kv_heads != 0) return SWQ_ERR_BAD_SHAPE;
    if (l->num_heads / l->num_kv_heads > kQ4MaxHeadGroup || !q4_head_dim(l->head_dim)) return SWQ_ERR_LIMIT;
    if (l->rotary_dims < 0 || l->rotary_dims > l->head_dim || l->rotary_dims % 2 != 0) return SWQ_ERR_BAD_SHAPE;
    if (!(l->norm_eps >= 0.f) || !l->q_norm_weight || !l->k_norm_weight) return SWQ_ERR_INVALID_ARGUMENT;
    return SWQ_OK;
}

// The sizes of a batch, without its device arrays.
inline int check_q4_sizes(const swq_q4_cache *c, const swq_q4_batch *b) {
    if (!b || b->reserved != 0 || b->sequences <= 0 || b->tokens < 0 || b->max_rows < 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (b->sequences > c->sequences) return SWQ_ERR_BAD_SHAPE;
    if (b->starts ? (b->max_tokens <= 0 && b->tokens > 0) : b->tokens % b->sequences != 0) return SWQ_ERR_BAD_SHAPE;
    return SWQ_OK;
}

inline int check_q4_batch(const swq_attention_layer *l, const swq_q4_cache *c, const swq_q4_batch *b) {
    int st = check_q4_layer(l);
    if (st == SWQ_OK) st = check_q4_cache(c);
    if (st == SWQ_OK) st = check_q4_sizes(c, b);
    if (st != SWQ_OK) return st;
    if (l->num_kv_heads != c->num_kv_heads || l->head_dim != c->head_dim) return SWQ_ERR_BAD_SHAPE;
    if (!b->rows) return SWQ_ERR_INVALID_ARGUMENT;
    if (l->rotary_dims > 0 && (!b->rope || b->rope_positions <= 0)) return SWQ_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(b->rope) % 16 != 0) return SWQ_ERR_MISALIGNED;
    return SWQ_OK;
}

inline int q4_max_tokens(const swq_q4_batch *b) {
    return b->starts ? std::min(b->max_tokens, b->tokens) : b->tokens / b->sequences;
}

inline Q4Batch q4_batch(const swq_attention_layer *l, const swq_q4_batch *b) {
    Q4Batch d{};
    d.B = b->sequences;
    d.N = b->tokens;
    d.max_tokens = q4_max_tokens(b);
    d.rope_positions = std::max(b->rope_positions, 1);
    d.rot = l->rotary_dims;
    d.starts = b->starts;
    d.rows = b->rows;
    d.positions = b->positions;
    d.rope = reinterpret_cast<const float2 *>(b->rope);
    return d;
}

// Workgroups along one sequence's tokens of a launch whose kernel goes round: `most` for one that brings
// max_tokens, at `heads` (sequence, head) pairs whose work fills `work` workgroups.  max_tokens is a bound, and a caller
// that does not know better gives the tokens of the whole call: then nearly all of `most` would find nothing
// (256 sequences of 512 tokens ask for 8 M workgroups of 512, 2^32 work-items, which no launch takes).  A batch
// of like lengths stays below 4 * work; the longest of a mixed one goes round.  128 sequences of 512 tokens of
// 32 heads of 64 in bf16: 714 us, without the longest given 785, with all of `most` 7,140.
inline int64_t q4_workgroups(int64_t most, int64_t heads, int64_t work) {
    return std::max<int64_t>(1, std::min(most, std::max<int64_t>(1 << 16, 4 * work) / heads));
}

inline int check_q4_dtype(int dt) { return dt == SWQ_F32 || dt == SWQ_BF16 ? SWQ_OK : SWQ_ERR_UNSUPPORTED_DTYPE; }

inline size_t q4_dtype_bytes(int dt) { return dt == SWQ_F32 ? 4 : 2; }

// The append launch (q4_cache.hip), for callers that have checked their arguments.
void launch_q4_append(const swq_attention_layer *l, const Q4View &c, const Q4Batch &b, const void *k, const void *v,
                      int dtype, hipStream_t s);

// ---- device ----

template <typename T>
__device__ __forceinline__ float q4_load(const T *p, int64_t i) {
    if constexpr (sizeof(T) == 4) return p[i];
    else return bf16_to_f32(p[i]);
}

template <typename T>
__device__ __forceinline__ void q4_store(T *p, int64_t i, float v) {
    if constexpr (sizeof(T) == 4) {
        p[i] = v;
    } else {
        p[i] = v == v ? f32_to_bf16_rne(v) : 0x7FC0;
    }
}

// 8 consecutive numbers, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T *p) {
    if constexpr (sizeof(T) == 4) {
        const float4 u = reinterpret_cast<const float4 *>(p)[0], v = reinterpret_cast<const float4 *>(p)[1];
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            T lo, hi;
            q4_store(&lo, 0, x[2 * i]);
            q4_store(&hi, 0, x[2 * i + 1]);
            w[i] = lo | static_cast<uint32_t>(hi) << 16;
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// cos and sin of dims 8 j .. 8 j + 7 of a row's turns (those below 2 half: the others' are not used).
// 64 bytes in a row where half allows: as 8 pairs the loads took more time than the rest of a query's
// work (4,096 tokens of 32 heads of 128: 28 us, now 21).
__device__ __forceinline__ void q4_turns(float2 (&cs)[8], const float2 *turn, int half, int j) {
    if (half % 8 == 0) {
        const float4 *t4 = reinterpret_cast<const float4 *>(turn + (8 * j < half ? 8 * j : 8 * j - half));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 t = t4[e];
            cs[2 * e] = make_float2(t.x, t.y);
            cs[2 * e + 1] = make_float2(t.z, t.w);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = 8 * j + e;
            cs[e] = turn[d < half ? d : min(d - half, half - 1)];
        }
    }
}

}  // namespace swq
