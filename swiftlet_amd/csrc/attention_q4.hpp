// What the launches of swq_attention_q4 share: arguments, a query head's norm and rotation, and
// the way 4-bit codes, scales and f32 numbers meet on the f16 matrix cores without losing bits.
//
//   codes   become f16 integers: nibbles 0 and 4 of a word or-ed into the f16 number 1024 and 1024
//           taken off again, nibbles 1 and 5 likewise but 16 times as large (they need no shift),
//           nibbles 2, 3, 6 and 7 the same after one shift: 9 operations for 8 codes.  The other
//           operand has 1/16 at the odd nibbles.  (Left as they lie, codes are f16 numbers below
//           the normal ones: 5 operations, but the matrix cores add their products with the
//           leading zeros of the mantissa, and outputs were off by 1.8e-5 where now by 1e-6.)
//   f32     operands (queries; p times a value scale) are two f16 numbers, high and low part, of
//           22 bits together; products with codes are exact, sums f32.  A power of two per head
//           (queries) or per wave (p * scale) keeps them inside f16's range.
//   scales  of keys multiply a group's sum of products, those of values p; biases meet the sum of
//           the queries' dims of a group, and p, on the VALU.
#pragma once

#include "q4_row.hpp"

namespace swq {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

struct AttnQ4Args {
    Q4View c;
    Q4Batch b;
    const void *q, *k, *v;
    const float *q_norm_w, *k_norm_w;
    void *out;
    float *weights;
    int32_t H, group;
    int32_t in_f32, out_f32;  // types of q, k, v and of out: f32, else bf16
    float eps, scale2;        // scale2: 1/sqrt(hd) * log2(e)
    // the cached rows in splits of `per`, and their partial results, by [row of out][split]: for
    // single tokens rows are (sequence, query head), for prompts (token, query head)
    int32_t per, splits;
    float *part;    // [rows][splits][hd]
    float2 *ml;     // [rows][splits]: reference exponent and sum
    float *scores;  // single tokens: [B][H][R] in units of log2, for the gathered weights
    // prompts
    int32_t planes_q, planes_v;  // f16 parts of queries and keys, and of p and values
    int32_t tiles, rows_per;     // tiles of (token, head) rows that are started, rows of one
    int32_t gparts;              // parts of the queries in the gathered weights
    void *qh, *ql;               // [N][H][hd] f16: queries, high and low part; qh NULL: not made
    float *qf;                   // [N][H]: what turns a product of them into log2 units
    void *qs;                    // [N][H][16] f16: sums of their groups as three parts, or NULL
    uint32_t *vmax;              // [B][KVH][2]: bits of the largest key and value, or NULL
    float *lse;                  // [N][H]: log2 of the sum of exponentials, or NULL
    float *gpart;                // [B][KVH][gparts][R]
};

__device__ __forceinline__ f4_t mfma16(h8_t a, h8_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The 8 codes of a word as operand: elements 0 .. 7 are nibbles 0 4 1 5 2 6 3 7, those of odd
// nibbles times 16.  magic: two f16 1024, which the caller keeps in a vector register so that
// masking and or-ing take one operation (kept_1024).
__device__ __forceinline__ uint32_t kept_1024() {
    uint32_t m = 0x64006400u;
    asm volatile("" : "+v"(m));
    return m;
}

__device__ __forceinline__ h8_t q4_operand(uint32_t w, uint32_t magic) {
    constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;
    const uint32_t s = w >> 8;
    const h2_t off = {static_cast<_Float16>(-1024.f), static_cast<_Float16>(-1024.f)};
    const h2_t a = __builtin_bit_cast(h2_t, (w & kEven) | magic) + off, b = __builtin_bit_cast(h2_t, (w & kOdd) | magic) + off;
    const h2_t c = __builtin_bit_cast(h2_t, (s & kEven) | magic) + off, d = __builtin_bit_cast(h2_t, (s & kOdd) | magic) + off;
    return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The same with codes about zero: 8 off those of even nibbles, 7 (times 16) off those of odd ones.  Sums of p * scale *
// code over rows then are of either sign, as the outputs are; with codes from 0 they grow with the rows, and so
// does what is left of their rounding once the biases are taken off (33,000 rows in a split: 9e-5 of the largest output,
// so 7e-7).  8 and 7 by turns, because their mean is the codes' and neither costs an operation.
constexpr float kQ4Even = 8.f, kQ4Odd = 7.f;
__device__ __forceinline__ h8_t q4_operand_signed(uint32_t w, uint32_t magic) {
    constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;
    const uint32_t s = w >> 8;
    const _Float16 e = static_cast<_Float16>(-1024.f - kQ4Even), o = static_cast<_Float16>(-1024.f - 16.f * kQ4Odd);
    const h2_t even = {e, e}, odd = {o, o};
    const h2_t a = __builtin_bit_cast(h2_t, (w & kEven) | magic) + even, b = __builtin_bit_cast(h2_t, (w & kOdd) | magic) + odd;
    const h2_t c = __builtin_bit_cast(h2_t, (s & kEven) | magic) + even, d = __builtin_bit_cast(h2_t, (s & kOdd) | magic) + odd;
    return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The same as q4_operand with 1024 added to each element.
__device__ __forceinline__ h8_t q4_operand_1024(uint32_t w, uint32_t magic) {
    constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;
    const uint32_t s = w >> 8;
    const uint4 u = make_uint4((w & kEven) | magic, (w & kOdd) | magic, (s & kEven) | magic, (s & kOdd) | magic);
    return __builtin_bit_cast(h8_t, u);
}

// Operand element of a nibble, and the nibble of an element.
__device__ __forceinline__ constexpr int q4_element(int nibble) { return nibble < 4 ? 2 * nibble : 2 * nibble - 7; }
__device__ __forceinline__ constexpr int q4_nibble(int element) { return element / 2 + 4 * (element & 1); }

// x = hi + lo with hi, lo f16.
__device__ __forceinline__ void split_f16(f32x2_t x, h2_t &hi, h2_t &lo) {
    hi = __builtin_convertvector(x, h2_t);
    // one mixed-precision fma each
    const f32x2_t rest = {fmaf(static_cast<float>(hi.x), -1.0f, x.x), fmaf(static_cast<float>(hi.y), -1.0f, x.y)};
    lo = __builtin_convertvector(rest, h2_t);
}

__device__ __forceinline__ float q4_load_any(const void *p, int64_t i, int is_f32) {
    return is_f32 ? static_cast<const float *>(p)[i] : bf16_to_f32(static_cast<const uint16_t *>(p)[i]);
}

__device__ __forceinline__ void q4_store_any(void *p, int64_t i, float v, int is_f32) {
    if (is_f32) q4_store(static_cast<float *>(p), i, v);
    else q4_store(static_cast<uint16_t *>(p), i, v);
}

__device__ __forceinline__ float q4_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Off by two units in the last place at most: expf, a sum and the hardware's reciprocal.
__device__ __forceinline__ float sigmoid_exact(float v) { return __builtin_amdgcn_rcpf(1.0f + expf(-v)); }

// Sum and maximum over L consecutive lanes (8, 16 or 32), to each of them.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp<0xB1, 0xF, true>(v);
    v += dpp<0x4E, 0xF, true>(v);
    v += dpp<0x141, 0xF, true>(v);
    if constexpr (L >= 16) v += dpp<0x140, 0xF, true>(v);
    if constexpr (L >= 32) v += __shfl_xor(v, 16, kWave);
    return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, dpp<0xB1, 0xF, true>(v));
    v = fmaxf(v, dpp<0x4E, 0xF, true>(v));
    v = fmaxf(v, dpp<0x141, 0xF, true>(v));
    if constexpr (L >= 16) v = fmaxf(v, dpp<0x140, 0xF, true>(v));
    if constexpr (L >= 32) v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return v;
}

// Four dims times the sigmoids of four bf16 gates, as bf16: the hardware's exponential and reciprocal,
// off by 2^-21, and its conversion to the nearest bf16 (a NaN stays one).
__device__ __forceinline__ uint2 gated_bf16(uint2 g, f4_t v) {
    typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
    const f4_t x = {__uint_as_float(g.x << 16), __uint_as_float(g.x & 0xFFFF0000u), __uint_as_float(g.y << 16), __uint_as_float(g.y & 0xFFFF0000u)};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= __builtin_amdgcn_rcpf(1.0f + q4_exp2(x[e] * -1.44269504f));
    return __builtin_bit_cast(uint2, __builtin_convertvector(v, b4_t));
}

// Four dims, attention * sigmoid(gate), at element `out` of the output; gate: of q_proj.
__device__ __forceinline__ void store_gated(const AttnQ4Args &a, int64_t out, int64_t gate, f4_t v) {
    if (a.in_f32) {
        const float4 g = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + gate);
        v *= f4_t{sigmoid_exact(g.x), sigmoid_exact(g.y), sigmoid_exact(g.z), sigmoid_exact(g.w)};
    } else {
        const uint2 g = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.q) + gate);
        v *= f4_t{sigmoid_exact(__uint_as_float(g.x << 16)), sigmoid_exact(__uint_as_float(g.x & 0xFFFF0000u)),
                  sigmoid_exact(__uint_as_float(g.y << 16)), sigmoid_exact(__uint_as_float(g.y & 0xFFFF0000u))};
    }
    if (a.out_f32) {
        *reinterpret_cast<f4_t *>(static_cast<float *>(a.out) + out) = v;
    } else {
        uint16_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q4_store(u, e, v[e]);
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + out) =
            make_uint2(u[0] | static_cast<uint32_t>(u[1]) << 16, u[2] | static_cast<uint32_t>(u[3]) << 16);
    }
}

// Single tokens (attention_q4_step.hip): a split of max_rows rows over workgroups, and its launches.
struct Q4StepPlan {
    int per, splits;
};
Q4StepPlan plan_q4_step(int64_t rows, int64_t heads, int hd);
int64_t most_q4_head_splits(int64_t rows, int64_t heads, int hd);  // heads * splits, of any number of rows and heads up to these
void launch_q4_step(const AttnQ4Args &a, hipStream_t s);

// Several tokens (attention_q4_prefill.hip): how the launches are cut for sequences of up to
// max_tokens tokens and `rows` rows, `all` (token, query head) rows of the batch.  Splits are made where
// tiles of 64 or 128 rows are fewer than 512: all * splits stays below 512 * 128 + all, which the
// workspace has room for; a batch that is padded a lot has fewer splits.
constexpr int kQ4PrefillMaxSplits = 32;
constexpr int64_t kQ4PartRows = 512 * 128;
constexpr int kQ4GatherMaxParts = 32;
constexpr int64_t kQ4GatherMost = 4 << 20;  // numbers of all parts' sums
struct Q4PrefillPlan {
    int planes_q, planes_v, rows_per, tiles, per, splits, gparts;
    bool prepares;  // queries in the attention's own launch
};
Q4PrefillPlan plan_q4_prefill(int64_t max_tokens, int64_t all, int64_t rows, int64_t heads, int group, int hd, int rot, int maxp, bool f32, bool weights);
void launch_q4_prefill(const AttnQ4Args &a, hipStream_t s);

}  // namespace swq
