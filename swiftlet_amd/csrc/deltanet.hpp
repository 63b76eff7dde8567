// What the gated DeltaNet launches share: where a token's projections lie, the checks of a layer, and the view of
// the tokens of many sequences that swq_deltanet_tokens hands its kernels.
#pragma once

#include "internal.hpp"

namespace swq {

constexpr int kDnMaxDv = 1024;
constexpr int kDnMaxConv = 8;

__device__ __forceinline__ float sigmoid_acc(float v) { return 1.0f / (1.0f + expf(-v)); }
__device__ __forceinline__ float silu_acc(float v) { return v * sigmoid_acc(v); }
// softplus as log1p(exp(.)) below 20
__device__ __forceinline__ float softplus_acc(float v) { return v > 20.f ? v : log1pf(expf(v)); }

// Element of a token's qkvz row that holds mixed channel c ([q | k | v] order).
template <typename A>
__device__ __forceinline__ int mixed_at(const A &a, int c) {
    if (a.layout == SWQ_DELTA_SPLIT) return c;
    const int chunk = 2 * a.dk + 2 * a.rep * a.dv;
    if (c < a.keyD) return (c / a.dk) * chunk + c % a.dk;
    if (c < 2 * a.keyD) {
        const int t = c - a.keyD;
        return (t / a.dk) * chunk + a.dk + t % a.dk;
    }
    const int t = c - 2 * a.keyD, hv = t / a.dv, i = t % a.dv;
    return (hv / a.rep) * chunk + 2 * a.dk + (hv % a.rep) * a.dv + i;
}

// Element of the same row that holds z[hv][i].
template <typename A>
__device__ __forceinline__ int z_at(const A &a, int hv, int i) {
    if (a.layout == SWQ_DELTA_SPLIT) return a.convD + hv * a.dv + i;
    const int chunk = 2 * a.dk + 2 * a.rep * a.dv;
    return (hv / a.rep) * chunk + 2 * a.dk + a.rep * a.dv + (hv % a.rep) * a.dv + i;
}

// Element of the ba row that holds b (which = 0) or a (which = 1) of value head hv.
template <typename A>
__device__ __forceinline__ int ba_at(const A &a, int hv, int which) {
    if (a.layout == SWQ_DELTA_SPLIT) return which * a.nv + hv;
    return (hv / a.rep) * 2 * a.rep + which * a.rep + hv % a.rep;
}

// Projections and outputs are f32 or bf16.
__device__ __forceinline__ float dn_load(const float *p, int64_t i) { return p[i]; }
__device__ __forceinline__ float dn_load(const uint16_t *p, int64_t i) { return bf16_to_f32(p[i]); }
__device__ __forceinline__ uint16_t dn_bf16(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));  // to the nearest; a NaN stays one
}
__device__ __forceinline__ void dn_store_as(void *p, int is_f32, int64_t i, float v) {
    if (is_f32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = dn_bf16(v);
}

constexpr int kCus = 256;

// A layer and the tokens of one swq_deltanet_tokens call.  What comes from device memory is clamped where it is
// read, so that no value of it leads out of a buffer.
struct DnTokens {
    const void *qkvz, *ba;
    int64_t qkvz_stride, ba_stride;  // elements from one token's row to the next
    const float *conv_w, *a_log, *dt_bias, *norm_w;
    uint8_t *states;
    int64_t slot_bytes, rec_at;  // bytes of a slot, and from its start to the recurrent state
    void *out;                   // [N][nv * dv]
    const int32_t *starts, *positions, *slot;
    int32_t B, N, max_tokens, slots;
    int32_t least, most;         // tokens of the sequences that a launch takes
    int32_t nk, nv, dk, dv, K, layout, rep, keyD, convD;
    int32_t out_f32;
    float eps;

    __device__ __forceinline__ int first(int b) const { return starts ? min(max(starts[b], 0), N) : b * max_tokens; }
    // Tokens of sequence b, 0 if the launch does not take it.
    __device__ __forceinline__ int count(int b) const {
        const int n = starts ? min(max(min(starts[b + 1], N) - first(b), 0), max_tokens) : max_tokens;
        return n >= least && n <= most ? n : 0;
    }
    // The sequence's state, or null for one that is left out.
    __device__ __forceinline__ uint8_t *state(int b) const {
        const int s = slot ? slot[b] : b;
        return s >= 0 && s < slots ? states + s * slot_bytes : nullptr;
    }
    __device__ __forceinline__ uint32_t position(int b) const { return static_cast<uint32_t>(max(positions[b], 0)); }
};

inline size_t dn_align(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// Prompts, a chunk of tokens at a time (deltanet_chunks.hip): which heads are taken, the workspace of a call, its
// launches.
constexpr int kDnChunk = 64;
bool deltanet_chunks_take(const swq_deltanet_layer *l);
bool deltanet_chunks_fit(const swq_deltanet_layer *l, int64_t sequences, int64_t tokens);  // launches of fewer than 2^32 work-items
size_t deltanet_chunks_bytes(const swq_deltanet_layer *l, int64_t sequences, int64_t tokens);
void launch_deltanet_chunks(const DnTokens &a, bool in_f32, void *ws, hipStream_t s);

int check_deltanet_layer(const swq_deltanet_layer *l);
size_t deltanet_ring_bytes(const swq_deltanet_layer *l);

}  // namespace swq
