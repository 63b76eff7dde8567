// Rows into a KV cache held in 4 bits, out of it as values, and the heaviest of them into a
// smaller cache.  The formats are swq.h's (swq_q4_cache).
#include <cmath>

#include "q4_row.hpp"

namespace swq {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWaves = kAppendThreads / kWave;

struct AppendArgs {
    Q4View c;
    Q4Batch b;
    const void *k, *v;
    const float *w;  // k_norm_weight
    float eps;
};

// One workgroup per block of 8 rows, kv head and sequence; a wave takes every fourth row of the
// block.  k words and all scales and biases belong to one row and are written by its wave; a v
// word holds 8 rows of one dim, so the codes meet in LDS, and words of which only some rows are
// new keep the others (the first and last block of a call).
template <int HD, typename T>
__global__ __launch_bounds__(kAppendThreads) void q4_append(const AppendArgs a) {
    constexpr int EPL = HD / kWave;
    __shared__ double s_rot[kAppendWaves][HD];
    __shared__ uint8_t s_v[kQ4Block][HD];
    const int h = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
    const int n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const int r1 = min(r0 + a.b.count(b), a.c.maxp);  // past the last row written
    const int half = a.b.rot / 2;
    uint32_t *kw = a.c.k_head(b, h), *vw = a.c.v_head(b, h);
    _Float16 *par = a.c.par_head(b, h);
    const T *kin = static_cast<const T *>(a.k), *vin = static_cast<const T *>(a.v);
    for (int blk = r0 / kQ4Block + blockIdx.x; blk * kQ4Block < r1; blk += gridDim.x) {
        for (int u = wave; u < kQ4Block; u += kAppendWaves) {
            const int row = blk * kQ4Block + u;
            if (row < r0 || row >= r1) continue;  // the same for the whole wave
            const int64_t at = (static_cast<int64_t>(n0 + row - r0) * a.c.KVH + h) * HD + lane * EPL;
            double x[EPL];
            uint32_t q[EPL];
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[e] = static_cast<double>(q4_load(kin, at + e));
            const float2 *turn = half > 0 ? a.b.rope + static_cast<int64_t>(a.b.position(b, row - r0)) * half : nullptr;
            Q4HeadTable<EPL> tab;
            tab.load(a.w, turn, half);
            q4_key_row<HD>(x, tab, a.eps, half, s_rot[wave], kw, par, a.c.R, row);
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[e] = static_cast<double>(q4_load(vin, at + e));
            q4_value_row<HD>(x, q, par, a.c.R, row);
#pragma unroll
            for (int e = 0; e < EPL; ++e) s_v[u][lane * EPL + e] = static_cast<uint8_t>(q[e]);
        }
        __syncthreads();
        const int u0 = max(r0 - blk * kQ4Block, 0), u1 = min(r1 - blk * kQ4Block, kQ4Block);
        for (int d = tid; d < HD; d += kAppendThreads) {
            uint32_t *p = vw + static_cast<int64_t>(blk) * HD + d;
            uint32_t word = u1 - u0 < kQ4Block ? *p : 0u;
            for (int u = u0; u < u1; ++u) word = (word & ~(15u << (4 * u))) | (static_cast<uint32_t>(s_v[u][d]) << (4 * u));
            *p = word;
        }
        __syncthreads();
    }
}

struct ReadArgs {
    Q4View c;
    const int32_t *first, *starts, *rows;
    int32_t count, B;
    void *k, *v;
};

// A thread per (row, kv head, 8 dims): one k word, and 8 v words of which it takes its row's codes.
template <typename T>
__global__ __launch_bounds__(256) void q4_read(const ReadArgs a) {
    const int b = blockIdx.y;
    const int oct = a.c.hd / 8, per_row = a.c.KVH * oct;
    const int s0 = a.starts ? min(max(a.starts[b], 0), a.count) : 0;
    const int n = a.starts ? max(min(a.starts[b + 1], a.count) - s0, 0) : a.count;
    const int64_t out0 = a.starts ? s0 : static_cast<int64_t>(b) * a.count;
    const int top = a.rows ? min(a.rows[b], a.c.maxp) : a.c.maxp;
    const int first = a.first ? a.first[b] : 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < static_cast<int64_t>(n) * per_row;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int t = static_cast<int>(i / per_row), h = static_cast<int>(i % per_row) / oct, j = static_cast<int>(i % oct);
        const int64_t row = static_cast<int64_t>(first) + t;
        const bool there = row >= 0 && row < top;
        const int64_t at = ((out0 + t) * a.c.KVH + h) * a.c.hd + 8 * j;
        const int ng = a.c.hd / kQ4Group, g = 8 * j / kQ4Group;
        const _Float16 *par = a.c.par_head(b, h) + row;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            T *out = static_cast<T *>(which ? a.v : a.k);
            if (!out) continue;
            float s = 0.f, z = 0.f;
            uint32_t word = 0;
            if (there) {
                s = static_cast<float>(par[(static_cast<int64_t>(2 * which) * ng + g) * a.c.R]);
                z = static_cast<float>(par[(static_cast<int64_t>(2 * which + 1) * ng + g) * a.c.R]);
                if (which) {
                    const uint32_t *p = a.c.v_head(b, h) + (row / 8) * a.c.hd + 8 * j;
#pragma unroll
                    for (int e = 0; e < 8; ++e) word |= ((p[e] >> (4 * (row & 7))) & 15u) << (4 * e);
                } else {
                    word = a.c.k_head(b, h)[row * oct + j];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) q4_store(out, at + e, there ? fmaf(s, static_cast<float>((word >> (4 * e)) & 15u), z) : 0.f);
        }
    }
}

struct EvictArgs {
    Q4View src, dst;
    const float *weights;
    const int32_t *rows;
    float *new_weights;
    int32_t *new_rows, *kept;
    int32_t budget, sink, recent;
};

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;

__device__ __forceinline__ uint32_t weight_key(float w) { return w == w ? orderable(w) : 0u; }

// The rows that one (sequence, kv head) keeps.  The smallest key among the kept of the middle is
// found eight bits at a time from histograms in LDS (their integer counts do not depend on the
// order of the adds), then the rows are numbered in order: those above it, and of those equal to
// it the first `need`.
__global__ __launch_bounds__(kSelectThreads) void q4_select(const EvictArgs a) {
    __shared__ uint32_t s_hist[256];
    __shared__ uint32_t s_wave[2][kSelectWaves];
    __shared__ uint32_t s_pick[2];
    const int h = blockIdx.x % a.src.KVH, b = blockIdx.x / a.src.KVH;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
    const int n = min(max(a.rows[b], 0), a.src.maxp);
    const float *w = a.weights + a.src.head(b, h) * a.src.maxp;
    int32_t *kept = a.kept + a.src.head(b, h) * a.budget;
    float *nw = a.new_weights ? a.new_weights + a.dst.head(b, h) * a.dst.maxp : nullptr;
    const bool all = n <= a.budget;
    const int m0 = all ? n : a.sink, m1 = all ? n : n - a.recent;  // the middle
    uint32_t need = all ? 0 : a.budget - a.sink - a.recent;        // of it, still to be found
    uint32_t key = 0, mask = 0;  // the bits of the border key that are known
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kSelectThreads) s_hist[i] = 0;
            __syncthreads();
            for (int t = m0 + tid; t < m1; t += kSelectThreads) {
                const uint32_t k = weight_key(w[t]);
                if ((k & mask) == key) atomicAdd(&s_hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (wave == 0) {  // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
                uint32_t c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[i] = s_hist[255 - 4 * lane - i];
                    sum += c[i];
                }
                uint32_t upto = sum;
                for (int off = 1; off < kWave; off <<= 1) {
                    const uint32_t o = __shfl_up(upto, off, kWave);
                    if (lane >= off) upto += o;
                }
                uint32_t above = upto - sum;
                if (above < need && upto >= need) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (above < need && above + c[i] >= need) {
                            s_pick[0] = 255 - 4 * lane - i;
                            s_pick[1] = need - above;
                            break;
                        }
                        above += c[i];
                    }
                }
            }
            __syncthreads();
            key |= s_pick[0] << shift;
            mask |= 255u << shift;
            need = s_pick[1];
        }
    }
    uint32_t taken = 0, equal = 0;  // before this tile
    for (int t0 = 0; t0 < n; t0 += kSelectThreads) {
        const int t = t0 + tid;
        const bool here = t < n, mid = here && t >= m0 && t < m1;
        const uint32_t k = mid ? weight_key(w[t]) : 0u;
        const bool eq = mid && need > 0 && k == key;
        const uint64_t eqs = __ballot(eq);
        if (lane == 0) s_wave[0][wave] = __popcll(eqs);
        __syncthreads();
        uint32_t before = equal, all_eq = 0;
        for (int i = 0; i < kSelectWaves; ++i) {
            if (i < wave) before += s_wave[0][i];
            all_eq += s_wave[0][i];
        }
        const uint64_t below = (1ull << lane) - 1;
        const bool take = here && (all || !mid || (need > 0 && (k > key || (eq && before + __popcll(eqs & below) < need))));
        const uint64_t takes = __ballot(take);
        if (lane == 0) s_wave[1][wave] = __popcll(takes);
        __syncthreads();
        uint32_t at = taken, all_take = 0;
        for (int i = 0; i < kSelectWaves; ++i) {
            if (i < wave) at += s_wave[1][i];
            all_take += s_wave[1][i];
        }
        at += __popcll(takes & below);
        if (take && at < static_cast<uint32_t>(a.budget)) {
            kept[at] = t;
            if (nw) nw[at] = w[t];
        }
        taken += all_take;
        equal += all_eq;
    }
    const int have = min(n, a.budget);
    for (int i = have + tid; i < a.budget; i += kSelectThreads) kept[i] = -1;
    if (nw)
        for (int i = have + tid; i < a.dst.maxp; i += kSelectThreads) nw[i] = 0.f;
    if (h == 0 && tid == 0) a.new_rows[b] = have;
}

// Their codes, scales and biases into the other cache, a workgroup per 8 rows of it and kv head.
template <int HD>
__global__ __launch_bounds__(256) void q4_gather(const EvictArgs a) {
    constexpr int NG = HD / kQ4Group, W = HD / 8;
    __shared__ int s_row[kQ4Block];
    const int h = blockIdx.y % a.src.KVH, b = blockIdx.y / a.src.KVH, tid = threadIdx.x;
    const int have = min(min(max(a.rows[b], 0), a.src.maxp), a.budget);
    const int32_t *kept = a.kept + a.src.head(b, h) * a.budget;
    const uint32_t *sk = a.src.k_head(b, h), *sv = a.src.v_head(b, h);
    uint32_t *dk = a.dst.k_head(b, h), *dv = a.dst.v_head(b, h);
    const _Float16 *sp = a.src.par_head(b, h);
    _Float16 *dp = a.dst.par_head(b, h);
    for (int blk = blockIdx.x; blk * kQ4Block < have; blk += gridDim.x) {
        const int j0 = blk * kQ4Block, n = min(kQ4Block, have - j0);
        if (tid < kQ4Block) s_row[tid] = tid < n ? min(max(kept[j0 + tid], 0), a.src.maxp - 1) : 0;
        __syncthreads();
        for (int i = tid; i < n * W; i += 256)
            dk[static_cast<int64_t>(j0) * W + i] = sk[static_cast<int64_t>(s_row[i / W]) * W + i % W];
        for (int i = tid; i < 4 * NG * n; i += 256) {
            const int64_t line = static_cast<int64_t>(i / n);
            dp[line * a.dst.R + j0 + i % n] = sp[line * a.src.R + s_row[i % n]];
        }
        for (int d = tid; d < HD; d += 256) {
            uint32_t word = 0;
            for (int u = 0; u < n; ++u) {
                const int r = s_row[u];
                word |= ((sv[static_cast<int64_t>(r / 8) * HD + d] >> (4 * (r & 7))) & 15u) << (4 * u);
            }
            dv[static_cast<int64_t>(blk) * HD + d] = word;
        }
        __syncthreads();
    }
}

template <typename T>
void append_typed(const AppendArgs &a, dim3 grid, hipStream_t s) {
    const dim3 block(kAppendThreads);
    switch (a.c.hd) {
        case 64: hipLaunchKernelGGL((q4_append<64, T>), grid, block, 0, s, a); break;
        case 128: hipLaunchKernelGGL((q4_append<128, T>), grid, block, 0, s, a); break;
        default: hipLaunchKernelGGL((q4_append<256, T>), grid, block, 0, s, a); break;
    }
}

}  // namespace

void launch_q4_append(const swq_attention_layer *l, const Q4View &c, const Q4Batch &b, const void *k, const void *v,
                      int dtype, hipStream_t s) {
    const AppendArgs a{c, b, k, v, l->k_norm_weight, l->norm_eps};
    // blocks that a sequence's tokens can touch: one more than they fill where the first row is
    // inside a block; a sequence that brings more goes round
    const dim3 grid((b.max_tokens + kQ4Block - 1) / kQ4Block + (b.max_tokens > 1), static_cast<uint32_t>(b.B) * c.KVH);
    if (dtype == SWQ_F32) append_typed<float>(a, grid, s);
    else append_typed<uint16_t>(a, grid, s);
}

}  // namespace swq

using namespace swq;

extern "C" size_t swq_q4_cache_bytes(int sequences, int num_kv_heads, int head_dim, int max_positions) {
    if (check_q4_shape(sequences, num_kv_heads, head_dim, max_positions) != SWQ_OK) return 0;
    return q4_layout(sequences, num_kv_heads, head_dim, max_positions).total;
}

extern "C" int swq_q4_rope_table(int rotary_dims, float rope_theta, int64_t first, int count, float *out) {
    if (rotary_dims <= 0 || rotary_dims % 2 != 0) return SWQ_ERR_BAD_SHAPE;
    if (!(rope_theta > 0.f) || first < 0 || first > (1LL << 31) || count <= 0 || !out) return SWQ_ERR_INVALID_ARGUMENT;
    const int half = rotary_dims / 2;
    for (int j = 0; j < half; ++j) {
        // the operands' roundings are swq_attention_step's
        const float ex = -static_cast<float>(2 * j) / static_cast<float>(rotary_dims);
        const float inv_freq = static_cast<float>(std::pow(static_cast<double>(rope_theta), static_cast<double>(ex)));
        for (int i = 0; i < count; ++i) {
            const float ang = static_cast<float>(first + i) * inv_freq;
            float *o = out + (static_cast<int64_t>(i) * half + j) * 2;
            o[0] = static_cast<float>(std::cos(static_cast<double>(ang)));
            o[1] = static_cast<float>(std::sin(static_cast<double>(ang)));
        }
    }
    return SWQ_OK;
}

extern "C" int swq_q4_append(const swq_attention_layer *layer, const swq_q4_cache *cache, const swq_q4_batch *batch,
                             const void *k_proj, const void *v_proj, int dtype, void *stream) {
    int st = check_q4_batch(layer, cache, batch);
    if (st == SWQ_OK) st = check_q4_dtype(dtype);
    if (st != SWQ_OK) return st;
    if (batch->tokens == 0) return SWQ_OK;
    if (!k_proj || !v_proj) return SWQ_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(k_proj) % 16 || reinterpret_cast<uintptr_t>(v_proj) % 16)
        return SWQ_ERR_MISALIGNED;
    launch_q4_append(layer, q4_view(cache), q4_batch(layer, batch), k_proj, v_proj, dtype, static_cast<hipStream_t>(stream));
    return launch_status();
}

extern "C" int swq_q4_read(const swq_q4_cache *cache, int sequences, const int32_t *first, const int32_t *starts,
                           const int32_t *rows, int count, void *k, void *v, int dtype, void *stream) {
    int st = check_q4_cache(cache);
    if (st == SWQ_OK) st = check_q4_dtype(dtype);
    if (st != SWQ_OK) return st;
    if (sequences <= 0 || count < 0 || (!k && !v)) return SWQ_ERR_INVALID_ARGUMENT;
    if (sequences > cache->sequences) return SWQ_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16)
        return SWQ_ERR_MISALIGNED;
    if (count == 0) return SWQ_OK;
    const ReadArgs a{q4_view(cache), first, starts, rows, count, sequences, k, v};
    const int64_t items = static_cast<int64_t>(count) * cache->num_kv_heads * (cache->head_dim / 8);
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>((items + 255) / 256, 4096)), sequences);
    if (dtype == SWQ_F32) hipLaunchKernelGGL(q4_read<float>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    else hipLaunchKernelGGL(q4_read<uint16_t>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return launch_status();
}

extern "C" int swq_q4_evict(const swq_q4_cache *src, int sequences, const float *weights, const int32_t *rows,
                            const swq_q4_cache *dst, int budget, int sink, int recent, float *new_weights,
                            int32_t *new_rows, int32_t *kept, void *stream) {
    int st = check_q4_cache(src);
    if (st == SWQ_OK) st = check_q4_cache(dst);
    if (st != SWQ_OK) return st;
    if (sequences <= 0 || budget <= 0 || sink < 0 || recent < 0 || !weights || !rows || !new_rows || !kept)
        return SWQ_ERR_INVALID_ARGUMENT;
    if (sequences > src->sequences || sequences > dst->sequences || src->num_kv_heads != dst->num_kv_heads ||
        src->head_dim != dst->head_dim || static_cast<int64_t>(sink) + recent > budget)
        return SWQ_ERR_BAD_SHAPE;
    if (budget > dst->max_positions) return SWQ_ERR_LIMIT;
    const uint8_t *s0 = static_cast<const uint8_t *>(src->data), *d0 = static_cast<const uint8_t *>(dst->data);
    const size_t sn = q4_layout(src->sequences, src->num_kv_heads, src->head_dim, src->max_positions).total;
    const size_t dn = q4_layout(dst->sequences, dst->num_kv_heads, dst->head_dim, dst->max_positions).total;
    if ((s0 < d0 + dn && d0 < s0 + sn) || weights == new_weights || rows == new_rows) return SWQ_ERR_INVALID_ARGUMENT;
    const EvictArgs a{q4_view(src), q4_view(dst), weights, rows, new_weights, new_rows, kept, budget, sink, recent};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t heads = static_cast<uint32_t>(sequences) * src->num_kv_heads;
    hipLaunchKernelGGL(q4_select, dim3(heads), dim3(kSelectThreads), 0, s, a);
    const dim3 grid((budget + kQ4Block - 1) / kQ4Block, heads);
    switch (src->head_dim) {
        case 64: hipLaunchKernelGGL(q4_gather<64>, grid, dim3(256), 0, s, a); break;
        case 128: hipLaunchKernelGGL(q4_gather<128>, grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL(q4_gather<256>, grid, dim3(256), 0, s, a); break;
    }
    return launch_status();
}
