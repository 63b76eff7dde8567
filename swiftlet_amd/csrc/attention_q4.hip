// Gated GQA attention over a KV cache held in 4 bits: many tokens of many sequences, causal after
// the rows that are there, with the attention that each row gathers if asked for.
#include <cmath>

#include "attention_q4.hpp"

namespace swq {
namespace {

constexpr int kRowTile = 256;  // rows of one softmax step, and threads

// One wave per (token, query head): q / rms * w, turned by the table.
template <int HD, typename T>
__global__ __launch_bounds__(256) void q4_queries(const AttnQ4Args a) {
    constexpr int EPL = HD / kWave;
    __shared__ float s_rot[4][HD];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    const int b = blockIdx.y, cnt = a.b.count(b);
    if (item >= static_cast<int64_t>(cnt) * a.H) return;
    const int i = static_cast<int>(item / a.H), h = static_cast<int>(item % a.H);
    const int64_t n = a.b.first(b) + i;
    const T *q = static_cast<const T *>(a.q) + (n * a.H + h) * 2 * HD + lane * EPL;
    float x[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = q4_load(q, e);
    const int half = a.b.rot / 2;
    Q4HeadTable<EPL> tab;
    tab.load(a.q_norm_w, half > 0 ? a.b.rope + static_cast<int64_t>(a.b.position(b, i)) * half : nullptr, half);
    q4_norm_rope<EPL>(x, tab, a.eps, half, s_rot[wave]);
#pragma unroll
    for (int e = 0; e < EPL; ++e) a.qn[(n * a.H + h) * HD + lane * EPL + e] = x[e];
}

template <int HD>
__device__ __forceinline__ float q4_score(const Q4View &c, const uint32_t *kw, const _Float16 *par, int row, const float *q) {
    constexpr int NG = HD / kQ4Group;
    float s = 0.f;
    for (int g = 0; g < NG; ++g) {
        const float sc = static_cast<float>(par[(static_cast<int64_t>(kQ4KScale) * NG + g) * c.R + row]);
        const float z = static_cast<float>(par[(static_cast<int64_t>(kQ4KBias) * NG + g) * c.R + row]);
        for (int j = 0; j < 8; ++j) {
            const uint32_t w = kw[static_cast<int64_t>(row) * (HD / 8) + 8 * g + j];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += fmaf(sc, static_cast<float>((w >> (4 * e)) & 15u), z) * q[64 * g + 8 * j + e];
        }
    }
    return s;
}

// One workgroup per (token, query head): a thread per row for the scores, then per dim for the
// values, with an online softmax from step to step.
template <int HD, typename T, typename O>
__global__ __launch_bounds__(kRowTile) void q4_attend(const AttnQ4Args a) {
    constexpr int NG = HD / kQ4Group;
    __shared__ float s_q[HD], s_p[kRowTile], s_red[2][4];
    const int h = blockIdx.y % a.H, b = blockIdx.y / a.H, kvh = h / a.group, tid = threadIdx.x;
    const int wave = tid / kWave, lane = tid & (kWave - 1);
    const int cnt = a.b.count(b), n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const uint32_t *kw = a.c.k_head(b, kvh), *vw = a.c.v_head(b, kvh);
    const _Float16 *par = a.c.par_head(b, kvh);
    for (int i = blockIdx.x; i < cnt; i += gridDim.x) {
        const int64_t n = n0 + i;
        const int rows = static_cast<int>(min(static_cast<int64_t>(r0) + i + 1, static_cast<int64_t>(a.c.maxp)));
        __syncthreads();
        for (int d = tid; d < HD; d += kRowTile) s_q[d] = a.qn[(n * a.H + h) * HD + d];
        float m = -INFINITY, l = 0.f, acc = 0.f;
        for (int t0 = 0; t0 < rows; t0 += kRowTile) {
            __syncthreads();
            const int row = t0 + tid;
            float s = row < rows ? q4_score<HD>(a.c, kw, par, row, s_q) * a.scale : -INFINITY;
            const float wm = wave_max_all(s);
            if (lane == 0) s_red[0][wave] = wm;
            __syncthreads();
            const float mn = fmaxf(fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3])), m);
            const float alpha = expf(m - mn);
            m = mn;
            const float p = row < rows ? expf(s - mn) : 0.f;
            s_p[tid] = p;
            const float ws = wave_sum(p);
            if (lane == 0) s_red[1][wave] = ws;
            __syncthreads();
            l = l * alpha + (s_red[1][0] + s_red[1][1] + s_red[1][2] + s_red[1][3]);
            acc *= alpha;
            if (tid < HD) {
                const int top = min(kRowTile, rows - t0);
                float add = 0.f;
                for (int u = 0; u < top; ++u) {
                    const int r = t0 + u;
                    const float sc = static_cast<float>(par[(static_cast<int64_t>(kQ4VScale) * NG + tid / kQ4Group) * a.c.R + r]);
                    const float z = static_cast<float>(par[(static_cast<int64_t>(kQ4VBias) * NG + tid / kQ4Group) * a.c.R + r]);
                    const uint32_t w = vw[static_cast<int64_t>(r / 8) * HD + tid];
                    add = fmaf(s_p[u], fmaf(sc, static_cast<float>((w >> (4 * (r & 7))) & 15u), z), add);
                }
                acc += add;
            }
        }
        if (tid < HD) {
            const float gate = q4_load(static_cast<const T *>(a.q), ((n * a.H + h) * 2 + 1) * HD + tid);
            const float o = rows > 0 ? acc / l : 0.f;
            q4_store(static_cast<O *>(a.out), (n * a.H + h) * HD + tid, o * (1.0f / (1.0f + expf(-gate))));
        }
        if (tid == 0) a.lse[n * a.H + h] = m + logf(l);
    }
}

// A thread per row of one kv head: the attention of every token and head that sees it.
template <int HD>
__global__ __launch_bounds__(256) void q4_gathered(const AttnQ4Args a) {
    const int kvh = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH;
    const int cnt = a.b.count(b), n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const int top = static_cast<int>(min(static_cast<int64_t>(r0) + cnt, static_cast<int64_t>(a.c.maxp)));
    const uint32_t *kw = a.c.k_head(b, kvh);
    const _Float16 *par = a.c.par_head(b, kvh);
    if (cnt <= 0) return;
    for (int row = blockIdx.x * 256 + threadIdx.x; row < top; row += gridDim.x * 256) {
        float sum = 0.f;
        for (int i = max(row - r0, 0); i < cnt; ++i)
            for (int u = 0; u < a.group; ++u) {
                const int64_t at = static_cast<int64_t>(n0 + i) * a.H + kvh * a.group + u;
                sum += expf(q4_score<HD>(a.c, kw, par, row, a.qn + at * HD) * a.scale - a.lse[at]);
            }
        float *w = a.weights + a.c.head(b, kvh) * a.c.maxp + row;
        *w = row < r0 ? *w + sum : sum;
    }
}

template <int HD, typename T>
void launch_typed(const AttnQ4Args &a, int out_dtype, hipStream_t s) {
    const dim3 block(256);
    const int64_t items = static_cast<int64_t>(a.b.max_tokens) * a.H;
    hipLaunchKernelGGL((q4_queries<HD, T>), dim3(static_cast<uint32_t>((items + 3) / 4), a.b.B), block, 0, s, a);
    const dim3 grid(std::min(a.b.max_tokens, 65535), static_cast<uint32_t>(a.b.B) * a.H);
    if (out_dtype == SWQ_F32) hipLaunchKernelGGL((q4_attend<HD, T, float>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((q4_attend<HD, T, uint16_t>), grid, block, 0, s, a);
    if (a.weights)
        hipLaunchKernelGGL(q4_gathered<HD>, dim3((a.c.maxp + 255) / 256, static_cast<uint32_t>(a.b.B) * a.c.KVH), block, 0, s, a);
}

template <int HD>
void launch(const AttnQ4Args &a, int dtype, int out_dtype, hipStream_t s) {
    if (dtype == SWQ_F32) launch_typed<HD, float>(a, out_dtype, s);
    else launch_typed<HD, uint16_t>(a, out_dtype, s);
}

}  // namespace
}  // namespace swq

using namespace swq;

namespace {

struct StepParts {
    size_t part, ml, scores, total;
};

StepParts step_parts(const swq_attention_layer *l, const swq_q4_cache *c, int sequences, int splits, bool weights) {
    const size_t heads = static_cast<size_t>(sequences) * l->num_heads;
    StepParts p{};
    p.part = q4_align(heads * splits * l->head_dim * sizeof(float));
    p.ml = q4_align(heads * splits * sizeof(float2));
    p.scores = weights ? q4_align(heads * q4_rows(c->max_positions) * sizeof(float)) : 0;
    p.total = p.part + p.ml + p.scores;
    return p;
}

size_t q4_step_workspace(const swq_attention_layer *l, const swq_q4_cache *c, const swq_q4_batch *b, int weights) {
    return step_parts(l, c, b->sequences, most_q4_splits(c->max_positions, static_cast<int64_t>(b->sequences) * c->num_kv_heads, c->head_dim), weights != 0).total;
}

size_t q4_prompt_workspace(const swq_attention_layer *l, const swq_q4_batch *b) {
    const size_t rows = static_cast<size_t>(std::max(b->tokens, 1)) * l->num_heads;
    return q4_align(rows * l->head_dim * sizeof(float)) + q4_align(rows * sizeof(float));
}

}  // namespace

extern "C" size_t swq_attention_q4_workspace_bytes(const swq_attention_layer *layer, const swq_q4_cache *cache,
                                                   const swq_q4_batch *batch, int weights) {
    if (check_q4_layer(layer) != SWQ_OK || !cache ||
        check_q4_shape(cache->sequences, cache->num_kv_heads, cache->head_dim, cache->max_positions) != SWQ_OK ||
        check_q4_sizes(cache, batch) != SWQ_OK || layer->head_dim != cache->head_dim ||
        layer->num_kv_heads != cache->num_kv_heads)
        return 0;
    return std::max(q4_step_workspace(layer, cache, batch, weights), q4_prompt_workspace(layer, batch));
}

extern "C" int swq_attention_q4(const swq_attention_layer *layer, const swq_q4_cache *cache, const swq_q4_batch *batch,
                                const void *q_proj, const void *k_proj, const void *v_proj, int dtype, float *weights,
                                void *out, int out_dtype, void *ws, size_t ws_bytes, void *stream) {
    int st = check_q4_batch(layer, cache, batch);
    if (st == SWQ_OK) st = check_q4_dtype(dtype);
    if (st == SWQ_OK) st = check_q4_dtype(out_dtype);
    if (st != SWQ_OK) return st;
    if (static_cast<int64_t>(batch->sequences) * layer->num_heads > 65535) return SWQ_ERR_LIMIT;
    if (batch->tokens == 0) return SWQ_OK;
    if (!q_proj || !out || !k_proj != !v_proj) return SWQ_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(q_proj) % 16 || reinterpret_cast<uintptr_t>(k_proj) % 16 ||
        reinterpret_cast<uintptr_t>(v_proj) % 16 || reinterpret_cast<uintptr_t>(out) % 16 ||
        reinterpret_cast<uintptr_t>(layer->q_norm_weight) % 16 ||
        reinterpret_cast<uintptr_t>(weights) % 4 || reinterpret_cast<uintptr_t>(ws) % 256)
        return SWQ_ERR_MISALIGNED;
    if (!ws || ws_bytes < swq_attention_q4_workspace_bytes(layer, cache, batch, weights != nullptr)) return SWQ_ERR_WORKSPACE;
    AttnQ4Args a{};
    a.c = q4_view(cache);
    a.b = q4_batch(layer, batch);
    a.q = q_proj;
    a.k = k_proj;
    a.v = v_proj;
    a.k_norm_w = layer->k_norm_weight;
    a.in_f32 = dtype == SWQ_F32;
    a.out_f32 = out_dtype == SWQ_F32;
    a.q_norm_w = layer->q_norm_weight;
    a.out = out;
    a.weights = weights;
    a.H = layer->num_heads;
    a.group = a.H / a.c.KVH;
    a.eps = layer->norm_eps;
    a.scale = 1.0f / std::sqrt(static_cast<float>(a.c.hd));
    a.scale2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(a.c.hd)));
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint8_t *p = static_cast<uint8_t *>(ws);
    if (a.b.max_tokens == 1) {
        const int64_t rows = batch->max_rows > 0 ? std::min(batch->max_rows, cache->max_positions) : cache->max_positions;
        const Q4StepPlan plan = plan_q4_step(rows, static_cast<int64_t>(a.b.B) * a.c.KVH, a.c.hd);
        const StepParts parts = step_parts(layer, cache, a.b.B, plan.splits, weights != nullptr);
        a.per = plan.per;
        a.splits = plan.splits;
        if (a.splits > 1 || weights) {
            a.part = reinterpret_cast<float *>(p);
            a.ml = reinterpret_cast<float2 *>(p + parts.part);
            if (weights) a.scores = reinterpret_cast<float *>(p + parts.part + parts.ml);
        }
        launch_q4_step(a, s);
        return launch_status();
    }
    const size_t rows = static_cast<size_t>(batch->tokens) * a.H;
    a.qn = reinterpret_cast<float *>(p);
    a.lse = reinterpret_cast<float *>(p + q4_align(rows * a.c.hd * sizeof(float)));
    if (k_proj) launch_q4_append(layer, a.c, a.b, k_proj, v_proj, dtype, s);
    switch (a.c.hd) {
        case 64: launch<64>(a, dtype, out_dtype, s); break;
        case 128: launch<128>(a, dtype, out_dtype, s); break;
        default: launch<256>(a, dtype, out_dtype, s); break;
    }
    return launch_status();
}
