// Gated GQA attention over a KV cache held in 4 bits: the entry point, its workspace, and which form a
// call takes.
#include <cmath>

#include "attention_q4.hpp"

namespace swq {
namespace {

// The workspace of either form, region after region at 256-byte boundaries.
struct StepParts {
    size_t part, ml, scores, total;
};

// head_splits: splits of all kv heads of all sequences.
StepParts step_parts(const swq_attention_layer *l, const swq_q4_cache *c, int sequences, int64_t head_splits, bool weights) {
    const size_t heads = static_cast<size_t>(sequences) * l->num_heads, triples = static_cast<size_t>(head_splits) * (l->num_heads / c->num_kv_heads);
    StepParts p{};
    p.part = q4_align(triples * l->head_dim * sizeof(float));
    p.ml = q4_align(triples * sizeof(float2));
    p.scores = weights ? q4_align(heads * q4_rows(c->max_positions) * sizeof(float)) : 0;
    p.total = p.part + p.ml + p.scores;
    return p;
}

struct PrefillParts {
    size_t q, qf, qs, vmax, lse, part, ml, gpart, total;
};

// part_rows: (token, query head, split) triples; 0 where nothing is split.
PrefillParts prefill_parts(const swq_attention_layer *l, const swq_q4_cache *c, int sequences, int64_t tokens, int64_t part_rows, int64_t gathered) {
    const size_t rows = static_cast<size_t>(tokens) * l->num_heads;
    PrefillParts p{};
    p.q = q4_align(rows * l->head_dim * 2);  // each of two
    p.qf = q4_align(rows * sizeof(float));
    p.qs = q4_align(rows * 16 * 2);
    p.vmax = q4_align(static_cast<size_t>(sequences) * c->num_kv_heads * 2 * sizeof(uint32_t));
    p.lse = q4_align(rows * sizeof(float));
    p.part = q4_align(static_cast<size_t>(part_rows) * l->head_dim * sizeof(float));
    p.ml = q4_align(static_cast<size_t>(part_rows) * sizeof(float2));
    p.gpart = q4_align(static_cast<size_t>(gathered) * sizeof(float));
    p.total = 2 * p.q + p.qf + p.qs + p.vmax + p.lse + p.part + p.ml + p.gpart;
    return p;
}

// What any call of up to these tokens can take.
size_t prefill_workspace(const swq_attention_layer *l, const swq_q4_cache *c, const swq_q4_batch *b, int weights) {
    const int64_t tokens = std::max(b->tokens, 1), rows = tokens * l->num_heads;
    const int64_t heads = static_cast<int64_t>(b->sequences) * c->num_kv_heads;
    const int64_t part_rows = std::min<int64_t>(rows * kQ4PrefillMaxSplits, kQ4PartRows + rows);
    const int64_t gathered = weights ? std::min<int64_t>(heads * q4_rows(c->max_positions) * kQ4GatherMaxParts, kQ4GatherMost) : 0;
    return prefill_parts(l, c, b->sequences, tokens, part_rows, gathered).total;
}

size_t step_workspace(const swq_attention_layer *l, const swq_q4_cache *c, const swq_q4_batch *b, int weights) {
    const int64_t splits = most_q4_head_splits(c->max_positions, static_cast<int64_t>(b->sequences) * c->num_kv_heads, c->head_dim);
    return step_parts(l, c, b->sequences, splits, weights != 0).total;
}

bool misaligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace
}  // namespace swq

using namespace swq;

extern "C" size_t swq_attention_q4_workspace_bytes(const swq_attention_layer *layer, const swq_q4_cache *cache,
                                                   const swq_q4_batch *batch, int weights) {
    if (check_q4_layer(layer) != SWQ_OK || !cache ||
        check_q4_shape(cache->sequences, cache->num_kv_heads, cache->head_dim, cache->max_positions) != SWQ_OK ||
        check_q4_sizes(cache, batch) != SWQ_OK || layer->head_dim != cache->head_dim ||
        layer->num_kv_heads != cache->num_kv_heads || static_cast<int64_t>(batch->tokens) * layer->num_heads > INT32_MAX)
        return 0;
    return std::max(step_workspace(layer, cache, batch, weights), prefill_workspace(layer, cache, batch, weights));
}

extern "C" int swq_attention_q4(const swq_attention_layer *layer, const swq_q4_cache *cache, const swq_q4_batch *batch,
                                const void *q_proj, const void *k_proj, const void *v_proj, int dtype, float *weights,
                                void *out, int out_dtype, void *ws, size_t ws_bytes, void *stream) {
    int st = check_q4_batch(layer, cache, batch);
    if (st == SWQ_OK) st = check_q4_dtype(dtype);
    if (st == SWQ_OK) st = check_q4_dtype(out_dtype);
    if (st != SWQ_OK) return st;
    if (static_cast<int64_t>(batch->tokens) * layer->num_heads > INT32_MAX) return SWQ_ERR_LIMIT;
    if (batch->tokens == 0) return SWQ_OK;
    if (!q_proj || !out || !k_proj != !v_proj) return SWQ_ERR_INVALID_ARGUMENT;
    if (misaligned(q_proj) || misaligned(k_proj) || misaligned(v_proj) || misaligned(out) || misaligned(layer->q_norm_weight) ||
        reinterpret_cast<uintptr_t>(weights) % 4 || reinterpret_cast<uintptr_t>(ws) % 256)
        return SWQ_ERR_MISALIGNED;
    if (!ws || ws_bytes < swq_attention_q4_workspace_bytes(layer, cache, batch, weights != nullptr)) return SWQ_ERR_WORKSPACE;
    AttnQ4Args a{};
    a.c = q4_view(cache);
    a.b = q4_batch(layer, batch);
    a.q = q_proj;
    a.k = k_proj;
    a.v = v_proj;
    a.q_norm_w = layer->q_norm_weight;
    a.k_norm_w = layer->k_norm_weight;
    a.in_f32 = dtype == SWQ_F32;
    a.out_f32 = out_dtype == SWQ_F32;
    a.out = out;
    a.weights = weights;
    a.H = layer->num_heads;
    a.group = a.H / a.c.KVH;
    a.eps = layer->norm_eps;
    a.scale2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(a.c.hd)));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t rows = batch->max_rows > 0 ? std::min(batch->max_rows, cache->max_positions) : cache->max_positions;
    const int64_t heads = static_cast<int64_t>(a.b.B) * a.c.KVH;
    uint8_t *p = static_cast<uint8_t *>(ws);
    if (a.b.max_tokens == 1) {
        const Q4StepPlan plan = plan_q4_step(rows, heads, a.c.hd);
        const StepParts parts = step_parts(layer, cache, a.b.B, heads * plan.splits, weights != nullptr);
        if (ws_bytes < parts.total) return SWQ_ERR_WORKSPACE;
        a.per = plan.per;
        a.splits = plan.splits;
        a.planes_q = a.in_f32 || a.out_f32 || weights ? 2 : 1;
        if (a.splits > 1 || weights) {
            a.part = reinterpret_cast<float *>(p);
            a.ml = reinterpret_cast<float2 *>(p + parts.part);
            if (weights) a.scores = reinterpret_cast<float *>(p + parts.part + parts.ml);
        }
        launch_q4_step(a, s);
        return launch_status();
    }
    const Q4PrefillPlan plan = plan_q4_prefill(a.b.max_tokens, static_cast<int64_t>(batch->tokens) * a.H, rows, heads, a.group, a.c.hd, layer->rotary_dims, cache->max_positions, a.in_f32 || a.out_f32, weights != nullptr);
    const PrefillParts parts = prefill_parts(layer, cache, a.b.B, batch->tokens,
                                             plan.splits > 1 ? static_cast<int64_t>(batch->tokens) * a.H * plan.splits : 0,
                                             plan.gparts > 1 ? heads * a.c.R * plan.gparts : 0);
    if (ws_bytes < parts.total) return SWQ_ERR_WORKSPACE;
    a.planes_q = plan.planes_q;
    a.planes_v = plan.planes_v;
    a.rows_per = plan.rows_per;
    a.tiles = plan.tiles;
    a.per = plan.per;
    a.splits = plan.splits;
    a.gparts = plan.gparts;
    if (!plan.prepares) a.qh = p;
    a.ql = p + parts.q;
    p += 2 * parts.q;
    a.qf = reinterpret_cast<float *>(p);
    p += parts.qf;
    if (a.planes_q == 2) a.qs = p;
    p += parts.qs;
    if (a.planes_v == 2) a.vmax = reinterpret_cast<uint32_t *>(p);
    p += parts.vmax;
    if (weights) a.lse = reinterpret_cast<float *>(p);
    p += parts.lse;
    a.part = reinterpret_cast<float *>(p);
    p += parts.part;
    a.ml = reinterpret_cast<float2 *>(p);
    p += parts.ml;
    a.gpart = reinterpret_cast<float *>(p);
    if (k_proj) launch_q4_append(layer, a.c, a.b, k_proj, v_proj, dtype, s);
    launch_q4_prefill(a, s);
    return launch_status();
}
