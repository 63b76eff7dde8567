// Attention over a 4-bit cache, one token per sequence: the rows of a (sequence, kv head) are split
// over workgroups, and each wave walks its own tiles of 32 rows.
#include <cmath>

#include "attention_q4.hpp"

namespace swq {
namespace {

constexpr int kStepThreads = 256;
constexpr int kStepWaves = kStepThreads / kWave;
constexpr int kTile = 32;    // rows of one step of a wave
constexpr int kHeadPad = 4;  // floats between heads' sums in LDS

// One tile's words and parameters, as loaded: lane (r = lane % 16, q = lane / 16).
template <int NG>
struct Q4Tile {
    uint2 k[2][NG];   // row 8 (r / 4) + 4 t + r % 4, words 2 q and 2 q + 1 of each group
    uint4 v[NG];      // rows 8 q .. 8 q + 7, dims 4 r .. 4 r + 3 of each group
    uint4 par[4][NG]; // rows 8 q .. 8 q + 7: k scale, k bias, v scale, v bias
};

template <int HD, typename T>
__global__ __launch_bounds__(kStepThreads, HD == 256 ? 2 : HD == 128 ? 3 : 4) void q4_step(const AttnQ4Args a) {
    constexpr int EPL = HD / kWave, NG = HD / kQ4Group, KS = HD / 32;
    constexpr int HP = HD + kHeadPad;
    constexpr int kQBytes = 2 * KS * kWave * 16, kOBytes = kStepWaves * kQ4MaxHeadGroup * HP * 4;
    // queries in operand order (used up to the last tile), then the waves' sums
    __shared__ __attribute__((aligned(16))) uint8_t s_buf[kQBytes > kOBytes ? kQBytes : kOBytes];
    __shared__ float s_qs[NG][kQ4MaxHeadGroup], s_f[kQ4MaxHeadGroup];
    __shared__ float s_rl[kStepWaves][2][kQ4MaxHeadGroup];
    __shared__ double s_rot[kStepWaves][HD];
    h8_t *s_q = reinterpret_cast<h8_t *>(s_buf);  // [plane][kstep][lane]
    float *s_o = reinterpret_cast<float *>(s_buf);  // [wave][head][HP]
    // Workgroups go to the 8 XCDs in turn: with the splits outermost and the heads turned by one from
    // split to split, no XCD gets the same splits, or the same sequences, of every head.
    const int split = blockIdx.y, head = (blockIdx.x + blockIdx.y) % gridDim.x;
    const int kvh = head % a.c.KVH, b = head / a.c.KVH;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int r = lane & 15, q = lane >> 4, G = a.group;
    if (a.b.count(b) <= 0) return;
    const int n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const int n = min(r0 + 1, a.c.maxp);  // rows that the token sees
    const int p0 = split * a.per, p1 = split == a.splits - 1 ? n : min(p0 + a.per, n);
    if (p0 >= n) return;
    const bool last = p1 == n;
    // In the last split two waves write the token's row before they, or another, load its tile.
    const bool writes = a.k && last && r0 < a.c.maxp;
    const int end = (p1 - p0 + kTile - 1) / kTile;  // tiles
    int tile = wave;

    const uint32_t *kw = a.c.k_head(b, kvh), *vw = a.c.v_head(b, kvh);
    const _Float16 *par = a.c.par_head(b, kvh);
    Q4Tile<NG> cur;
    auto load_k = [&](int t) {
        const int64_t t0 = p0 + static_cast<int64_t>(t) * kTile;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int g = 0; g < NG; ++g)
                cur.k[x][g] = *reinterpret_cast<const uint2 *>(kw + (t0 + 8 * (r >> 2) + 4 * x + (r & 3)) * (HD / 8) + 8 * g + 2 * q);
#pragma unroll
        for (int w = kQ4KScale; w <= kQ4KBias; ++w)
#pragma unroll
            for (int g = 0; g < NG; ++g)
                cur.par[w][g] = *reinterpret_cast<const uint4 *>(par + (static_cast<int64_t>(w) * NG + g) * a.c.R + t0 + 8 * q);
    };
    auto load_v = [&](int t) {
        const int64_t t0 = p0 + static_cast<int64_t>(t) * kTile;
#pragma unroll
        for (int w = kQ4VScale; w <= kQ4VBias; ++w)
#pragma unroll
            for (int g = 0; g < NG; ++g)
                cur.par[w][g] = *reinterpret_cast<const uint4 *>(par + (static_cast<int64_t>(w) * NG + g) * a.c.R + t0 + 8 * q);
#pragma unroll
        for (int g = 0; g < NG; ++g)
            cur.v[g] = *reinterpret_cast<const uint4 *>(vw + (t0 / 8 + q) * HD + 64 * g + 4 * r);
    };
    const bool waits = writes && tile == end - 1;  // its first tile is the one with the new row
    if (tile < end && !waits) {
        load_k(tile);
        load_v(tile);
    }

    const int half = a.b.rot / 2;
    const float2 *turn = half > 0 ? a.b.rope + static_cast<int64_t>(a.b.position(b, 0)) * half : nullptr;
    const int askers = writes ? kStepWaves - 2 : kStepWaves;  // waves that prepare queries
    if (wave >= askers) {
        const int64_t at = (static_cast<int64_t>(n0) * a.c.KVH + kvh) * HD + lane * EPL;
        double x[EPL];
        _Float16 *pw = a.c.par_head(b, kvh);
        if (wave == askers) {
            Q4HeadTable<EPL> tab;
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[e] = static_cast<double>(q4_load(static_cast<const T *>(a.k), at + e));
            tab.load(a.k_norm_w, turn, half);
            q4_key_row<HD>(x, tab, a.eps, half, s_rot[wave], a.c.k_head(b, kvh), pw, a.c.R, r0);
        } else {
            uint32_t code[EPL], old[EPL];
            uint32_t *vp = a.c.v_head(b, kvh) + static_cast<int64_t>(r0 / kQ4Block) * HD + lane * EPL;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                x[e] = static_cast<double>(q4_load(static_cast<const T *>(a.v), at + e));
                old[e] = vp[e];
            }
            q4_value_row<HD>(x, code, pw, a.c.R, r0);
            const int sh = 4 * (r0 & 7);
#pragma unroll
            for (int e = 0; e < EPL; ++e) vp[e] = (old[e] & ~(15u << sh)) | (code[e] << sh);
        }
    } else {
        constexpr int AT_ONCE = 4;  // heads of a wave whose loads are in flight together
        Q4HeadTable<EPL> tab;
        tab.load(a.q_norm_w, turn, half);
        for (int base = 0; base < G; base += AT_ONCE * askers) {
            float x[AT_ONCE][EPL];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int u = min(base + k * askers + wave, G - 1);
                const T *src = static_cast<const T *>(a.q) + (static_cast<int64_t>(n0) * a.H + kvh * G + u) * 2 * HD + lane * EPL;
#pragma unroll
                for (int e = 0; e < EPL; ++e) x[k][e] = q4_load(src, e);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int u = base + k * askers + wave;
                if (u >= G) break;
                q4_norm_rope<EPL>(x[k], tab, a.eps, half, reinterpret_cast<float *>(s_rot[wave]));
                float top = 0.f, qs = 0.f;
#pragma unroll
                for (int e = 0; e < EPL; ++e) top = fmaxf(top, fabsf(x[k][e]));
                top = wave_max_all(top);
                int ex = 0;
                if (top > 0.f && top < INFINITY) frexpf(top, &ex);
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    x[k][e] = ldexpf(x[k][e], 10 - ex);  // below 2^10
                    qs += x[k][e];
                }
                if (lane == 0) s_f[u] = ldexpf(a.scale2, ex - 10);
                qs = segment_sum(qs, kQ4Group / EPL);
                if (lane % (kQ4Group / EPL) == 0) s_qs[lane * EPL / kQ4Group][u] = qs;
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    const int d = lane * EPL + e, j = (d & 63) >> 3, nb = d & 7;  // word of its group, nibble
                    const float v = nb & 1 ? x[k][e] * 0.0625f : x[k][e];
                    const _Float16 hi = static_cast<_Float16>(v), lo = static_cast<_Float16>(v - static_cast<float>(hi));
                    _Float16 *dst = reinterpret_cast<_Float16 *>(s_q + (2 * (d >> 6) + (j & 1)) * kWave + (j >> 1) * 16 + u) + q4_element(nb);
                    dst[0] = hi;
                    dst[KS * kWave * 8] = lo;
                }
            }
        }
    }
    // heads past the group are columns of their own in both products: what they hold reaches nothing
    if (writes) __syncthreads();  // the row's stores are done
    else lds_barrier();
    if (waits) {
        load_k(tile);
        load_v(tile);
    }

    float qs[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) qs[g] = s_qs[g][r];
    const float f = r < G ? s_f[r] : 0.f;
    float m = -INFINITY, l = 0.f, ref = -INFINITY, cap = 0.f, ce = -24.f;  // 2^ce bounds the value scales so far
    float pb[NG];
    f4_t o[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        pb[g] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][e] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    float *sc_out = a.scores && r < G ? a.scores + (static_cast<int64_t>(b) * a.H + kvh * G + r) * a.c.R : nullptr;
    constexpr int stride = kStepWaves;
    const uint32_t magic = kept_1024();
    for (; tile < end; tile += stride) {
        const int t0 = p0 + tile * kTile;
        // scores; the queries come from LDS each time, which leaves registers for another wave
        int ql = lane;
        asm volatile("" : "+v"(ql));
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const h8_t ks = __builtin_bit_cast(h8_t, cur.par[kQ4KScale][g]), kb = __builtin_bit_cast(h8_t, cur.par[kQ4KBias][g]);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const h8_t c = q4_operand(u ? cur.k[x][g].y : cur.k[x][g].x, magic);
                    d = mfma16(c, s_q[(2 * g + u) * kWave + ql], d);
                    d = mfma16(c, s_q[(KS + 2 * g + u) * kWave + ql], d);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[4 * x + i] = fmaf(static_cast<float>(kb[4 * x + i]), qs[g], p[4 * x + i]);
                    p[4 * x + i] = fmaf(static_cast<float>(ks[4 * x + i]), d[i], p[4 * x + i]);
                }
            }
            if constexpr (NG > 2) __builtin_amdgcn_sched_barrier(0);
        }
        const int next = tile + stride < end ? tile + stride : tile;  // the last tile once more: never used
        load_k(next);
        if (t0 + kTile > p1) {  // rows past the end count nothing, whatever they hold
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = t0 + 8 * q + i < p1 ? p[i] : -INFINITY;
            uint4 keep;
            const int left = p1 - t0 - 8 * q;  // of this lane's 8 rows
            keep.x = (left > 0 ? 0xFFFFu : 0u) | (left > 1 ? 0xFFFF0000u : 0u);
            keep.y = (left > 2 ? 0xFFFFu : 0u) | (left > 3 ? 0xFFFF0000u : 0u);
            keep.z = (left > 4 ? 0xFFFFu : 0u) | (left > 5 ? 0xFFFF0000u : 0u);
            keep.w = (left > 6 ? 0xFFFFu : 0u) | (left > 7 ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int w = kQ4VScale; w <= kQ4VBias; ++w)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    cur.par[w][g].x &= keep.x;
                    cur.par[w][g].y &= keep.y;
                    cur.par[w][g].z &= keep.z;
                    cur.par[w][g].w &= keep.w;
                }
        }
        if (sc_out) {
            *reinterpret_cast<float4 *>(sc_out + t0 + 8 * q) = make_float4(p[0] * f, p[1] * f, p[2] * f, p[3] * f);
            *reinterpret_cast<float4 *>(sc_out + t0 + 8 * q + 4) = make_float4(p[4] * f, p[5] * f, p[6] * f, p[7] * f);
        }
        float mt = f * fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        h2_t st = {static_cast<_Float16>(0.f), static_cast<_Float16>(0.f)};
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 u = cur.par[kQ4VScale][g];
                st = __builtin_elementwise_max(st, __builtin_bit_cast(h2_t, i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w));
            }
        float top = fmaxf(static_cast<float>(st.x), static_cast<float>(st.y));
        if (__any(mt > m || top > cap)) {
            mt = fmaxf(mt, __shfl_xor(mt, 16, kWave));
            mt = fmaxf(mt, __shfl_xor(mt, 32, kWave));
            m = fmaxf(m, mt);
            top = wave_max_all(top);
            if (top > cap) {
                int ex = 0;
                frexpf(top, &ex);
                ce = static_cast<float>(ex);
                cap = ldexpf(1.0f, ex);
            }
            const float to = m + (ce - 15.0f);
            const float alpha = q4_exp2(ref - to);
            ref = to;
            l *= alpha;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                pb[g] *= alpha;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[g][e] *= alpha;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = q4_exp2(fmaf(p[i], f, -ref));
            l += p[i];
        }
        float pe[8];  // in operand order, 1/16 where the codes are 16 times as large
#pragma unroll
        for (int j = 0; j < 8; ++j) pe[j] = q4_nibble(j) & 1 ? p[q4_nibble(j)] * 0.0625f : p[q4_nibble(j)];
        // values
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const h8_t vs = __builtin_bit_cast(h8_t, cur.par[kQ4VScale][g]), vb = __builtin_bit_cast(h8_t, cur.par[kQ4VBias][g]);
            h8_t hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const f32x2_t x = {pe[j] * static_cast<float>(vs[q4_nibble(j)]), pe[j + 1] * static_cast<float>(vs[q4_nibble(j + 1)])};
                h2_t h, w;
                split_f16(x, h, w);
                hi[j] = h.x;
                hi[j + 1] = h.y;
                lo[j] = w.x;
                lo[j + 1] = w.y;
            }
            const uint32_t vw4[4] = {cur.v[g].x, cur.v[g].y, cur.v[g].z, cur.v[g].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const h8_t c = q4_operand(vw4[e], magic);
                o[g][e] = mfma16(c, hi, o[g][e]);
                o[g][e] = mfma16(c, lo, o[g][e]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) pb[g] = fmaf(p[i], static_cast<float>(vb[i]), pb[g]);
            if constexpr (NG > 2) __builtin_amdgcn_sched_barrier(0);
        }
        load_v(next);
    }
    // the waves' sums meet
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        pb[g] += __shfl_xor(pb[g], 16, kWave);
        pb[g] += __shfl_xor(pb[g], 32, kWave);
    }
    if (q == 0) {
        s_rl[wave][0][r] = ref;
        s_rl[wave][1][r] = l;
    }
    lds_barrier();  // and every wave is done with the queries
    float top = s_rl[0][0][r];
#pragma unroll
    for (int w = 1; w < kStepWaves; ++w) top = fmaxf(top, s_rl[w][0][r]);
    const float mine = q4_exp2(ref - top);
    float *mo = s_o + (wave * kQ4MaxHeadGroup + r) * HP + 16 * q;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4 v;
            v.x = mine * (o[g][0][i] + pb[g]);
            v.y = mine * (o[g][1][i] + pb[g]);
            v.z = mine * (o[g][2][i] + pb[g]);
            v.w = mine * (o[g][3][i] + pb[g]);
            *reinterpret_cast<float4 *>(mo + 64 * g + 4 * i) = v;
        }
    lds_barrier();
    const int64_t head0 = static_cast<int64_t>(b) * a.H + kvh * G;
    for (int i = tid; i < G * (HD / 4); i += kStepThreads) {
        const int u = i / (HD / 4), d = i % (HD / 4) * 4;
        float4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kStepWaves; ++w) {
            const float4 v = *reinterpret_cast<const float4 *>(s_o + (w * kQ4MaxHeadGroup + u) * HP + d);
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        float R = s_rl[0][0][u], L = 0.f;
#pragma unroll
        for (int w = 1; w < kStepWaves; ++w) R = fmaxf(R, s_rl[w][0][u]);
#pragma unroll
        for (int w = 0; w < kStepWaves; ++w) L += q4_exp2(s_rl[w][0][u] - R) * s_rl[w][1][u];
        if (a.part) {
            *reinterpret_cast<float4 *>(a.part + ((head0 + u) * a.splits + split) * HD + d) = s;
            if (d == 0) a.ml[(head0 + u) * a.splits + split] = make_float2(R, L);
        } else {
            const int64_t at = static_cast<int64_t>(n0) * a.H + kvh * G + u;
            const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float gate = q4_load(static_cast<const T *>(a.q), (2 * at + 1) * HD + d + e);
                q4_store_any(a.out, at * HD + d + e, v[e] / L * sigmoid_exact(gate), a.out_f32);
            }
        }
    }
}

// The splits merged: a workgroup per (sequence, query head) for the output, then workgroups per 1,024
// rows of a kv head for the gathered weights.
constexpr int kMergeThreads = 256;
constexpr int kMergeRows = 1024;
constexpr int kMaxSplits = 1024;

template <int HD>
__global__ __launch_bounds__(kMergeThreads) void q4_step_merge(const AttnQ4Args a) {
    constexpr int LPS = HD / 4, SPR = kMergeThreads / LPS, U = 8;
    __shared__ float s_w[kMaxSplits];
    __shared__ float s_red[kMergeThreads / kWave];
    __shared__ float4 s_acc[SPR][LPS];
    __shared__ float s_lse[kQ4MaxHeadGroup];
    const int kvh = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH, G = a.group;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
    if (a.b.count(b) <= 0) return;
    const int n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const int n = min(r0 + 1, a.c.maxp);
    const int splits = min((n + a.per - 1) / a.per, a.splits);
    if (static_cast<int>(blockIdx.x) < G) {
        const int64_t head = static_cast<int64_t>(b) * a.H + kvh * G + blockIdx.x;
        const float2 *ml = a.ml + head * a.splits;
        const float *src = a.part + head * a.splits * HD + (tid % LPS) * 4;
        const int s0 = tid / LPS;
        float4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const float4 *>(src + static_cast<int64_t>(min(s0 + u * SPR, splits - 1)) * HD);
        float R = -INFINITY;
        for (int s = tid; s < splits; s += kMergeThreads) R = fmaxf(R, ml[s].x);
        R = wave_max_all(R);
        if (lane == 0) s_red[wave] = R;
        lds_barrier();
#pragma unroll
        for (int w = 0; w < kMergeThreads / kWave; ++w) R = fmaxf(R, s_red[w]);
        float L = 0.f;
        for (int s = tid; s < splits; s += kMergeThreads) {
            const float2 x = ml[s];
            const float w = q4_exp2(x.x - R);
            s_w[s] = w;
            L += w * x.y;
        }
        L = wave_sum_all(L);
        lds_barrier();
        if (lane == 0) s_red[wave] = L;
        float4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int base = 0; base < splits; base += U * SPR) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = base + s0 + u * SPR;
                if (s < splits) {
                    const float w = s_w[s];
                    acc.x += w * v[u].x;
                    acc.y += w * v[u].y;
                    acc.z += w * v[u].z;
                    acc.w += w * v[u].w;
                }
            }
            if (base + U * SPR < splits) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    v[u] = *reinterpret_cast<const float4 *>(src + static_cast<int64_t>(min(base + (U + u) * SPR + s0, splits - 1)) * HD);
            }
        }
        s_acc[s0][tid % LPS] = acc;
        lds_barrier();
        if (tid < HD) {
            L = 0.f;
#pragma unroll
            for (int w = 0; w < kMergeThreads / kWave; ++w) L += s_red[w];
            float t = 0.f;
#pragma unroll
            for (int s = 0; s < SPR; ++s) t += reinterpret_cast<const float *>(s_acc[s])[tid];
            const int64_t at = static_cast<int64_t>(n0) * a.H + kvh * G + blockIdx.x;
            const float gate = q4_load_any(a.q, (2 * at + 1) * HD + tid, a.in_f32);
            q4_store_any(a.out, at * HD + tid, t / L * sigmoid_exact(gate), a.out_f32);
        }
        return;
    }
    for (int chunk = blockIdx.x - G; chunk * kMergeRows < n; chunk += gridDim.x - G) {
        __syncthreads();
        for (int u = wave; u < G; u += kMergeThreads / kWave) {
            const float2 *ml = a.ml + (static_cast<int64_t>(b) * a.H + kvh * G + u) * a.splits;
            float R = -INFINITY, L = 0.f;
            for (int s = lane; s < splits; s += kWave) R = fmaxf(R, ml[s].x);
            R = wave_max_all(R);
            for (int s = lane; s < splits; s += kWave) L += q4_exp2(ml[s].x - R) * ml[s].y;
            L = wave_sum_all(L);
            if (lane == 0) s_lse[u] = R + log2f(L);
        }
        __syncthreads();
        const int row = chunk * kMergeRows + tid * 4;
        if (row < n) {
            float4 s = {0.f, 0.f, 0.f, 0.f};
            for (int u = 0; u < G; ++u) {
                const float z = s_lse[u];
                const float4 x = *reinterpret_cast<const float4 *>(a.scores + (static_cast<int64_t>(b) * a.H + kvh * G + u) * a.c.R + row);
                s.x += q4_exp2(x.x - z);
                s.y += q4_exp2(x.y - z);
                s.z += q4_exp2(x.z - z);
                s.w += q4_exp2(x.w - z);
            }
            float *w = a.weights + a.c.head(b, kvh) * a.c.maxp + row;
            const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row + e < n) w[e] = row + e < r0 ? w[e] + v[e] : v[e];
        }
    }
}

template <int HD, typename T>
void launch_typed(const AttnQ4Args &a, hipStream_t s) {
    const uint32_t heads = static_cast<uint32_t>(a.b.B) * a.c.KVH;
    hipLaunchKernelGGL((q4_step<HD, T>), dim3(heads, a.splits), dim3(kStepThreads), 0, s, a);
    if (a.part) {
        const int chunks = a.weights ? (a.c.maxp + kMergeRows - 1) / kMergeRows : 0;
        hipLaunchKernelGGL(q4_step_merge<HD>, dim3(a.group + chunks, heads), dim3(kMergeThreads), 0, s, a);
    }
}

}  // namespace

Q4StepPlan plan_q4_step(int64_t rows, int64_t heads) {
    const int64_t total = rows * heads;
    int64_t per = std::min(total / 512, std::max<int64_t>(512, total / 2048));
    per = std::max<int64_t>((per + 127) / 128 * 128, 128);
    per = std::max<int64_t>(per, (rows + kMaxSplits - 1) / kMaxSplits);
    per = (per + kTile - 1) / kTile * kTile;
    return {static_cast<int>(per), static_cast<int>((rows + per - 1) / per)};
}

int most_q4_splits(int64_t rows, int64_t heads) {
    // rows per split are at least 128, and at least a 2,048th of rows * heads
    return static_cast<int>(std::min<int64_t>({(rows + 127) / 128, 2048 / heads + 2, kMaxSplits}));
}

void launch_q4_step(const AttnQ4Args &a, hipStream_t s) {
    switch (a.c.hd) {
        case 64: a.in_f32 ? launch_typed<64, float>(a, s) : launch_typed<64, uint16_t>(a, s); break;
        case 128: a.in_f32 ? launch_typed<128, float>(a, s) : launch_typed<128, uint16_t>(a, s); break;
        default: a.in_f32 ? launch_typed<256, float>(a, s) : launch_typed<256, uint16_t>(a, s); break;
    }
}

}  // namespace swq
