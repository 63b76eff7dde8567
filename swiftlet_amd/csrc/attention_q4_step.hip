// Attention over a 4-bit cache, one token per sequence: the rows of a (sequence, kv head) are split
// over workgroups, and each wave walks its own tiles of 32 rows.
#include <cmath>

#include "attention_q4.hpp"

namespace swq {
namespace {

constexpr int kStepThreads = 256;
constexpr int kStepWaves = kStepThreads / kWave;
constexpr int kTile = 32;    // rows of one step of a team
constexpr int kHeadPad = 4;  // floats between heads' sums in LDS

// What one wave reads of a tile: GW * 64 dims of 32 rows; lane (r = lane % 16, q = lane / 16).
template <int GW>
struct Q4Tile {
    uint2 k[GW][2];    // row 8 (r / 4) + 4 t + r % 4, words 2 q and 2 q + 1 of each group
    uint4 v[GW];       // rows 8 q .. 8 q + 7, dims 4 r .. 4 r + 3 of each group
    uint4 par[4][GW];  // rows 8 q .. 8 q + 7: k scale, k bias, v scale, v bias
};

// Four dims of head u: to the partial results of `split`, or, of the only one, to the output.
template <int HD>
__device__ __forceinline__ void finish(const AttnQ4Args &a, int64_t head0, int n0, int h0, int u, int split, int d, f4_t s, float M, float L) {
    if (a.part) {
        *reinterpret_cast<f4_t *>(a.part + ((head0 + u) * a.splits + split) * HD + d) = s;
        if (d == 0) a.ml[(head0 + u) * a.splits + split] = make_float2(M, L);
    } else {
        const int64_t at = static_cast<int64_t>(n0) * a.H + h0 + u;
        store_gated(a, at * HD + d, (2 * at + 1) * HD + d, s * (1.0f / L));
    }
}

// A wave has GW groups of 64 dims of the head (groups as the cache's scales have them): the whole
// head at hd 64 and 128, half of it at 256.  The waves of a head, a team, walk the same tiles, the
// teams of a workgroup different ones.  A step of a team:
//   scores  K's codes are the left operand (rows: 16 of the tile's 32 positions, twice), the queries
//           of the kv head's group the right one (columns: heads): lane (h, q) gets head h's sums of
//           positions 8 q .. 8 q + 7, times scale, plus bias * the sum of the query's dims.  Where a
//           team is two waves their partial scores meet in LDS, a barrier a step (two buffers);
//   softmax online, on both waves of the team alike.  p is taken against the running maximum and
//           against the largest value scale so far, so that p * scale fits f16;
//   values  V's codes are the left operand (rows: dims), p * scale the right one (columns: heads),
//           straight from the registers that the scores left: no transpose, and the running
//           maximum's factor is the lane's own.  Codes are taken about zero (q4_operand_signed), and p *
//           (bias + 8 or 7 scale) is summed on the VALU.
// Heads past the group are columns that nothing reads.  The next tile's loads are issued as soon as
// their registers are free.
//   P = 1   (bf16 in and out, no gathered weights): queries and p * scale as one f16 number instead of
//           two, and K's codes with the 1024 left on, whose share of a score is the same for all rows
//           and starts the sum.  32 sequences of up to 16,384 rows of 8 heads of 128: 81 us, with two 9 more.
//           (Not for V's: there the 1024 would swallow the bits of an average that is near zero.)
// Wide batches are bound by instruction issue beside the loads: those 81 us are 3.8 TB/s of cache, with
// VALU and matrix instructions for some 50 of them on every SIMD; three waves are all that 160 registers
// leave (bounded to 128 they spill: 163 us).  Small ones are a chain, 9 us at 500 rows of 2 heads of 256 in
// f32: by a workgroup's own clock rows and addresses 0.9, queries 1.9, one step 1.6, the teams' sums 1.2.
template <int HD, int P, typename T>
__global__ __launch_bounds__(kStepThreads, HD == 64 ? 4 : 3) void q4_step(const AttnQ4Args a) {
    constexpr int EPL = HD / kWave, NG = HD / kQ4Group, GW = NG > 1 ? 2 : 1, TW = NG / GW, TEAMS = kStepWaves / TW;
    constexpr int HP = HD + kHeadPad;
    __shared__ h8_t s_q[P][NG][2][kWave];  // queries in operand order: [high, low][group][step][lane]
    __shared__ float s_off[P == 1 ? NG : 1][kQ4MaxHeadGroup];
    __shared__ float s_qs[NG][kQ4MaxHeadGroup], s_f[kQ4MaxHeadGroup];
    __shared__ float s_ml[TEAMS][2][kQ4MaxHeadGroup];
    // one after another, a barrier between them: heads to be rotated, partial scores, teams' sums
    constexpr int kRotWave = 256;  // doubles of a wave: a key, or all the heads that it takes at once
    constexpr int kRot = kStepWaves * kRotWave * 8, kPart = TW > 1 ? 2 * kStepWaves * 2 * kWave * 16 : 0;
    constexpr int SETS = TEAMS > 2 ? 2 : TEAMS;  // two teams' sums at a time
    constexpr int kSums = SETS * kQ4MaxHeadGroup * HP * 4;
    __shared__ __attribute__((aligned(16))) uint8_t s_buf[kRot > kPart ? (kRot > kSums ? kRot : kSums) : (kPart > kSums ? kPart : kSums)];
    double(*s_rot)[kRotWave] = reinterpret_cast<double(*)[kRotWave]>(s_buf);
    f4_t(*s_part)[kStepWaves][2][kWave] = reinterpret_cast<f4_t(*)[kStepWaves][2][kWave]>(s_buf);
    float *s_o = reinterpret_cast<float *>(s_buf);  // [team % SETS][head][HP]
    // Workgroups go to the 8 XCDs in turn: with the splits outermost and the heads turned by one from
    // split to split, no XCD gets the same splits, or the same sequences, of every head.
    const int split = blockIdx.y, head = (blockIdx.x + blockIdx.y) % gridDim.x;
    const int kvh = head % a.c.KVH, b = head / a.c.KVH;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int r = lane & 15, q = lane >> 4, G = a.group;
    const int g0 = wave % TW * GW, team = wave / TW;  // first group
    if (a.b.count(b) <= 0) return;
    const int n0 = a.b.first(b);
    // 8 dims of a query per lane, a word's: HD / 8 lanes per head, 512 / HD heads of a wave at once.  Its
    // loads go first: they need no row count, and nothing that they would queue behind.
    constexpr int LPH = HD / 8, HPW = kWave / LPH;
    float x[8], w[8];
    auto load_query = [&](int base) {
        const int u = base + wave * HPW + lane / LPH;
        load8<T>(x, static_cast<const T *>(a.q) + (static_cast<int64_t>(n0) * a.H + kvh * G + min(u, G - 1)) * 2 * HD + 8 * (lane % LPH));
    };
    load_query(0);
    load8<float>(w, a.q_norm_w + 8 * (lane % LPH));
    const int r0 = a.b.row0(b, a.c.maxp);
    const int n = min(r0 + 1, a.c.maxp);  // rows that the token sees
    const int p0 = split * a.per, p1 = split == a.splits - 1 ? n : min(p0 + a.per, n);
    if (p0 >= n) return;
    const bool last = p1 == n;
    // In the last split two waves write the token's row before its tile is loaded.
    const bool writes = a.k && last && r0 < a.c.maxp;
    const int end = (p1 - p0 + kTile - 1) / kTile;  // tiles

    const int half = a.b.rot / 2;
    const float2 *turn = half > 0 ? a.b.rope + static_cast<int64_t>(a.b.position(b, 0)) * half : nullptr;
    float2 cs[8];
    if (8 * (lane % LPH) < 2 * half) q4_turns(cs, turn, half, lane % LPH);

    const uint32_t *kw = a.c.k_head(b, kvh) + (8 * (r >> 2) + (r & 3)) * (HD / 8) + 8 * g0 + 2 * q;
    const uint32_t *vw = a.c.v_head(b, kvh) + q * HD + 64 * g0 + 4 * r;
    const _Float16 *par = a.c.par_head(b, kvh) + static_cast<int64_t>(g0) * a.c.R + 8 * q;
    Q4Tile<GW> cur;
    auto load_k = [&](int t) {
        const int64_t t0 = p0 + static_cast<int64_t>(t) * kTile;
#pragma unroll
        for (int g = 0; g < GW; ++g) {
#pragma unroll
            for (int x = 0; x < 2; ++x) cur.k[g][x] = *reinterpret_cast<const uint2 *>(kw + (t0 + 4 * x) * (HD / 8) + 8 * g);
#pragma unroll
            for (int w = kQ4KScale; w <= kQ4KBias; ++w)
                cur.par[w][g] = *reinterpret_cast<const uint4 *>(par + (static_cast<int64_t>(w) * NG + g) * a.c.R + t0);
        }
    };
    auto load_v = [&](int t) {
        const int64_t t0 = p0 + static_cast<int64_t>(t) * kTile;
#pragma unroll
        for (int g = 0; g < GW; ++g) {
#pragma unroll
            for (int w = kQ4VScale; w <= kQ4VBias; ++w)
                cur.par[w][g] = *reinterpret_cast<const uint4 *>(par + (static_cast<int64_t>(w) * NG + g) * a.c.R + t0);
            cur.v[g] = *reinterpret_cast<const uint4 *>(vw + t0 / 8 * HD + 64 * g);
        }
    };
    const bool waits = writes && team >= end - 1;  // its first tile is the one with the new row
    if (!waits) {
        load_k(min(team, end - 1));
        load_v(min(team, end - 1));
    }

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
        const int j = lane % LPH;
        float *lds = reinterpret_cast<float *>(s_rot[wave]) + lane / LPH * HD;
        for (int base = 0; base < G; base += askers * HPW) {
            const int u = base + wave * HPW + lane / LPH;
            if (base > 0) load_query(base);
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
            ss = lanes_sum<LPH>(ss);
            const float sc = 1.0f / __fsqrt_rn(ss / static_cast<float>(HD) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] *= sc * w[e];
                lds[8 * j + e] = x[e];
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = 8 * j + e;
                const float o = lds[i < half ? i + half : i < 2 * half ? i - half : i];
                if (i < 2 * half) x[e] = i < half ? x[e] * cs[e].x - o * cs[e].y : x[e] * cs[e].x + o * cs[e].y;
                top = fmaxf(top, fabsf(x[e]));
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            top = lanes_max<LPH>(top);
            int ex = 0;
            if (top > 0.f && top < INFINITY) frexpf(top, &ex);
            float qs = 0.f;
            h8_t hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = ldexpf(x[e], 10 - ex);  // below 2^10
                qs += v;
                const float y = e & 1 ? v * 0.0625f : v;
                hi[q4_element(e)] = static_cast<_Float16>(y);
                lo[q4_element(e)] = static_cast<_Float16>(y - static_cast<float>(hi[q4_element(e)]));
            }
            float off = 0.f;
            if constexpr (P == 1) {  // the sum of what the products will take
                float even = 0.f, odd = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    even += static_cast<float>(hi[q4_element(e)]);
                    odd += static_cast<float>(hi[q4_element(e + 1)]);
                }
                qs = fmaf(odd, 16.0f, even);
                off = lanes_sum<8>(even + odd) * -1024.0f;
            }
            qs = lanes_sum<8>(qs);
            if (u < G) {
                // word j % 8 of group j / 8: lane row (j % 8) / 2 of step j % 2
                s_q[0][j / 8][j & 1][((j & 7) >> 1) * 16 + u] = hi;
                if constexpr (P == 2) s_q[P - 1][j / 8][j & 1][((j & 7) >> 1) * 16 + u] = lo;
                if ((j & 7) == 0) s_qs[j / 8][u] = qs;
                if (P == 1 && (j & 7) == 0) s_off[j / 8][u] = off;
                if (j == 0) s_f[u] = ldexpf(a.scale2, ex - 10);
            }
        }
    }
    if (writes) __syncthreads();  // the row's stores are done
    else lds_barrier();
    if (waits) {
        load_k(min(team, end - 1));
        load_v(min(team, end - 1));
    }

    const float f = r < G ? s_f[r] : 0.f;
    float qs[GW], pb[GW], off[GW];
    f4_t o[GW][4];
#pragma unroll
    for (int g = 0; g < GW; ++g) {
        qs[g] = s_qs[g0 + g][r];
        off[g] = P == 1 ? s_off[P == 1 ? g0 + g : 0][r] : 0.f;
        pb[g] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][e] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    float m = -INFINITY, l = 0.f, ref = -INFINITY, cap = 0.f, ce = -24.f;  // 2^ce bounds the value scales so far
    float *sc_out = a.scores && r < G && g0 == 0 ? a.scores + (static_cast<int64_t>(b) * a.H + kvh * G + r) * a.c.R : nullptr;
    const uint32_t magic = kept_1024();
    const int steps = (end + TEAMS - 1) / TEAMS;
    for (int step = 0; step < steps; ++step) {
        const int tile = step * TEAMS + team, t0 = p0 + tile * kTile;
        const bool have = tile < end;
        const int next = min(tile + TEAMS, end - 1);  // past the end the last one again: never used
        float p[8];
        int ql = lane;  // the queries come from LDS each time, which leaves registers for another wave
        asm volatile("" : "+v"(ql));
        if (have) {
#pragma unroll
            for (int g = 0; g < GW; ++g) {
                const h8_t ks = __builtin_bit_cast(h8_t, cur.par[kQ4KScale][g]), kb = __builtin_bit_cast(h8_t, cur.par[kQ4KBias][g]);
                f4_t d[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) d[x] = f4_t{off[g], off[g], off[g], off[g]};
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t word = u ? cur.k[g][x].y : cur.k[g][x].x;
                        const h8_t c = P == 1 ? q4_operand_1024(word, magic) : q4_operand(word, magic);
                        d[x] = mfma16(c, s_q[0][g0 + g][u][ql], d[x]);
                        if constexpr (P == 2) d[x] = mfma16(c, s_q[P - 1][g0 + g][u][ql], d[x]);
                    }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float z = static_cast<float>(kb[4 * x + i]);
                        p[4 * x + i] = g == 0 ? z * qs[g] : fmaf(z, qs[g], p[4 * x + i]);
                        p[4 * x + i] = fmaf(static_cast<float>(ks[4 * x + i]), d[x][i], p[4 * x + i]);
                    }
            }
            load_k(next);
            if constexpr (TW > 1) {
                s_part[step & 1][wave][0][lane] = f4_t{p[0], p[1], p[2], p[3]};
                s_part[step & 1][wave][1][lane] = f4_t{p[4], p[5], p[6], p[7]};
            }
        }
        if constexpr (TW > 1) lds_barrier();
        if (!have) continue;
        if constexpr (TW > 1) {
            f4_t sum[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                sum[x] = s_part[step & 1][team * TW][x][lane];
#pragma unroll
                for (int w = 1; w < TW; ++w) sum[x] += s_part[step & 1][team * TW + w][x][lane];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = sum[i / 4][i % 4];
        }
        if (t0 + kTile > p1) {  // rows past the end count nothing, whatever they hold
            uint4 keep;
            const int left = p1 - t0 - 8 * q;  // of this lane's 8 rows
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = i < left ? p[i] : -INFINITY;
            keep.x = (left > 0 ? 0xFFFFu : 0u) | (left > 1 ? 0xFFFF0000u : 0u);
            keep.y = (left > 2 ? 0xFFFFu : 0u) | (left > 3 ? 0xFFFF0000u : 0u);
            keep.z = (left > 4 ? 0xFFFFu : 0u) | (left > 5 ? 0xFFFF0000u : 0u);
            keep.w = (left > 6 ? 0xFFFFu : 0u) | (left > 7 ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int w = kQ4VScale; w <= kQ4VBias; ++w)
#pragma unroll
                for (int g = 0; g < GW; ++g) {
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
        for (int g = 0; g < GW; ++g) {
            const uint4 u = cur.par[kQ4VScale][g];
            st = __builtin_elementwise_max(st, __builtin_elementwise_max(
                __builtin_elementwise_max(__builtin_bit_cast(h2_t, u.x), __builtin_bit_cast(h2_t, u.y)),
                __builtin_elementwise_max(__builtin_bit_cast(h2_t, u.z), __builtin_bit_cast(h2_t, u.w))));
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
            for (int g = 0; g < GW; ++g) {
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
#pragma unroll
        for (int g = 0; g < GW; ++g) {
            const h8_t vs = __builtin_bit_cast(h8_t, cur.par[kQ4VScale][g]), vb = __builtin_bit_cast(h8_t, cur.par[kQ4VBias][g]);
            h8_t hi, lo;
            if constexpr (P == 1) {
#pragma unroll
                for (int j = 0; j < 8; ++j) hi[j] = static_cast<_Float16>(fmaf(pe[j], static_cast<float>(vs[q4_nibble(j)]), 0.f));
            } else {
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
            }
            const uint32_t vw4[4] = {cur.v[g].x, cur.v[g].y, cur.v[g].z, cur.v[g].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const h8_t c = q4_operand_signed(vw4[e], magic);
                o[g][e] = mfma16(c, hi, o[g][e]);
                if constexpr (P == 2) o[g][e] = mfma16(c, lo, o[g][e]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) pb[g] = fmaf(p[i], fmaf(i & 1 ? kQ4Odd : kQ4Even, static_cast<float>(vs[i]), static_cast<float>(vb[i])), pb[g]);
        }
        load_v(next);
    }
    // sums over the tile's rows meet, in units of the maximum alone
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
#pragma unroll
    for (int g = 0; g < GW; ++g) {
        pb[g] += __shfl_xor(pb[g], 16, kWave);
        pb[g] += __shfl_xor(pb[g], 32, kWave);
    }
    float unit = ref > -INFINITY ? q4_exp2(ce - 15.0f) : 0.f;
    l *= unit;
    const int64_t head0 = static_cast<int64_t>(b) * a.H + kvh * G;
    {
        if (q == 0 && g0 == 0) {
            s_ml[team][0][r] = m;
            s_ml[team][1][r] = l;
        }
        lds_barrier();
        float M = s_ml[0][0][r], L = 0.f;
#pragma unroll
        for (int w = 1; w < TEAMS; ++w) M = fmaxf(M, s_ml[w][0][r]);
        unit *= q4_exp2(m - M);
        float *mo = s_o + (team % SETS * kQ4MaxHeadGroup + r) * HP + 64 * g0 + 16 * q;
#pragma unroll
        for (int set = TEAMS / SETS - 1; set >= 0; --set) {
            if (team / SETS == set) {
#pragma unroll
                for (int g = 0; g < GW; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f4_t x = {unit * (o[g][0][i] + pb[g]), unit * (o[g][1][i] + pb[g]), unit * (o[g][2][i] + pb[g]), unit * (o[g][3][i] + pb[g])};
                        f4_t *to = reinterpret_cast<f4_t *>(mo + 64 * g + 4 * i);
                        if (set < TEAMS / SETS - 1) x += *to;
                        *to = x;
                    }
            }
            if (set > 0) lds_barrier();
        }
        lds_barrier();
        for (int i = tid; i < G * (HD / 4); i += kStepThreads) {
            const int u = i / (HD / 4), d = i % (HD / 4) * 4;
            f4_t s = *reinterpret_cast<const f4_t *>(s_o + u * HP + d);
#pragma unroll
            for (int w = 1; w < SETS; ++w) s += *reinterpret_cast<const f4_t *>(s_o + (w * kQ4MaxHeadGroup + u) * HP + d);
            M = s_ml[0][0][u];
            L = 0.f;
#pragma unroll
            for (int w = 1; w < TEAMS; ++w) M = fmaxf(M, s_ml[w][0][u]);
#pragma unroll
            for (int w = 0; w < TEAMS; ++w) L += q4_exp2(s_ml[w][0][u] - M) * s_ml[w][1][u];
            finish<HD>(a, head0, n0, kvh * G, u, split, d, s, M, L);
        }
    }
}

// The splits merged: a workgroup per (sequence, query head) for the output, then workgroups per 1,024
// rows of a kv head for the gathered weights.  A chain of loads and two exchanges: 4 us, with the weights
// of 33,000 rows of 2 heads (4.2 MB of scores) 7.
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
    const dim3 grid(heads, a.splits), block(kStepThreads);
    if (sizeof(T) == 2 && a.planes_q == 1) hipLaunchKernelGGL((q4_step<HD, sizeof(T) == 2 ? 1 : 2, T>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((q4_step<HD, 2, T>), grid, block, 0, s, a);
    if (a.part) {
        const int chunks = a.weights ? (a.c.maxp + kMergeRows - 1) / kMergeRows : 0;
        hipLaunchKernelGGL(q4_step_merge<HD>, dim3(a.group + chunks, heads), dim3(kMergeThreads), 0, s, a);
    }
}

}  // namespace

// Rows of one step of a workgroup: a tile of each team.
static int64_t step_unit(int hd) { return hd == 256 ? 2 * kTile : 4 * kTile; }

// Rows of a split: 512 workgroups (two per CU) where rows are few, 512 rows where that leaves more, and
// no more than 2,048 workgroups.  16 sequences of up to 8,192 rows of 2 heads of 256: 512 rows 25.3 us,
// 256 28.8; one of 33,000: 192 rows 16.6 + 7.1 for the merge, 128 17.4 + 9.1, 64 21.0 + 15.1; 32 of up to
// 16,384 of 8 heads of 128, where all have 512 rows at least: 2,048 rows 80 us, 1,024 81, 512 96.
Q4StepPlan plan_q4_step(int64_t rows, int64_t heads, int hd) {
    const int64_t unit = step_unit(hd);
    const int64_t total = rows * heads;
    int64_t per = std::min(total / 512, std::max<int64_t>(512, total / 2048));
    per = std::max<int64_t>((per + unit - 1) / unit * unit, unit);
    per = std::max<int64_t>(per, (rows + kMaxSplits - 1) / kMaxSplits);
    per = (per + kTile - 1) / kTile * kTile;
    return {static_cast<int>(per), static_cast<int>((rows + per - 1) / per)};
}

int64_t most_q4_head_splits(int64_t rows, int64_t heads, int hd) {
    const int64_t unit = step_unit(hd);
    // rows per split are at least a step's, and at least a 2,048th of rows * heads, rounded down from 512
    // or more (which can make 4 splits more)
    return std::min<int64_t>({heads * ((rows + unit - 1) / unit), 2052 + 2 * heads, heads * kMaxSplits});
}

void launch_q4_step(const AttnQ4Args &a, hipStream_t s) {
    switch (a.c.hd) {
        case 64: a.in_f32 ? launch_typed<64, float>(a, s) : launch_typed<64, uint16_t>(a, s); break;
        case 128: a.in_f32 ? launch_typed<128, float>(a, s) : launch_typed<128, uint16_t>(a, s); break;
        default: a.in_f32 ? launch_typed<256, float>(a, s) : launch_typed<256, uint16_t>(a, s); break;
    }
}

}  // namespace swq
