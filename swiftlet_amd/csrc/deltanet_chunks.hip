// The gated DeltaNet block over prompts (swq_deltanet_tokens): 64 tokens of a sequence at a time on the matrix cores.
//
// With c_i the sum of log g up to token i of a chunk, S the state [dk][dv] before it and rows k_i, q_i, v_i:
//   d = U - W S              what each token writes, U = T (b v), W = T (b e^c k), T = (1 + A)^-1,
//                            A_ij = b_i e^(c_i - c_j) k_i.k_j for i > j
//   o = e^c (q S) + P d      P_ij = e^(c_i - c_j) q_i.k_j for i >= j
//   S = e^c_last S + k^T (e^(c_last - c) d)
// which is the token after token recurrence written out.  Three launches:
//   prepare  per (chunk, value head), all chunks at once: convolution, norms, gates, A, T, W, U, P;
//   chain    per (sequence, value head, 16 to 64 columns of S), chunk after chunk: d, o, S;
//   finish   the gated norm, and the ring's rows.
//
// Numbers.  f32 numbers meet on the f16 matrix cores as two f16 numbers each, x = hi + lo / 2048 with lo = (x - hi) *
// 2048, and three products (hi hi, and hi lo + lo hi in sums of their own): 22 bits.  k, q, W and T stay inside
// f16's range by themselves: |k|, |q| <= 1, and b, g <= 1, so that a step of the rule lengthens nothing.  v, d and S do
// not: a power of two per (sequence, head, column group), from the largest v and S, brings them to about 1; S
// grows by sqrt(tokens) at most from there.  Sums are f32, c is summed and subtracted in 64 bits, and T is made by f32
// substitution and f32 matrix instructions.  Where projections and out are bf16, q S and P d take the high parts alone:
// their terms are off by 2^-12, an eighth of what the projections' own rounding makes them.
//
// Layout.  A matrix instruction's result has a lane's 4 numbers in consecutive rows of one column; its operands have 8
// numbers along the contraction.  The order of a contraction is free, so operands take the order in which two
// results lie: position j of lane group g is element 16 (j / 4) + 4 g + j % 4 of 32.  Every result then is the next
// product's operand after rounding alone, and all operands lie in the workspace as lanes load them, 16 bytes each.
#include <algorithm>

#include "deltanet.hpp"
#include "route.hpp"

namespace swq {
namespace {

typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr int kC = kDnChunk;
constexpr int kRowTiles = kC / 16;
constexpr int kPrepThreads = 512;
constexpr int kChainThreads = 512;
constexpr int kFinishThreads = 256;
constexpr int kVBlock = 128;  // columns of v that are prepared at once
constexpr float kLo = 2048.f, kLoInv = 1.f / 2048.f;

// The workspace: operands of every (chunk, key head) and (chunk, value head).
struct DnChunks {
    uint4 *k, *q, *w, *p;  // f16 operands; k, w two planes, q, p `planes`
    f4_t *u;               // [chunk][nv][dv / 16][4][64]
    float *decay;          // [chunk][nv][2][64]: e^c_i and e^(c_last - c_i)
    float *vmax;           // [chunk][nv]
    float *o;              // [N][nv * dv]: the outputs before their norm
    int32_t cap;           // chunks that there is room for
    int32_t planes;
};

__device__ __forceinline__ f4_t mfma16(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4_t mfma4(float a, float b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Values that are in their registers before any branch that follows.  The compiler counts the wait states from a matrix
// instruction to the first use of its result over the branch's longer way alone where both meet again, and on the
// shorter one the last elements were used before they were there; so no branch stands between the two, and chunks
// that do not exist are loaded as the last one again.
__device__ __forceinline__ void here(f4_t &v) { asm volatile("" : "+v"(v)); }

__device__ __forceinline__ void split4(f4_t x, h4_t &hi, h4_t &lo) {
    hi = __builtin_convertvector(x, h4_t);
    lo = __builtin_convertvector((x - __builtin_convertvector(hi, f4_t)) * kLo, h4_t);
}
__device__ __forceinline__ h8_t join(h4_t a, h4_t b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ h8_t as_h8(uint4 u) { return __builtin_bit_cast(h8_t, u); }
__device__ __forceinline__ uint4 as_u4(h8_t h) { return __builtin_bit_cast(uint4, h); }
__device__ __forceinline__ uint2 as_u2(h4_t h) { return __builtin_bit_cast(uint2, h); }

// Operand of 8 f32 numbers, high and low parts.
struct Op {
    h8_t hi, lo;
};
__device__ __forceinline__ Op op_of(f4_t a, f4_t b) {
    h4_t ah, al, bh, bl;
    split4(a, ah, al);
    split4(b, bh, bl);
    return {join(ah, bh), join(al, bl)};
}
// Products of 22-bit numbers: the high parts' sum and that of the mixed ones, 2048 times as large.
struct Acc {
    f4_t main, cross;
    __device__ __forceinline__ void clear() { main = cross = f4_t{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void add(h8_t ah, h8_t al, h8_t bh, h8_t bl) {
        main = mfma16(ah, bh, main);
        cross = mfma16(ah, bl, cross);
        cross = mfma16(al, bh, cross);
    }
    __device__ __forceinline__ f4_t sum() const { return main + cross * kLoInv; }
};

// A power of two that brings m to 1 .. 2, and its inverse; 1 where m is 0 or no number.
__device__ __forceinline__ float scale_of(float m, float &inverse) {
    int e = static_cast<int>((__float_as_uint(m) >> 23) & 255u);
    if (e == 255 || !(m > 0.f)) e = 127;
    e = min(max(e, 2), 252);
    inverse = __uint_as_float(static_cast<uint32_t>(e) << 23);
    return __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}

// The chunk's place: sequence b, chunk m of it.  Sequence b has its chunks from first(b) / 64 + b on, so that those of
// no two sequences meet where starts rise, and none lies past cap wherever starts point.
__device__ __forceinline__ int chunk_base(const DnTokens &a, int b) { return a.first(b) / kC + b; }
__device__ __forceinline__ bool find_chunk(const DnTokens &a, int chunk, int &b, int &m) {
    const int lane = threadIdx.x & (kWave - 1);
    int below = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
        const bool is = b0 + lane < a.B && chunk_base(a, min(b0 + lane, a.B - 1)) <= chunk;
        below += __builtin_popcountll(__ballot(is));
    }
    b = max(below - 1, 0);
    m = chunk - chunk_base(a, b);
    return m >= 0 && m < (a.count(b) + kC - 1) / kC && a.state(b) != nullptr;
}

__device__ __forceinline__ f4_t load4(const float *p) { return *reinterpret_cast<const f4_t *>(p); }
__device__ __forceinline__ f4_t load4(const uint16_t *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return f4_t{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u)};
}

// silu by the hardware's exponential and reciprocal: off by less than 2^-22 of the larger of 1 and the value.
__device__ __forceinline__ float silu_hw(float v) { return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504f)); }

// Four bf16 or f32 numbers as they are loaded.
template <typename T>
struct Four;
template <>
struct Four<float> {
    f4_t v;
    __device__ __forceinline__ void load(const float *p) { v = *reinterpret_cast<const f4_t *>(p); }
    __device__ __forceinline__ f4_t get() const { return v; }
};
template <>
struct Four<uint16_t> {
    uint2 u;
    __device__ __forceinline__ void load(const uint16_t *p) { u = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ f4_t get() const {
        return f4_t{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u)};
    }
};

// Convolution and silu of a tile of 16 tokens, N of them per lane from `tau` on (places in the sequence) and 4 mixed channels
// from ch on, whose elements lie at `at`: a row's channels side by side over the lanes, a token's earlier rows in
// registers.  Zeros for tokens that the sequence does not have.  KM: rows of the kernel that are held, 4 or 8; shorter
// kernels have zero weights in front.
template <int KM, int N, typename T>
__device__ __forceinline__ void conv_tile(const DnTokens &a, const T *x, const float *ring, uint32_t pos, int tokens, int tau, int at, int ch, f4_t (&y)[N]) {
    Four<T> rows[N + KM - 1];
#pragma unroll
    for (int i = 0; i < N + KM - 1; ++i) rows[i].load(x + min(max(tau + i - (KM - 1), 0), tokens - 1) * a.qkvz_stride + at);
    f4_t w[KM];
    if (KM == 4 && a.K == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f4_t k = load4(a.conv_w + 4 * (ch + e));
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j][e] = k[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < KM; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[j][e] = j >= KM - a.K ? a.conv_w[static_cast<int64_t>(ch + e) * a.K + j - (KM - a.K)] : 0.f;
    }
    f4_t win[KM];
#pragma unroll
    for (int j = 0; j < KM - 1; ++j) win[j + 1] = rows[j].get();
    if (tau < KM - 1) {
        // rows before the sequence's first, from its ring; those of zero weights are any
#pragma unroll
        for (int j = 0; j < KM - 1; ++j)
            if (tau + j < KM - 1)
                win[j + 1] = j >= KM - a.K ? load4(ring + static_cast<int64_t>((pos + static_cast<uint32_t>(tau + 1 + j - (KM - a.K))) % a.K) * a.convD + ch) : f4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int j = 0; j < KM - 1; ++j) win[j] = win[j + 1];
        win[KM - 1] = rows[i + KM - 1].get();
        f4_t acc = w[0] * win[0];
#pragma unroll
        for (int j = 1; j < KM; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(w[j][e], win[j][e], acc[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[i][e] = tau + i < tokens ? silu_hw(acc[e]) : 0.f;
    }
}

// Block (row tile, column tile) of a lower triangular matrix of 4 x 4 blocks of 16 x 16, rows 20 apart.
constexpr int kTriRow = 20;
__device__ __forceinline__ constexpr int tri(int rt, int ct) { return (rt * (rt + 1) / 2 + ct) * 16 * kTriRow; }

// A block product's operands for the f32 instruction at contraction step s: element (lane % 16, 4 (lane / 16) + s).
__device__ __forceinline__ float tri_a(const float *blk, int lane, int s) { return blk[(lane & 15) * kTriRow + 4 * (lane >> 4) + s]; }
// Element (4 (lane / 16) + s, lane % 16).
__device__ __forceinline__ float tri_b(const float *blk, int lane, int s) { return blk[(4 * (lane >> 4) + s) * kTriRow + (lane & 15)]; }
__device__ __forceinline__ f4_t tri_mul(const float *x, const float *y, int lane, f4_t c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = mfma4(tri_a(x, lane, s), tri_b(y, lane, s), c);
    return c;
}
// x times a result y.
__device__ __forceinline__ f4_t tri_mul(const float *x, f4_t y, int lane, f4_t c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = mfma4(tri_a(x, lane, s), y[s], c);
    return c;
}
__device__ __forceinline__ void tri_put(float *blk, f4_t v, int lane) {
#pragma unroll
    for (int r = 0; r < 4; ++r) blk[(4 * (lane >> 4) + r) * kTriRow + (lane & 15)] = v[r];
}

// The inverse of 1 + blk (strictly lower triangular), in its place: each lane a column, by substitution.
__device__ __forceinline__ void tri_invert(float *blk, int lane) {
    const int n = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float v = i == n ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) v = fmaf(-blk[i * kTriRow + j], x[j], v);
        x[i] = v;
    }
    // every lane has read before any writes: they are one wave
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (lane < 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) blk[i * kTriRow + n] = x[i];
    }
}

// One workgroup per (chunk, value head).  Waves 0 to 3 take a key tile of 16 tokens each, waves 4 to 7 a query
// tile, then P and the values while the others make T.
template <int DK, bool HQ, int KM, typename T>
__global__ __launch_bounds__(kPrepThreads, 4) void deltanet_prepare_kernel(const DnTokens a, const DnChunks w) {
    constexpr int KS = DK / 32, DT = DK / 16, PL = HQ ? 2 : 1;
    __shared__ uint4 s_kv[kRowTiles * (kVBlock / 32) * 2 * kWave];  // keys by tokens; then values, transposed
    __shared__ uint4 s_kt[DT * 2 * 2 * kWave];                      // queries by tokens; then keys, transposed
    __shared__ __align__(16) float s_t[10 * 16 * kTriRow];
    __shared__ double s_c[kC];
    __shared__ float s_beta[kC], s_grown[kC], s_max[8];
    const int hv = blockIdx.x % a.nv, hk = hv / a.rep, ri = hv % a.rep;
    const int64_t chunk = blockIdx.x / a.nv;
    int b, m;
    if (!find_chunk(a, static_cast<int>(chunk), b, m)) return;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, g = lane >> 4;
    const int tokens = a.count(b), n0 = a.first(b), tile = wave & 3;
    const bool keys = wave < 4;
    const T *x0 = static_cast<const T *>(a.qkvz) + n0 * a.qkvz_stride;
    const float *ring = reinterpret_cast<const float *>(a.state(b));
    const uint32_t pos = a.position(b);
    const int v_base = 2 * a.keyD + hv * a.dv;
    const f4_t zero = {0.f, 0.f, 0.f, 0.f};

    // gates, and their logarithms' sums, in units of log 2
    if (wave == 0) {
        const int t = min(m * kC + lane, tokens - 1);
        const T *ba = static_cast<const T *>(a.ba) + (n0 + static_cast<int64_t>(t)) * a.ba_stride;
        const bool is = m * kC + lane < tokens;
        const float log_g = -expf(a.a_log[hv]) * softplus_acc(dn_load(ba, ba_at(a, hv, 1)) + a.dt_bias[hv]);
        // below 2^-149 a decay is 0 like any other, and sums stay exact beside it
        double c = is ? 1.4426950408889634 * static_cast<double>(fmaxf(log_g, -110.f)) : 0.0;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const double up = __shfl_up(c, d, kWave);
            if (lane >= d) c += up;
        }
        s_c[lane] = c;
        s_beta[lane] = is ? sigmoid_acc(dn_load(ba, ba_at(a, hv, 0))) : 0.f;
        const float grown = __builtin_amdgcn_exp2f(static_cast<float>(c));
        s_grown[lane] = grown;
        const double last = __shfl(c, kWave - 1, kWave);
        float *decay = w.decay + (chunk * a.nv + hv) * 2 * kC;
        decay[lane] = grown;
        decay[kC + lane] = __builtin_amdgcn_exp2f(static_cast<float>(last - c));
    }

    auto kv_at = [&](int t, int ks, int plane) { return ((t * KS + ks) * 2 + plane) * kWave; };
    auto kt_at = [&](int dt, int ks, int plane) { return ((dt * 2 + ks) * 2 + plane) * kWave; };
    // four tokens of four channels of a tile, transposed: `token` of the tile, `ch` of the operand's rows
    auto put_transposed = [&](uint4 *to, int token, int ch, const f4_t *v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h4_t hi, lo;
            split4(f4_t{v[0][e], v[1][e], v[2][e], v[3][e]}, hi, lo);
            uint2 *at = reinterpret_cast<uint2 *>(to + kt_at(ch / 16, tile >> 1, 0) + 16 * (token / 4) + ch % 16 + e) + (tile & 1);
            at[0] = as_u2(hi);
            at[2 * kWave] = as_u2(lo);
        }
    };

    // keys and queries, normalised: N tokens and 4 channels per lane
    constexpr int N = DK / 16;
    const int ch = 4 * (lane % (DK / 4)), t0 = N * (lane / (DK / 4));
    f4_t y[N];
    {
        const int c = (keys ? a.keyD : 0) + hk * DK + ch;
        conv_tile<KM, N>(a, x0, ring, pos, tokens, m * kC + 16 * tile + t0, mixed_at(a, c), c, y);
        uint4 *to = keys ? s_kv : s_kt;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float ss = y[i][0] * y[i][0] + y[i][1] * y[i][1] + y[i][2] * y[i][2] + y[i][3] * y[i][3];
            ss = segment_sum(ss, DK / 4);
            y[i] *= 1.0f / __fsqrt_rn(ss + DK * 1e-6f);
            h4_t hi, lo;
            split4(y[i], hi, lo);
            uint2 *at = reinterpret_cast<uint2 *>(to + kv_at(tile, ch / 32, 0) + t0 + i + 16 * (ch % 16 / 4)) + ch / 16 % 2;
            at[0] = as_u2(hi);
            at[2 * kWave] = as_u2(lo);
        }
    }
    // a wave reads its own tile back as operands, the queries' before keys take their place
    asm volatile("" ::: "memory");
    Op x[KS];
    auto read_back = [&](const uint4 *from) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x[ks] = {as_h8(from[kv_at(tile, ks, 0) + lane]), as_h8(from[kv_at(tile, ks, 1) + lane])};
    };
    if (!keys) read_back(s_kt);
    lds_barrier();
    if (keys) {
#pragma unroll
        for (int i = 0; i < N; i += 4) put_transposed(s_kt, t0 + i, ch, y + i);
        read_back(s_kv);
    } else if (ri == 0) {
        uint4 *q = w.q + (chunk * a.nk + hk) * (kRowTiles * KS * PL * kWave) + tile * KS * PL * kWave + lane;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            q[ks * PL * kWave] = as_u4(x[ks].hi);
            if (HQ) q[(ks * PL + 1) * kWave] = as_u4(x[ks].lo);
        }
    }

    // k_i.k_j and k_j.q_i of the lower triangle's tiles
    auto fade = [&](int i, int j) { return __builtin_amdgcn_exp2f(static_cast<float>(s_c[i] - s_c[j])); };
    if (keys) {
        for (int jt = 0; jt <= tile; ++jt) {
            Acc acc;
            acc.clear();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) acc.add(x[ks].hi, x[ks].lo, as_h8(s_kv[kv_at(jt, ks, 0) + lane]), as_h8(s_kv[kv_at(jt, ks, 1) + lane]));
            f4_t d = acc.sum();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * tile + 4 * g + e, j = 16 * jt + col;
                d[e] = i > j ? d[e] * s_beta[i] * fade(i, j) : 0.f;
            }
            tri_put(s_t + tri(tile, jt), d, lane);
        }
        // the diagonal block's inverse, by the wave that has just written it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        tri_invert(s_t + tri(tile, tile), lane);
    } else {
        uint4 *p = w.p + (chunk * a.nv + hv) * (kRowTiles * 2 * PL * kWave) + tile * 2 * PL * kWave + lane;
        for (int ks2 = 0; ks2 <= tile / 2; ++ks2) {
            f4_t d[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int jt = 2 * ks2 + half;
                d[half] = zero;
                if (jt > tile) continue;
                Acc acc;
                acc.clear();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const h8_t kh = as_h8(s_kv[kv_at(jt, ks, 0) + lane]);
                    if constexpr (HQ) acc.add(kh, as_h8(s_kv[kv_at(jt, ks, 1) + lane]), x[ks].hi, x[ks].lo);
                    else acc.main = mfma16(kh, x[ks].hi, acc.main);
                }
                d[half] = HQ ? acc.sum() : acc.main;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 16 * tile + col, j = 16 * jt + 4 * g + e;
                    d[half][e] = i >= j ? d[half][e] * fade(i, j) : 0.f;
                }
            }
            const Op o = op_of(d[0], d[1]);
            p[ks2 * PL * kWave] = as_u4(o.hi);
            if (HQ) p[(ks2 * PL + 1) * kWave] = as_u4(o.lo);
        }
    }
    lds_barrier();

    // T below the diagonal blocks, while waves 4 to 7 have the values
    constexpr int VN = kVBlock / 16;
    const int vch = 4 * (lane % (kVBlock / 4)), vt0 = VN * (lane / (kVBlock / 4));
    f4_t v[VN];
    auto values = [&](int c0) {  // columns c0 .. of this wave's tile, and their largest
        float most = 0.f;
        const int c = v_base + min(c0 + vch, a.dv - 4);
        conv_tile<KM, VN>(a, x0, ring, pos, tokens, m * kC + 16 * tile + vt0, mixed_at(a, c), c, v);
#pragma unroll
        for (int i = 0; i < VN; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(v[i][e]));
        most = wave_max_all(most);
        if (lane == 0) s_max[wave] = most;
    };
    if (keys) {
        if (wave < 2) {
            const int i = 2 * wave + 1, j = 2 * wave;
            const f4_t t = tri_mul(s_t + tri(i, j), s_t + tri(j, j), lane, zero);
            tri_put(s_t + tri(i, j), -tri_mul(s_t + tri(i, i), t, lane, zero), lane);
        }
    } else {
        values(0);
    }
    lds_barrier();
    float vmax = fmaxf(fmaxf(s_max[4], s_max[5]), fmaxf(s_max[6], s_max[7]));
    float v_inv;
    float v_scale = scale_of(vmax, v_inv);
    auto put_values = [&]() {
#pragma unroll
        for (int i = 0; i < VN; ++i) v[i] *= v_scale;
#pragma unroll
        for (int i = 0; i < VN; i += 4) put_transposed(s_kv, vt0 + i, vch, v + i);
    };
    if (wave < 2) {
        // columns of the lower left 32 x 32 part
        const int q = wave;
        f4_t x2 = zero, x3 = zero;
        for (int s = q; s < 2; ++s) {
            x2 = tri_mul(s_t + tri(2, s), s_t + tri(s, q), lane, x2);
            x3 = tri_mul(s_t + tri(3, s), s_t + tri(s, q), lane, x3);
        }
        const f4_t t2 = -tri_mul(s_t + tri(2, 2), x2, lane, zero);
        const f4_t t3 = -tri_mul(s_t + tri(3, 3), x3, lane, tri_mul(s_t + tri(3, 2), x2, lane, zero));
        // the blocks are read by this wave (and, of the first column, by the other) until here
        lds_barrier();
        tri_put(s_t + tri(2, q), t2, lane);
        tri_put(s_t + tri(3, q), t3, lane);
    } else {
        if (!keys) put_values();
        lds_barrier();
    }
    lds_barrier();

    // T's rows as operands: 8 of T_ij times b_j (and e^c_j) for i of this wave's tile
    Op tu[2], tw[2];
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
        f4_t u[2], e_u[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int jt = 2 * ks2 + half, j = 16 * jt + 4 * g;
            u[half] = jt <= tile ? *reinterpret_cast<const f4_t *>(s_t + tri(tile, jt) + col * kTriRow + 4 * g) : zero;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u[half][e] *= s_beta[j + e];
                e_u[half][e] = u[half][e] * s_grown[j + e];
            }
        }
        tu[ks2] = op_of(u[0], u[1]);
        tw[ks2] = op_of(e_u[0], e_u[1]);
    }
    const int half_of = wave >> 2, last = tile / 2;  // contraction steps past `last` are zeros
    {
        uint4 *to = w.w + (chunk * a.nv + hv) * (kRowTiles * KS * 2 * kWave) + tile * KS * 2 * kWave + lane;
        uint4 *k_to = w.k + (chunk * a.nk + hk) * (DT * 2 * 2 * kWave) + lane;
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
            const int ks = half_of * (KS / 2) + i;
            f4_t d[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int dt = 2 * ks + half;
                Acc acc;
                acc.clear();
                for (int ks2 = 0; ks2 < 2; ++ks2) {
                    const uint4 kh = s_kt[kt_at(dt, ks2, 0) + lane], kl = s_kt[kt_at(dt, ks2, 1) + lane];
                    if (ks2 <= last) acc.add(as_h8(kh), as_h8(kl), tw[ks2].hi, tw[ks2].lo);
                    if (ri == 0 && (dt & 3) == tile) {
                        k_to[(dt * 2 + ks2) * 2 * kWave] = kh;
                        k_to[((dt * 2 + ks2) * 2 + 1) * kWave] = kl;
                    }
                }
                d[half] = acc.sum();
            }
            const Op o = op_of(d[0], d[1]);
            to[ks * 2 * kWave] = as_u4(o.hi);
            to[(ks * 2 + 1) * kWave] = as_u4(o.lo);
        }
    }
    f4_t *u_to = w.u + (chunk * a.nv + hv) * (a.dv / 16 * kRowTiles * kWave) + lane;
    for (int c0 = 0;;) {
        for (int i = half_of; i < kVBlock / 16 && c0 + 16 * i < a.dv; i += 2) {
            Acc acc;
            acc.clear();
            for (int ks2 = 0; ks2 <= last; ++ks2)
                acc.add(tu[ks2].hi, tu[ks2].lo, as_h8(s_kv[kt_at(i, ks2, 0) + lane]), as_h8(s_kv[kt_at(i, ks2, 1) + lane]));
            u_to[((c0 / 16 + i) * kRowTiles + tile) * kWave] = acc.sum() * v_inv;
        }
        c0 += kVBlock;
        if (c0 >= a.dv) break;
        // heads of more than 128 values: the next of them
        lds_barrier();
        if (!keys) values(c0);
        lds_barrier();
        const float now = fmaxf(fmaxf(s_max[4], s_max[5]), fmaxf(s_max[6], s_max[7]));
        vmax = fmaxf(vmax, now);
        v_scale = scale_of(now, v_inv);
        if (!keys) put_values();
        lds_barrier();
    }
    if (tid == 0) w.vmax[chunk * a.nv + hv] = vmax;
}

// One workgroup per (sequence, value head, CT * 16 columns of the state).  Waves 0 to 3 hold the state's rows and make
// d and the next state; waves 4 to 7 make the outputs, off the chain from chunk to chunk.
template <int DK, int CT, bool HQ>
__global__ __launch_bounds__(kChainThreads) void deltanet_chain_kernel(const DnTokens a, const DnChunks w, int groups) {
    constexpr int KS = DK / 32, DT = DK / 64, PL = HQ ? 2 : 1;  // DT: row tiles of the state per wave
    __shared__ uint4 s_s[CT * KS * 2 * kWave], s_d[CT * 2 * PL * kWave], s_e[CT * 2 * 2 * kWave];
    __shared__ float s_max[8];
    // workgroups of one key head on one XCD (they are handed out round robin): its L2 then has what they share
    const int xcd = blockIdx.x & 7, rest = blockIdx.x >> 3;
    const int unit = rest / (groups * a.rep) * 8 + xcd, within = rest % (groups * a.rep);
    if (unit >= a.B * a.nk) return;
    const int b = unit / a.nk, hk = unit % a.nk, hv = hk * a.rep + within / groups, c0 = within % groups * CT * 16;
    const int tokens = a.count(b);
    uint8_t *slot = a.state(b);
    if (tokens <= 0 || !slot) return;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, g = lane >> 4;
    const int chunks = (tokens + kC - 1) / kC, tile = wave & 3;
    const int64_t n0 = a.first(b), first = chunk_base(a, b);
    const f4_t zero = {0.f, 0.f, 0.f, 0.f};

    // the state's columns, a lane's 4 rows side by side in memory
    f4_t st[DT][CT];
    float *state = reinterpret_cast<float *>(slot + a.rec_at) + (static_cast<int64_t>(hv) * a.dv + c0 + col) * DK + 4 * g;
    float most = 0.f;
    if (wave < 4) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                st[t][c] = *reinterpret_cast<const f4_t *>(state + static_cast<int64_t>(16 * c) * DK + 16 * (wave * DT + t));
#pragma unroll
                for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(st[t][c][e]));
            }
    }
    for (int i = tid; i < chunks; i += kChainThreads) most = fmaxf(most, w.vmax[(first + i) * a.nv + hv]);
    most = wave_max_all(most);
    if (lane == 0) s_max[wave] = most;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, s_max[i]);
    float inverse;
    const float scale = scale_of(most, inverse);

    auto put_state = [&]() {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int dt = wave * DT + t;
                h4_t hi, lo;
                split4(st[t][c], hi, lo);
                reinterpret_cast<uint2 *>(s_s + ((c * KS + dt / 2) * 2) * kWave + lane)[dt & 1] = as_u2(hi);
                reinterpret_cast<uint2 *>(s_s + ((c * KS + dt / 2) * 2 + 1) * kWave + lane)[dt & 1] = as_u2(lo);
            }
    };
    if (wave < 4) {
        const uint4 *wp = w.w + (first * a.nv + hv) * (kRowTiles * KS * 2 * kWave) + tile * KS * 2 * kWave + lane;
        const f4_t *up = w.u + ((first * a.nv + hv) * (a.dv / 16) + c0 / 16) * kRowTiles * kWave + tile * kWave + lane;
        const uint4 *kp = w.k + (first * a.nk + hk) * (4 * DT * 2 * 2 * kWave) + wave * DT * 2 * 2 * kWave + lane;
        const float *dp = w.decay + (first * a.nv + hv) * 2 * kC;
        const int64_t w_step = static_cast<int64_t>(a.nv) * kRowTiles * KS * 2 * kWave, u_step = static_cast<int64_t>(a.nv) * (a.dv / 16) * kRowTiles * kWave,
                      k_step = static_cast<int64_t>(a.nk) * 4 * DT * 2 * 2 * kWave, d_step = static_cast<int64_t>(a.nv) * 2 * kC;
        uint4 wr[KS][2], kr[DT][2][2];
        f4_t ur[CT], late;
        float grown;
        auto load_w = [&]() {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int p = 0; p < 2; ++p) wr[ks][p] = wp[(ks * 2 + p) * kWave];
#pragma unroll
            for (int c = 0; c < CT; ++c) ur[c] = up[c * kRowTiles * kWave];
            late = *reinterpret_cast<const f4_t *>(dp + kC + 16 * tile + 4 * g);
            grown = dp[kC - 1];
        };
        auto load_k = [&]() {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                    for (int p = 0; p < 2; ++p) kr[t][ks2][p] = kp[((t * 2 + ks2) * 2 + p) * kWave];
        };
        load_w();
        load_k();
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c) st[t][c] *= scale;
        put_state();
        for (int m = 0; m < chunks; ++m) {
            lds_barrier();
            const float keep = grown;
            const bool more = m + 1 < chunks;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                Acc acc;
                acc.clear();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    acc.add(as_h8(wr[ks][0]), as_h8(wr[ks][1]), as_h8(s_s[((c * KS + ks) * 2) * kWave + lane]), as_h8(s_s[((c * KS + ks) * 2 + 1) * kWave + lane]));
                const f4_t d = ur[c] * scale - acc.sum();
                h4_t hi, lo;
                split4(d, hi, lo);
                reinterpret_cast<uint2 *>(s_d + ((c * 2 + tile / 2) * PL) * kWave + lane)[tile & 1] = as_u2(hi);
                if (HQ) reinterpret_cast<uint2 *>(s_d + ((c * 2 + tile / 2) * PL + 1) * kWave + lane)[tile & 1] = as_u2(lo);
                split4(d * late, hi, lo);
                reinterpret_cast<uint2 *>(s_e + ((c * 2 + tile / 2) * 2) * kWave + lane)[tile & 1] = as_u2(hi);
                reinterpret_cast<uint2 *>(s_e + ((c * 2 + tile / 2) * 2 + 1) * kWave + lane)[tile & 1] = as_u2(lo);
            }
            wp += more ? w_step : 0;
            up += more ? u_step : 0;
            dp += more ? d_step : 0;
            load_w();
            lds_barrier();
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                h8_t e[2][2];
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                    for (int p = 0; p < 2; ++p) e[ks2][p] = as_h8(s_e[((c * 2 + ks2) * 2 + p) * kWave + lane]);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    Acc acc;
                    acc.main = st[t][c] * keep;
                    acc.cross = zero;
#pragma unroll
                    for (int ks2 = 0; ks2 < 2; ++ks2) acc.add(as_h8(kr[t][ks2][0]), as_h8(kr[t][ks2][1]), e[ks2][0], e[ks2][1]);
                    st[t][c] = acc.sum();
                }
            }
            kp += more ? k_step : 0;
            load_k();
            put_state();
        }
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c)
                *reinterpret_cast<f4_t *>(state + static_cast<int64_t>(16 * c) * DK + 16 * (wave * DT + t)) = st[t][c] * inverse;
    } else {
        const uint4 *qp = w.q + (first * a.nk + hk) * (kRowTiles * KS * PL * kWave) + tile * KS * PL * kWave + lane;
        const uint4 *pp = w.p + (first * a.nv + hv) * (kRowTiles * 2 * PL * kWave) + tile * 2 * PL * kWave + lane;
        const float *dp = w.decay + (first * a.nv + hv) * 2 * kC;
        const int64_t q_step = static_cast<int64_t>(a.nk) * kRowTiles * KS * PL * kWave, p_step = static_cast<int64_t>(a.nv) * kRowTiles * 2 * PL * kWave,
                      d_step = static_cast<int64_t>(a.nv) * 2 * kC;
        const int last = tile / 2;
        uint4 qr[KS][PL], pr[2][PL];
        f4_t grown;
        auto load_q = [&]() {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int p = 0; p < PL; ++p) qr[ks][p] = qp[(ks * PL + p) * kWave];
            grown = *reinterpret_cast<const f4_t *>(dp + 16 * tile + 4 * g);
        };
        auto load_p = [&]() {
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                for (int p = 0; p < PL; ++p) pr[ks2][p] = ks2 <= last ? pp[(ks2 * PL + p) * kWave] : make_uint4(0, 0, 0, 0);
        };
        load_q();
        load_p();
        const float back = inverse / __fsqrt_rn(static_cast<float>(DK));
        float *o = w.o + (n0 + 16 * tile + 4 * g) * a.nv * a.dv + hv * a.dv + c0 + col;
        for (int m = 0; m < chunks; ++m) {
            lds_barrier();
            const bool more = m + 1 < chunks;
            f4_t part[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                Acc acc;
                acc.clear();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const h8_t sh = as_h8(s_s[((c * KS + ks) * 2) * kWave + lane]);
                    if constexpr (HQ) acc.add(as_h8(qr[ks][0]), as_h8(qr[ks][PL - 1]), sh, as_h8(s_s[((c * KS + ks) * 2 + 1) * kWave + lane]));
                    else acc.main = mfma16(as_h8(qr[ks][0]), sh, acc.main);
                }
                part[c] = (HQ ? acc.sum() : acc.main) * grown;
            }
            qp += more ? q_step : 0;
            dp += more ? d_step : 0;
            load_q();
            lds_barrier();
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                Acc acc;
                acc.main = part[c];
                acc.cross = zero;
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2) {
                    const h8_t dh = as_h8(s_d[((c * 2 + ks2) * PL) * kWave + lane]);
                    if constexpr (HQ) acc.add(as_h8(pr[ks2][0]), as_h8(pr[ks2][PL - 1]), dh, as_h8(s_d[((c * 2 + ks2) * PL + PL - 1) * kWave + lane]));
                    else acc.main = mfma16(as_h8(pr[ks2][0]), dh, acc.main);
                }
                f4_t v = (HQ ? acc.sum() : acc.main) * back;
                here(v);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (m * kC + 16 * tile + 4 * g + e < tokens) o[static_cast<int64_t>(m * kC + e) * a.nv * a.dv + 16 * c] = v[e];
            }
            pp += more ? p_step : 0;
            load_p();
        }
    }
}

// The gated norm of a chunk's outputs, and the ring's rows of a sequence's last one.  `parts` workgroups share a chunk;
// a row (token, value head) has `lanes` lanes of 4 values, up to 4 times.
template <typename T>
__global__ __launch_bounds__(kFinishThreads) void deltanet_finish_kernel(const DnTokens a, const DnChunks w, int parts, int lanes) {
    const int part = blockIdx.x % parts;
    int b, m;
    if (!find_chunk(a, static_cast<int>(blockIdx.x / parts), b, m)) return;
    const int tid = threadIdx.x, tokens = a.count(b), lane = tid % lanes, here = min(tokens - m * kC, kC);
    const int64_t n0 = a.first(b) + static_cast<int64_t>(m) * kC;
    const T *x = static_cast<const T *>(a.qkvz) + n0 * a.qkvz_stride;
    for (int row = part * (kFinishThreads / lanes) + tid / lanes; row < here * a.nv; row += parts * (kFinishThreads / lanes)) {
        const int t = row / a.nv, hv = row % a.nv;
        const int64_t at = (n0 + t) * a.nv * a.dv + hv * a.dv;
        f4_t v[4], z[4];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * (lane + i * lanes);
            if (e >= a.dv) continue;
            v[i] = load4(w.o + at + e);
            z[i] = load4(x + t * a.qkvz_stride + z_at(a, hv, e));
            ss += v[i][0] * v[i][0] + v[i][1] * v[i][1] + v[i][2] * v[i][2] + v[i][3] * v[i][3];
        }
        const float sc = 1.0f / __fsqrt_rn(segment_sum(ss, lanes) / static_cast<float>(a.dv) + a.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * (lane + i * lanes);
            if (e >= a.dv) continue;
            const f4_t nw = {a.norm_w[e], a.norm_w[e + 1], a.norm_w[e + 2], a.norm_w[e + 3]};
            f4_t y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = v[i][k] * (sc * nw[k]) * silu_acc(z[i][k]);
            if (a.out_f32) {
                *reinterpret_cast<f4_t *>(static_cast<float *>(a.out) + at + e) = y;
            } else {
                const uint32_t lo = dn_bf16(y[0]) | static_cast<uint32_t>(dn_bf16(y[1])) << 16, hi = dn_bf16(y[2]) | static_cast<uint32_t>(dn_bf16(y[3])) << 16;
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at + e) = make_uint2(lo, hi);
            }
        }
    }
    if ((m + 1) * kC < tokens) return;
    float *ring = reinterpret_cast<float *>(a.state(b));
    const uint32_t pos = a.position(b);
    const T *first = static_cast<const T *>(a.qkvz) + a.first(b) * a.qkvz_stride;
    for (int ch = part * kFinishThreads + tid; ch < a.convD; ch += parts * kFinishThreads) {
        const int at = mixed_at(a, ch);
        for (int i = max(tokens - a.K, 0); i < tokens; ++i)
            ring[static_cast<int64_t>((pos + static_cast<uint32_t>(i)) % a.K) * a.convD + ch] = dn_load(first, i * a.qkvz_stride + at);
    }
}

// Whether outputs are made of two planes: unless projections and outputs are bf16.
int planes_of(const DnTokens &a, bool in_f32) { return in_f32 || a.out_f32 ? 2 : 1; }

// Parts of the workspace, at 256-byte boundaries; o only where the outputs are no f32.
struct Parts {
    size_t k, q, w, p, u, decay, vmax, o, total;
};
Parts parts_of(int64_t nk, int64_t nv, int64_t dk, int64_t dv, int64_t cap, int64_t tokens, int planes, bool with_o) {
    Parts s{};
    s.k = dn_align(cap * nk * dk * kC * 2 * 2);
    s.q = dn_align(cap * nk * dk * kC * planes * 2);
    s.w = dn_align(cap * nv * dk * kC * 2 * 2);
    s.p = dn_align(cap * nv * kC * kC * planes * 2);
    s.u = dn_align(cap * nv * dv * kC * 4);
    s.decay = dn_align(cap * nv * 2 * kC * 4);
    s.vmax = dn_align(cap * nv * 4);
    s.o = with_o ? dn_align(tokens * nv * dv * 4) : 0;
    s.total = s.k + s.q + s.w + s.p + s.u + s.decay + s.vmax + s.o;
    return s;
}
int64_t cap_of(int64_t sequences, int64_t tokens) { return tokens / kC + sequences; }

template <int DK, bool HQ, typename T>
void launch_prepare(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>(w.cap * a.nv)), block(kPrepThreads);
    if (a.K <= 4) hipLaunchKernelGGL((deltanet_prepare_kernel<DK, HQ, 4, T>), grid, block, 0, s, a, w);
    else hipLaunchKernelGGL((deltanet_prepare_kernel<DK, HQ, 8, T>), grid, block, 0, s, a, w);
}

template <int DK, bool HQ>
void launch_chain(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    const int64_t units = (static_cast<int64_t>(a.B) * a.nk + 7) / 8 * 8 * a.rep;
    const int groups = a.dv / 16;
    hipLaunchKernelGGL((deltanet_chain_kernel<DK, 1, HQ>), dim3(static_cast<uint32_t>(units * groups)), dim3(kChainThreads), 0, s, a, w, groups);
}

template <bool HQ>
void launch(const DnTokens &a, const DnChunks &w, bool in_f32, hipStream_t s) {
    if (a.dk == 64) {
        if (in_f32) launch_prepare<64, HQ, float>(a, w, s);
        else launch_prepare<64, HQ, uint16_t>(a, w, s);
        launch_chain<64, HQ>(a, w, s);
    } else {
        if (in_f32) launch_prepare<128, HQ, float>(a, w, s);
        else launch_prepare<128, HQ, uint16_t>(a, w, s);
        launch_chain<128, HQ>(a, w, s);
    }
    int lanes = 4;
    while (lanes < kWave && 4 * lanes < a.dv) lanes *= 2;
    const int parts = std::max(1, std::min(32, kC * a.nv * lanes / kFinishThreads / 8));
    const dim3 grid(static_cast<uint32_t>(w.cap) * parts), block(kFinishThreads);
    if (in_f32) hipLaunchKernelGGL(deltanet_finish_kernel<float>, grid, block, 0, s, a, w, parts, lanes);
    else hipLaunchKernelGGL(deltanet_finish_kernel<uint16_t>, grid, block, 0, s, a, w, parts, lanes);
}

}  // namespace

bool deltanet_chunks_take(const swq_deltanet_layer *l) {
    return (l->key_head_dim == 64 || l->key_head_dim == 128) && l->value_head_dim % 16 == 0;
}

bool deltanet_chunks_fit(const swq_deltanet_layer *l, int64_t sequences, int64_t tokens) {
    const int64_t most = 1LL << 23, chunks = cap_of(sequences, tokens), heads = (sequences * l->num_key_heads + 7) * (l->num_value_heads / l->num_key_heads);
    return chunks * std::max(l->num_value_heads, 32) < most && heads * (l->value_head_dim / 16) < most;
}

size_t deltanet_chunks_bytes(const swq_deltanet_layer *l, int64_t sequences, int64_t tokens) {
    return parts_of(l->num_key_heads, l->num_value_heads, l->key_head_dim, l->value_head_dim, cap_of(sequences, tokens), tokens, 2, true).total;
}

void launch_deltanet_chunks(const DnTokens &a, bool in_f32, void *ws, hipStream_t s) {
    DnChunks w{};
    w.cap = static_cast<int32_t>(cap_of(a.B, a.N));
    w.planes = planes_of(a, in_f32);
    const Parts parts = parts_of(a.nk, a.nv, a.dk, a.dv, w.cap, a.N, w.planes, !a.out_f32);
    uint8_t *p = static_cast<uint8_t *>(ws);
    auto take = [&](size_t n) {
        uint8_t *at = p;
        p += n;
        return at;
    };
    w.k = reinterpret_cast<uint4 *>(take(parts.k));
    w.q = reinterpret_cast<uint4 *>(take(parts.q));
    w.w = reinterpret_cast<uint4 *>(take(parts.w));
    w.p = reinterpret_cast<uint4 *>(take(parts.p));
    w.u = reinterpret_cast<f4_t *>(take(parts.u));
    w.decay = reinterpret_cast<float *>(take(parts.decay));
    w.vmax = reinterpret_cast<float *>(take(parts.vmax));
    w.o = a.out_f32 ? static_cast<float *>(a.out) : reinterpret_cast<float *>(p);
    if (w.planes == 2) launch<true>(a, w, in_f32, s);
    else launch<false>(a, w, in_f32, s);
}

}  // namespace swq
