// The gated DeltaNet block over prompts (swq_deltanet_tokens): 64 tokens of a sequence at a time on the matrix cores.
//
// With c_i the sum of log g up to token i of a chunk, S the state [dk][dv] before it and rows k_i, q_i, v_i:
//   d = U - W S              what each token writes, U = T (b v), W = T (b e^c k), T = (1 + A)^-1,
//                            A_ij = b_i e^(c_i - c_j) k_i.k_j for i > j
//   o = e^c (q S) + P d      P_ij = e^(c_i - c_j) q_i.k_j for i >= j
//   S = e^c_last S + k^T (e^(c_last - c) d)
// which is the token after token recurrence written out.  Four launches:
//   keys     per (chunk, key head), all chunks at once: convolution and norms of k and q, k.k and k.q, gates;
//   solve    per (chunk, value head), all chunks at once: convolution of v, A, T, W, U, P;
//   chain    per (sequence, value head, 16 or 32 columns of S), chunk after chunk: d, o, S;
//   finish   all chunks at once: the gated norm, and the ring's rows.
//
// Numbers.  f32 numbers meet on the f16 matrix cores as two f16 numbers each, x = hi + lo / 2048, and three products (hi
// hi, hi lo, lo hi; those with a lo are summed apart): 22 bits.  lo is 2048 times what hi leaves, as large as hi, so it
// keeps its bits wherever hi is a normal f16 number, and below that 2^-36 of 1 remains.  Powers of two bring numbers to the top
// of that range.  k, q, P and T are bounded by 1 and W by 8 (|k|, |q| <= 1 and b, g <= 1: a step of the rule lengthens
// nothing) and take fixed ones.  v, d and S have no bound.  In T (b v) each chunk's v are brought below 2^15, beside which
// numbers down to 2^-28 of the largest keep 22 bits.  In the chain one power per (sequence, head, columns), from the largest v
// and S, leaves room for what S can become: the writes of n tokens add at most their largest times sqrt(n) to its norm.
// For 64 tokens numbers down to 2^-24 of the largest keep 22 bits, for 2,048 down to 2^-22, for 2^20 2^-17; smaller
// ones lose a bit with each power of two.  Sums are f32, c is summed and subtracted in 64 bits, and T is made by f32
// substitution and f32 matrix instructions.  That holds whatever the types of the projections and of out: bf16 outputs are
// the f32 ones rounded once.
//
// What is not finite.  0 times it is no 0, and the triangles above T's and P's diagonals would carry it to earlier tokens.
// So keys, gates and values that are not finite are taken as 0 (log g: g = 1), and e^c is NaN from the first such token of
// a chunk on: outputs of that token and all after it are, and S is from the chunk's end on, as a whole where
// one value alone would spoil its row.  Queries reach their own token's outputs alone and need nothing.
//
// No branch stands between a matrix instruction and its result's first use (see `here`): chunks that do not exist are
// loaded as the last one again.
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
// Chunks of a prompt alone that go through all launches before the next do, 163 MB of operands at 16 key and 32 value heads
// of 128, which the caches hold from one launch to the next.  4,096 (16,384) tokens: spans of 16 277 us (1,129), 32 251
// (966), 64 303 (1,195), the whole prompt at once 303 (1,116).  It was found at these heads and does not follow others': 8
// value heads of 128 bring 41 MB.
constexpr int kSpan = 32;
constexpr int kRowTiles = kC / 16;
constexpr int kPrepThreads = 512;
constexpr int kChainThreads = 768;
constexpr int kFinishThreads = 256;
constexpr int kVBlock = 128;  // columns of v that are prepared at once
// What low parts are multiplied by, and T, W, P and q as operands: decays make the entries of T, W and P small beside 1 where
// the numbers they meet may be large; q's is P's, as their products meet in a sum.  W stays below 2^14.
constexpr float kLow = 2048.f, kScaleT = 2048.f;

// The workspace: operands of every (chunk, key head) and (chunk, value head).
struct DnChunks {
    uint4 *k, *q, *w, *p;  // f16 operands, two planes each
    f4_t *u;               // [chunk][nv][dv / 16][4][64]
    float *decay;          // [chunk][nv][2][64]: e^c_i, NaN from the first token with anything not finite on, and e^(c_last - c_i)
    double *sums;          // [chunk][nv][64]: c, in units of log 2
    float *beta;           // [chunk][nv][64]
    float *vmax;           // [chunk][nv]
    f4_t *dots;            // [chunk][nk][2][10][64]: k_i.k_j and k_j.q_i, tiles of the lower triangle
    f4_t *o;               // the outputs before their norm, as the results lie: [chunk][nv][dv / 16][4][64]
    int32_t cap;           // chunks that there is room for
    int32_t chunk0, span;  // a launch's chunks: those of a sequence from chunk0 on, span at most
    int32_t least;         // tokens of a sequence that comes through here
};

__device__ __forceinline__ f4_t mfma16(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4_t mfma4(float a, float b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ void split4(f4_t x, h4_t &hi, h4_t &lo) {
    hi = __builtin_convertvector(x, h4_t);
#pragma unroll
    for (int e = 0; e < 4; ++e) lo[e] = static_cast<_Float16>(kLow * fmaf(static_cast<float>(hi[e]), -1.0f, x[e]));
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
// A sum of products in 22 bits: of high parts, and of those that have a low part.
struct Sum {
    f4_t hi = {0.f, 0.f, 0.f, 0.f}, lo = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ f4_t get() const {
        f4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(lo[e], 1.f / kLow, hi[e]);
        return v;
    }
};
__device__ __forceinline__ void mfma22(h8_t ah, h8_t al, h8_t bh, h8_t bl, Sum &c) {
    c.lo = mfma16(ah, bl, mfma16(al, bh, c.lo));
    c.hi = mfma16(ah, bh, c.hi);
}

// A power of two that brings m to 2^top .. 2^(top + 1), and its inverse; 1 where m is 0 or no number.
__device__ __forceinline__ float scale_of(float m, int top, float &inverse) {
    int e = static_cast<int>((__float_as_uint(m) >> 23) & 255u);
    e = e == 255 || !(m > 0.f) ? 127 : min(max(e - top, 1), 253);
    inverse = __uint_as_float(static_cast<uint32_t>(e) << 23);
    return __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}

// Sequence b has its chunks' places in the workspace from first(b) / 64 + b on, so that those of no two sequences meet where
// starts rise, and none lies past cap wherever starts point.  A long prompt alone goes a span of chunks at a time, in the
// same places again.
__device__ __forceinline__ int chunk_base(const DnTokens &a, int b) { return a.B == 1 ? 0 : a.first(b) / kC + b; }

// A chunk: of sequence b the m-th, the sequence's first token, how many it has, tokens before them, its state.
struct Chunk {
    int b, m, n0, tokens;
    uint32_t pos;
    uint8_t *state;
};
// Whether the chunk exists.  Each lane loads all of a sequence, so that one of them is found in one round trip.
__device__ __forceinline__ bool find_chunk(const DnTokens &a, const DnChunks &w, int chunk, Chunk &c) {
    const int lane = threadIdx.x & (kWave - 1);
    int n0 = 0, tokens = 0, slot = -1, pos = 0;
    c.b = -1;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
        const int b = min(b0 + lane, a.B - 1);
        const int n = a.first(b), t = a.count(b), s = a.slot ? a.slot[b] : b, p = a.positions[b];
        const bool is = b0 + lane < a.B && (a.B == 1 || n / kC + b <= chunk);
        const uint64_t all = __ballot(is);
        if (all == 0) continue;
        const int from = 63 - __builtin_clzll(all);  // the last that starts no later
        c.b = b0 + from;
        n0 = __builtin_amdgcn_readlane(n, from);
        tokens = __builtin_amdgcn_readlane(t, from);
        slot = __builtin_amdgcn_readlane(s, from);
        pos = __builtin_amdgcn_readlane(p, from);
    }
    c.m = chunk - (a.B == 1 ? 0 : n0 / kC + c.b) + w.chunk0;
    c.n0 = n0;
    c.tokens = tokens;
    c.pos = static_cast<uint32_t>(max(pos, 0));
    c.state = slot >= 0 && slot < a.slots ? a.states + slot * a.slot_bytes : nullptr;
    return c.b >= 0 && c.m < (tokens + kC - 1) / kC && c.state != nullptr;
}

// The bits of |v|; those of what is not finite are kNotFinite or more.
constexpr uint32_t kNotFinite = 0x7F800000u;
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

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

// Sum over 16, 32 or 64 consecutive lanes, to each of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp<0xB1, 0xF, true>(v);   // quad_perm [1,0,3,2]
    v += dpp<0x4E, 0xF, true>(v);   // quad_perm [2,3,0,1]
    v += dpp<0x141, 0xF, true>(v);  // row_half_mirror
    v += dpp<0x140, 0xF, true>(v);  // row_mirror
    if constexpr (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LANES == 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// Convolution and silu of a tile of 16 tokens, N of them per lane from `tau` on (places in the sequence) and 4 mixed channels
// from ch on, whose elements lie at `at`: a row's channels side by side over the lanes, a token's earlier rows in
// registers.  Zeros for tokens that the sequence does not have.  tau0: the wave's first token.  KM: rows of the kernel that
// are held, 4 or 8; shorter kernels have zero weights in front.  SHORT: and zeros for the rows that meet them, which may be
// not finite and no business of the token's.
template <int KM, int N, bool SHORT, typename T>
__device__ __forceinline__ void conv_tile(const DnTokens &a, const T *x, const float *ring, uint32_t pos, int tokens, int tau0, int t0, int at, int ch,
                                          f4_t (&y)[N]) {
    Four<T> rows[N + KM - 1];
    const int tau = tau0 + t0;
    if (tau0 >= KM - 1 && tau0 + 16 <= tokens) {
        // the usual tile: a scalar address per row
        const uint32_t off = static_cast<uint32_t>(t0) * static_cast<uint32_t>(a.qkvz_stride) + at;
        const T *p = x + (tau0 - (KM - 1)) * a.qkvz_stride;
#pragma unroll
        for (int i = 0; i < N + KM - 1; ++i, p += a.qkvz_stride) rows[i].load(p + off);
    } else {
#pragma unroll
        for (int i = 0; i < N + KM - 1; ++i) rows[i].load(x + min(max(tau + i - (KM - 1), 0), tokens - 1) * a.qkvz_stride + at);
    }
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
    auto taps = [&](int j0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < KM - 1; ++j) win[j] = win[j + 1];
            win[KM - 1] = rows[i + KM - 1].get();
            f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KM; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = fmaf(w[j][e], j >= j0 ? win[j][e] : 0.f, acc[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][e] = tau + i < tokens ? silu_hw(acc[e]) : 0.f;
        }
    };
    if (!SHORT || a.K == KM) taps(0);
    else taps(KM - a.K);
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

// Where operands of a tile lie in LDS, by tokens [tile][contraction step][plane] and transposed [row tile][tokens / 32][plane], 64
// places of 16 bytes each.  Operands are read with lane l's at place l but for the low bits of its row, which are mixed
// with what sets lanes apart that write at once: 16 of them would meet in a bank.
template <int DK>
__device__ __forceinline__ constexpr int by_tokens(int tile, int ks, int plane) { return ((tile * (DK / 32) + ks) * 2 + plane) * kWave; }
__device__ __forceinline__ constexpr int token_place(int ks, int token, int g) { return 16 * g + (token ^ (4 * ks + g)); }
__device__ __forceinline__ constexpr int transposed(int dt, int ks2, int plane) { return ((dt * 2 + ks2) * 2 + plane) * kWave; }
__device__ __forceinline__ constexpr int row_place(int dt, int row, int g) { return 16 * g + (row ^ (dt & 3)); }

// N tokens from t0 of the tile and four channels from ch of the operand's rows, transposed, N a multiple of 4.
template <int N>
__device__ __forceinline__ void put_transposed(uint4 *to, int tile, int t0, int ch, const f4_t (&v)[N]) {
    const int dt = ch / 16;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        uint2 *at = reinterpret_cast<uint2 *>(to + transposed(dt, tile >> 1, 0)) + (tile & 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h4_t hi, lo;
            split4(f4_t{v[i][e], v[i + 1][e], v[i + 2][e], v[i + 3][e]}, hi, lo);
            const int place = row_place(dt, ch % 16 + e, (t0 + i) / 4);
            at[2 * place] = as_u2(hi);
            at[2 * (place + kWave)] = as_u2(lo);
        }
    }
}

// One workgroup per (chunk, key head): waves 0 to 3 take a key tile of 16 tokens each, waves 4 to 7 a query tile; then
// their products.  The gates of the key head's value heads beside it.  32 chunks of 16 heads of 128 take 19 us: one round of
// two workgroups to a CU, so what bounds it is its own chain of loads, convolution, norms and products.
template <int DK, int KM, typename T>
__global__ __launch_bounds__(kPrepThreads, 4) void deltanet_keys_kernel(const DnTokens a, const DnChunks w) {
    constexpr int KS = DK / 32, DT = DK / 16, N = DK / 16;
    __shared__ uint4 s_k[kRowTiles * KS * 2 * kWave];  // keys by tokens
    __shared__ uint4 s_q[DT * 2 * 2 * kWave];          // queries by tokens; then keys, transposed
    __shared__ int s_bad[kRowTiles];                   // the first token of each tile whose key is not finite, or kC
    const int hk = blockIdx.x % a.nk;
    const int64_t chunk = blockIdx.x / a.nk;
    Chunk it;
    if (!find_chunk(a, w, static_cast<int>(chunk), it)) return;
    const int m = it.m, tokens = it.tokens, n0 = it.n0;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int tile = wave & 3;
    const bool keys = wave < 4;

    // N tokens and 4 channels per lane, normalised
    const int ch = 4 * (lane % (DK / 4)), t0 = N * (lane / (DK / 4));
    f4_t y[N];
    {
        const int c = (keys ? a.keyD : 0) + hk * DK + ch, head = a.layout == SWQ_DELTA_SPLIT ? hk * DK + (keys ? a.keyD : 0) : hk * (2 * DK + 2 * a.rep * a.dv) + (keys ? DK : 0);
        conv_tile<KM, N, true>(a, static_cast<const T *>(a.qkvz) + n0 * a.qkvz_stride, reinterpret_cast<const float *>(it.state), it.pos, tokens,
                               m * kC + 16 * tile, t0, head + ch, c, y);
        float most = 0.f;  // of the sums: what is not finite makes them so
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float ss = lanes_sum<DK / 4>(y[i][0] * y[i][0] + y[i][1] * y[i][1] + y[i][2] * y[i][2] + y[i][3] * y[i][3]);
            y[i] *= (keys ? 1.f : kScaleT) * __builtin_amdgcn_rsqf(ss + DK * 1e-6f);
            most = fmaxf(most, ss < INFINITY ? 0.f : 1.f);
        }
        if (keys) {
            int bad = kC;
            if (__any(most > 0.f)) {
#pragma unroll
                for (int i = N - 1; i >= 0; --i) {
                    float odd = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd += abs_bits(y[i][e]) >= kNotFinite ? 1.f : 0.f;
                    if (lanes_sum<DK / 4>(odd) > 0.f) {
                        y[i] = f4_t{0.f, 0.f, 0.f, 0.f};
                        bad = 16 * tile + t0 + i;
                    }
                }
                for (int d = 1; d < kWave; d <<= 1) bad = min(bad, __shfl_xor(bad, d, kWave));
            }
            if (lane == 0) s_bad[tile] = bad;
        }
        uint2 *to = reinterpret_cast<uint2 *>((keys ? s_k : s_q) + by_tokens<DK>(tile, ch / 32, 0)) + ch / 16 % 2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            h4_t hi, lo;
            split4(y[i], hi, lo);
            const int place = token_place(ch / 32, t0 + i, ch % 16 / 4);
            to[2 * place] = as_u2(hi);
            to[2 * (place + kWave)] = as_u2(lo);
        }
    }
    // a wave reads its own tile back as operands, the queries' before keys take their place
    asm volatile("" ::: "memory");
    Op x[KS];
    auto read_back = [&](const uint4 *from) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int place = token_place(ks, lane & 15, lane >> 4);
            x[ks] = {as_h8(from[by_tokens<DK>(tile, ks, 0) + place]), as_h8(from[by_tokens<DK>(tile, ks, 1) + place])};
        }
    };
    if (!keys) read_back(s_q);
    lds_barrier();
    if (keys) {
        put_transposed(s_q, tile, t0, ch, y);
        read_back(s_k);
    } else {
        uint4 *q = w.q + (chunk * a.nk + hk) * (kRowTiles * KS * 2 * kWave) + tile * KS * 2 * kWave + lane;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            q[ks * 2 * kWave] = as_u4(x[ks].hi);
            q[(ks * 2 + 1) * kWave] = as_u4(x[ks].lo);
        }
    }
    // k_i.k_j and k_j.q_i of the lower triangle's tiles, as the results lie
    f4_t *dots = w.dots + (chunk * a.nk + hk) * (2 * 10 * kWave) + (keys ? 0 : 10 * kWave) + tile * (tile + 1) / 2 * kWave + lane;
    for (int jt = 0; jt <= tile; ++jt) {
        Sum sum;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int place = token_place(ks, lane & 15, lane >> 4);
            const h8_t kh = as_h8(s_k[by_tokens<DK>(jt, ks, 0) + place]), kl = as_h8(s_k[by_tokens<DK>(jt, ks, 1) + place]);
            if (keys) mfma22(x[ks].hi, x[ks].lo, kh, kl, sum);
            else mfma22(kh, kl, x[ks].hi, x[ks].lo, sum);
        }
        f4_t d = sum.get() * (keys ? 1.f : 1.f / kScaleT);
        here(d);
        dots[jt * kWave] = d;
    }
    // gates, and their logarithms' sums, in units of log 2
    for (int r = wave; r < a.rep; r += kPrepThreads / kWave) {
        const int hv = hk * a.rep + r, t = min(m * kC + lane, tokens - 1);
        const T *ba = static_cast<const T *>(a.ba) + (n0 + static_cast<int64_t>(t)) * a.ba_stride;
        const bool is = m * kC + lane < tokens;
        const float log_g = -expf(a.a_log[hv]) * softplus_acc(dn_load(ba, ba_at(a, hv, 1)) + a.dt_bias[hv]), b = sigmoid_acc(dn_load(ba, ba_at(a, hv, 0)));
        const bool none = log_g != log_g || b != b;
        const uint64_t nones = __ballot(is && none);
        const int bad = min(min(min(s_bad[0], s_bad[1]), min(s_bad[2], s_bad[3])), nones ? __builtin_ctzll(nones) : kC);
        // below 2^-149 a decay is 0 like any other, and sums stay exact beside it
        double c = is && !none ? 1.4426950408889634 * static_cast<double>(fmaxf(log_g, -110.f)) : 0.0;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const double up = __shfl_up(c, d, kWave);
            if (lane >= d) c += up;
        }
        const double last = __shfl(c, kWave - 1, kWave);
        const int64_t head = chunk * a.nv + hv;
        w.sums[head * kC + lane] = c;
        w.beta[head * kC + lane] = is && !none ? b : 0.f;
        w.decay[head * 2 * kC + lane] = lane < bad ? __builtin_amdgcn_exp2f(static_cast<float>(c)) : NAN;
        w.decay[head * 2 * kC + kC + lane] = __builtin_amdgcn_exp2f(static_cast<float>(last - c));
    }
    lds_barrier();
    uint4 *k_to = w.k + (chunk * a.nk + hk) * (DT * 2 * 2 * kWave);
#pragma unroll
    for (int i = 0; i < DT * 2 * 2 * kWave / kPrepThreads; ++i) {
        const int part = i * (kPrepThreads / kWave) + wave;  // four to a row tile
        k_to[part * kWave + lane] = s_q[part * kWave + row_place(part / 4, lane & 15, lane >> 4)];
    }
}

// One workgroup per (chunk, value head): waves 0 to 3 make A and T, waves 4 to 7 P and the values; then all W and U.  32 chunks of
// 32 heads of 128 take 42 us: two rounds of two workgroups to a CU (128 registers, of which 10 to 17 are spilled, 50 to 57 with
// kernels of 5 to 8 rows; 4 waves with twice the columns each spill more: 53 when this took 40), 10 to 16 thousand clocks up to the inverted diagonal blocks, 5 for the others, 4 each for W and U.
template <int DK, int KM, typename T>
__global__ __launch_bounds__(kPrepThreads, 4) void deltanet_solve_kernel(const DnTokens a, const DnChunks w) {
    constexpr int KS = DK / 32, DT = DK / 16, N = kVBlock / 16;
    __shared__ uint4 s_v[kVBlock / 16 * 2 * 2 * kWave];  // values, transposed
    __shared__ __align__(16) float s_t[10 * 16 * kTriRow];
    __shared__ float s_max[4];
    __shared__ int s_bad[4];  // the first token of each tile that has a value which is not finite, or kC
    // a key head's value heads on one XCD (workgroups are handed out round robin), which they share dots and keys in
    const uint32_t unit = blockIdx.x / 8 / a.rep * 8 + blockIdx.x % 8;
    const int hk = unit % a.nk, hv = hk * a.rep + blockIdx.x / 8 % a.rep;
    const int64_t chunk = unit / a.nk, head = chunk * a.nv + hv;
    if (chunk >= w.cap) return;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), col = lane & 15, g = lane >> 4;
    const int tile = wave & 3;
    const bool keys = wave < 4;
    const f4_t zero = {0.f, 0.f, 0.f, 0.f};
    const double *c = w.sums + head * kC;
    const float *beta = w.beta + head * kC;
    float *decay = w.decay + head * 2 * kC;
    const f4_t *dots_at = w.dots + (chunk * a.nk + hk) * (2 * 10 * kWave) + (keys ? 0 : 10 * kWave) + tile * (tile + 1) / 2 * kWave + lane;
    f4_t dots[kRowTiles];
#pragma unroll
    for (int jt = 0; jt < kRowTiles; ++jt) dots[jt] = dots_at[min(jt, tile) * kWave];
    asm volatile("" ::: "memory");  // in flight while the chunk is looked up
    Chunk it;
    if (!find_chunk(a, w, static_cast<int>(chunk), it)) return;
    const int m = it.m, tokens = it.tokens, n0 = it.n0;

    const int ch = 4 * (lane % (kVBlock / 4)), t0 = N * (lane / (kVBlock / 4));
    f4_t v[N];
    auto values = [&](int c0) {  // columns c0 .. of this wave's tile, and their largest
        const int off = min(c0 + ch, a.dv - 4), v_at = a.layout == SWQ_DELTA_SPLIT ? 2 * a.keyD + hv * a.dv : hk * (2 * DK + 2 * a.rep * a.dv) + 2 * DK + (hv - hk * a.rep) * a.dv;
        // from the first value that is not finite on the head gives none, so it does not matter how far a shorter kernel carries it
        conv_tile<KM, N, false>(a, static_cast<const T *>(a.qkvz) + n0 * a.qkvz_stride, reinterpret_cast<const float *>(it.state), it.pos, tokens,
                                m * kC + 16 * tile, t0, v_at + off, 2 * a.keyD + hv * a.dv + off, v);
        uint32_t most = 0;
        auto largest = [&]() {
            most = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, abs_bits(v[i][e]));
        };
        largest();
        int bad = kC;
        if (__any(most >= kNotFinite)) {
#pragma unroll
            for (int i = N - 1; i >= 0; --i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (abs_bits(v[i][e]) >= kNotFinite) {
                        v[i][e] = 0.f;
                        bad = 16 * tile + t0 + i;
                    }
            for (int d = 1; d < kWave; d <<= 1) bad = min(bad, __shfl_xor(bad, d, kWave));
            largest();
        }
        const float m = wave_max_all(__uint_as_float(most));
        if (lane == 0) {
            s_max[tile] = m;
            s_bad[tile] = c0 ? min(bad, s_bad[tile]) : bad;
        }
    };
    // e^(c_i - c_j) is a row's share times a column's about the tile's first row, both at most 1; within the diagonal
    // tile it is taken as it is
    auto pow2 = [](double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x)); };
    const double mid = c[16 * tile];
    if (keys) {
        double ci[4];
        float bi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ci[e] = c[16 * tile + 4 * g + e];
            bi[e] = beta[16 * tile + 4 * g + e];
        }
#pragma unroll
        for (int jt = 0; jt < kRowTiles - 1; ++jt) {
            if (jt >= tile) continue;
            f4_t d = dots[jt] * pow2(mid - c[16 * jt + col]);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] *= bi[e] * pow2(ci[e] - mid);
            tri_put(s_t + tri(tile, jt), d, lane);
        }
        f4_t d = dots[kRowTiles - 1];  // the diagonal tile in any wave
        const double cj = c[16 * tile + col];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = 4 * g + e > col ? d[e] * bi[e] * pow2(ci[e] - cj) : 0.f;
        tri_put(s_t + tri(tile, tile), d, lane);
        // the diagonal block's inverse, by the wave that has just written it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        tri_invert(s_t + tri(tile, tile), lane);
    } else {
        values(0);
        const double ci = c[16 * tile + col];
        const float row = kScaleT * pow2(ci - mid);
        uint4 *p = w.p + head * (kRowTiles * 2 * 2 * kWave) + tile * 2 * 2 * kWave + lane;
#pragma unroll
        for (int ks2 = 0; ks2 < 2; ++ks2) {
            f4_t d[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int jt = 2 * ks2 + half;
                d[half] = dots[jt];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = 16 * jt + 4 * g + e;
                    const float share = jt < tile ? row * pow2(mid - c[j]) : kScaleT * pow2(ci - c[j]);
                    d[half][e] = 16 * tile + col >= j ? d[half][e] * share : 0.f;
                }
            }
            const Op o = op_of(d[0], d[1]);
            p[ks2 * 2 * kWave] = as_u4(o.hi);
            p[(ks2 * 2 + 1) * kWave] = as_u4(o.lo);
        }
    }
    lds_barrier();

    // T below the diagonal blocks, 16 x 16 and then 32 x 32, while waves 4 to 7 put the values
    float vmax = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3])), v_inv;
    float v_scale = scale_of(vmax, 14, v_inv);
    auto put_values = [&]() {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= v_scale;
        put_transposed(s_v, tile, t0, ch, v);
    };
    float low[2][2][4];  // blocks (2 .. 3, 0 .. 1) of A as operands, before another wave's results take their places
    if (wave < 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int s = 0; s < 4; ++s) low[i][j][s] = tri_a(s_t + tri(2 + i, j), lane, s);
        const int i = 2 * wave + 1, j = 2 * wave;
        const f4_t t = tri_mul(s_t + tri(i, j), s_t + tri(j, j), lane, zero);
        tri_put(s_t + tri(i, j), -tri_mul(s_t + tri(i, i), t, lane, zero), lane);
    } else if (!keys) {
        put_values();
    }
    lds_barrier();
    if (wave < 2) {
        const int q = wave;  // a column of blocks
        f4_t x2 = zero, x3 = zero;
        for (int j = q; j < 2; ++j) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float t = tri_b(s_t + tri(j, q), lane, s);
                x2 = mfma4(j ? low[0][1][s] : low[0][0][s], t, x2);
                x3 = mfma4(j ? low[1][1][s] : low[1][0][s], t, x3);
            }
        }
        here(x2);
        here(x3);
        tri_put(s_t + tri(2, q), -tri_mul(s_t + tri(2, 2), x2, lane, zero), lane);
        tri_put(s_t + tri(3, q), -tri_mul(s_t + tri(3, 3), x3, lane, tri_mul(s_t + tri(3, 2), x2, lane, zero)), lane);
    }
    const int half_of = wave >> 2;
    const uint4 *k_at = w.k + (chunk * a.nk + hk) * (DT * 2 * 2 * kWave) + lane;
    uint4 k[2][2][2];
    auto load_k = [&](int ks) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                for (int p = 0; p < 2; ++p) k[half][ks2][p] = k_at[transposed(2 * ks + half, ks2, p)];
    };
    load_k(half_of * (KS / 2));
    lds_barrier();

    // T's rows as operands: 8 of T_ij times b_j (and e^c_j) for i of this wave's tile
    Op tu[2], tw[2];
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
        f4_t u[2], e_u[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int jt = 2 * ks2 + half, j = 16 * jt + 4 * g;
            u[half] = *reinterpret_cast<const f4_t *>(s_t + tri(tile, min(jt, tile)) + col * kTriRow + 4 * g) * (jt <= tile ? kScaleT : 0.f);
            u[half] *= load4(beta + j);
            f4_t grown = load4(decay + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) grown[e] = fmaxf(grown[e], 0.f);  // 0 for NaN, whose tokens T has zeros for in earlier rows
            e_u[half] = u[half] * grown;
        }
        tu[ks2] = op_of(u[0], u[1]);
        tw[ks2] = op_of(e_u[0], e_u[1]);
    }
    uint4 *w_to = w.w + head * (kRowTiles * KS * 2 * kWave) + tile * KS * 2 * kWave + lane;
#pragma unroll
    for (int i = 0; i < KS / 2; ++i) {
        const int ks = half_of * (KS / 2) + i;
        Sum d[2];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2) mfma22(as_h8(k[half][ks2][0]), as_h8(k[half][ks2][1]), tw[ks2].hi, tw[ks2].lo, d[half]);
        if (i + 1 < KS / 2) load_k(ks + 1);
        const Op o = op_of(d[0].get(), d[1].get());
        w_to[ks * 2 * kWave] = as_u4(o.hi);
        w_to[(ks * 2 + 1) * kWave] = as_u4(o.lo);
    }
    f4_t *u_to = w.u + head * (a.dv / 16 * kRowTiles * kWave) + lane;
    for (int c0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kVBlock / 32; ++i) {
            const int ct = 2 * i + half_of;
            Sum sum;
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2)
                mfma22(tu[ks2].hi, tu[ks2].lo, as_h8(s_v[transposed(ct, ks2, 0) + row_place(ct, col, g)]), as_h8(s_v[transposed(ct, ks2, 1) + row_place(ct, col, g)]), sum);
            f4_t d = sum.get() * (v_inv * (1.f / kScaleT));
            here(d);
            if (c0 + 16 * ct < a.dv) u_to[((c0 / 16 + ct) * kRowTiles + tile) * kWave] = d;
        }
        c0 += kVBlock;
        if (c0 >= a.dv) break;
        // heads of more than 128 values: the next of them
        lds_barrier();
        if (!keys) values(c0);
        lds_barrier();
        const float now = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        vmax = fmaxf(vmax, now);
        v_scale = scale_of(now, 14, v_inv);
        if (!keys) put_values();
        lds_barrier();
    }
    if (tid == 0) w.vmax[head] = vmax;
    const int bad = min(min(s_bad[0], s_bad[1]), min(s_bad[2], s_bad[3]));
    if (bad < kC) {
        lds_barrier();  // all waves have used what they read of it
        if (tid >= bad && tid < kC) decay[tid] = NAN;
    }
}

// One workgroup per (sequence, value head, CT * 16 columns of the state), three quarters of waves at three tasks: waves 0 to
// 3 make d of a quarter of the chunk's tokens each, waves 4 to 7 the next state, of whose rows they hold a quarter each, and
// waves 8 to 11 the outputs, off the chain from chunk to chunk.  While one kind computes, the others have their loads
// and stores issued.  A chunk takes 1.4 us at 256 workgroups: each reads its head's operands for itself, 20 TB/s from the
// L2s in all, of 22 to 28 that loads alone reach.  Outputs in a launch of their own, from S and d stored per chunk, took 145
// us instead of 109 for 64 chunks (both with outputs of 11 bits, which are 22 now).
template <int DK, int CT>
__global__ __launch_bounds__(kChainThreads, 3) void deltanet_chain_kernel(const DnTokens a, const DnChunks w, int groups) {
    constexpr int KS = DK / 32, DT = DK / 64;  // DT: row tiles of the state per wave
    __shared__ uint4 s_s[CT * KS * 2 * kWave], s_d[CT * 2 * 2 * kWave], s_e[CT * 2 * 2 * kWave];
    __shared__ float s_max[kChainThreads / kWave];
    // workgroups of one key head on one XCD (they are handed out round robin): its L2 then has what they share
    const int xcd = blockIdx.x & 7, rest = blockIdx.x >> 3;
    const int unit = rest / (groups * a.rep) * 8 + xcd, within = rest % (groups * a.rep);
    if (unit >= a.B * a.nk) return;
    const int b = unit / a.nk, hk = unit % a.nk, hv = hk * a.rep + within / groups, ct0 = within % groups * CT;
    const int tokens = a.count(b) - w.chunk0 * kC;
    uint8_t *slot = a.state(b);
    if (tokens <= 0 || !slot) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), part = wave & 3;
    const uint32_t lane = threadIdx.x & (kWave - 1), col = lane & 15, g = lane >> 4;
    const int chunks = min((tokens + kC - 1) / kC, w.span), cts = a.dv / 16;
    const int64_t first = chunk_base(a, b), head0 = first * a.nv + hv, key0 = first * a.nk + hk;
    const int64_t decay_step = static_cast<int64_t>(a.nv) * 2 * kC;
    const f4_t zero = {0.f, 0.f, 0.f, 0.f};
    const bool rows = wave / 4 == 1;  // of the state

    // the state's columns, a lane's 4 rows side by side in memory
    f4_t st[DT][CT];
    float *state = reinterpret_cast<float *>(slot + a.rec_at) + (static_cast<int64_t>(hv) * a.dv + 16 * ct0 + col) * DK + 4 * g;
    float most = 0.f;
    if (rows) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                st[t][c] = *reinterpret_cast<const f4_t *>(state + static_cast<int64_t>(16 * c) * DK + 16 * (part * DT + t));
#pragma unroll
                for (int e = 0; e < 4; ++e) most = fmaxf(most, abs_bits(st[t][c][e]) < kNotFinite ? fabsf(st[t][c][e]) : 0.f);
            }
    }
    for (int i = tid; i < chunks; i += kChainThreads) most = fmaxf(most, w.vmax[(first + i) * a.nv + hv]);
    most = wave_max_all(most);
    if (lane == 0) s_max[wave] = most;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kChainThreads / kWave; ++i) most = fmaxf(most, s_max[i]);
    // (1 + sqrt(dk + n)) times the largest, with n tokens' writes, stays below f16's largest
    float inverse;
    const float scale = scale_of(most, 14 - (33 - __builtin_clz(min(tokens, chunks * kC) + DK - 1)) / 2, inverse);

    // What a chunk brings is in flight for more than a chunk before it is used.  Chunks that do not exist are loaded as the
    // last one again: no branch.
    if (rows) {
        uint4 kr[2][DT][2][2];
        float grown[2];
        const uint4 *k_at = w.k + key0 * (4 * DT * 2 * 2 * kWave) + part * DT * 2 * 2 * kWave;
        const float *decay_at = w.decay + head0 * 2 * kC + kC - 1;
        const int64_t k_step = static_cast<int64_t>(a.nk) * 4 * DT * 2 * 2 * kWave;
        auto load = [&](int s, bool more) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                    for (int p = 0; p < 2; ++p) kr[s][t][ks2][p] = k_at[((t * 2 + ks2) * 2 + p) * kWave + lane];
            grown[s] = *decay_at;
            k_at += more ? k_step : 0;
            decay_at += more ? decay_step : 0;
        };
        load(0, 1 < chunks);
        load(1, 2 < chunks);
        auto put_state = [&]() {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const int dt = part * DT + t, at = (c * KS + dt / 2) * 2;
                    h4_t hi, lo;
                    split4(st[t][c], hi, lo);
                    reinterpret_cast<uint2 *>(s_s + at * kWave + lane)[dt & 1] = as_u2(hi);
                    reinterpret_cast<uint2 *>(s_s + (at + 1) * kWave + lane)[dt & 1] = as_u2(lo);
                }
        };
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c) st[t][c] *= scale;
        put_state();
        auto turn = [&](int s, int m) {
            lds_barrier();
            if (m > 0) load(s ^ 1, m + 2 < chunks);  // in place of the last chunk's
            const float keep = grown[s];
            lds_barrier();
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                h8_t e[2][2];
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                    for (int p = 0; p < 2; ++p) e[ks2][p] = as_h8(s_e[((c * 2 + ks2) * 2 + p) * kWave + lane]);
#pragma unroll
                for (int t = 0; t < DT; ++t) st[t][c] *= keep;
                f4_t low[DT];
#pragma unroll
                for (int t = 0; t < DT; ++t) low[t] = zero;
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                    for (int p = 0; p < 3; ++p)
#pragma unroll
                        for (int t = 0; t < DT; ++t) {
                            f4_t &to = p < 2 ? low[t] : st[t][c];
                            to = mfma16(as_h8(kr[s][t][ks2][p == 0]), e[ks2][p == 1], to);
                        }
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int x = 0; x < 4; ++x) st[t][c][x] = fmaf(low[t][x], 1.f / kLow, st[t][c][x]);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int c = 0; c < CT; ++c) here(st[t][c]);
            put_state();
        };
        for (int m = 0; m < chunks; m += 2) {
            turn(0, m);
            if (m + 1 < chunks) turn(1, m + 1);
        }
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c)
                *reinterpret_cast<f4_t *>(state + static_cast<int64_t>(16 * c) * DK + 16 * (part * DT + t)) = st[t][c] * inverse;
    } else if (wave < 4) {
        uint4 wr[2][KS][2];
        f4_t ur[2][CT], late[2];
        const uint4 *w_at = w.w + head0 * (kRowTiles * KS * 2 * kWave) + part * KS * 2 * kWave;
        const f4_t *u_at = w.u + (head0 * cts + ct0) * kRowTiles * kWave + part * kWave;
        const float *decay_at = w.decay + head0 * 2 * kC + kC + 16 * part;
        const int64_t w_step = static_cast<int64_t>(a.nv) * kRowTiles * KS * 2 * kWave, u_step = static_cast<int64_t>(a.nv) * cts * kRowTiles * kWave;
        auto load = [&](int s, bool more) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int p = 0; p < 2; ++p) wr[s][ks][p] = w_at[(ks * 2 + p) * kWave + lane];
#pragma unroll
            for (int c = 0; c < CT; ++c) ur[s][c] = u_at[c * kRowTiles * kWave + lane];
            late[s] = load4(decay_at + 4 * g);
            w_at += more ? w_step : 0;
            u_at += more ? u_step : 0;
            decay_at += more ? decay_step : 0;
        };
        load(0, 1 < chunks);
        load(1, 2 < chunks);
        auto turn = [&](int s, int m) {
            lds_barrier();
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                // a sum for each kind of product: one after another of the same sum would wait for each other
                f4_t sum[3] = {zero, zero, zero};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int p = 0; p < 3; ++p) sum[p] = mfma16(as_h8(wr[s][ks][p == 0]), as_h8(s_s[((c * KS + ks) * 2 + (p == 1)) * kWave + lane]), sum[p]);
                const f4_t d = ur[s][c] * scale - Sum{sum[2], sum[1] + sum[0]}.get() * (1.f / kScaleT);
                h4_t hi, lo;
                split4(d * late[s], hi, lo);
                reinterpret_cast<uint2 *>(s_e + ((c * 2 + part / 2) * 2) * kWave + lane)[part & 1] = as_u2(hi);
                reinterpret_cast<uint2 *>(s_e + ((c * 2 + part / 2) * 2 + 1) * kWave + lane)[part & 1] = as_u2(lo);
                split4(d, hi, lo);
                reinterpret_cast<uint2 *>(s_d + (c * 2 + part / 2) * 2 * kWave + lane)[part & 1] = as_u2(hi);
                reinterpret_cast<uint2 *>(s_d + ((c * 2 + part / 2) * 2 + 1) * kWave + lane)[part & 1] = as_u2(lo);
            }
            lds_barrier();
            load(s, m + 3 < chunks);
        };
        for (int m = 0; m < chunks; m += 2) {
            turn(0, m);
            if (m + 1 < chunks) turn(1, m + 1);
        }
    } else {
        uint4 qr[2][KS][2], pr[2][2][2];
        f4_t grown[2];
        const uint4 *q_at = w.q + key0 * (kRowTiles * KS * 2 * kWave) + part * KS * 2 * kWave, *p_at = w.p + head0 * (kRowTiles * 2 * 2 * kWave) + part * 2 * 2 * kWave;
        const float *decay_at = w.decay + head0 * 2 * kC + 16 * part;
        const int64_t q_step = static_cast<int64_t>(a.nk) * kRowTiles * KS * 2 * kWave, p_step = static_cast<int64_t>(a.nv) * kRowTiles * 2 * 2 * kWave;
        auto load_q = [&](int s, bool more) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int p = 0; p < 2; ++p) qr[s][ks][p] = q_at[(ks * 2 + p) * kWave + lane];
            grown[s] = load4(decay_at + 4 * g);
            q_at += more ? q_step : 0;
            decay_at += more ? decay_step : 0;
        };
        auto load_p = [&](int s, bool more) {
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                for (int p = 0; p < 2; ++p) pr[s][ks2][p] = p_at[(ks2 * 2 + p) * kWave + lane];
            p_at += more ? p_step : 0;
        };
        load_q(0, 1 < chunks);
        load_p(0, 1 < chunks);
        load_q(1, 2 < chunks);
        load_p(1, 2 < chunks);
        const float back = inverse / (kScaleT * __fsqrt_rn(static_cast<float>(DK)));
        f4_t *o = w.o + (head0 * cts + ct0) * kRowTiles * kWave + part * kWave + lane;
        const int64_t o_step = static_cast<int64_t>(a.nv) * cts * kRowTiles * kWave;
        auto turn = [&](int s, int m) {
            lds_barrier();
            f4_t v[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                Sum sum;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const h8_t sh = as_h8(s_s[(c * KS + ks) * 2 * kWave + lane]);
                    mfma22(as_h8(qr[s][ks][0]), as_h8(qr[s][ks][1]), sh, as_h8(s_s[((c * KS + ks) * 2 + 1) * kWave + lane]), sum);
                }
                v[c] = sum.get() * grown[s];
            }
            lds_barrier();
            load_q(s, m + 3 < chunks);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                Sum sum{v[c]};
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2) {
                    const h8_t dh = as_h8(s_d[(c * 2 + ks2) * 2 * kWave + lane]);
                    mfma22(as_h8(pr[s][ks2][0]), as_h8(pr[s][ks2][1]), dh, as_h8(s_d[((c * 2 + ks2) * 2 + 1) * kWave + lane]), sum);
                }
                v[c] = sum.get() * back;
            }
            load_p(s, m + 3 < chunks);
#pragma unroll
            for (int c = 0; c < CT; ++c) o[c * kRowTiles * kWave] = v[c];
            o += o_step;
        };
        for (int m = 0; m < chunks; m += 2) {
            turn(0, m);
            if (m + 1 < chunks) turn(1, m + 1);
        }
    }
}

// One workgroup per (chunk, value head): the gated norm, and the ring's rows of a sequence's last chunk, also of one that has
// gone token after token.  CW * 32 columns at
// most, CW * 8 lanes of 4 columns to a token; the outputs come as the matrix instructions leave them, and through LDS.  32
// chunks of 32 heads of 128 take 18 us for 67 MB: one round of workgroups, loads and stores in turn.
template <int CW, typename T>
__global__ __launch_bounds__(kFinishThreads) void deltanet_finish_kernel(const DnTokens a, const DnChunks w) {
    constexpr int L = CW * 8, ROWS = kFinishThreads / L, R = kC / ROWS, kRow = CW * 32 + 4;
    __shared__ __align__(16) float s_o[kC * kRow];
    const int hv = blockIdx.x % a.nv, hk = hv / a.rep, ri = hv - hk * a.rep;
    const int64_t chunk = blockIdx.x / a.nv, head = chunk * a.nv + hv;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), col = lane & 15, g = lane >> 4, cts = a.dv / 16;
    constexpr int PARTS = CW * 2 * kRowTiles * kWave / kFinishThreads;
    f4_t o[PARTS];
    const int64_t o0 = head * cts * kRowTiles * kWave + lane;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const int at = i * (kFinishThreads / kWave) + tid / kWave, ct = min(at / kRowTiles, cts - 1), rt = at % kRowTiles;
        o[i] = w.o[o0 + (ct * kRowTiles + rt) * kWave];
    }
    asm volatile("" ::: "memory");  // in flight while the chunk is looked up
    Chunk it;
    if (!find_chunk(a, w, static_cast<int>(chunk), it)) return;
    const int m = it.m, tokens = it.tokens, here_tokens = min(tokens - m * kC, kC);
    const int64_t n0 = it.n0 + static_cast<int64_t>(m) * kC;

    if (tokens >= w.least) {
        // output gates and the norm's weights, as they will be used
        const int e = min(4 * (tid % L), a.dv - 4), row0 = tid / L;
        const bool real = 4 * (tid % L) < a.dv;
        const T *zr = static_cast<const T *>(a.qkvz) + n0 * a.qkvz_stride + z_at(a, hv, 0) + e;
        Four<T> z[R];
#pragma unroll
        for (int i = 0; i < R; ++i) z[i].load(zr + min(row0 + i * ROWS, here_tokens - 1) * a.qkvz_stride);
        f4_t nw;
#pragma unroll
        for (int k = 0; k < 4; ++k) nw[k] = a.norm_w[e + k];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int at = i * (kFinishThreads / kWave) + tid / kWave, ct = min(at / kRowTiles, cts - 1), rt = at % kRowTiles;
#pragma unroll
            for (int k = 0; k < 4; ++k) s_o[(16 * rt + 4 * g + k) * kRow + 16 * ct + col] = o[i][k];
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int t = row0 + i * ROWS;
            const f4_t ot = *reinterpret_cast<const f4_t *>(s_o + t * kRow + e);
            const float ss = real ? ot[0] * ot[0] + ot[1] * ot[1] + ot[2] * ot[2] + ot[3] * ot[3] : 0.f;
            const float sc = __builtin_amdgcn_rsqf(lanes_sum<L>(ss) / static_cast<float>(a.dv) + a.eps);
            const f4_t zi = z[i].get();
            f4_t y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = ot[k] * (sc * nw[k]) * silu_hw(zi[k]);
            if (t >= here_tokens || !real) continue;
            const int64_t at = ((n0 + t) * a.nv + hv) * a.dv + e;
            if (a.out_f32) {
                *reinterpret_cast<f4_t *>(static_cast<float *>(a.out) + at) = y;
            } else {
                const uint32_t lo = dn_bf16(y[0]) | static_cast<uint32_t>(dn_bf16(y[1])) << 16, hi = dn_bf16(y[2]) | static_cast<uint32_t>(dn_bf16(y[3])) << 16;
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at) = make_uint2(lo, hi);
            }
        }
    }
    if ((m + 1) * kC < tokens) return;
    // the ring: this head's values, and with the first value head of a key head its queries and keys
    float *ring = reinterpret_cast<float *>(it.state);
    const T *last = static_cast<const T *>(a.qkvz) + (it.n0 + static_cast<int64_t>(tokens) - 1) * a.qkvz_stride;
    const int channels = a.dv + (ri == 0 ? 2 * a.dk : 0), rows = min(tokens, a.K);
    for (int i = tid; i < channels * rows; i += kFinishThreads) {
        const int ago = i / channels, c = i - ago * channels;
        const int ch = c < a.dv ? 2 * a.keyD + hv * a.dv + c : hk * a.dk + (c - a.dv) % a.dk + (c - a.dv >= a.dk ? a.keyD : 0);
        ring[static_cast<int64_t>((it.pos + static_cast<uint32_t>(tokens - 1 - ago)) % a.K) * a.convD + ch] = dn_load(last - ago * a.qkvz_stride, mixed_at(a, ch));
    }
}

// Parts of the workspace, at 256-byte boundaries.
struct Parts {
    size_t k, q, w, p, u, decay, sums, beta, vmax, dots, o, total;
};
Parts parts_of(int64_t nk, int64_t nv, int64_t dk, int64_t dv, int64_t cap) {
    Parts s{};
    s.k = dn_align(cap * nk * dk * kC * 2 * 2);
    s.q = dn_align(cap * nk * dk * kC * 2 * 2);
    s.w = dn_align(cap * nv * dk * kC * 2 * 2);
    s.p = dn_align(cap * nv * kC * kC * 2 * 2);
    s.u = dn_align(cap * nv * dv * kC * 4);
    s.decay = dn_align(cap * nv * 2 * kC * 4);
    s.sums = dn_align(cap * nv * kC * 8);
    s.beta = dn_align(cap * nv * kC * 4);
    s.vmax = dn_align(cap * nv * 4);
    s.dots = dn_align(cap * nk * 2 * 10 * 256 * 4);
    s.o = dn_align(cap * nv * dv * kC * 4);
    s.total = s.k + s.q + s.w + s.p + s.u + s.decay + s.sums + s.beta + s.vmax + s.dots + s.o;
    return s;
}
// Chunks that have places in the workspace: for one sequence those of a span.
int64_t cap_of(int64_t sequences, int64_t tokens) {
    return sequences == 1 ? std::min<int64_t>((tokens + kC - 1) / kC, kSpan) : tokens / kC + sequences;
}

template <int DK, int KM, typename T>
void launch_prepare_km(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    hipLaunchKernelGGL((deltanet_keys_kernel<DK, KM, T>), dim3(static_cast<uint32_t>(w.cap * a.nk)), dim3(kPrepThreads), 0, s, a, w);
    hipLaunchKernelGGL((deltanet_solve_kernel<DK, KM, T>), dim3(static_cast<uint32_t>((w.cap * a.nk + 7) / 8 * 8 * a.rep)), dim3(kPrepThreads), 0, s, a, w);
}
template <int DK, typename T>
void launch_prepare(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    if (a.K <= 4) launch_prepare_km<DK, 4, T>(a, w, s);
    else launch_prepare_km<DK, 8, T>(a, w, s);
}

template <typename T>
void launch_finish(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>(w.cap * a.nv)), block(kFinishThreads);
    if (a.dv <= 64) hipLaunchKernelGGL((deltanet_finish_kernel<2, T>), grid, block, 0, s, a, w);
    else if (a.dv <= 128) hipLaunchKernelGGL((deltanet_finish_kernel<4, T>), grid, block, 0, s, a, w);
    else hipLaunchKernelGGL((deltanet_finish_kernel<8, T>), grid, block, 0, s, a, w);
}

template <int DK>
void launch_chain(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    const int64_t units = (static_cast<int64_t>(a.B) * a.nk + 7) / 8 * 8 * a.rep;
    // 32 columns to a workgroup where those of 16 would not find a CU each: at 32 value heads of 128 four prompts of 2,500
    // tokens in all take 154 us instead of 178, but one of 4,096 257 instead of 244
    const int cts = a.dv / 16, ct = cts % 2 == 0 && static_cast<int64_t>(a.B) * a.nv * cts > kCus ? 2 : 1;
    const dim3 grid(static_cast<uint32_t>(units * (cts / ct))), block(kChainThreads);
    if (ct == 1) hipLaunchKernelGGL((deltanet_chain_kernel<DK, 1>), grid, block, 0, s, a, w, cts / ct);
    else hipLaunchKernelGGL((deltanet_chain_kernel<DK, 2>), grid, block, 0, s, a, w, cts / ct);
}

template <int DK, typename T>
void launch(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    launch_prepare<DK, T>(a, w, s);
    launch_chain<DK>(a, w, s);
    DnTokens all = a;
    all.least = 1;
    launch_finish<T>(all, w, s);
}
template <typename T>
void launch_dk(const DnTokens &a, const DnChunks &w, hipStream_t s) {
    if (a.dk == 64) launch<64, T>(a, w, s);
    else launch<128, T>(a, w, s);
}

}  // namespace

bool deltanet_chunks_take(const swq_deltanet_layer *l) {
    return (l->key_head_dim == 64 || l->key_head_dim == 128) && l->value_head_dim % 16 == 0 && l->value_head_dim <= 256;
}

bool deltanet_chunks_fit(const swq_deltanet_layer *l, int64_t sequences, int64_t tokens) {
    const int64_t most = 1LL << 23, chunks = cap_of(sequences, tokens), heads = (sequences * l->num_key_heads + 7) * (l->num_value_heads / l->num_key_heads);
    return chunks * l->num_value_heads < most && 2 * heads * (l->value_head_dim / 16) < most;
}

size_t deltanet_chunks_bytes(const swq_deltanet_layer *l, int64_t sequences, int64_t tokens) {
    return parts_of(l->num_key_heads, l->num_value_heads, l->key_head_dim, l->value_head_dim, cap_of(sequences, tokens)).total;
}

void launch_deltanet_chunks(const DnTokens &a, bool in_f32, void *ws, hipStream_t s) {
    DnChunks w{};
    w.cap = static_cast<int32_t>(cap_of(a.B, a.N));
    w.least = a.least;
    const Parts parts = parts_of(a.nk, a.nv, a.dk, a.dv, w.cap);
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
    w.sums = reinterpret_cast<double *>(take(parts.sums));
    w.beta = reinterpret_cast<float *>(take(parts.beta));
    w.vmax = reinterpret_cast<float *>(take(parts.vmax));
    w.dots = reinterpret_cast<f4_t *>(take(parts.dots));
    w.o = reinterpret_cast<f4_t *>(take(parts.o));
    const int chunks = a.B == 1 ? (a.max_tokens + kC - 1) / kC : 1;  // of a sequence alone
    w.span = a.B == 1 ? kSpan : INT32_MAX;
    for (w.chunk0 = 0; w.chunk0 < chunks; w.chunk0 += kSpan) {
        if (a.B == 1) w.cap = std::min(chunks - w.chunk0, kSpan);
        if (in_f32) launch_dk<float>(a, w, s);
        else launch_dk<uint16_t>(a, w, s);
    }
}

}  // namespace swq
