// Attention over a 4-bit cache, several tokens per sequence: tiles of (token, query head) rows of one
// kv head against tiles of cached rows, whose values are unpacked into LDS once for all rows.
#include <cmath>

#include "attention_q4.hpp"

namespace swq {
namespace {

constexpr float kLow = -1e30f;  // below every score: exponents against it stay numbers

// ---- queries ----------------------------------------------------------------

// q / rms * w, turned, times a power of two that brings the row's largest below 2^8 (the sum of a group
// fits f16); as f16 high (and low) parts, the 8 dims of a chunk in the order of a cache word's operand,
// and, with two parts, the groups' sums: three parts, 32 bits.  8 dims per lane, and
// ROWS consecutive (token, head) rows whose loads are in flight together and which read a token's turns
// once: four where that gives each compute unit two workgroups, else one (77 tokens of 16 heads of 256: 5
// us, with four 8; 4,096 tokens of 32 heads of 128: 21, with one 28).
template <int HD, int PQ, int ROWS, typename T>
__global__ __launch_bounds__(256) void q4_queries(const AttnQ4Args a) {
    constexpr int LPH = HD / 8, HPB = 256 / LPH;
    __shared__ float s_rot[HPB][HD];
    const int b = blockIdx.y, tid = threadIdx.x, slot = tid / LPH, j = tid % LPH;
    if (a.vmax && blockIdx.x == 0)  // for q4_largest
        for (int u = tid; u < 2 * a.c.KVH; u += 256) a.vmax[a.c.head(b, 0) * 2 + u] = 0;
    const int cnt = a.b.count(b);
    if (cnt <= 0) return;
    const uint32_t all = static_cast<uint32_t>(cnt) * a.H;  // the host keeps it below 2^31
    const int64_t first = static_cast<int64_t>(a.b.first(b)) * a.H;
    const int half = a.b.rot / 2;
    float w[8];
    load8<float>(w, a.q_norm_w + 8 * j);
    for (uint32_t base = blockIdx.x * (HPB * ROWS); base < all; base += gridDim.x * (HPB * ROWS)) {
        const uint32_t row = base + slot * ROWS;
        float x[ROWS][8];
        float2 cs[8];
        uint32_t turned = ~0u;  // the token whose turns cs holds
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const uint32_t it = min(row + k, all - 1);
            load8<T>(x[k], static_cast<const T *>(a.q) + (first + it) * 2 * HD + 8 * j);
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const uint32_t token = min(row + k, all - 1) / a.H;
            if (8 * j < 2 * half && token != turned) {
                q4_turns(cs, a.b.rope + static_cast<int64_t>(a.b.position(b, token)) * half, half, j);
                turned = token;
            }
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[k][e] * x[k][e];
            ss = lanes_sum<LPH>(ss);
            const float sc = 1.0f / __fsqrt_rn(ss / static_cast<float>(HD) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[k][e] *= sc * w[e];
                s_rot[slot][8 * j + e] = x[k][e];
            }
            __builtin_amdgcn_wave_barrier();  // a head's lanes are of one wave
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = 8 * j + e;
                if (d < 2 * half) {
                    const float o = s_rot[slot][d < half ? d + half : d - half];
                    x[k][e] = d < half ? x[k][e] * cs[e].x - o * cs[e].y : x[k][e] * cs[e].x + o * cs[e].y;
                }
                top = fmaxf(top, fabsf(x[k][e]));
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            top = lanes_max<LPH>(top);
            int ex = 0;
            if (top > 0.f && top < INFINITY) frexpf(top, &ex);
            h8_t hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = ldexpf(x[k][e], 8 - ex);
                hi[q4_element(e)] = static_cast<_Float16>(v);
                lo[q4_element(e)] = static_cast<_Float16>(v - static_cast<float>(hi[q4_element(e)]));
            }
            float qs = 0.f;
            if constexpr (PQ == 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) qs += static_cast<float>(hi[e]) + static_cast<float>(lo[e]);
                qs = lanes_sum<8>(qs);
            }
            if (row + k >= all) continue;
            const int64_t at = first + row + k;
            if (PQ == 2 && j % 8 == 0) {
                _Float16 *to = static_cast<_Float16 *>(a.qs) + at * 16;
#pragma unroll
                for (int g = 0; g < 4; g += HD / kQ4Group) {  // zeros for groups that heads of less than 256 lack
                    float rest = g == 0 ? qs : 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const _Float16 h = i < 3 ? static_cast<_Float16>(rest) : static_cast<_Float16>(0.f);
                        rest -= static_cast<float>(h);
                        to[4 * i + g + j / 8] = h;
                    }
                }
            }
            reinterpret_cast<h8_t *>(a.qh)[at * LPH + j] = hi;
            if constexpr (PQ == 2) reinterpret_cast<h8_t *>(a.ql)[at * LPH + j] = lo;
            if (j == 0) a.qf[at] = ldexpf(a.scale2, ex - 8);
        }
    }
}

// The largest |bias| + 15 scale of a sequence's keys and of its values, by kv head: what high and low
// parts are scaled by.  Maxima of non-negative numbers, whose bits order as they do.
__global__ __launch_bounds__(256) void q4_largest(const AttnQ4Args a) {
    const int h = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH, ng = a.c.hd / kQ4Group;
    const int cnt = a.b.count(b);
    if (cnt <= 0) return;
    const int n = static_cast<int>(min(static_cast<int64_t>(a.b.row0(b, a.c.maxp)) + cnt, static_cast<int64_t>(a.c.maxp)));
    const _Float16 *par = a.c.par_head(b, h);
    float top[2] = {0.f, 0.f};
    // 8 rows of one group and kind per thread
    const int octs = (n + 7) / 8;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < octs * 2 * ng; i += gridDim.x * 256) {
        const int oct = i % octs, line = i / octs, w = line / ng, g = line % ng;
        const _Float16 *p = par + (static_cast<int64_t>(2 * w) * ng + g) * a.c.R + 8 * oct;
        const h8_t s = __builtin_bit_cast(h8_t, *reinterpret_cast<const uint4 *>(p));
        const h8_t z = __builtin_bit_cast(h8_t, *reinterpret_cast<const uint4 *>(p + static_cast<int64_t>(ng) * a.c.R));
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (8 * oct + e < n) t = fmaxf(t, fabsf(static_cast<float>(z[e])) + 15.0f * static_cast<float>(s[e]));
        top[0] = fmaxf(top[0], w == 0 ? t : 0.f);
        top[1] = fmaxf(top[1], w == 1 ? t : 0.f);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float t = wave_max_all(top[w]);
        if ((threadIdx.x & (kWave - 1)) == 0 && t > 0.f) atomicMax(a.vmax + 2 * a.c.head(b, h) + w, __float_as_uint(t));
    }
}

// The exponent that brings numbers up to `bits` (an f32's) to 2^14 .. 2^15.
__device__ __forceinline__ int q4_lift(uint32_t bits) {
    const float t = __uint_as_float(bits);
    int ex = 0;
    if (t > 0.f && t < INFINITY) frexpf(t, &ex);
    return 15 - ex;
}

// ---- tiles of values in LDS -------------------------------------------------

// Where chunk c (8 numbers, 16 bytes) of a line of CH chunks lies: xor-ed with bits of the line.  LDS
// serves 16 lanes of 16 bytes at once, lanes 0-3, 12-15, 20-23 and 24-27 together and so on: with chunk
// q = lane / 16 of line r = lane % 16, these are 16 different places of 256 bytes for the lines below,
// and for the lines or chunks that a wave writes.  KEY: line r is cached row 8 (r / 4) + r % 4 of the
// tile (bit 2 of the row is no part of it); else a dim or a query.
template <int CH, bool KEY>
__device__ __forceinline__ int q4_place(int line, int c) {
    const int r = KEY ? (line & 3) | (line >> 1 & 12) : line & 15;
    const int high = (r >> 3) | ((r >> 2 ^ r >> 3) & 1) << 1;  // 0, 2, 3, 1 for r / 4 = 0 .. 3
    const int f = CH == 4 ? high : CH == 8 ? (high & 1) | (r & 2) | (high & 2) << 1 : r;
    return line * CH + (c ^ f);
}

// A word's codes as f16 integers, pairs of nibbles (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void q4_codes(uint32_t w, uint32_t magic, h2_t (&c)[4]) {
    constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;
    const uint32_t s = w >> 8;
    const h2_t off = {static_cast<_Float16>(-1024.f), static_cast<_Float16>(-1024.f)};
    const h2_t down = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    const h2_t off16 = {static_cast<_Float16>(-64.f), static_cast<_Float16>(-64.f)};
    c[0] = __builtin_bit_cast(h2_t, (w & kEven) | magic) + off;
    c[1] = __builtin_elementwise_fma(__builtin_bit_cast(h2_t, (w & kOdd) | magic), down, off16);
    c[2] = __builtin_bit_cast(h2_t, (s & kEven) | magic) + off;
    c[3] = __builtin_elementwise_fma(__builtin_bit_cast(h2_t, (s & kOdd) | magic), down, off16);
}

// One plane: scale * code + bias rounded to f16 once (2^-12 of the value, none past f16's largest; exact
// below f16's normal numbers, where all three are multiples of 2^-24).  Two: in f32, times 2^lift, as high and low part.
template <int PLANES>
__device__ __forceinline__ void q4_values(uint32_t w, uint32_t magic, const h2_t (&s)[4], const h2_t (&z)[4], float unit, h8_t &hi, h8_t &lo) {
    h2_t c[4];
    q4_codes(w, magic, c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (PLANES == 1) {
            const h2_t v = __builtin_elementwise_fma(c[k], s[k], z[k]);
            hi[2 * k] = v.x;
            hi[2 * k + 1] = v.y;
        } else {
            const f32x2_t v = {unit * fmaf(static_cast<float>(c[k].x), static_cast<float>(s[k].x), static_cast<float>(z[k].x)),
                               unit * fmaf(static_cast<float>(c[k].y), static_cast<float>(s[k].y), static_cast<float>(z[k].y))};
            h2_t h, l;
            split_f16(v, h, l);
            hi[2 * k] = h.x;
            hi[2 * k + 1] = h.y;
            lo[2 * k] = l.x;
            lo[2 * k + 1] = l.y;
        }
    }
}

__device__ __forceinline__ h2_t pair_ll(uint32_t a, uint32_t b) { return __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(b, a, 0x05040100u)); }
__device__ __forceinline__ h2_t pair_hh(uint32_t a, uint32_t b) { return __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(b, a, 0x07060302u)); }

// ---- attention --------------------------------------------------------------

// Whether a bf16 call's queries are prepared where they are used: pairs of dims that turn together, `half`
// apart, are then the same lane's, chunks 4 u + q and 4 (u + half / 32) + q.  A launch less and the queries
// read once: 4,096 tokens of 16 heads of 256 240 us, now 224 (all launches), 4 x 1,000 of 32 heads of 128
// 131, now 112; 512 after 16,384 rows in two splits, which prepare them twice, 193 and 194.
bool prepares_queries(int rot) { return rot == 0 || rot == 64 || rot == 128 || rot == 256; }

template <int HU, int KS>
__device__ __forceinline__ void turn_chunks(float (&x)[KS][8], const float2 *turn, int half, int q) {
    if constexpr (2 * HU <= KS) {
#pragma unroll
        for (int u = 0; u < HU; ++u) {
            float2 cs[8];
            q4_turns(cs, turn, half, 4 * u + q);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float m = x[u][e], n = x[u + HU][e];
                x[u][e] = m * cs[e].x - n * cs[e].y;
                x[u + HU][e] = n * cs[e].x + m * cs[e].y;
            }
        }
    }
}

// What q4_queries makes of one row, by the four lanes that have it as operand: chunks 4 u + q as f16, and
// what turns a product of them into log2 units.
template <int HD>
__device__ __forceinline__ float prepare_queries(const AttnQ4Args &a, const uint16_t *src, const float2 *turn, int q, h8_t (&out)[HD / 32]) {
    constexpr int KS = HD / 32;
    const int half = a.b.rot / 2;
    float x[KS][8], ss = 0.f, top = 0.f;
#pragma unroll
    for (int u = 0; u < KS; ++u) load8<uint16_t>(x[u], src + 8 * (4 * u + q));
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[u][e] * x[u][e];
    ss += __shfl_xor(ss, 16, kWave);
    ss += __shfl_xor(ss, 32, kWave);
    const float sc = 1.0f / __fsqrt_rn(ss / static_cast<float>(HD) + a.eps);
#pragma unroll
    for (int u = 0; u < KS; ++u) {
        float w[8];
        load8<float>(w, a.q_norm_w + 8 * (4 * u + q));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u][e] *= sc * w[e];
    }
    if (half == 32) turn_chunks<1>(x, turn, half, q);
    else if (half == 64) turn_chunks<2>(x, turn, half, q);
    else if (half == 128) turn_chunks<4>(x, turn, half, q);
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[u][e]));
    top = fmaxf(top, __shfl_xor(top, 16, kWave));
    top = fmaxf(top, __shfl_xor(top, 32, kWave));
    int ex = 0;
    if (top > 0.f && top < INFINITY) frexpf(top, &ex);
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) out[u][q4_element(e)] = static_cast<_Float16>(ldexpf(x[u][e], 8 - ex));
    return ldexpf(a.scale2, ex - 8);
}

// A workgroup takes M = 16 WAVES rows (token, query head of the kv head's group; heads of one token next
// to each other) and the cached rows of one split that the last of them sees, NT at a time.  The tile's
// words are loaded two tiles ahead into registers, unpacked one tile ahead into the other of two LDS
// buffers, one barrier per tile.  Each wave has 16 rows as columns of both products: scores = K Q
// (K's rows permuted so that the result's registers are the next operand), out = V^T P, so that
// maxima, sums and rescaling belong to the lane's own column.  p is taken against a reference that only
// moves when a score passes it by 2^15: most tiles need no maximum across lanes and no rescaling.
// Bound, at hd 256, by what two waves per SIMD and a barrier a tile let overlap: 4,096 tokens of 16 heads of
// 256 in bf16 take 220 us traced, 625 TFLOP/s, their queries prepared here; of those clocks VALU has 46%, LDS (each
// wave reads the whole tile's operands for its 16 rows) 44%, the matrix units 31%.  512 after 8,192 rows, queries
// in two parts: 158.  32 rows per wave halve the LDS bytes but leave one wave per SIMD (slower); scores of the
// next tile beside the softmax (237 us, when this took 217) cost more registers.
// Heads of up to 128 in bf16: two workgroups per CU, their registers bounded to 128 (4,096 tokens of 32
// heads of 128 250 us with the other launches, else 284; of 64 154, else 182).  Registers are spilled once a row
// tile, none in the loop over cached rows: 23 (<128, 1, 1, 32, 8>), 51 (4 waves), 4 and 18 at hd 64, and at
// hd 256, which has 256, 29 (<256, 2, 1, 32, 8>), 55 (4 waves) and 18 (<256, 1, 1, 32, 4>).
template <int HD, int PQ, int PV, int NT, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, HD <= 128 && PQ == 1 ? 4 : 2) void q4_prefill(const AttnQ4Args a) {
    constexpr int NG = HD / kQ4Group, KS = HD / 32, DT = HD / 16, PAIRS = NT / 32, M = 16 * WAVES;
    constexpr int THREADS = WAVES * kWave, KCH = HD / 8, VCH = NT / 8;
    // words of a thread: of keys KW, THREADS apart; of values VW of one block and group, 64 / VW dims apart
    constexpr int KW = NT * KCH / THREADS, VW = VCH * HD / THREADS;
    static_assert(KW >= 1 && (VW == 1 || VW == 2 || VW == 4), "a thread's value words share a block and a group");
    constexpr uint32_t KB = NT * KCH * 16, VB = HD * VCH * 16;  // bytes of one plane of a tile
    // Keys: [buffer][plane] of values.  Or, with two parts of the queries and one of p and values, codes: their
    // products are exact, a product and a plane less for a scale and score on the VALU (bf16 with gathered
    // weights, 512 tokens after 8,192 rows: 157 us, with planes 173; but in f32 2,048 tokens of 32 heads of 128
    // 175 against 169: there the VALU has enough to do with values and p).  Beside the codes lie, by buffer,
    // scales by group and row, and the biases of a row's groups twice, as the sums' parts lie.
    constexpr bool CODES = PQ == 2 && PV == 1;
    constexpr int KP = CODES ? 1 : PQ;
    __shared__ __attribute__((aligned(16))) uint8_t s_k[2 * KP * KB];
    __shared__ __attribute__((aligned(16))) _Float16 s_ks[CODES ? 2 : 1][CODES ? NG : 1][CODES ? NT : 8];
    __shared__ __attribute__((aligned(16))) _Float16 s_kz[CODES ? 2 : 1][CODES ? NT : 1][8];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[2 * PV * VB];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int r = lane & 15, q = lane >> 4, G = a.group;
    // heads innermost; tiles of rows from the last, which sees the most cached rows, to the first: a CU
    // that is done takes the longest that is left.  Workgroups go to the 8 XCDs in turn, and in each to
    // its 4 shader engines in turn, which wait for one another: from tile to tile the heads are turned by
    // 8, so that a head keeps its XCD (its rows are in that L2) and no engine gets all of a sequence's
    // (1,000, 750, 500 and 250 tokens of 32 heads of 128: 81 us, turned 53)
    const int heads = a.b.B * a.c.KVH;
    const int rank = blockIdx.x / heads;
    const int head = static_cast<int>((blockIdx.x + 8u * rank) % static_cast<uint32_t>(heads));
    const int split = rank % a.splits, slot = a.tiles - 1 - rank / a.splits;
    const int kvh = head % a.c.KVH, b = head / a.c.KVH;
    const int cnt = a.b.count(b);
    const int n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const uint32_t all = static_cast<uint32_t>(cnt) * G;  // rows: the host keeps tokens * H below 2^31
    const uint32_t *kw = a.c.k_head(b, kvh), *vw = a.c.v_head(b, kvh);
    const _Float16 *par = a.c.par_head(b, kvh);
    const uint32_t magic = kept_1024();
    const int seq_rows = static_cast<int>(min(static_cast<int64_t>(r0) + cnt, static_cast<int64_t>(a.c.maxp)));
    const int klift = KP == 2 ? q4_lift(a.vmax[2 * a.c.head(b, kvh)]) : 0, vlift = PV == 2 ? q4_lift(a.vmax[2 * a.c.head(b, kvh) + 1]) : 0;
    const float kunit = ldexpf(1.0f, klift), vunit = ldexpf(1.0f, vlift);

    for (uint32_t base = static_cast<uint32_t>(slot) * M; base < all; base += static_cast<uint32_t>(a.tiles) * M) {
        // rows that the workgroup's last valid one sees, and this split's share of them
        const uint32_t end_row = min(base + M, all) - 1;
        const int sees = min(r0 + static_cast<int>(end_row / G) + 1, a.c.maxp);
        const int kv0 = split * a.per, kv1 = split == a.splits - 1 ? sees : min(kv0 + a.per, sees);
        if (kv0 >= kv1) continue;
        // this lane's column
        const uint32_t column = min(base + wave * 16 + r, all - 1);
        const bool valid = base + wave * 16 + r < all;
        const int vis = valid ? min(r0 + static_cast<int>(column / G) + 1, a.c.maxp) : 0;
        int low = vis;
        float f;
        h8_t qh[KS], ql[PQ == 2 ? KS : 1], qs = h8_t{};
        {
            const int64_t at = static_cast<int64_t>(n0 + column / G) * a.H + kvh * G + column % G;
            int lq = q;  // as below: addresses kept from row tile to row tile were spilled
            asm volatile("" : "+v"(lq));
            if (PQ == 1 && !a.qh) {
                const float2 *turn = a.b.rope + static_cast<int64_t>(a.b.position(b, column / G)) * (a.b.rot / 2);
                f = prepare_queries<HD>(a, static_cast<const uint16_t *>(a.q) + at * 2 * HD, turn, lq, qh);
            } else {
                f = ldexpf(a.qf[at], -klift);
                if (CODES && q < 2) qs = static_cast<const h8_t *>(a.qs)[2 * at + q];
#pragma unroll
                for (int u = 0; u < KS; ++u) {
                    qh[u] = reinterpret_cast<const h8_t *>(a.qh)[at * KCH + 4 * u + lq];
                    if constexpr (PQ == 2) ql[u] = reinterpret_cast<const h8_t *>(a.ql)[at * KCH + 4 * u + lq];
                }
            }
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) low = min(low, __shfl_xor(low, off, kWave));
        low = __builtin_amdgcn_readfirstlane(low);
        float ref = kLow, l = 0.f;
        f4_t o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = f4_t{0.f, 0.f, 0.f, 0.f};

        uint32_t rk[KW], rv[VW];
        _Float16 rks[KW], rkz[KW];  // key scale and bias of the word's row
        uint4 rvs, rvz;             // value scales and biases of the block's rows
        // The words of a tile lie one after another, keys and values alike.  Of 64 rows the second 32
        // may lie past the cache's: then they are the first again.  Addresses: the tile's, the same for
        // all lanes, and the lane's 32-bit offset in it.
        constexpr uint32_t VGAP = kQ4Group / VW;
        const uint32_t vblk = tid / (VGAP * NG), vdim = tid / VGAP % NG * kQ4Group + tid % VGAP;
        auto fetch = [&](int t0) {
            int tf = tid;
            if constexpr (CODES && HD == 256) asm volatile("" : "+v"(tf));
            const uint32_t vblk = tf / (VGAP * NG), vdim = tf / VGAP % NG * kQ4Group + tf % VGAP;
            const bool beyond = NT > 32 && t0 + 32 >= a.c.R;
            const uint32_t *pk = kw + static_cast<int64_t>(t0) * KCH, *pv = vw + static_cast<int64_t>(t0 / 8) * HD;
            const _Float16 *ps = par + t0, *pz = ps + static_cast<int64_t>(NG) * a.c.R;
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const uint32_t line = i * (THREADS / KCH) + tf / KCH, back = beyond && line >= 32 ? 32 : 0;
                rk[i] = pk[(line - back) * KCH + tf % KCH];
                const uint32_t at = (tf % KCH / 8) * a.c.R + (line - back);
                rks[i] = ps[at];
                rkz[i] = pz[at];
            }
            const uint32_t blk = vblk - (beyond && vblk >= 4 ? 4 : 0);
            pv += blk * HD + vdim;
#pragma unroll
            for (int i = 0; i < VW; ++i) rv[i] = pv[i * VGAP];
            const uint32_t at = vdim / kQ4Group * a.c.R + 8 * blk;
            rvs = *reinterpret_cast<const uint4 *>(ps + static_cast<int64_t>(kQ4VScale) * NG * a.c.R + at);
            rvz = *reinterpret_cast<const uint4 *>(ps + static_cast<int64_t>(kQ4VBias) * NG * a.c.R + at);
        };
        auto unpack_k = [&](int buf) {
            int tk = tid;
            if constexpr (CODES && HD == 256) asm volatile("" : "+v"(tk));
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const int line = i * (THREADS / KCH) + tk / KCH, j = tk % KCH;
                const h2_t s1 = {rks[i], rks[i]}, z1 = {rkz[i], rkz[i]};
                const h2_t s[4] = {s1, s1, s1, s1}, z[4] = {z1, z1, z1, z1};
                h8_t hi, lo;
                if constexpr (!CODES) {
                    q4_values<KP>(rk[i], magic, s, z, kunit, hi, lo);
                } else {
                    h2_t c[4];
                    q4_codes(rk[i], magic, c);
                    hi = h8_t{c[0].x, c[0].y, c[1].x, c[1].y, c[2].x, c[2].y, c[3].x, c[3].y};
                    if (j % 8 == 0) {
                        s_ks[buf][j / 8][line] = rks[i];
#pragma unroll
                        for (int g = 0; g < 4; g += NG) {  // zeros for groups that heads of less than 256 lack
                            const _Float16 b0 = g == 0 ? rkz[i] : static_cast<_Float16>(0.f);
                            s_kz[buf][line][g + j / 8] = b0;
                            s_kz[buf][line][4 + g + j / 8] = b0;
                        }
                    }
                }
                uint8_t *dst = s_k + buf * (KP * KB) + 16 * q4_place<KCH, true>(line, j);
                *reinterpret_cast<h8_t *>(dst) = hi;
                if constexpr (KP == 2) *reinterpret_cast<h8_t *>(dst + KB) = lo;
            }
        };
        auto unpack_v = [&](int t0, int buf) {
            if (t0 + NT > seq_rows) {  // rows past the sequence's: 0, whatever they hold
                const int left = seq_rows - t0 - 8 * static_cast<int>(vblk);
                uint4 keep;
                keep.x = (left > 0 ? 0xFFFFu : 0u) | (left > 1 ? 0xFFFF0000u : 0u);
                keep.y = (left > 2 ? 0xFFFFu : 0u) | (left > 3 ? 0xFFFF0000u : 0u);
                keep.z = (left > 4 ? 0xFFFFu : 0u) | (left > 5 ? 0xFFFF0000u : 0u);
                keep.w = (left > 6 ? 0xFFFFu : 0u) | (left > 7 ? 0xFFFF0000u : 0u);
                rvs.x &= keep.x; rvs.y &= keep.y; rvs.z &= keep.z; rvs.w &= keep.w;
                rvz.x &= keep.x; rvz.y &= keep.y; rvz.z &= keep.z; rvz.w &= keep.w;
            }
            const h2_t s[4] = {pair_ll(rvs.x, rvs.z), pair_hh(rvs.x, rvs.z), pair_ll(rvs.y, rvs.w), pair_hh(rvs.y, rvs.w)};
            const h2_t z[4] = {pair_ll(rvz.x, rvz.z), pair_hh(rvz.x, rvz.z), pair_ll(rvz.y, rvz.w), pair_hh(rvz.y, rvz.w)};
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                h8_t hi, lo;
                q4_values<PV>(rv[i], magic, s, z, vunit, hi, lo);
                uint8_t *dst = s_v + buf * (PV * VB) + 16 * q4_place<VCH, false>(vdim + i * VGAP, vblk);
                *reinterpret_cast<h8_t *>(dst) = hi;
                if constexpr (PV == 2) *reinterpret_cast<h8_t *>(dst + VB) = lo;
            }
        };

        __syncthreads();  // a row tile before this one is done with the buffers
        const int final = kv0 + (kv1 - 1 - kv0) / NT * NT;  // the last tile: past it, it is unpacked again
        fetch(kv0);
        unpack_k(0);
        unpack_v(kv0, 0);
        fetch(min(kv0 + NT, final));
        int buf = 0;
        for (int t0 = kv0; t0 < kv1; t0 += NT, buf ^= 1) {
            lds_barrier();
            f4_t s[PAIRS][2];
            // The chains of the tile's products by turns; key chunks are read a few ahead of them.  Step u's chunk lies 64 u
            // xor-ed into the first one's address, the rows of the second product 4 lines on.
            constexpr int NK = PAIRS * 2 * KS, AHEAD = PQ == 2 ? 2 : 4;
            uint32_t kat = buf * (KP * KB) + 16 * q4_place<KCH, true>(8 * (r >> 2) + (r & 3), q);
            asm volatile("" : "+v"(kat));  // no step's address is kept from tile to tile
            auto key = [&](int n, int plane) {
                const int pr = n / 2 % PAIRS, x = n % 2, u = n / (2 * PAIRS);
                return *reinterpret_cast<const h8_t *>(s_k + (kat ^ (64u * u)) + plane * KB + (32 * pr + 4 * x) * KCH * 16);
            };
            h8_t kf[AHEAD][KP];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n)
#pragma unroll
                for (int p = 0; p < KP; ++p) kf[n][p] = key(n, p);
            if constexpr (CODES) {
                // sums of codes by group, times the rows' scales; the biases and the sums of the queries are one
                // more product
#pragma unroll
                for (int n = 0; n < 2 * PAIRS; ++n)
                    s[n / 2][n % 2] = mfma16(*reinterpret_cast<const h8_t *>(s_kz[buf][32 * (n / 2) + 8 * (r >> 2) + 4 * (n % 2) + (r & 3)]), qs, f4_t{0.f, 0.f, 0.f, 0.f});
            }
            f4_t d[PAIRS][2];
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                const int pr = n / 2 % PAIRS, x = n % 2, u = n / (2 * PAIRS);
                if constexpr (CODES) {
                    d[pr][x] = mfma16(kf[n % AHEAD][0], qh[u], u % 2 == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : d[pr][x]);
                    d[pr][x] = mfma16(kf[n % AHEAD][0], ql[u], d[pr][x]);
                } else {
                    f4_t c = u == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : s[pr][x];
                    c = mfma16(kf[n % AHEAD][0], qh[u], c);
                    if constexpr (PQ == 2) {
                        c = mfma16(kf[n % AHEAD][0], ql[u], c);
                        c = mfma16(kf[n % AHEAD][1], qh[u], c);
                    }
                    s[pr][x] = c;
                }
                if (n + AHEAD < NK) {
#pragma unroll
                    for (int p = 0; p < KP; ++p) kf[n % AHEAD][p] = key(n + AHEAD, p);
                }
                if (CODES && u % 2 == 1 && n % (2 * PAIRS) == 2 * PAIRS - 1) {  // a group is complete
#pragma unroll
                    for (int p = 0; p < PAIRS; ++p) {
                        const h8_t ks = *reinterpret_cast<const h8_t *>(&s_ks[CODES ? buf : 0][CODES ? u / 2 : 0][CODES ? 32 * p + 8 * q : 0]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) s[p][i / 4][i % 4] = fmaf(static_cast<float>(ks[i]), d[p][i / 4][i % 4], s[p][i / 4][i % 4]);
                    }
                }
            }
            unpack_k(buf ^ 1);
            unpack_v(min(t0 + NT, final), buf ^ 1);
            fetch(min(t0 + 2 * NT, final));
            if (t0 + NT > low || t0 + NT > kv1) {
                const int lim = min(vis, kv1) - t0 - 8 * q;
#pragma unroll
                for (int pr = 0; pr < PAIRS; ++pr)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[pr][x][i] = 32 * pr + 4 * x + i < lim ? s[pr][x][i] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int pr = 0; pr < PAIRS; ++pr)
#pragma unroll
                for (int x = 0; x < 2; ++x) top = fmaxf(top, fmaxf(fmaxf(s[pr][x][0], s[pr][x][1]), fmaxf(s[pr][x][2], s[pr][x][3])));
            top *= f;
            if (__any(top > ref + 15.0f)) {
                top = fmaxf(top, __shfl_xor(top, 16, kWave));
                top = fmaxf(top, __shfl_xor(top, 32, kWave));
                const float to = fmaxf(ref, top - 7.0f);
                const float alpha = q4_exp2(ref - to);
                ref = to;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= alpha;
            }
            constexpr int NV = DT * PAIRS, AHEAD_V = PV == 2 ? 2 : 4;
            const uint32_t vat = buf * (PV * VB) + 16 * q4_place<VCH, false>(r, q);
            auto value = [&](int n, int plane) {
                return *reinterpret_cast<const h8_t *>(s_v + (vat ^ (64u * (n % PAIRS))) + plane * VB + n / PAIRS * 16 * VCH * 16);
            };
            h8_t vf[AHEAD_V][PV];
#pragma unroll
            for (int n = 0; n < AHEAD_V; ++n)
#pragma unroll
                for (int p = 0; p < PV; ++p) vf[n][p] = value(n, p);
            h8_t ph[PAIRS], pl[PV == 2 ? PAIRS : 1];
#pragma unroll
            for (int pr = 0; pr < PAIRS; ++pr) {
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = q4_exp2(fmaf(s[pr][i / 4][i % 4], f, -ref));
                // to the lane's sum eight rows at a time: 33,000 rows in a split with sharp scores are off by 4e-6, one by one 1e-5
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const f32x2_t x = {p[q4_nibble(j)], p[q4_nibble(j + 1)]};
                    h2_t h, w;
                    if constexpr (PV == 2) {
                        split_f16(x, h, w);
                        pl[pr][j] = w.x;
                        pl[pr][j + 1] = w.y;
                    } else {
                        h = __builtin_convertvector(x, h2_t);
                    }
                    ph[pr][j] = h.x;
                    ph[pr][j + 1] = h.y;
                }
            }
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int d = n / PAIRS, pr = n % PAIRS;
                o[d] = mfma16(vf[n % AHEAD_V][0], ph[pr], o[d]);
                if constexpr (PV == 2) {
                    o[d] = mfma16(vf[n % AHEAD_V][0], pl[pr], o[d]);
                    o[d] = mfma16(vf[n % AHEAD_V][1], ph[pr], o[d]);
                }
                if (n + AHEAD_V < NV) {
#pragma unroll
                    for (int p = 0; p < PV; ++p) vf[n % AHEAD_V][p] = value(n + AHEAD_V, p);
                }
            }
        }
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        const bool last = a.splits == 1;
        const float unit = last ? (l > 0.f || l != l ? 1.0f / (vunit * l) : 0.f) : 1.0f / vunit;
        const int64_t at = static_cast<int64_t>(n0 + column / G) * a.H + kvh * G + column % G;
        if (valid && q == 0) {
            if (!last) a.ml[at * a.splits + split] = make_float2(ref, l);
            else if (a.lse) a.lse[at] = ref + log2f(l);
        }
        // Up to 128 dims of the wave's 16 rows at a time through its share of the tiles' LDS, so that rows
        // leave, and gates come, in whole lines.
        constexpr int PART = HD == 256 ? 128 : 64, CPR = PART / 4, RPI = kWave / CPR;
        static_assert(sizeof(s_k) >= WAVES / 2 * 16 * PART * 4 && sizeof(s_v) >= WAVES / 2 * 16 * PART * 4, "16 rows for each wave");
        constexpr int ITS = 16 / RPI, PARTS = HD / PART;
        // Where one part is used for p and values, inputs and output are bf16.  The gates of a part are all
        // on their way before any is used, the first part's across the barrier.
        const int at32 = static_cast<int>(at);
        int el = lane;  // no address of what follows is kept across the tiles
        asm volatile("" : "+v"(el));
        uint32_t to[ITS];  // (token, head) of the rows that this lane writes; the host keeps them below 2^31
        uint2 gates[ITS];
        const int d0 = el % CPR * 4;
#pragma unroll
        for (int it = 0; it < ITS; ++it) to[it] = __shfl(at32, it * RPI + el / CPR, kWave);
        const bool any = base + wave * 16 < all;  // of this wave's rows
        auto load_gates = [&](uint2 (&g)[ITS], int part) {
            if constexpr (PV == 1) {
#pragma unroll
                for (int it = 0; it < ITS; ++it)
                    g[it] = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.q) + static_cast<uint64_t>(to[it]) * (2 * HD) + HD + part * PART + d0);
            }
        };
        if (last && any) load_gates(gates, 0);
        __syncthreads();
        if (!any) continue;
        uint8_t *mine = wave < WAVES / 2 ? s_k + wave * (16 * PART * 4) : s_v + (wave - WAVES / 2) * (16 * PART * 4);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
#pragma unroll
            for (int d = 0; d < PART / 16; ++d) *reinterpret_cast<f4_t *>(mine + ((el & 15) * CPR + ((4 * d + (el >> 4)) ^ (el & 15))) * 16) = o[part * (PART / 16) + d] * unit;
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            uint2 next[ITS];
            if (last && part + 1 < PARTS) load_gates(next, part + 1);
#pragma unroll
            for (int it = 0; it < ITS; ++it) {
                const int row = it * RPI + el / CPR, c = el % CPR;
                const f4_t v = *reinterpret_cast<const f4_t *>(mine + (row * CPR + (c ^ row)) * 16);
                if (base + wave * 16 + row >= all) continue;
                const int d = part * PART + d0;
                if (!last) {
                    *reinterpret_cast<f4_t *>(a.part + (static_cast<uint64_t>(to[it]) * a.splits + split) * HD + d) = v;
                } else if constexpr (PV == 1) {
                    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + static_cast<uint64_t>(to[it]) * HD + d) = gated_bf16(gates[it], v);
                } else {
                    store_gated(a, static_cast<int64_t>(to[it]) * HD + d, (2 * static_cast<int64_t>(to[it]) + 1) * HD + d, v);
                }
            }
            if constexpr (PV == 1) {
#pragma unroll
                for (int it = 0; it < ITS; ++it) gates[it] = next[it];
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// The splits of each (token, query head) merged: HD / 4 lanes per row, 4 dims each.
template <int HD>
__global__ __launch_bounds__(256) void q4_prefill_merge(const AttnQ4Args a) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;  // lanes per row, rows per workgroup
    const int b = blockIdx.y, cnt = a.b.count(b);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / LPR;
    if (item >= static_cast<int64_t>(cnt) * a.H) return;
    const int r0 = a.b.row0(b, a.c.maxp), i = static_cast<int>(item / a.H), d = threadIdx.x % LPR * 4;
    const int64_t at = static_cast<int64_t>(a.b.first(b) + i) * a.H + item % a.H;
    // splits that hold rows which this row's tile of rows sees
    const int64_t row = static_cast<int64_t>(i) * a.group + item % a.H % a.group, all = static_cast<int64_t>(cnt) * a.group;
    const int64_t end_row = min((row / a.rows_per + 1) * a.rows_per, all) - 1;
    const int sees = static_cast<int>(min(static_cast<int64_t>(r0) + end_row / a.group + 1, static_cast<int64_t>(a.c.maxp)));
    const int splits = min((sees + a.per - 1) / a.per, a.splits);
    const float2 *ml = a.ml + at * a.splits;
    float top = kLow;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s].x);
    f4_t sum = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float w = q4_exp2(ml[s].x - top);
        l += w * ml[s].y;
        sum += w * *reinterpret_cast<const f4_t *>(a.part + (at * a.splits + s) * HD + d);
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    store_gated(a, at * HD + d, (2 * at + 1) * HD + d, sum * inv);
    if (d == 0 && a.lse) a.lse[at] = top + log2f(l);
}

// ---- gathered weights -------------------------------------------------------

// A workgroup has kGatherRows cached rows of a kv head, 32 per wave, their codes as f16 integers in
// registers, and walks the rows of queries that see any of them, 16 at a time: those go through LDS
// once for all waves, the next 16 on their way meanwhile.  A group's products with the queries' two parts
// are exact and take the rows' scales on the VALU; the biases meet the groups' sums, which are in three
// parts, in one more matrix product.  Sums of p stay with the lane until the end.  512 tokens of 16 heads
// after 8,192 rows of 2 kv heads of 256: 115 us, 616 TFLOP/s in the two products, with values as two parts
// and so three products 143 (16 cached rows per wave and queries read by each from L1: 911).
constexpr int kGatherRows = 128;

template <int HD>
__global__ __launch_bounds__(256, 2) void q4_gathered(const AttnQ4Args a) {
    constexpr int NG = HD / kQ4Group, KS = HD / 32, KCH = HD / 8, NC = 16 * KCH / 256 > 0 ? 16 * KCH / 256 : 1;
    __shared__ h8_t s_q[2][2][16 * KCH];  // [buffer][high, low]
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int r = lane & 15, q = lane >> 4, G = a.group;
    const int kvh = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH;
    const int cnt = a.b.count(b);
    if (cnt <= 0) return;
    const int n0 = a.b.first(b), r0 = a.b.row0(b, a.c.maxp);
    const int top = static_cast<int>(min(static_cast<int64_t>(r0) + cnt, static_cast<int64_t>(a.c.maxp)));
    const uint32_t magic = kept_1024();
    const uint32_t all = static_cast<uint32_t>(cnt) * G;
    const int part = blockIdx.z, parts = gridDim.z;  // of the queries
    for (int t0 = blockIdx.x * kGatherRows; t0 < top; t0 += gridDim.x * kGatherRows) {
        const int w0 = t0 + 32 * wave;
        typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
        h8_t kc[2][KS], kb[2];  // biases of a row: twice in lanes q = 0, once in 1, as the sums' parts lie
        h4_t ks[2][NG];         // scales of the four rows whose scores the lane gets
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int64_t line = min(w0 + 16 * x + r, a.c.R - 1);
            const _Float16 *par = a.c.par_head(b, kvh);
            kb[x] = h8_t{};
#pragma unroll
            for (int u = 0; u < KS; ++u) {
                h2_t c[4];
                q4_codes(a.c.k_head(b, kvh)[line * KCH + 4 * u + q], magic, c);
                kc[x][u] = h8_t{c[0].x, c[0].y, c[1].x, c[1].y, c[2].x, c[2].y, c[3].x, c[3].y};
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                ks[x][g] = *reinterpret_cast<const h4_t *>(par + static_cast<int64_t>(g) * a.c.R + min(w0 + 16 * x + 4 * q, a.c.R - 4));
                const _Float16 z = par[static_cast<int64_t>(kQ4KBias * NG + g) * a.c.R + line];
                if (q < 2) kb[x][g] = z;
                if (q == 0) kb[x][4 + g] = z;
            }
        }
        float sum[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[x][e] = 0.f;
        // the first 16 rows of queries that see row t0; this part's share of those from there on
        const uint32_t from = static_cast<uint32_t>(max(t0 - r0, 0)) * G / 16 + part, blocks = (all + 15) / 16;
        uint4 ch[NC], cl[NC];
        h8_t qs;
        float f, z;
        int vis;
        const bool copies = 16 * KCH >= 256 || tid < 16 * KCH;
        auto fetch = [&](uint32_t blk) {
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const uint32_t id = k * 256 + tid, row = min(blk * 16 + id / KCH, all - 1);
                const int64_t at = (static_cast<int64_t>(n0 + row / G) * a.H + kvh * G + row % G) * KCH + id % KCH;
                if (copies) {
                    ch[k] = static_cast<const uint4 *>(a.qh)[at];
                    cl[k] = static_cast<const uint4 *>(a.ql)[at];
                }
            }
            const uint32_t row = min(blk * 16 + r, all - 1), i = row / G;
            const int64_t at = static_cast<int64_t>(n0 + i) * a.H + kvh * G + row % G;
            f = a.qf[at];
            z = a.lse[at];
            qs = static_cast<const h8_t *>(a.qs)[2 * at + (q & 1)];
            vis = blk * 16 + r < all ? min(r0 + static_cast<int>(i) + 1, a.c.maxp) : 0;
        };
        auto put = [&](int buf) {
            if (copies) {
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const int id = k * 256 + tid;
                    s_q[buf][0][q4_place<KCH, false>(id / KCH, id % KCH)] = __builtin_bit_cast(h8_t, ch[k]);
                    s_q[buf][1][q4_place<KCH, false>(id / KCH, id % KCH)] = __builtin_bit_cast(h8_t, cl[k]);
                }
            }
        };
        __syncthreads();  // the rows before these are done with the buffers
        if (from < blocks) {
            fetch(from);
            put(0);
        }
        int buf = 0;
        for (uint32_t blk = from; blk < blocks; blk += parts, buf ^= 1) {
            const float cf = f, cz = z;
            const int cv = vis;
            const bool more = blk + parts < blocks;
            f4_t s[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) s[x] = mfma16(kb[x], qs, f4_t{0.f, 0.f, 0.f, 0.f});
            lds_barrier();
            if (more) fetch(blk + parts);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f4_t d[2];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int u = 2 * g + v;
                    const h8_t qh = s_q[buf][0][q4_place<KCH, false>(r, 4 * u + q)], ql = s_q[buf][1][q4_place<KCH, false>(r, 4 * u + q)];
#pragma unroll
                    for (int x = 0; x < 2; ++x) d[x] = mfma16(kc[x][u], qh, v == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : d[x]);
#pragma unroll
                    for (int x = 0; x < 2; ++x) d[x] = mfma16(kc[x][u], ql, d[x]);
                }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[x][e] = fmaf(static_cast<float>(ks[x][g][e]), d[x][e], s[x][e]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = q4_exp2(fmaf(s[x][e], cf, -cz));
                    sum[x][e] += w0 + 16 * x + 4 * q + e < cv ? p : 0.f;
                }
            if (more) put(buf ^ 1);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[x][e] = lanes_sum<16>(sum[x][e]);
        if (r == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = w0 + 16 * (i / 4) + 4 * q + i % 4;
                const float v = sum[i / 4][i % 4];
                if (t >= top) continue;
                if (parts > 1) {
                    a.gpart[(a.c.head(b, kvh) * parts + part) * a.c.R + t] = v;
                } else {
                    float *w = a.weights + a.c.head(b, kvh) * a.c.maxp + t;
                    *w = t < r0 ? *w + v : v;
                }
            }
        }
    }
}

__global__ __launch_bounds__(256) void q4_gathered_merge(const AttnQ4Args a, int parts) {
    const int kvh = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH, cnt = a.b.count(b);
    if (cnt <= 0) return;
    const int r0 = a.b.row0(b, a.c.maxp);
    const int top = static_cast<int>(min(static_cast<int64_t>(r0) + cnt, static_cast<int64_t>(a.c.maxp)));
    for (int t = blockIdx.x * 256 + threadIdx.x; t < top; t += gridDim.x * 256) {
        float s = 0.f;
        for (int p = 0; p < parts; ++p) s += a.gpart[(a.c.head(b, kvh) * parts + p) * a.c.R + t];
        float *w = a.weights + a.c.head(b, kvh) * a.c.maxp + t;
        *w = t < r0 ? *w + s : s;
    }
}

// ---- launches ---------------------------------------------------------------

template <int HD, int PQ, typename T>
void launch_queries(const AttnQ4Args &a, hipStream_t s) {
    constexpr int HPB = 256 / (HD / 8);
    const int64_t items = static_cast<int64_t>(a.b.max_tokens) * a.H, all = static_cast<int64_t>(a.b.N) * a.H;
    const bool four = items * a.b.B >= 4 * HPB * 512;
    const int64_t per = four ? 4 * HPB : HPB;
    const dim3 grid(static_cast<uint32_t>(q4_workgroups((items + per - 1) / per, a.b.B, all / per + a.b.B)), a.b.B);
    if (four) hipLaunchKernelGGL((q4_queries<HD, PQ, 4, T>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((q4_queries<HD, PQ, 1, T>), grid, dim3(256), 0, s, a);
}

template <int HD, int WAVES>
void launch_tiles(const AttnQ4Args &a, dim3 grid, hipStream_t s) {
    constexpr int NT = HD == 64 ? 64 : 32;
    const dim3 block(WAVES * kWave);
    if (a.planes_q == 1) hipLaunchKernelGGL((q4_prefill<HD, 1, 1, NT, WAVES>), grid, block, 0, s, a);
    else if (a.planes_v == 1) hipLaunchKernelGGL((q4_prefill<HD, 2, 1, NT, WAVES>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((q4_prefill<HD, 2, 2, NT, WAVES>), grid, block, 0, s, a);
}

template <int HD>
void launch_head_dim(const AttnQ4Args &a, hipStream_t s) {
    const uint32_t heads = static_cast<uint32_t>(a.b.B) * a.c.KVH;
    const int rows = static_cast<int>(std::min<int64_t>(a.c.maxp, 1 << 20));
    if (a.planes_q == 2) a.in_f32 ? launch_queries<HD, 2, float>(a, s) : launch_queries<HD, 2, uint16_t>(a, s);
    else if (a.qh) launch_queries<HD, 1, uint16_t>(a, s);  // one part: bf16 in and out
    if (a.vmax) hipLaunchKernelGGL(q4_largest, dim3(std::min(((rows + 7) / 8 * 2 * (HD / kQ4Group) + 255) / 256, 256), heads), dim3(256), 0, s, a);
    const dim3 grid(static_cast<uint32_t>(static_cast<int64_t>(a.tiles) * a.splits * heads)), block(256);
    a.rows_per == 64 ? launch_tiles<HD, 4>(a, grid, s) : launch_tiles<HD, 8>(a, grid, s);
    if (a.splits > 1) {
        constexpr int RPB = 256 / (HD / 4);
        const int64_t items = static_cast<int64_t>(a.b.max_tokens) * a.H;
        hipLaunchKernelGGL(q4_prefill_merge<HD>, dim3(static_cast<uint32_t>((items + RPB - 1) / RPB), a.b.B), block, 0, s, a);
    }
    if (a.weights) {
        hipLaunchKernelGGL(q4_gathered<HD>, dim3((rows + kGatherRows - 1) / kGatherRows, heads, a.gparts), block, 0, s, a);
        if (a.gparts > 1) hipLaunchKernelGGL(q4_gathered_merge, dim3(std::min((rows + 255) / 256, 1024), heads), block, 0, s, a, a.gparts);
    }
}

}  // namespace

Q4PrefillPlan plan_q4_prefill(int64_t max_tokens, int64_t all, int64_t rows, int64_t heads, int group, int hd, int rot, int maxp, bool f32, bool weights) {
    Q4PrefillPlan p{};
    p.planes_q = f32 || weights ? 2 : 1;
    p.planes_v = f32 ? 2 : 1;
    p.prepares = p.planes_q == 1 && prepares_queries(rot);
    // 128 rows share a tile's values; where that leaves half of the compute units without work however
    // the cached rows are split, 64, whose steps are shorter (77 tokens of 16 heads of 256 in f32: 26 us,
    // with 64 rows 21.6)
    p.rows_per = (max_tokens * group + 127) / 128 * heads * std::max<int64_t>(1, rows / 256) <= 128 ? 64 : 128;
    p.tiles = static_cast<int>(q4_workgroups((max_tokens * group + p.rows_per - 1) / p.rows_per, heads, all / p.rows_per + heads));
    // as many workgroups as the CUs hold, if the cached rows can be split that often with 256 rows each:
    // two per CU where registers are bounded for that (512 tokens after 16,384 rows, 32 heads of 128: 193
    // us, with one 220), else one (16 heads of 256: 196, with two 212)
    const int64_t groups = p.tiles * heads;
    const int64_t want = std::max<int64_t>(1, (hd <= 128 && p.planes_q == 1 ? 512 : 256) / groups), most = std::max<int64_t>(1, rows / 256);
    // a padded batch has more rows than its longest sequence accounts for
    const int64_t splits = std::min<int64_t>({want, most, kQ4PrefillMaxSplits, (kQ4PartRows + all) / all});
    p.per = static_cast<int>(((rows + splits - 1) / splits + 63) / 64 * 64);
    p.splits = static_cast<int>((rows + p.per - 1) / p.per);
    // the gathered weights: three rounds of two workgroups per CU, the queries dealt out where the cached
    // rows are few (512 tokens after 8,192 rows: 118 us, in one round of 408 workgroups 127, in four 121)
    const int64_t cols = (rows + kGatherRows - 1) / kGatherRows * heads;
    p.gparts = weights ? static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({1536 / cols, (max_tokens * group + 127) / 128, kQ4GatherMaxParts,
                                                                               kQ4GatherMost / (heads * q4_rows(maxp))}))) : 0;
    return p;
}

void launch_q4_prefill(const AttnQ4Args &a, hipStream_t s) {
    switch (a.c.hd) {
        case 64: launch_head_dim<64>(a, s); break;
        case 128: launch_head_dim<128>(a, s); break;
        default: launch_head_dim<256>(a, s); break;
    }
}

}  // namespace swq
