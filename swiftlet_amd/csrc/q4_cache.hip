// Rows into a KV cache held in 4 bits, out of it as values, and the heaviest of them into a
// smaller cache.  The formats are swq.h's (swq_q4_cache).
#include <cmath>

#include "q4_row.hpp"

namespace swq {
namespace {

constexpr int kAppendThreads = 256;

struct AppendArgs {
    Q4View c;
    Q4Batch b;
    const void *k, *v;
    const float *w;  // k_norm_weight
    float eps;
};

// A workgroup per block of 8 rows, kv head and sequence (two blocks at hd 64).  HD / 8 lanes have a row,
// 8 dims each, so that a lane's codes are one k word, a wave takes 2 to 8 rows at once and sums cross few
// lanes.  A v word holds 8 rows of one dim: those codes meet in LDS, and words of which only some rows
// are new keep the others (the first and last block of a call).  All in 64 bits up to the format's own
// roundings.  Bound by that arithmetic (8,192 tokens of 8 heads of 128, 43 MB: 36 us, VALU
// instructions for 24 of them); one row per wave and a division per value took 58.
template <int HD, typename T>
__global__ __launch_bounds__(kAppendThreads) void q4_append(const AppendArgs a) {
    constexpr int LPR = HD / 8, PER = kQ4Block * LPR;  // lanes of a row, of a block's keys or values
    constexpr int ROUNDS = 2 * PER > kAppendThreads ? 2 : 1, BLOCKS = ROUNDS == 1 ? kAppendThreads / (2 * PER) : 1, NG = HD / kQ4Group;
    __shared__ double s_rot[kAppendThreads / LPR][HD];
    __shared__ uint2 s_v[BLOCKS][kQ4Block][LPR];
    const int h = blockIdx.y % a.c.KVH, b = blockIdx.y / a.c.KVH, tid = threadIdx.x, j = tid % LPR;
    const Q4Rows rows = a.b.written(b, a.c.maxp);
    const int half = a.b.rot / 2, block_end = rows.block_end();
    uint32_t *kw = a.c.k_head(b, h), *vw = a.c.v_head(b, h);
    _Float16 *par = a.c.par_head(b, h);
    for (int blk0 = rows.block0() + blockIdx.x * BLOCKS; blk0 < block_end; blk0 += gridDim.x * BLOCKS) {
#pragma unroll
        for (int round = 0; round < ROUNDS; ++round) {
            const bool values = ROUNDS == 2 ? round == 1 : tid / PER % 2 == 1;  // the same for a whole wave
            const int which = ROUNDS == 2 ? 0 : tid / (2 * PER), u = tid % PER / LPR, row = (blk0 + which) * kQ4Block + u;
            const bool here = rows.has(row);
            const int n = rows.token(row);
            const int64_t at = (static_cast<int64_t>(n) * a.c.KVH + h) * HD + 8 * j;
            float in[8];
            load8<T>(in, static_cast<const T *>(values ? a.v : a.k) + at);
            uint32_t q[8];
            _Float16 scale, bias;
            if (!values) {
                double x[8];
                float2 cs[8];
                float w[8];
                if (8 * j < 2 * half) q4_turns(cs, a.b.rope + static_cast<int64_t>(a.b.position(b, n - rows.n0)) * half, half, j);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = a.w[8 * j + e];
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = static_cast<double>(in[e]);
                    ss += x[e] * x[e];
                }
                if constexpr (LPR == 32) {
                    ss = reduce_f64<16>(ss, [](double p, double r) { return p + r; });
                    ss += __shfl_xor(ss, 16, kWave);
                } else {
                    ss = reduce_f64<LPR>(ss, [](double p, double r) { return p + r; });
                }
                const double inv = 1.0 / sqrt(ss / HD + static_cast<double>(a.eps));
                double *rot = s_rot[tid / LPR];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = x[e] * inv * static_cast<double>(w[e]);
                    rot[8 * j + e] = x[e];
                }
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (8 * j < 2 * half) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = 8 * j + e;
                        if (d < 2 * half) {
                            const double o = rot[d < half ? d + half : d - half];
                            const double c = static_cast<double>(cs[e].x), s = static_cast<double>(cs[e].y);
                            x[e] = d < half ? x[e] * c - o * s : x[e] * c + o * s;
                        }
                    }
                }
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                q4_quantise<8>(x, q, scale, bias);
            } else {
                q4_quantise(in, q, scale, bias);
            }
            if (here && j % 8 == 0) {
                _Float16 *p = par + (static_cast<int64_t>(values ? kQ4VScale : kQ4KScale) * NG + j / 8) * a.c.R + row;
                p[0] = scale;
                p[static_cast<int64_t>(NG) * a.c.R] = bias;
            }
            if (values) {
                s_v[which][u][j] = make_uint2(q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24);
            } else if (here) {
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) word |= q[e] << (4 * e);
                kw[static_cast<int64_t>(row) * LPR + j] = word;
            }
        }
        __syncthreads();
        for (int i = tid; i < BLOCKS * HD; i += kAppendThreads) {
            const int which = i / HD, d = i % HD, blk = blk0 + which;
            const int u0 = max(rows.r0 - blk * kQ4Block, 0), u1 = min(rows.r1 - blk * kQ4Block, kQ4Block);
            if (u0 < u1) {
                uint32_t *p = vw + static_cast<int64_t>(blk) * HD + d;
                uint32_t word = 0, mask = 0;
#pragma unroll
                for (int u = 0; u < kQ4Block; ++u) {
                    word |= static_cast<uint32_t>(reinterpret_cast<const uint8_t *>(s_v[which][u])[d]) << (4 * u);
                    mask |= u >= u0 && u < u1 ? 15u << (4 * u) : 0u;
                }
                *p = mask == 0xFFFFFFFFu ? word : (*p & ~mask) | (word & mask);
            }
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

// A thread per (kReadRows rows, kv head, 8 dims): their k words, and the block's 8 v words, of which it
// takes its rows' codes.  Bound by the bytes it writes: 8,192 rows of 8 heads of 128 to f32 (77 MB) 18 us,
// 4.3 TB/s; a row or a block of 8 per thread take as long there, but 8 rows 8 us where two take 5 (2,048
// rows of 2 heads of 256, too few waves).
constexpr int kReadRows = 2;

template <typename T>
__global__ __launch_bounds__(256) void q4_read(const ReadArgs a) {
    const int b = blockIdx.y;
    const uint32_t oct = a.c.hd / 8, per_row = a.c.KVH * oct;
    const int s0 = a.starts ? min(max(a.starts[b], 0), a.count) : 0;
    const int n = a.starts ? max(min(a.starts[b + 1], a.count) - s0, 0) : a.count;
    if (n <= 0) return;
    const int64_t out0 = a.starts ? s0 : static_cast<int64_t>(b) * a.count;
    const int64_t first = a.first ? a.first[b] : 0;
    const int top = a.rows ? min(a.rows[b], a.c.maxp) : a.c.maxp;
    const int64_t base = first & ~static_cast<int64_t>(kReadRows - 1);  // an even row: a pair is of one block
    const int64_t pairs = (first + n - base + kReadRows - 1) / kReadRows;
    const int ng = a.c.hd / kQ4Group;
    const uint32_t each = per_row < 256 ? 256 / per_row : 1;  // pairs of a workgroup, which follow one another
    for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * each; c0 < pairs; c0 += static_cast<int64_t>(gridDim.x) * each) {
        for (uint32_t i = threadIdx.x; i < each * per_row; i += 256) {
            const uint32_t u = i / per_row, v = i - u * per_row, h = v / oct, j = v - h * oct;
            const int64_t row0 = base + (c0 + u) * kReadRows, t0 = row0 - first;
            if (c0 + u >= pairs) continue;
            const bool inside = row0 >= 0 && row0 < top;
            const _Float16 *par = a.c.par_head(b, h) + row0 + static_cast<int64_t>(j / 8) * a.c.R;
            const uint32_t *kp = a.c.k_head(b, h) + row0 * oct + j, *vp = a.c.v_head(b, h) + (row0 / 8) * a.c.hd + 8 * j;
            const int lift = 4 * static_cast<int>(row0 & 7);
            uint32_t kw[kReadRows] = {}, sz[4] = {};
            uint4 v0{}, v1{};
            if (inside) {
                if (a.k) {
                    kw[0] = kp[0];
                    kw[1] = kp[oct];
                }
                if (a.v) {
                    v0 = reinterpret_cast<const uint4 *>(vp)[0];
                    v1 = reinterpret_cast<const uint4 *>(vp)[1];
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) sz[w] = *reinterpret_cast<const uint32_t *>(par + static_cast<int64_t>(w) * ng * a.c.R);
            }
            const uint32_t vw[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int r = 0; r < kReadRows; ++r) {
                if (t0 + r < 0 || t0 + r >= n) continue;
                const bool there = inside && row0 + r < top;
                const int64_t at = ((out0 + t0 + r) * a.c.KVH + h) * a.c.hd + 8 * j;
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    T *out = static_cast<T *>(which ? a.v : a.k);
                    if (!out) continue;
                    const float s = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(sz[2 * which] >> (16 * r))));
                    const float z = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(sz[2 * which + 1] >> (16 * r))));
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t q = which ? vw[e] >> (lift + 4 * r) : kw[r] >> (4 * e);
                        x[e] = there ? fmaf(s, static_cast<float>(q & 15u), z) : 0.f;
                    }
                    store8(out + at, x);
                }
            }
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
constexpr int kSelectKeep = 48;  // rows of a thread that are in registers at once
constexpr int kSelectRows = kSelectThreads * kSelectKeep;
constexpr int kSelectBins = 2048;
constexpr int kSelectList = 4096;  // rows that are left to decide on, when they are few
static_assert(kSelectKeep * kSelectWaves <= kSelectThreads && kSelectBins == 2 * kSelectThreads, "a thread per count, two bins per thread");

// What rows are ordered by: the weight (NaN lowest), then the lower row; all different.
__device__ __forceinline__ uint32_t weight_key(float w) { return w == w ? orderable(w == 0.f ? 0.f : w) : 0u; }
__device__ __forceinline__ uint64_t rank_key(uint32_t key, int row) { return static_cast<uint64_t>(key) << 32 | ~static_cast<uint32_t>(row); }

// Sum over the lanes before this one, and over all of them.
__device__ __forceinline__ uint32_t lanes_before(uint32_t v, uint32_t &all) {
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t s = v;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const uint32_t o = __shfl_up(s, off, kWave);
        if (lane >= off) s += o;
    }
    all = __builtin_amdgcn_readlane(s, kWave - 1);
    return s - v;
}

// The rows that one (sequence, kv head) keeps: those of the middle whose rank_key reaches a border, and
// all before and behind it.  The border is found eleven bits at a time from the top from histograms in
// LDS, whose integer counts do not depend on the order of the adds, until all rows that share its known
// bits are kept; once those are few they are listed, and the later passes go over the list alone.  Then
// the kept rows are counted and numbered in order.  Weights stay in registers, 48 rows of each thread;
// caches of more than 49,152 rows are gone through in parts, read again by each pass.  One workgroup per
// head, because all its rows decide together: 33,000 rows to 4,096 34 us on two CUs, bound by their VALU
// (every row is looked at by the first one or two passes, the count and the writing); 8,193 rows of 64
// heads to 2,047 16 us.
__global__ __launch_bounds__(kSelectThreads) void q4_select(const EvictArgs a) {
    __shared__ uint32_t s_hist[kSelectBins];
    __shared__ uint64_t s_list[kSelectList];
    __shared__ uint32_t s_count[kSelectKeep * kSelectWaves];  // by chunk of 1,024 rows and wave
    __shared__ uint32_t s_wave[kSelectWaves];
    __shared__ uint32_t s_pick[3], s_listed;
    const int h = blockIdx.x % a.src.KVH, b = blockIdx.x / a.src.KVH;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
    const int n = min(max(a.rows[b], 0), a.src.maxp);
    const float *w = a.weights + a.src.head(b, h) * a.src.maxp;
    int32_t *kept = a.kept + a.src.head(b, h) * a.budget;
    float *nw = a.new_weights ? a.new_weights + a.dst.head(b, h) * a.dst.maxp : nullptr;
    const bool all = n <= a.budget;
    const int m0 = all ? n : a.sink, m1 = all ? n : n - a.recent;  // the middle
    uint32_t need = all ? 0 : a.budget - a.sink - a.recent;        // of it, still to be found
    const int parts = (n + kSelectRows - 1) / kSelectRows;
    float x[kSelectKeep];
    // the rows of a part, 1,024 at a time; f(i, row, weight)
    auto load = [&](int part) {
#pragma unroll
        for (int i = 0; i < kSelectKeep; ++i) {
            const int t = part * kSelectRows + i * kSelectThreads + tid;
            x[i] = t < n ? w[t] : 0.f;
        }
    };
    if (parts > 0) load(0);
    uint64_t border = need > 0 ? 0 : ~0ull, mask = 0;  // its known bits
    bool listed = false;
    uint32_t left = static_cast<uint32_t>(m1 - m0);  // rows that share them
    for (int shift = 53; need > 0 && need < left; shift = max(shift - 11, 0)) {
        s_hist[tid] = s_hist[tid + kSelectThreads] = 0;
        if (tid == 0) s_listed = 0;
        __syncthreads();
        auto count = [&](bool in, uint32_t bin) {
            const uint64_t who = __ballot(in);
            if (who == 0) return;
            const int lead = __builtin_ctzll(who);
            if (__ballot(in && bin == static_cast<uint32_t>(__builtin_amdgcn_readlane(bin, lead))) == who) {  // one add for all
                if (lane == lead) atomicAdd(&s_hist[bin], static_cast<uint32_t>(__popcll(who)));
            } else if (in) {
                atomicAdd(&s_hist[bin], 1u);
            }
        };
        const uint32_t digit = shift == 0 ? 511u : 2047u;  // 53, 42, 31, 20, 9, 0
        if (listed) {
            for (uint32_t i = tid; i < ((left + 63) & ~63u); i += kSelectThreads) {
                const uint64_t k = i < left ? s_list[i] : 0;
                count(i < left && (k & mask) == border, static_cast<uint32_t>(k >> shift) & digit);
            }
        } else {
            for (int part = 0; part < parts; ++part) {
                if (parts > 1) load(part);
#pragma unroll
                for (int i = 0; i < kSelectKeep; ++i) {
                    if (part * kSelectRows + i * kSelectThreads >= n) break;
                    const int t = part * kSelectRows + i * kSelectThreads + tid;
                    const uint64_t k = rank_key(weight_key(x[i]), t);
                    count(t >= m0 && t < m1 && (k & mask) == border, static_cast<uint32_t>(k >> shift) & digit);
                }
            }
        }
        __syncthreads();
        // thread t: bins 2047 - 2 t and the one below, from the top
        const uint32_t c0 = s_hist[kSelectBins - 1 - 2 * tid], c1 = s_hist[kSelectBins - 2 - 2 * tid];
        uint32_t total, above = lanes_before(c0 + c1, total);
        if (lane == 0) s_wave[wave] = total;
        __syncthreads();
        for (int i = 0; i < wave; ++i) above += s_wave[i];
        if (above < need && above + c0 + c1 >= need) {
            const bool second = above + c0 < need;
            s_pick[0] = kSelectBins - 1 - 2 * tid - second;
            s_pick[1] = need - above - (second ? c0 : 0u);
            s_pick[2] = second ? c1 : c0;
        }
        __syncthreads();
        border |= static_cast<uint64_t>(s_pick[0]) << shift;
        mask |= static_cast<uint64_t>(digit) << shift;
        need = s_pick[1];
        const uint32_t share = s_pick[2];
        if (listed) {
            __syncthreads();  // all have read the pick; the list stays, `left` is its length
            if (need == share) left = need;
        } else {
            left = share;
            if (need < left && left <= kSelectList) {
                for (int part = 0; part < parts; ++part) {
                    if (parts > 1) load(part);
#pragma unroll
                    for (int i = 0; i < kSelectKeep; ++i) {
                        if (part * kSelectRows + i * kSelectThreads >= n) break;
                        const int t = part * kSelectRows + i * kSelectThreads + tid;
                        const uint64_t k = rank_key(weight_key(x[i]), t);
                        const bool in = t >= m0 && t < m1 && (k & mask) == border;
                        const uint64_t who = __ballot(in);
                        if (who == 0) continue;
                        uint32_t at = 0;
                        if (lane == __builtin_ctzll(who)) at = atomicAdd(&s_listed, static_cast<uint32_t>(__popcll(who)));
                        at = __builtin_amdgcn_readlane(at, __builtin_ctzll(who)) + __popcll(who & ((1ull << lane) - 1));
                        if (in) s_list[at] = k;  // in any order: only counts are taken of it
                    }
                }
                listed = true;
            }
            __syncthreads();
        }
    }
    uint32_t taken = 0;  // before this part
    const uint64_t below = (1ull << lane) - 1;
    for (int part = 0; part < parts; ++part) {
        if (parts > 1) load(part);
        uint64_t takes = 0;  // of this thread's rows, a bit each
        for (int i = tid; i < kSelectKeep * kSelectWaves; i += kSelectThreads) s_count[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSelectKeep; ++i) {
            if (part * kSelectRows + i * kSelectThreads >= n) break;
            const int t = part * kSelectRows + i * kSelectThreads + tid;
            const bool mid = t >= m0 && t < m1;
            const bool take = t < n && (!mid || rank_key(weight_key(x[i]), t) >= border);
            takes |= static_cast<uint64_t>(take) << i;
            const uint32_t c = __popcll(__ballot(take));
            if (lane == 0) s_count[i * kSelectWaves + wave] = c;
        }
        __syncthreads();
        uint32_t total = 0;
        if (wave < kSelectKeep * kSelectWaves / kWave) {
            const uint32_t before = lanes_before(s_count[tid], total);
            s_count[tid] = before;
            if (lane == 0) s_wave[wave] = total;
        }
        __syncthreads();
        uint32_t sum = taken;
#pragma unroll
        for (int i = 0; i < kSelectKeep; ++i) {
            if (part * kSelectRows + i * kSelectThreads >= n) break;
            if (i > 0 && i * kSelectWaves % kWave == 0) sum += s_wave[i * kSelectWaves / kWave - 1];
            const bool take = takes >> i & 1;
            const uint32_t at = sum + s_count[i * kSelectWaves + wave] + __popcll(__ballot(take) & below);
            if (take && at < static_cast<uint32_t>(a.budget)) {
                kept[at] = part * kSelectRows + i * kSelectThreads + tid;
                if (nw) nw[at] = x[i];
            }
        }
        for (int i = 0; i < kSelectKeep * kSelectWaves / kWave; ++i) taken += s_wave[i];
        __syncthreads();
    }
    const int have = min(n, a.budget);
    for (int i = have + tid; i < a.budget; i += kSelectThreads) kept[i] = -1;
    if (nw)
        for (int i = have + tid; i < a.dst.maxp; i += kSelectThreads) nw[i] = 0.f;
    if (h == 0 && tid == 0) a.new_rows[b] = have;
}

// Their codes, scales and biases into the other cache, a workgroup per 2,048 / HD rows of it and kv head:
// each thread takes a k word, a v word, which has its codes from 8 rows anywhere, and half of them a
// parameter; all its loads are in flight together.  8 x 2,047 rows of 8 heads of 128 (38 MB read and
// written) 14 us, 4,096 of 2 heads of 256 5.
template <int HD>
__global__ __launch_bounds__(256) void q4_gather(const EvictArgs a) {
    constexpr int NG = HD / kQ4Group, W = HD / 8, ROWS = 256 / W;
    static_assert(4 * NG * ROWS <= 256 && ROWS % kQ4Block == 0, "a thread each");
    __shared__ int s_row[ROWS];
    const int h = blockIdx.y % a.src.KVH, b = blockIdx.y / a.src.KVH, tid = threadIdx.x;
    const int have = min(min(max(a.rows[b], 0), a.src.maxp), a.budget);
    const int32_t *kept = a.kept + a.src.head(b, h) * a.budget;
    const uint32_t *sk = a.src.k_head(b, h), *sv = a.src.v_head(b, h);
    uint32_t *dk = a.dst.k_head(b, h), *dv = a.dst.v_head(b, h);
    const _Float16 *sp = a.src.par_head(b, h);
    _Float16 *dp = a.dst.par_head(b, h);
    for (int j0 = blockIdx.x * ROWS; j0 < have; j0 += gridDim.x * ROWS) {
        const int n = min(ROWS, have - j0);
        if (tid < ROWS) s_row[tid] = min(max(kept[j0 + min(tid, n - 1)], 0), a.src.maxp - 1);  // past the last: it again
        __syncthreads();
        const int blk = tid / HD, d = tid % HD, left = n - blk * kQ4Block;
        const int64_t line = tid / ROWS % (4 * NG);
        const uint32_t k = sk[static_cast<int64_t>(s_row[tid / W]) * W + tid % W];
        const _Float16 p = sp[line * a.src.R + s_row[tid % ROWS]];
        uint32_t c[kQ4Block], word = 0;
#pragma unroll
        for (int u = 0; u < kQ4Block; ++u) c[u] = sv[static_cast<int64_t>(s_row[blk * kQ4Block + u] / 8) * HD + d];
#pragma unroll
        for (int u = 0; u < kQ4Block; ++u) word |= u < left ? ((c[u] >> (4 * (s_row[blk * kQ4Block + u] & 7))) & 15u) << (4 * u) : 0u;
        if (tid / W < n) dk[static_cast<int64_t>(j0) * W + tid] = k;
        if (tid < 4 * NG * ROWS && tid % ROWS < n) dp[line * a.dst.R + j0 + tid % ROWS] = p;
        if (left > 0) dv[static_cast<int64_t>(j0 / kQ4Block + blk) * HD + d] = word;
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
    const int64_t heads = static_cast<int64_t>(b.B) * c.KVH;
    const int64_t blocks = q4_workgroups((b.max_tokens + kQ4Block - 1) / kQ4Block + (b.max_tokens > 1), heads, b.N / kQ4Block * static_cast<int64_t>(c.KVH) + 2 * heads);
    const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(heads));
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
    if (sequences <= 0 || count < 0 || (count > 0 && !k && !v)) return SWQ_ERR_INVALID_ARGUMENT;
    if (sequences > cache->sequences) return SWQ_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16)
        return SWQ_ERR_MISALIGNED;
    if (count == 0) return SWQ_OK;
    const ReadArgs a{q4_view(cache), first, starts, rows, count, sequences, k, v};
    // count rows may begin and end inside a pair
    const int64_t pairs = static_cast<int64_t>(count) / kReadRows + 1, each = std::max(1, 256 / (cache->num_kv_heads * (cache->head_dim / 8)));
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>((pairs + each - 1) / each, 4096)), sequences);
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
    const size_t heads = static_cast<size_t>(sequences) * src->num_kv_heads;
    struct Span {
        const void *at;
        size_t bytes;
        bool over(const Span &o) const {
            const uintptr_t a = reinterpret_cast<uintptr_t>(at), b = reinterpret_cast<uintptr_t>(o.at);
            return at && a < b + o.bytes && b < a + bytes;
        }
    };
    const Span in[] = {{weights, heads * src->max_positions * sizeof(float)}, {rows, sequences * sizeof(int32_t)}};
    const Span out[] = {{new_weights, heads * dst->max_positions * sizeof(float)}, {new_rows, sequences * sizeof(int32_t)}, {kept, heads * budget * sizeof(int32_t)}};
    for (const Span &o : out)
        for (const Span &i : in)
            if (o.over(i)) return SWQ_ERR_INVALID_ARGUMENT;
    const Span from{src->data, q4_layout(src->sequences, src->num_kv_heads, src->head_dim, src->max_positions).total};
    const Span to{dst->data, q4_layout(dst->sequences, dst->num_kv_heads, dst->head_dim, dst->max_positions).total};
    if (from.over(to)) return SWQ_ERR_INVALID_ARGUMENT;
    const EvictArgs a{q4_view(src), q4_view(dst), weights, rows, new_weights, new_rows, kept, budget, sink, recent};
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(q4_select, dim3(static_cast<uint32_t>(heads)), dim3(kSelectThreads), 0, s, a);
    const int per = 2048 / src->head_dim;
    const dim3 grid((budget + per - 1) / per, static_cast<uint32_t>(heads));
    switch (src->head_dim) {
        case 64: hipLaunchKernelGGL(q4_gather<64>, grid, dim3(256), 0, s, a); break;
        case 128: hipLaunchKernelGGL(q4_gather<128>, grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL(q4_gather<256>, grid, dim3(256), 0, s, a); break;
    }
    return launch_status();
}
