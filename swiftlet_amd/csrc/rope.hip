// Rotary positions: tables of cos and sin for contexts of any length (swq_rope_table), and queries and keys turned
// by them (swq_rope), normalised before where the block does so (QwenCPUModel.swift:308-343, whose rotation is the
// half layout with plain angles).
//
// Table: the angle of position p and pair j is p * freq[j].  The frequencies are made on the host in 64 bits, in
// turns; a position's part of a whole turn is then one multiplication, a rounding and an fma in 64 bits, and what is
// left small enough for 32: no argument reduction of a large angle.
//
// Turning: a pass over the data, so the memory is the bound.  A lane takes two runs of V elements (16 bytes each), side by
// side over the lanes: the two halves of V pairs, neighbouring pairs, or elements that are only normalised or copied; a
// row (token, head) has as many lanes, and its sum of squares meets by DPP.
#include <algorithm>
#include <cmath>

#include "internal.hpp"
#include "tile.hpp"

namespace swq {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTableBlocks = 4096;  // that rows are shared among
constexpr int kRopeMaxParts = 4;
constexpr int kRopeMaxDim = 512;
// From so many bytes of outputs on, the caches' size, they are stored past them: 16 query and 2 key heads of 256 (bf16) of
// 16,384 tokens, 151 MB in, as many out, take 51 us so and 66 otherwise, the same inputs again (62 where they change).
constexpr int64_t kRopeStream = 32 << 20;

struct RopeTable {
    double turns[kRopeMaxDim / 2];  // per position
    const int32_t *positions;
    int64_t first;
    float2 *out;
    int32_t count, pairs;
    float magnitude;
};

// A thread keeps its pair and goes from row to row.  Within a quarter turn's eighths sine and cosine are polynomials in the
// square of r, that part of a quarter turn: through the Chebyshev nodes of [0, 1/4] in 64 bits, off by 2^-27 at most, and by 1.3
// 2^-24 with their f32 arithmetic.  The table of 262,144 positions and 32 pairs, 67 MB: 14 us, stores at 4.9 TB/s
// beside some 30 operations an element (fills reach 6.9).
__global__ __launch_bounds__(kRopeThreads) void rope_table_kernel(const RopeTable a) {
    const int step = kRopeThreads / a.pairs, j = threadIdx.x % a.pairs, own = threadIdx.x / a.pairs;
    if (own >= step) return;
    const double f = a.turns[j];
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * step + own; row < a.count; row += static_cast<int64_t>(gridDim.x) * step) {
        const double p = static_cast<double>(a.positions ? static_cast<int64_t>(a.positions[row]) : a.first + row);
        const double part = fma(p, f, -rint(p * f));  // of a turn, -1/2 to 1/2
        const float q = rintf(4.f * static_cast<float>(part)), r = static_cast<float>(fma(4.0, part, -static_cast<double>(q))), z = r * r;
        const float s = fmaf(r, 1.57079637f, r * fmaf(z, fmaf(z, fmaf(z, -0.00460214913f, 0.0796802193f), -0.64596349f), -4.37113883e-8f));
        const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0.000903628068f, -0.0208600704f), 0.253669202f), -1.23370051f), 1.f);
        const int n = static_cast<int>(q);
        const float x = n & 1 ? s : c, y = n & 1 ? c : s;
        a.out[row * a.pairs + j] = make_float2((n + 1) & 2 ? -x * a.magnitude : x * a.magnitude, n & 2 ? -y * a.magnitude : y * a.magnitude);
    }
}

struct RopePart {
    const void *x;
    void *out;
    int64_t token_stride, head_stride, out_token_stride, out_head_stride;
    const float *norm;
    uint32_t heads, first_block;
};

struct RopeArgs {
    RopePart part[kRopeMaxParts];
    int32_t parts, tokens, hd, rot, interleaved, table_rows, lanes_log2, units, pairs;
    float sign, eps;
    const float2 *table;
    const int32_t *rows;
};

typedef uint32_t RopeWords __attribute__((ext_vector_type(4)));
template <bool STREAM>
__device__ __forceinline__ void rope_put(void *p, RopeWords w) {
    if constexpr (STREAM) __builtin_nontemporal_store(w, static_cast<RopeWords *>(p));
    else *static_cast<RopeWords *>(p) = w;
}

template <typename T, int V>
struct RopeRun;  // V elements in one access
template <int V>
struct RopeRun<float, V> {
    static __device__ __forceinline__ void load(const float *p, float (&v)[V]) {
        if constexpr (V == 4) {
            const float4 u = *reinterpret_cast<const float4 *>(p);
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else {
            v[0] = *p;
        }
    }
    template <bool STREAM>
    static __device__ __forceinline__ void store(float *p, const float (&v)[V]) {
        if constexpr (V == 4) rope_put<STREAM>(p, RopeWords{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
        else *p = v[0];
    }
};
template <int V>
struct RopeRun<uint16_t, V> {
    static __device__ __forceinline__ uint16_t narrow(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
    static __device__ __forceinline__ void load(const uint16_t *p, float (&v)[V]) {
        if constexpr (V == 8) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __uint_as_float(w[e] << 16);
                v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
            }
        } else {
            v[0] = bf16_to_f32(*p);
        }
    }
    template <bool STREAM>
    static __device__ __forceinline__ void store(uint16_t *p, const float (&v)[V]) {
        if constexpr (V == 8) {
            RopeWords w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = narrow(v[2 * e]) | static_cast<uint32_t>(narrow(v[2 * e + 1])) << 16;
            rope_put<STREAM>(p, w);
        } else {
            *p = narrow(v[0]);
        }
    }
};

// A lane's share of rows: U units of two runs each.  NEAR: pairs of neighbours in runs of more than an element.
template <typename T, int V, int U, bool NEAR>
struct RopeLane {
    const RopeArgs &a;
    const int lane, lanes;

    __device__ __forceinline__ int unit(int u) const { return lane + u * lanes; }
    // Where the runs of a unit lie, neighbours side by side over the lanes.
    __device__ __forceinline__ int run(int u, int half) const {
        const int i = unit(u);
        if (i >= a.pairs) return a.rot + V * (i - a.pairs + half * (a.units - a.pairs));
        return V == 1 && a.interleaved ? 2 * i + half : V * i + half * (a.rot / 2);
    }
    // Whether a row has that run: at V = 1 the last may be missing.
    __device__ __forceinline__ bool has(int u, int half) const { return unit(u) < a.units && (V > 1 || run(u, half) < a.hd); }
    __device__ __forceinline__ bool turns(int u) const { return unit(u) < a.pairs; }
};

// U: units of a row per lane.  NEAR and STREAM: V > 1 alone; a branch for pairs of neighbours would keep v in memory.  V = 1 takes
// heads of any size and alignment and both layouts.  Each part has blocks of its own.  All loads before any store: 66 us
// instead of 85 for 16,384 tokens; two (four) rows per lane take 68 (83).
template <typename T, int V, int U, bool NEAR, bool STREAM>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeArgs a) {
    int n = 0;
#pragma unroll
    for (int k = 1; k < kRopeMaxParts; ++k)
        if (k < a.parts && blockIdx.x >= a.part[k].first_block) n = k;
    const RopePart &p = a.part[n];
    const int lanes = 1 << a.lanes_log2;
    const RopeLane<T, V, U, NEAR> l{a, static_cast<int>(threadIdx.x) & (lanes - 1), lanes};
    const uint32_t row = ((blockIdx.x - p.first_block) * kRopeThreads + threadIdx.x) >> a.lanes_log2;  // of fewer than 2^26
    const bool there = row < static_cast<uint32_t>(a.tokens) * p.heads;
    const uint32_t r = there ? row : 0, at_token = r / p.heads;
    const int64_t token = at_token, h = r - at_token * p.heads;
    const T *x = static_cast<const T *>(p.x) + token * p.token_stride + h * p.head_stride;
    T *out = static_cast<T *>(p.out) + token * p.out_token_stride + h * p.out_head_stride;
    const int t = a.rows ? min(max(a.rows[token], 0), a.table_rows - 1) : static_cast<int>(token);
    const float2 *table = a.table + static_cast<int64_t>(t) * (a.rot / 2);
    float v[U][2][V], w[U][2][V];
    float2 turn[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (there && l.has(u, half)) {
                RopeRun<T, V>::load(x + l.run(u, half), v[u][half]);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) v[u][half][e] = 0.f;
            }
        }
        if (l.turns(u)) {
#pragma unroll
            for (int e = 0; e < V; ++e) turn[u][e] = table[NEAR ? l.run(u, 2 * e / V) / 2 + 2 * e % V / 2 : V * l.unit(u) + e];
        }
    }
    if (p.norm) {
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (l.has(u, half))
#pragma unroll
                    for (int e = 0; e < V; ++e) w[u][half][e] = p.norm[l.run(u, half) + e];
#pragma unroll
            for (int e = 0; e < V; ++e) ss += v[u][0][e] * v[u][0][e] + v[u][1][e] * v[u][1][e];
        }
        const float scale = 1.0f / __fsqrt_rn(segment_sum(ss, lanes) / static_cast<float>(a.hd) + a.eps);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (l.has(u, half))
#pragma unroll
                    for (int e = 0; e < V; ++e) v[u][half][e] *= scale * w[u][half][e];
    }
    auto rotate = [&](float2 cs, float &lo, float &hi) {
        const float s = a.sign * cs.y, c0 = lo * cs.x - hi * s, c1 = hi * cs.x + lo * s;
        lo = c0, hi = c1;
    };
    if (!there) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (l.turns(u)) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (NEAR) rotate(turn[u][e], v[u][2 * e / V][2 * e % V], v[u][2 * e / V][2 * e % V + 1]);
                else rotate(turn[u][e], v[u][0][e], v[u][1][e]);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
            if (l.has(u, half)) RopeRun<T, V>::template store<STREAM>(out + l.run(u, half), v[u][half]);
    }
}

bool whole(const RopePart &p, int hd, int size) {
    auto off = [&](int64_t s) { return s * size % 16 != 0; };
    return reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && !off(p.token_stride) && !off(p.head_stride) &&
           !off(p.out_token_stride) && !off(p.out_head_stride);
}

template <typename T>
void launch_rope(RopeArgs a, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    bool vec = a.rot / 2 % V == 0 && (a.hd - a.rot) % (2 * V) == 0;
    for (int k = 0; k < a.parts; ++k) vec = vec && whole(a.part[k], a.hd, sizeof(T));
    const int v = vec ? V : 1;
    a.pairs = a.rot / 2 / v;
    a.units = a.pairs + (a.hd - a.rot + 2 * v - 1) / (2 * v);
    a.lanes_log2 = 0;
    while ((1 << a.lanes_log2) < std::min(a.units, kWave)) ++a.lanes_log2;
    int64_t rows = 0;
    for (int k = 0; k < a.parts; ++k) rows += static_cast<int64_t>(a.tokens) * a.part[k].heads;
    const bool stream = rows * a.hd * static_cast<int64_t>(sizeof(T)) > kRopeStream;
    const int64_t per = kRopeThreads >> a.lanes_log2;
    uint32_t blocks = 0;
    for (int k = 0; k < a.parts; ++k) {
        a.part[k].first_block = blocks;
        blocks += static_cast<uint32_t>((static_cast<int64_t>(a.tokens) * a.part[k].heads + per - 1) / per);
    }
    const dim3 grid(blocks), block(kRopeThreads);
    if (!vec) hipLaunchKernelGGL((rope_kernel<T, 1, (kRopeMaxDim / 2 + kWave - 1) / kWave, false, false>), grid, block, 0, s, a);
    else if (stream && a.interleaved) hipLaunchKernelGGL((rope_kernel<T, V, 1, true, true>), grid, block, 0, s, a);
    else if (stream) hipLaunchKernelGGL((rope_kernel<T, V, 1, false, true>), grid, block, 0, s, a);
    else if (a.interleaved) hipLaunchKernelGGL((rope_kernel<T, V, 1, true, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rope_kernel<T, V, 1, false, false>), grid, block, 0, s, a);
}

}  // namespace
}  // namespace swq

using namespace swq;

extern "C" int swq_rope_table(int rotary_dims, double rope_theta, const swq_rope_scaling *scaling, const int32_t *positions, int64_t first, int count,
                              float *table, void *stream) {
    if (rotary_dims <= 0 || rotary_dims % 2 != 0) return SWQ_ERR_BAD_SHAPE;
    if (rotary_dims > kRopeMaxDim) return SWQ_ERR_LIMIT;
    if (!(rope_theta > 0.0) || !std::isfinite(rope_theta) || count < 0) return SWQ_ERR_INVALID_ARGUMENT;
    const int kind = scaling ? scaling->kind : SWQ_ROPE_PLAIN;
    const double d = rotary_dims, factor = kind == SWQ_ROPE_PLAIN ? 1.0 : scaling->factor;
    if (kind < SWQ_ROPE_PLAIN || kind > SWQ_ROPE_YARN || (scaling && scaling->reserved != 0)) return SWQ_ERR_INVALID_ARGUMENT;
    if (!(factor > 0.0) || !std::isfinite(factor)) return SWQ_ERR_INVALID_ARGUMENT;
    double theta = rope_theta, low = 0.0, high = 0.0, magnitude = 1.0;
    if (kind == SWQ_ROPE_NTK) {
        if (rotary_dims <= 2) return SWQ_ERR_BAD_SHAPE;
        theta *= std::pow(factor, d / (d - 2.0));
    } else if (kind == SWQ_ROPE_YARN) {
        const double fast = scaling->beta_fast, slow = scaling->beta_slow;
        if (scaling->original_positions <= 0 || !(fast > 0.0) || !(slow > 0.0) || !std::isfinite(fast) || rope_theta == 1.0 ||
            !(scaling->magnitude >= 0.0) || !std::isfinite(scaling->magnitude))
            return SWQ_ERR_INVALID_ARGUMENT;
        // the pair that turns so often over the original positions
        auto pair_of = [&](double turns) { return d * std::log(scaling->original_positions / (6.283185307179586 * turns)) / (2.0 * std::log(rope_theta)); };
        low = std::max(std::floor(pair_of(fast)), 0.0);
        high = std::min(std::ceil(pair_of(slow)), d - 1.0);
        magnitude = scaling->magnitude > 0.0 ? scaling->magnitude : factor > 1.0 ? 1.0 + 0.1 * std::log(factor) : 1.0;
    }
    if (count == 0) return SWQ_OK;
    if (!table) return SWQ_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(table) % 8 != 0 || reinterpret_cast<uintptr_t>(positions) % 4 != 0) return SWQ_ERR_MISALIGNED;
    RopeTable a{};
    a.positions = positions;
    a.first = first;
    a.out = reinterpret_cast<float2 *>(table);
    a.pairs = rotary_dims / 2;
    a.count = count;
    a.magnitude = static_cast<float>(magnitude);
    for (int j = 0; j < a.pairs; ++j) {
        double f = std::pow(theta, -2.0 * j / d);
        if (kind == SWQ_ROPE_LINEAR) f /= factor;
        if (kind == SWQ_ROPE_YARN) {
            const double share = std::min(std::max((j - low) / std::max(high - low, 0.001), 0.0), 1.0);
            f = (1.0 - share) * f + share * f / factor;
        }
        a.turns[j] = f / 6.283185307179586;
    }
    const int step = kRopeThreads / a.pairs, blocks = std::min((count - 1) / step + 1, kRopeTableBlocks);
    hipLaunchKernelGGL(rope_table_kernel, dim3(blocks), dim3(kRopeThreads), 0, static_cast<hipStream_t>(stream), a);
    return launch_status();
}

extern "C" int swq_rope(const swq_rope_heads *parts, int n, int tokens, int head_dim, int rotary_dims, int layout, int inverse, float norm_eps,
                        const float *table, int table_rows, const int32_t *rows, int dtype, void *stream) {
    if (!parts || n <= 0 || tokens < 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (n > kRopeMaxParts) return SWQ_ERR_LIMIT;
    if (head_dim <= 0 || rotary_dims <= 0 || rotary_dims % 2 != 0 || rotary_dims > head_dim) return SWQ_ERR_BAD_SHAPE;
    if (head_dim > kRopeMaxDim) return SWQ_ERR_LIMIT;
    if ((layout != SWQ_ROPE_HALF && layout != SWQ_ROPE_INTERLEAVED) || (inverse != 0 && inverse != 1) || !(norm_eps >= 0.f)) return SWQ_ERR_INVALID_ARGUMENT;
    if (dtype != SWQ_F32 && dtype != SWQ_BF16) return SWQ_ERR_UNSUPPORTED_DTYPE;
    const int size = dtype == SWQ_F32 ? 4 : 2;
    RopeArgs a{};
    int64_t heads = 0;
    for (int k = 0; k < n; ++k) {
        const swq_rope_heads &p = parts[k];
        if (p.reserved != 0 || p.heads <= 0) return SWQ_ERR_INVALID_ARGUMENT;
        if (tokens > 0 && (!p.x || !p.out)) return SWQ_ERR_INVALID_ARGUMENT;
        if (reinterpret_cast<uintptr_t>(p.x) % size != 0 || reinterpret_cast<uintptr_t>(p.out) % size != 0 || reinterpret_cast<uintptr_t>(p.norm_weight) % 4 != 0)
            return SWQ_ERR_MISALIGNED;
        a.part[k] = {p.x, p.out, p.token_stride, p.head_stride, p.out_token_stride, p.out_head_stride, p.norm_weight, static_cast<uint32_t>(p.heads), 0};
        heads += p.heads;
        if (heads > 65536) return SWQ_ERR_LIMIT;
    }
    // a launch has fewer than 2^32 work-items, 64 a row at most
    if (tokens * heads >= (1LL << 32) / kWave - kRopeMaxParts * kRopeThreads) return SWQ_ERR_LIMIT;
    if (tokens == 0) return SWQ_OK;
    if (!table || table_rows <= 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (!rows && table_rows < tokens) return SWQ_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(table) % 8 != 0 || reinterpret_cast<uintptr_t>(rows) % 4 != 0) return SWQ_ERR_MISALIGNED;
    a.parts = n;
    a.tokens = tokens;
    a.hd = head_dim;
    a.rot = rotary_dims;
    a.interleaved = layout == SWQ_ROPE_INTERLEAVED;
    a.table_rows = table_rows;
    a.sign = inverse ? -1.f : 1.f;
    a.eps = norm_eps;
    a.table = reinterpret_cast<const float2 *>(table);
    a.rows = rows;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == SWQ_F32) launch_rope<float>(a, s);
    else launch_rope<uint16_t>(a, s);
    return launch_status();
}
