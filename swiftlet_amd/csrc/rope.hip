// Rotary positions: tables of cos and sin for contexts of any length (swq_rope_table), and queries and keys turned
// by them (swq_rope), normalised before where the block does so (QwenCPUModel.swift:308-343, whose rotation is the
// half layout with plain angles).
//
// Table: the angle of position p and pair j is p * freq[j].  The frequencies are made on the host in 64 bits, in
// turns; a position's part of a whole turn is then one multiplication, a rounding and an fma in 64 bits, and what is
// left is small enough for 32: no argument reduction of a large angle.
//
// Turning: a pass over the data, so the memory is the bound.  A lane takes two runs of V elements (16 bytes each):
// the two halves of V pairs (half layout), V neighbouring pairs (interleaved) or 2 V elements that are only
// normalised or copied; a row (token, head) has as many lanes, and its sum of squares meets by DPP.
#include <algorithm>
#include <cmath>

#include "internal.hpp"
#include "tile.hpp"

namespace swq {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxParts = 4;
constexpr int kRopeMaxDim = 512;

struct RopeTable {
    double turns[kRopeMaxDim / 2];  // per position
    const int32_t *positions;
    int64_t first;
    float2 *out;
    int64_t total;
    int32_t pairs;
    float magnitude;
};

__global__ __launch_bounds__(kRopeThreads) void rope_table_kernel(const RopeTable a) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRopeThreads + threadIdx.x; i < a.total; i += static_cast<int64_t>(gridDim.x) * kRopeThreads) {
        const int64_t row = i / a.pairs;
        const int j = static_cast<int>(i - row * a.pairs);
        const double p = static_cast<double>(a.positions ? static_cast<int64_t>(a.positions[row]) : a.first + row), f = a.turns[j];
        const double part = fma(p, f, -rint(p * f));  // of a turn, -1/2 to 1/2
        const float x = static_cast<float>(2.0 * part), rest = 3.14159265f * static_cast<float>(2.0 * part - static_cast<double>(x));
        float s, c;
        sincospif(x, &s, &c);
        a.out[i] = make_float2(fmaf(-rest, s, c) * a.magnitude, fmaf(rest, c, s) * a.magnitude);
    }
}

struct RopePart {
    const void *x;
    void *out;
    int64_t token_stride, head_stride, out_token_stride, out_head_stride;
    const float *norm;
    int32_t first_head;  // of all parts' heads together
};

struct RopeArgs {
    RopePart part[kRopeMaxParts];
    int32_t parts, heads, tokens, hd, rot, interleaved, table_rows, lanes_log2, units, pairs;
    float sign, eps;
    const float2 *table;
    const int32_t *rows;
};

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
    static __device__ __forceinline__ void store(float *p, const float (&v)[V]) {
        if constexpr (V == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
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
    static __device__ __forceinline__ void store(uint16_t *p, const float (&v)[V]) {
        if constexpr (V == 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = narrow(v[2 * e]) | static_cast<uint32_t>(narrow(v[2 * e + 1])) << 16;
            *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *p = narrow(v[0]);
        }
    }
};

// U: units of a row per lane.  V = 1 takes heads of any size and alignment; its last unit may be half a one.
template <typename T, int V, int U>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeArgs a) {
    const int lanes = 1 << a.lanes_log2;
    const uint32_t row = (blockIdx.x * kRopeThreads + threadIdx.x) >> a.lanes_log2;  // of fewer than 2^26
    const int lane = threadIdx.x & (lanes - 1);
    const bool there = row < static_cast<uint32_t>(a.tokens) * a.heads;
    const uint32_t r = there ? row : 0, at_token = r / a.heads;
    const int64_t token = at_token;
    const int head = static_cast<int>(r - at_token * a.heads);
    int n = 0;
#pragma unroll
    for (int k = 1; k < kRopeMaxParts; ++k)
        if (k < a.parts && head >= a.part[k].first_head) n = k;
    const RopePart p = a.part[n];
    const int h = head - p.first_head;
    const T *x = static_cast<const T *>(p.x) + token * p.token_stride + h * p.head_stride;
    T *out = static_cast<T *>(p.out) + token * p.out_token_stride + h * p.out_head_stride;

    float v[U][2][V];
    int at[U][2];
    bool has[U], both[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int unit = lane + u * lanes;
        has[u] = there && unit < a.units;
        both[u] = has[u];
        if (unit < a.pairs) {
            at[u][0] = a.interleaved ? 2 * V * unit : V * unit;
            at[u][1] = a.interleaved ? at[u][0] + V : a.rot / 2 + V * unit;
        } else {
            at[u][0] = a.rot + 2 * V * (unit - a.pairs);
            at[u][1] = at[u][0] + V;
            if (V == 1) both[u] = has[u] && at[u][1] < a.hd;
        }
        if (has[u]) RopeRun<T, V>::load(x + at[u][0], v[u][0]);
        if (both[u]) RopeRun<T, V>::load(x + at[u][1], v[u][1]);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) v[u][1][e] = 0.f;
    }
    const int t = a.rows ? min(max(a.rows[token], 0), a.table_rows - 1) : static_cast<int>(token);
    const float2 *turn = a.table + static_cast<int64_t>(t) * (a.rot / 2);
    if (p.norm) {
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (has[u])
#pragma unroll
                for (int e = 0; e < V; ++e) ss += v[u][0][e] * v[u][0][e] + v[u][1][e] * v[u][1][e];
        const float scale = 1.0f / __fsqrt_rn(segment_sum(ss, lanes) / static_cast<float>(a.hd) + a.eps);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (half ? both[u] : has[u])
#pragma unroll
                    for (int e = 0; e < V; ++e) v[u][half][e] *= scale * p.norm[at[u][half] + e];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!has[u]) continue;
        const int unit = lane + u * lanes;
        if (unit < a.pairs) {
            float *flat = &v[u][0][0];  // interleaved: pairs lie side by side over both runs
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 cs = turn[V * unit + e];
                const float s = a.sign * cs.y;
                float &lo = a.interleaved ? flat[2 * e] : v[u][0][e], &hi = a.interleaved ? flat[2 * e + 1] : v[u][1][e];
                const float c0 = lo * cs.x - hi * s, c1 = hi * cs.x + lo * s;
                lo = c0, hi = c1;
            }
        }
        RopeRun<T, V>::store(out + at[u][0], v[u][0]);
        if (both[u]) RopeRun<T, V>::store(out + at[u][1], v[u][1]);
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
    const int64_t threads = (static_cast<int64_t>(a.tokens) * a.heads) << a.lanes_log2;
    const dim3 grid(static_cast<uint32_t>((threads + kRopeThreads - 1) / kRopeThreads)), block(kRopeThreads);
    if (vec) hipLaunchKernelGGL((rope_kernel<T, V, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rope_kernel<T, 1, (kRopeMaxDim / 2 + 1 + kWave - 1) / kWave>), grid, block, 0, s, a);
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
    a.total = static_cast<int64_t>(count) * a.pairs;
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
    const int64_t blocks = std::min<int64_t>((a.total + kRopeThreads - 1) / kRopeThreads, 1 << 20);
    hipLaunchKernelGGL(rope_table_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kRopeThreads), 0, static_cast<hipStream_t>(stream), a);
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
        a.part[k] = {p.x, p.out, p.token_stride, p.head_stride, p.out_token_stride, p.out_head_stride, p.norm_weight, static_cast<int32_t>(heads)};
        heads += p.heads;
        if (heads > 65536) return SWQ_ERR_LIMIT;
    }
    // a launch has fewer than 2^32 work-items, 64 a row at most
    if (tokens * heads >= (1LL << 32) / kWave - kRopeThreads) return SWQ_ERR_LIMIT;
    if (tokens == 0) return SWQ_OK;
    if (!table || table_rows <= 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (!rows && table_rows < tokens) return SWQ_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(table) % 8 != 0 || reinterpret_cast<uintptr_t>(rows) % 4 != 0) return SWQ_ERR_MISALIGNED;
    a.parts = n;
    a.heads = static_cast<int32_t>(heads);
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
