// One head's new row into a 4-bit cache, by one wave: EPL = hd / 64 consecutive dims per lane, in 64
// bits up to the format's own roundings.
#pragma once

#include "q4_cache.hpp"

namespace swq {

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = dpp_u32<CTRL>(static_cast<uint32_t>(u)), hi = dpp_u32<CTRL>(static_cast<uint32_t>(u >> 32));
    return __builtin_bit_cast(double, lo | (hi << 32));
}

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
    return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(v)));
}

__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(double, lo | (static_cast<uint64_t>(hi) << 32));
}

// op over LANES consecutive lanes (8, 16, 32 or 64), to each of them: through DPP within 16, then
// through scalar registers (a ds_bpermute per step and half costs four times as long).
template <int LANES, typename Op>
__device__ __forceinline__ double reduce_f64(double v, Op op) {
    v = op(v, dpp_f64<0xB1>(v));   // quad_perm [1,0,3,2]
    v = op(v, dpp_f64<0x4E>(v));   // quad_perm [2,3,0,1]
    v = op(v, dpp_f64<0x141>(v));  // row_half_mirror
    if constexpr (LANES >= 16) v = op(v, dpp_f64<0x140>(v));  // row_mirror
    if constexpr (LANES > 16) {
        const double a = op(lane_f64(v, 0), lane_f64(v, 16)), b = op(lane_f64(v, 32), lane_f64(v, 48));
        v = LANES == 64 ? op(a, b) : (threadIdx.x & 32 ? b : a);
    }
    return v;
}

// This lane's elements of a norm weight and of the rotation at them: element i < 2 * half turns with
// its partner i +- half by angle i % half.
template <int EPL>
struct Q4HeadTable {
    float w[EPL];
    float2 cs[EPL];
    __device__ __forceinline__ void load(const float *weight, const float2 *turn, int half) {
        const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int i = lane * EPL + e;
            w[e] = weight[i];
            cs[e] = half > 0 ? turn[i < half ? i : i < 2 * half ? i - half : 0] : make_float2(1.f, 0.f);
        }
    }
};

// f16 by way of f32, both roundings as the format has them: the compiler would make one of the two.
__device__ __forceinline__ _Float16 f16_by_f32(double x) {
    float f = static_cast<float>(x);
    asm volatile("" : "+v"(f));
    return static_cast<_Float16>(f);
}

// A group's scale: x to f16, or the largest number with which no value, bias + 15 scale at most, passes f16's
// largest.  One below x's is not always enough: a bias of that size may have been rounded up by 16.
__device__ __forceinline__ _Float16 q4_scale(double x, _Float16 bias) {
    _Float16 s = f16_by_f32(x);
    if (fmaf(15.0f, static_cast<float>(s), static_cast<float>(bias)) >= 65504.0f) {
        const double b = static_cast<double>(static_cast<float>(bias));
        auto over = [&](_Float16 v) { return fma(15.0, static_cast<double>(static_cast<float>(v)), b) > 65504.0; };  // exact
        if (over(s)) {
            s = f16_by_f32((65504.0 - b) / 15.0);  // to one of the two numbers about it
            if (over(s)) s = __builtin_bit_cast(_Float16, static_cast<uint16_t>(__builtin_bit_cast(uint16_t, s) - 1));
        }
    }
    return s;
}

// The codes of values whose group has scale and bias.  (y - b) / s is first taken in f32 with a
// reciprocal: codes are at most 15 and a bit and the difference, the reciprocal and the product each
// round once, so it is off by less than 16 * 4 * 2^-24 = 4e-6.  Where that leaves the nearest integer in
// doubt an exact division decides, so that a value on a border between two codes goes to the even one.
template <int EPL, typename X>
__device__ __forceinline__ void q4_codes(const X (&y)[EPL], uint32_t (&q)[EPL], _Float16 scale, _Float16 bias) {
    const X b = static_cast<X>(static_cast<float>(bias));
    const float s = static_cast<float>(scale), inv = s > 0.f ? 1.0f / s : 0.f;
    bool doubt = false;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        const float t = static_cast<float>(y[e] - b) * inv, n = rintf(t);
        doubt |= fabsf(t - n) > 0.49999f;
        q[e] = static_cast<uint32_t>(fminf(fmaxf(n, 0.f), 15.f));
    }
    if (__any(doubt)) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
            q[e] = s > 0.f ? static_cast<uint32_t>(fmin(fmax(rint((static_cast<double>(y[e]) - static_cast<double>(b)) / static_cast<double>(s)), 0.0), 15.0))
                           : 0u;
    }
}

// 4-bit codes of EPL consecutive dims per lane, 64 / EPL lanes to a group: the scale and bias of this
// lane's group, the codes into q.
template <int EPL>
__device__ __forceinline__ void q4_quantise(const double (&x)[EPL], uint32_t (&q)[EPL], _Float16 &scale, _Float16 &bias) {
    double y[EPL], lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        y[e] = x[e] == x[e] ? fmin(fmax(x[e], -65504.0), 65504.0) : 0.0;
        lo = fmin(lo, y[e]);
        hi = fmax(hi, y[e]);
    }
    lo = reduce_f64<kQ4Group / EPL>(lo, [](double a, double b) { return fmin(a, b); });
    hi = reduce_f64<kQ4Group / EPL>(hi, [](double a, double b) { return fmax(a, b); });
    bias = f16_by_f32(lo);
    scale = q4_scale((hi - lo) / 15.0, bias);
    q4_codes<EPL>(y, q, scale, bias);
}

// The same of numbers that come in 32 bits, 8 per lane: only their difference needs more.
__device__ __forceinline__ void q4_quantise(const float (&x)[8], uint32_t (&q)[8], _Float16 &scale, _Float16 &bias) {
    float y[8], lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        y[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -65504.f), 65504.f) : 0.f;
        lo = fminf(lo, y[e]);
        hi = fmaxf(hi, y[e]);
    }
    lo = fminf(lo, dpp_f32<0xB1>(lo));
    hi = fmaxf(hi, dpp_f32<0xB1>(hi));
    lo = fminf(lo, dpp_f32<0x4E>(lo));
    hi = fmaxf(hi, dpp_f32<0x4E>(hi));
    lo = fminf(lo, dpp_f32<0x141>(lo));
    hi = fmaxf(hi, dpp_f32<0x141>(hi));
    bias = static_cast<_Float16>(lo);
    scale = q4_scale((static_cast<double>(hi) - static_cast<double>(lo)) / 15.0, bias);
    q4_codes<8>(y, q, scale, bias);
}

// Scale and bias of this lane's group to parameters `which` and which + 1 of `row`.
template <int HD>
__device__ __forceinline__ void q4_put_params(_Float16 *par, int64_t R, int which, int64_t row, _Float16 scale, _Float16 bias) {
    constexpr int EPL = HD / kWave, NG = HD / kQ4Group;
    const int lane = threadIdx.x & (kWave - 1), g = lane * EPL / kQ4Group;
    if (lane % (kQ4Group / EPL) == 0) {
        par[(static_cast<int64_t>(which) * NG + g) * R + row] = scale;
        par[(static_cast<int64_t>(which + 1) * NG + g) * R + row] = bias;
    }
}

// A key: x / rms * w, turned, quantised, its words and parameters written.  lds: HD doubles of this
// wave; half: of the rotated dims.
template <int HD>
__device__ __forceinline__ void q4_key_row(double (&x)[HD / kWave], const Q4HeadTable<HD / kWave> &tab, float eps, int half,
                                           double *lds, uint32_t *kw, _Float16 *par, int64_t R, int64_t row) {
    constexpr int EPL = HD / kWave;
    const int lane = threadIdx.x & (kWave - 1);
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) ss += x[e] * x[e];
    ss = reduce_f64<kWave>(ss, [](double a, double b) { return a + b; });
    const double inv = 1.0 / sqrt(ss / HD + static_cast<double>(eps));
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        x[e] = x[e] * inv * static_cast<double>(tab.w[e]);
        lds[lane * EPL + e] = x[e];
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (half > 0) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int i = lane * EPL + e;
            if (i < 2 * half) {
                const double o = lds[i < half ? i + half : i - half];
                const double c = static_cast<double>(tab.cs[e].x), s = static_cast<double>(tab.cs[e].y);
                x[e] = i < half ? x[e] * c - o * s : x[e] * c + o * s;
            }
        }
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint32_t q[EPL], word = 0;
    _Float16 scale, bias;
    q4_quantise<EPL>(x, q, scale, bias);
#pragma unroll
    for (int e = 0; e < EPL; ++e) word |= q[e] << (4 * ((lane * EPL + e) & 7));
    word |= dpp_u32<0xB1>(word);  // the lanes of one word: 2, 4 or 8
    if constexpr (EPL <= 2) word |= dpp_u32<0x4E>(word);
    if constexpr (EPL == 1) word |= dpp_u32<0x141>(word);
    if (lane % (8 / EPL) == 0) kw[row * (HD / 8) + lane * EPL / 8] = word;
    q4_put_params<HD>(par, R, kQ4KScale, row, scale, bias);
}

// A value row quantised, its parameters written; its codes into q, for the words of its block.
template <int HD>
__device__ __forceinline__ void q4_value_row(const double (&x)[HD / kWave], uint32_t (&q)[HD / kWave], _Float16 *par, int64_t R,
                                             int64_t row) {
    _Float16 scale, bias;
    q4_quantise<HD / kWave>(x, q, scale, bias);
    q4_put_params<HD>(par, R, kQ4VScale, row, scale, bias);
}

}  // namespace swq
