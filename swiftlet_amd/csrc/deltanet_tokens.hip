// The gated DeltaNet block over the tokens of many sequences (swq_deltanet_tokens): the entry point, the token after
// token form, and the ring's rows.  The block is deltanet.hip's, numerics of QwenCPUModel.deltaNetForward
// (QwenCPUModel.swift:371-496); the state's layout too, so that a sequence may go on with either call.
//
// Token after token: one workgroup per (sequence, value head).  The head's matrix [dv][dk] is loaded once, stays in
// registers over the sequence's tokens (its first 128 rows, 64 at dk 256; others pass through memory) and is stored once;
// the convolution's rows stay in registers as well, and the next token's inputs are in flight while one is computed.
#include <algorithm>

#include "deltanet.hpp"
#include "route.hpp"

namespace swq {
namespace {

constexpr int kTokThreads = 512;
constexpr int kTokWaves = kTokThreads / kWave;
constexpr int kRingThreads = 256;

__device__ __forceinline__ float lds_sum_sq(const float *v, int n, int lane) {
    float ss = 0.f;
    for (int i = lane; i < n; i += kWave) ss += v[i] * v[i];
    return wave_sum_all(ss);
}

// WIDE: kernels of up to 8 rows and any number of channels per head; else 4 rows and a channel per thread, as
// the usual heads of 128 have.  Kernels shorter than that have zero weights in front, and zeros for the rows that meet
// them, which change no bit of the sums.  ONE: no sequence brings more than a token, and the ring takes its row here (a
// workgroup then overwrites no row that another still reads; with more tokens it would).  MANY: registers for two
// workgroups to a CU, where there are more workgroups than CUs: 64 single tokens at 32 heads of 128 take 51 us instead of 56
// (the same states again, in part from the caches; 64 where they change, 4.3 TB/s), 32 sequences of 4 55 instead of 69; one of 8
// would take 29 instead of 27.  Several tokens spill 4 registers so, 6 at dk 256.
template <int DK, bool WIDE, bool ONE, bool MANY, typename T>
__global__ __launch_bounds__(kTokThreads, MANY ? 4 : 2) void deltanet_tokens_kernel(const DnTokens a) {
    constexpr int C4 = DK / 4;          // float4 chunks per state row
    constexpr int G = C4 < 4 ? C4 : C4 > 32 ? 8 : 4;  // lanes per row
    constexpr int CPL = C4 / G;         // chunks per lane
    constexpr int RPW = kWave / G;      // rows per wave and pass
    constexpr int KM = WIDE ? kDnMaxConv : 4;                                           // rows of the convolution
    constexpr int MC = WIDE ? (2 * DK + kDnMaxDv + kTokThreads - 1) / kTokThreads : 1;  // channels per thread
    __shared__ __align__(16) float s_q[DK], s_k[DK];
    __shared__ float s_v[kDnMaxDv], s_o[kDnMaxDv];
    __shared__ float s_gb[2];
    const int b = blockIdx.x / a.nv, hv = blockIdx.x % a.nv, hk = hv / a.rep, ri = hv % a.rep;
    const int tokens = ONE ? min(a.count(b), 1) : a.count(b);
    uint8_t *slot = a.state(b);
    if (tokens <= 0 || !slot) return;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t n0 = a.first(b);
    const uint32_t pos = a.position(b);
    float *ring = reinterpret_cast<float *>(slot);

    // the state rows of the first pass, before anything that waits
    const int gl = lane % G;
    float *st_head = reinterpret_cast<float *>(slot + a.rec_at) + static_cast<int64_t>(hv) * a.dv * DK;
    const int row_first = wave * RPW + lane / G;
    float4 s0[CPL];
    if (row_first < a.dv) {
        const float4 *sr = reinterpret_cast<const float4 *>(st_head + static_cast<int64_t>(row_first) * DK);
#pragma unroll
        for (int m = 0; m < CPL; ++m) s0[m] = sr[gl + G * m];
    }
    const float nw0 = tid < a.dv ? a.norm_w[tid] : 0.f;

    // this thread's channels: weights, earlier rows, the first token's inputs
    const int nch = 2 * DK + a.dv;
    const T *x = static_cast<const T *>(a.qkvz) + n0 * a.qkvz_stride;
    const T *ba = static_cast<const T *>(a.ba) + n0 * a.ba_stride;
    int at[MC];
    float w[MC][KM], hist[MC][KM - 1], xn[MC];
#pragma unroll
    for (int c = 0; c < MC; ++c) {
        const int t = tid + c * kTokThreads;
        if (t >= nch) continue;
        const int ch = t < DK ? hk * DK + t : t < 2 * DK ? a.keyD + hk * DK + (t - DK) : 2 * a.keyD + hv * a.dv + (t - 2 * DK);
        at[c] = mixed_at(a, ch);
#pragma unroll
        for (int j = 0; j < KM; ++j) {
            const int jj = j - (KM - a.K);
            w[c][j] = jj >= 0 ? a.conv_w[static_cast<int64_t>(ch) * a.K + jj] : 0.f;
            // row j of the last KM - 1: position pos - (KM - 1) + j, in slot (pos + 1 + jj) % K
            if (j < KM - 1) hist[c][j] = jj >= 0 ? ring[static_cast<int64_t>((pos + 1 + jj) % a.K) * a.convD + ch] : 0.f;
        }
        xn[c] = dn_load(x, at[c]);
        if constexpr (ONE) {
            if (t >= 2 * DK || ri == 0) ring[static_cast<int64_t>(pos % a.K) * a.convD + ch] = xn[c];
        }
    }
    const int z_first = z_at(a, hv, min(tid, a.dv - 1)), b_at = ba_at(a, hv, 0), a_at = ba_at(a, hv, 1);
    float z0 = dn_load(x, z_first), bn = dn_load(ba, b_at), an = dn_load(ba, a_at);
    const float dt = a.dt_bias[hv], a_log = a.a_log[hv];

    for (int i = 0; i < tokens; ++i) {
        const float z = z0, bv = bn, av = an;
        float xc[MC];
#pragma unroll
        for (int c = 0; c < MC; ++c) xc[c] = xn[c];
        if (!ONE && i + 1 < tokens) {
            const T *nx = x + (i + 1) * a.qkvz_stride, *nb = ba + (i + 1) * a.ba_stride;
#pragma unroll
            for (int c = 0; c < MC; ++c)
                if (tid + c * kTokThreads < nch) xn[c] = dn_load(nx, at[c]);
            z0 = dn_load(nx, z_first);
            bn = dn_load(nb, b_at);
            an = dn_load(nb, a_at);
        }
        // 1. convolution and silu (multiply and add rounded separately as the reference does)
#pragma unroll
        for (int c = 0; c < MC; ++c) {
            const int t = tid + c * kTokThreads;
            if (t >= nch) continue;
            float acc = 0.f;
#pragma unroll
            for (int j = 0; j < KM - 1; ++j) acc = __fadd_rn(acc, __fmul_rn(w[c][j], hist[c][j]));
            acc = __fadd_rn(acc, __fmul_rn(w[c][KM - 1], xc[c]));
            (t < DK ? s_q[t] : t < 2 * DK ? s_k[t - DK] : s_v[t - 2 * DK]) = silu_acc(acc);
            if constexpr (!ONE) {
#pragma unroll
                for (int j = 0; j < KM - 1; ++j) hist[c][j] = j < KM - a.K ? 0.f : j < KM - 2 ? hist[c][j + 1] : xc[c];
            }
        }
        // 2. gates
        if (tid == 0) {
            s_gb[0] = expf(-expf(a_log) * softplus_acc(av + dt));
            s_gb[1] = sigmoid_acc(bv);
        }
        lds_barrier();  // only LDS is handed over, here and below
        const float ssq = lds_sum_sq(s_q, DK, lane), ssk = lds_sum_sq(s_k, DK, lane);
        const float inv = 1.0f / __fsqrt_rn(static_cast<float>(DK));
        const float scq = 1.0f / __fsqrt_rn(ssq / static_cast<float>(DK) + 1e-6f);
        const float sck = 1.0f / __fsqrt_rn(ssk / static_cast<float>(DK) + 1e-6f);
        const float g = s_gb[0], beta = s_gb[1];

        // 3. recurrence: G lanes per row, chunk m of lane j is chunk j + G * m of the row
        auto part = [&](const float *from, int m, float by, float and_by) {
            const float4 x = *reinterpret_cast<const float4 *>(from + 4 * (gl + G * m));
            return make_float4(x.x * by * and_by, x.y * by * and_by, x.z * by * and_by, x.w * by * and_by);
        };
        auto turn = [&](float4(&s)[CPL], int row) {
            float mem = 0.f;
#pragma unroll
            for (int m = 0; m < CPL; ++m) {
                const float4 k = part(s_k, m, sck, inv);
                s[m].x *= g;
                s[m].y *= g;
                s[m].z *= g;
                s[m].w *= g;
                mem += s[m].x * k.x + s[m].y * k.y + s[m].z * k.z + s[m].w * k.w;
            }
            mem = segment_sum(mem, G);
            const float delta = (s_v[row] - mem) * beta;
            if constexpr (MANY) asm volatile("" ::: "memory");  // read again, for fewer registers
            float o = 0.f;
#pragma unroll
            for (int m = 0; m < CPL; ++m) {
                const float4 k = part(s_k, m, sck, inv), q = part(s_q, m, scq, inv * inv);
                s[m].x += k.x * delta;
                s[m].y += k.y * delta;
                s[m].z += k.z * delta;
                s[m].w += k.w * delta;
                o += s[m].x * q.x + s[m].y * q.y + s[m].z * q.z + s[m].w * q.w;
            }
            o = segment_sum(o, G);
            if (gl == 0) s_o[row] = o;
        };
        if (row_first < a.dv) turn(s0, row_first);
        for (int row = row_first + kTokWaves * RPW; row < a.dv; row += kTokWaves * RPW) {
            float4 *sr = reinterpret_cast<float4 *>(st_head + static_cast<int64_t>(row) * DK);
            float4 s[CPL];
#pragma unroll
            for (int m = 0; m < CPL; ++m) s[m] = sr[gl + G * m];
            turn(s, row);
#pragma unroll
            for (int m = 0; m < CPL; ++m) sr[gl + G * m] = s[m];
        }
        lds_barrier();

        // 4. gated RMSNorm: y = o * (scale * w) * silu(z)
        const float sso = lds_sum_sq(s_o, a.dv, lane);
        const float sc = 1.0f / __fsqrt_rn(sso / static_cast<float>(a.dv) + a.eps);
        const int64_t row = (n0 + i) * a.nv * a.dv + hv * a.dv;
        for (int e = tid; e < a.dv; e += kTokThreads) {
            const float y = s_o[e] * (sc * (e == tid ? nw0 : a.norm_w[e]));
            dn_store_as(a.out, a.out_f32, row + e, y * silu_acc(e == tid ? z : dn_load(x + i * a.qkvz_stride, z_at(a, hv, e))));
        }
    }
    if (row_first < a.dv) {
        float4 *sr = reinterpret_cast<float4 *>(st_head + static_cast<int64_t>(row_first) * DK);
#pragma unroll
        for (int m = 0; m < CPL; ++m) sr[gl + G * m] = s0[m];
    }
}

// The last K rows of what each sequence brought into its ring, after every launch that reads the earlier ones.
template <typename T>
__global__ __launch_bounds__(kRingThreads) void deltanet_ring_kernel(const DnTokens a, int parts) {
    const int b = blockIdx.x / parts, ch = (blockIdx.x % parts) * kRingThreads + threadIdx.x;
    const int tokens = a.count(b);
    uint8_t *slot = a.state(b);
    if (tokens <= 0 || !slot || ch >= a.convD) return;
    const uint32_t pos = a.position(b);
    const T *x = static_cast<const T *>(a.qkvz) + a.first(b) * a.qkvz_stride + mixed_at(a, ch);
    for (int i = max(tokens - a.K, 0); i < tokens; ++i)
        reinterpret_cast<float *>(slot)[static_cast<int64_t>((pos + static_cast<uint32_t>(i)) % a.K) * a.convD + ch] = dn_load(x, i * a.qkvz_stride);
}

template <int DK, typename T>
void launch_tokens(const DnTokens &a, hipStream_t s) {
    const dim3 grid(a.B * a.nv), block(kTokThreads);
    const bool one = a.max_tokens == 1, wide = a.K > 4 || 2 * a.dk + a.dv > kTokThreads, many = a.B * a.nv > kCus;
    if (wide && one) hipLaunchKernelGGL((deltanet_tokens_kernel<DK, true, true, false, T>), grid, block, 0, s, a);
    else if (wide) hipLaunchKernelGGL((deltanet_tokens_kernel<DK, true, false, false, T>), grid, block, 0, s, a);
    else if (one) hipLaunchKernelGGL((deltanet_tokens_kernel<DK, false, true, true, T>), grid, block, 0, s, a);
    else if (many) hipLaunchKernelGGL((deltanet_tokens_kernel<DK, false, false, true, T>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((deltanet_tokens_kernel<DK, false, false, false, T>), grid, block, 0, s, a);
    if (!one && a.most == INT32_MAX) {  // else deltanet_chunks.hip's last launch does it
        const int parts = (a.convD + kRingThreads - 1) / kRingThreads;
        hipLaunchKernelGGL(deltanet_ring_kernel<T>, dim3(a.B * parts), dim3(kRingThreads), 0, s, a, parts);
    }
}

template <typename T>
void launch_tokens_dk(const DnTokens &a, hipStream_t s) {
    switch (a.dk) {
        case 8: launch_tokens<8, T>(a, s); break;
        case 16: launch_tokens<16, T>(a, s); break;
        case 32: launch_tokens<32, T>(a, s); break;
        case 64: launch_tokens<64, T>(a, s); break;
        case 128: launch_tokens<128, T>(a, s); break;
        default: launch_tokens<256, T>(a, s); break;
    }
}

// Sizes of a call without its device arrays.
int check_sizes(const swq_deltanet_layer *l, const swq_deltanet_batch *b) {
    const int st = check_deltanet_layer(l);
    if (st != SWQ_OK) return st;
    if (!b || b->reserved != 0 || b->sequences <= 0 || b->tokens < 0 || b->slots <= 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (b->qkvz_stride < 0 || b->ba_stride < 0) return SWQ_ERR_INVALID_ARGUMENT;
    if (b->starts ? (b->max_tokens <= 0 && b->tokens > 0) : b->tokens % b->sequences != 0) return SWQ_ERR_BAD_SHAPE;
    const int64_t val = 1LL * l->num_value_heads * l->value_head_dim, conv = 2LL * l->num_key_heads * l->key_head_dim + val;
    if ((b->qkvz_stride && b->qkvz_stride < conv + val) || (b->ba_stride && b->ba_stride < 2LL * l->num_value_heads))
        return SWQ_ERR_BAD_SHAPE;
    if (!b->slot && b->slots < b->sequences) return SWQ_ERR_BAD_SHAPE;
    // rows that 32 bits address, and launches of fewer than 2^32 work-items
    if (conv + val > INT32_MAX || (1LL << 32) / kTokThreads <= 1LL * b->sequences * l->num_value_heads ||
        (1LL << 32) <= b->sequences * (conv + kRingThreads) || (deltanet_chunks_take(l) && !deltanet_chunks_fit(l, b->sequences, b->tokens)))
        return SWQ_ERR_LIMIT;
    return SWQ_OK;
}

// Most tokens of one sequence.
int most_tokens(const swq_deltanet_batch *b) { return b->starts ? std::min(b->max_tokens, b->tokens) : b->tokens / b->sequences; }

// From so many tokens of a sequence on, those of a batch go a chunk at a time; from more where workgroups are as many as
// CUs, which token after token keeps busy.  At 32 value heads of 128 (bf16), 1 sequence of 8 (12, 16) takes 28 us (38, 49) token
// after token and 34 us in chunks, 4 of them 28 (38, 47) and 46, 8 of 16 (24) 50 (71) and 67, 32 of them 138 (195) and 187 (196).
constexpr int kChunksFrom = 12, kChunksFromMany = 24;
// Beside a sequence of so many, those of up to kFew go token after token all the same, in launches of their own: with one of
// 600 tokens, 31 of 1 (4) take 116 us (134) so and 223 (232) in chunks, but a single one of 1 69 and 63, of 8 88 and 64.
// Of 8 tokens 8 (31) would take 99 (162) so and 103 (239) in chunks, where they go: the rule does not count them.
constexpr int kFew = 4;

bool misaligned(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

}  // namespace
}  // namespace swq

using namespace swq;

extern "C" size_t swq_deltanet_slot_bytes(const swq_deltanet_layer *l) { return dn_align(swq_deltanet_state_bytes(l)); }

extern "C" size_t swq_deltanet_tokens_workspace_bytes(const swq_deltanet_layer *l, const swq_deltanet_batch *b) {
    if (check_sizes(l, b) != SWQ_OK) return 0;
    return most_tokens(b) >= kChunksFrom && deltanet_chunks_take(l) ? deltanet_chunks_bytes(l, b->sequences, b->tokens) : 256;
}

extern "C" int swq_deltanet_tokens(const swq_deltanet_layer *l, const swq_deltanet_batch *b, const void *qkvz, const void *ba, int dtype,
                                   void *states, size_t states_bytes, void *out, int out_dtype, void *ws, size_t ws_bytes, void *stream) {
    const int st = check_sizes(l, b);
    if (st != SWQ_OK) return st;
    if ((dtype != SWQ_F32 && dtype != SWQ_BF16) || (out_dtype != SWQ_F32 && out_dtype != SWQ_BF16)) return SWQ_ERR_UNSUPPORTED_DTYPE;
    if (b->tokens == 0) return SWQ_OK;
    if (!qkvz || !ba || !states || !out || !b->positions) return SWQ_ERR_INVALID_ARGUMENT;
    const int in = dtype == SWQ_F32 ? 4 : 2;
    if (misaligned(qkvz, in) || misaligned(ba, in) || misaligned(out, out_dtype == SWQ_F32 ? 4 : 2) || misaligned(states, 256) ||
        misaligned(ws, 256))
        return SWQ_ERR_MISALIGNED;
    if (states_bytes / swq_deltanet_slot_bytes(l) < static_cast<size_t>(b->slots)) return SWQ_ERR_WORKSPACE;
    if (!ws || ws_bytes < swq_deltanet_tokens_workspace_bytes(l, b)) return SWQ_ERR_WORKSPACE;
    DnTokens a{};
    a.qkvz = qkvz;
    a.ba = ba;
    a.conv_w = l->conv_weight;
    a.a_log = l->a_log;
    a.dt_bias = l->dt_bias;
    a.norm_w = l->norm_weight;
    a.states = static_cast<uint8_t *>(states);
    a.slot_bytes = static_cast<int64_t>(swq_deltanet_slot_bytes(l));
    a.rec_at = static_cast<int64_t>(deltanet_ring_bytes(l));
    a.out = out;
    a.starts = b->starts;
    a.positions = b->positions;
    a.slot = b->slot;
    a.B = b->sequences;
    a.N = b->tokens;
    a.max_tokens = most_tokens(b);
    a.slots = b->slots;
    a.nk = l->num_key_heads;
    a.nv = l->num_value_heads;
    a.dk = l->key_head_dim;
    a.dv = l->value_head_dim;
    a.K = l->conv_kernel;
    a.layout = l->layout;
    a.rep = a.nv / a.nk;
    a.keyD = a.nk * a.dk;
    a.convD = 2 * a.keyD + a.nv * a.dv;
    a.qkvz_stride = b->qkvz_stride ? b->qkvz_stride : a.convD + a.nv * a.dv;
    a.ba_stride = b->ba_stride ? b->ba_stride : 2 * a.nv;
    a.out_f32 = out_dtype == SWQ_F32;
    a.eps = l->norm_eps;
    hipStream_t s = static_cast<hipStream_t>(stream);
    // chunks are loaded and stored four elements at a time
    const bool four = !misaligned(qkvz, 4 * in) && a.qkvz_stride % 4 == 0 && a.qkvz_stride < 1 << 24 && !misaligned(out, a.out_f32 ? 16 : 8) && !misaligned(a.conv_w, 16);
    const bool chunks = a.max_tokens >= (a.B * a.nv < kCus ? kChunksFrom : kChunksFromMany) && four && deltanet_chunks_take(l);
    // where no sequence can be of another length, nothing is launched for the short ones
    a.least = 1;
    a.most = !chunks ? INT32_MAX : a.B > 1 && a.starts ? kFew : 0;
    if (a.most) {
        if (dtype == SWQ_F32) launch_tokens_dk<float>(a, s);
        else launch_tokens_dk<uint16_t>(a, s);
    }
    if (chunks) {
        a.least = a.most + 1;
        a.most = INT32_MAX;
        launch_deltanet_chunks(a, dtype == SWQ_F32, ws, s);
    }
    return launch_status();
}
