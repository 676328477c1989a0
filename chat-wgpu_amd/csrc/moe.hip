// A mixture-of-experts layer over split Q4_0 experts, the whole of it for rows
// (tokens) of a step: y = [residual +] sum_e p_e Wd_e (silu(Wg_e x) * (Wu_e x)).

#include "cw_internal.hpp"

namespace {

using namespace cwi;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxExperts = 512, kMaxTop = 32;
constexpr int kChunk = 1024;  // rows that go through the layer together

struct MoeArgs {
    cw_moe m;
    const float *x, *residual;
    const int *positions;
    int rows;
    float *y;
    int *experts;     // the caller's, or null
    float *weights;
    int *ids;         // [rows][top_k]; -1: a padding row's
    float *p;         // [rows][top_k]
    float *h;         // [rows][top_k][hidden]
};

// One Q4_0 block times 32 values: d * sum of (q - 8) x
__device__ __forceinline__ float dot_block(const uint8_t *q, uint16_t d, const float *x) {
    float s = 0.0f;
    for (int j = 0; j < 16; ++j) {
        s = __builtin_fmaf((float)((int)(q[j] & 15) - 8), x[j], s);
        s = __builtin_fmaf((float)((int)(q[j] >> 4) - 8), x[j + 16], s);
    }
    return (float)__builtin_bit_cast(_Float16, d) * s;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Row n of a matrix [.][nb] of blocks times x, by a wave
__device__ __forceinline__ float dot_row(const uint16_t *s, const uint8_t *q, size_t n, int nb,
                                         const float *x, int lane) {
    float acc = 0.0f;
    for (int b = lane; b < nb; b += 64)
        acc += dot_block(q + (n * nb + b) * 16, s[n * nb + b], x + 32 * b);
    return wave_sum(acc);
}

__global__ __launch_bounds__(kThreads) void moe_route_kernel(MoeArgs a) {
    __shared__ double score[kMaxExperts];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int E = a.m.n_experts, K = a.m.top_k, dim = a.m.dim;
    if (a.positions && a.positions[r] < 0) {
        if ((int)threadIdx.x < K) a.ids[r * K + threadIdx.x] = -1;
        return;
    }
    const float *x = a.x + (size_t)r * dim;
    for (int e = wave; e < E; e += kWaves) {
        double s = 0.0;
        for (int i = lane; i < dim; i += 64) s += (double)x[i] * (double)a.m.router[(size_t)e * dim + i];
        for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
        if (lane == 0) score[e] = s;
    }
    __syncthreads();
    if (wave) return;
    double v[kMaxExperts / 64];
    double most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kMaxExperts / 64; ++j) {
        const int e = lane + 64 * j;
        v[j] = e < E ? score[e] : 0.0;
        if (e < E) most = fmax(most, v[j]);
    }
    for (int d = 32; d >= 1; d >>= 1) most = fmax(most, __shfl_xor(most, d));
    double all = 0.0, sum = 0.0;
#pragma unroll
    for (int j = 0; j < kMaxExperts / 64; ++j) {
        const int e = lane + 64 * j;
        if (e < E) all += exp(v[j] - most);
        if (!(v[j] >= -INFINITY)) v[j] = -INFINITY;  // NaN is chosen last
    }
    for (int d = 32; d >= 1; d >>= 1) all += __shfl_xor(all, d);
    double mine = 0.0;
    int taken = 0;
    for (int k = 0; k < K; ++k) {
        double best = -INFINITY;
        int at = E;
#pragma unroll
        for (int j = 0; j < kMaxExperts / 64; ++j) {
            const int e = lane + 64 * j;
            if (e < E && !(taken >> j & 1) && (v[j] > best || at == E)) {
                best = v[j];
                at = e;
            }
        }
        for (int d = 32; d >= 1; d >>= 1) {
            const double o = __shfl_xor(best, d);
            const int i = __shfl_xor(at, d);
            if (i < E && (at == E || o > best || (o == best && i < at))) {
                best = o;
                at = i;
            }
        }
        if (lane == (at & 63)) taken |= 1 << (at >> 6);
        const double p = exp(best - most) / all;
        sum += p;
        if (lane == k) {
            mine = p;
            a.ids[r * K + k] = at;
        }
    }
    if (lane < K) a.p[r * K + lane] = (float)(a.m.normalise ? mine / sum : mine);
    if (lane < K && a.experts) a.experts[r * K + lane] = a.ids[r * K + lane];
    if (lane < K && a.weights) a.weights[r * K + lane] = a.p[r * K + lane];
}

__global__ __launch_bounds__(kThreads) void moe_up_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63, pair = blockIdx.y, e = a.ids[pair];
    const int n = blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (e < 0 || n >= a.m.hidden) return;
    const float *x = a.x + (size_t)(pair / a.m.top_k) * a.m.dim;
    const size_t row = (size_t)e * a.m.hidden + n;
    const int nb = a.m.dim / 32;
    const float g = dot_row(a.m.gate_scales, a.m.gate_quants, row, nb, x, lane);
    const float u = dot_row(a.m.up_scales, a.m.up_quants, row, nb, x, lane);
    if (lane == 0) a.h[(size_t)pair * a.m.hidden + n] = g / (1.0f + expf(-g)) * u;
}

__global__ __launch_bounds__(kThreads) void moe_down_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63, r = blockIdx.y, K = a.m.top_k;
    const int n = blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (n >= a.m.dim || a.ids[r * K] < 0) return;
    float y = 0.0f;
    for (int k = 0; k < K; ++k) {
        const size_t row = (size_t)a.ids[r * K + k] * a.m.dim + n;
        const float z = dot_row(a.m.down_scales, a.m.down_quants, row, a.m.hidden / 32,
                                a.h + ((size_t)r * K + k) * a.m.hidden, lane);
        y = __builtin_fmaf(a.p[r * K + k], z, y);
    }
    if (lane == 0) {
        const size_t o = (size_t)r * a.m.dim + n;
        a.y[o] = a.residual ? a.residual[o] + y : y;
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

using namespace cwi;

extern "C" int cw_moe_rows(cw_ctx *ctx, const cw_moe *moe, const float *x, int rows,
                           const int *positions, const float *residual, float *y, int *experts,
                           float *weights) {
    CW_CHECK_ARG(ctx && moe && x && y, "cw_moe_rows: null argument");
    const cw_moe &m = *moe;
    CW_CHECK_ARG(m.router && m.gate_scales && m.gate_quants && m.up_scales && m.up_quants &&
                     m.down_scales && m.down_quants,
                 "cw_moe_rows: null weights");
    CW_CHECK_ARG(rows > 0 && rows <= 65536, "cw_moe_rows: rows=%d outside [1, 65536]", rows);
    for (const int n : {m.dim, m.hidden})
        CW_CHECK_ARG(n > 0 && n % 32 == 0 && n <= 32768,
                     "cw_moe_rows: dim=%d and hidden=%d must be multiples of 32, at most 32768",
                     m.dim, m.hidden);
    CW_CHECK_ARG(m.n_experts > 0 && m.n_experts <= kMaxExperts, "cw_moe_rows: n_experts=%d (at most %d)",
                 m.n_experts, kMaxExperts);
    CW_CHECK_ARG(m.top_k > 0 && m.top_k <= std::min(m.n_experts, kMaxTop),
                 "cw_moe_rows: top_k=%d of %d experts (at most %d)", m.top_k, m.n_experts, kMaxTop);
    CW_CHECK_ARG(m.normalise == 0 || m.normalise == 1, "cw_moe_rows: normalise=%d", m.normalise);
    CW_CHECK_ARG(aligned16(x) && aligned16(m.router) && aligned16(m.gate_quants) &&
                     aligned16(m.up_quants) && aligned16(m.down_quants),
                 "cw_moe_rows: x, router and quants must be 16-byte aligned");
    const size_t n = (size_t)rows * m.dim;
    CW_CHECK_ARG(x + n <= y || y + n <= x, "cw_moe_rows: x and y overlap");
    CW_HIP(hipSetDevice(ctx->device));
    const int chunk = std::min(rows, kChunk), K = m.top_k;
    const size_t pairs = (size_t)chunk * K;
    void *scratch = nullptr;
    CW_TRY(ctx_scratch(ctx, pairs * (8 + 4 * (size_t)m.hidden), &scratch));
    MoeArgs a{};
    a.m = m;
    a.ids = static_cast<int *>(scratch);
    a.p = reinterpret_cast<float *>(a.ids + pairs);
    a.h = a.p + pairs;
    for (int r0 = 0; r0 < rows; r0 += chunk) {
        a.rows = std::min(chunk, rows - r0);
        a.x = x + (size_t)r0 * m.dim;
        a.residual = residual ? residual + (size_t)r0 * m.dim : nullptr;
        a.positions = positions ? positions + r0 : nullptr;
        a.y = y + (size_t)r0 * m.dim;
        a.experts = experts ? experts + (size_t)r0 * K : nullptr;
        a.weights = weights ? weights + (size_t)r0 * K : nullptr;
        CW_TRY(launch(ctx, "moe_route", moe_route_kernel, dim3(a.rows), dim3(kThreads), 0, a));
        CW_TRY(launch(ctx, "moe_up", moe_up_kernel, dim3((m.hidden + kWaves - 1) / kWaves, a.rows * K),
                      dim3(kThreads), 0, a));
        CW_TRY(launch(ctx, "moe_down", moe_down_kernel, dim3((m.dim + kWaves - 1) / kWaves, a.rows),
                      dim3(kThreads), 0, a));
    }
    return CW_OK;
}
