// Attention of many rows over a paged cache of several requests: decode steps,
// pieces of prompts and trees of drafted tokens in one call.
//
// o_h = sum_p softmax_p(q_h . k_p / sqrt(hd)) v_p over the positions that a row
// sees: its request's cached ones, and of the request's own rows (nodes) those
// its mask shows.

#include <cmath>

#include "paged_device.hpp"

namespace {

using namespace cwi;

constexpr int kThreads = 256;

struct TreeArgs {
    const float *q;
    size_t q_stride;
    float *out;
    size_t out_stride;
    const void *kc, *vc;
    PageMap map;
    const int *first_row, *cached;
    int n_seq, rows;
    const uint32_t *mask;
    int mask_words;
    int n_heads, n_kv;
    float scale;  // log2(e) / sqrt(hd)
};

// Whether node i of a request sees its node j (row: the node's row of the mask)
__device__ __forceinline__ bool sees(const TreeArgs &a, int row, int i, int j) {
    if (!a.mask) return j <= i;
    return (j >> 5) < a.mask_words &&
           (a.mask[(size_t)row * a.mask_words + (j >> 5)] >> (j & 31) & 1);
}

// One (row, head) a workgroup: wave w takes positions w, w + 4, ..., a lane
// HD / 64 elements of each (or one, of HD lanes); the waves' (max, sum, o) meet
// in LDS.
template <typename KVT, int HD>
__global__ __launch_bounds__(kThreads) void tree_row_kernel(TreeArgs a) {
    constexpr int E = HD > 64 ? HD / 64 : 1, W = kThreads / 64;
    __shared__ float so[W][HD], sm[W], sl[W];
    const int r = blockIdx.x, h = blockIdx.y, g = h / (a.n_heads / a.n_kv);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the request whose rows hold r
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (a.first_row[m] <= r) lo = m;
        else hi = m;
    }
    const SeqRows s = seq_rows(a.first_row, a.cached, a.rows, lo);
    const int i = r - s.r0;
    if (i < 0 || i >= s.n) return;
    const int e0 = lane * E;
    const bool on = e0 < HD;
    float q[E], o[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e)
        q[e] = on ? a.q[(size_t)r * a.q_stride + (size_t)h * HD + e0 + e] : 0.0f;
    float m = -INFINITY, l = 0.0f;
    bool lost = false;  // a position without a block
    const KVT *kc = static_cast<const KVT *>(a.kc), *vc = static_cast<const KVT *>(a.vc);
    for (int p = wave; p < s.cached + s.n; p += W) {
        const int slot = slot_of(a.map, lo, p);
        lost |= slot < 0;
        if (slot < 0 || (p >= s.cached && !sees(a, r, i, p - s.cached))) continue;
        const size_t at = ((size_t)slot * a.n_kv + g) * HD + e0;
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (on) d = __builtin_fmaf(q[e], (float)kc[at + e], d);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) d += __shfl_xor(d, off);
        d *= a.scale;
        const float mn = fmaxf(m, d), ref = mn == -INFINITY ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(d - ref);
        m = mn;
        l = __builtin_fmaf(l, f, w);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (on) o[e] = __builtin_fmaf(o[e], f, w * (float)vc[at + e]);
    }
    if (on)
#pragma unroll
        for (int e = 0; e < E; ++e) so[wave][e0 + e] = o[e];
    if (lane == 0) sm[wave] = m, sl[wave] = lost ? NAN : l;
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w]);
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < W; ++w) L += sl[w] * __builtin_amdgcn_exp2f(sm[w] - ref);
    for (int e = threadIdx.x; e < HD; e += kThreads) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += so[w][e] * __builtin_amdgcn_exp2f(sm[w] - ref);
        a.out[(size_t)r * a.out_stride + (size_t)h * HD + e] = L == 0.0f ? 0.0f : v / L;
    }
}

template <typename KVT>
int launch_rows(cw_ctx *ctx, const TreeArgs &a, int hd) {
    auto fn = hd == 16 ? tree_row_kernel<KVT, 16> : hd == 32 ? tree_row_kernel<KVT, 32>
            : hd == 64 ? tree_row_kernel<KVT, 64> : hd == 128 ? tree_row_kernel<KVT, 128>
                       : tree_row_kernel<KVT, 256>;
    return launch(ctx, "attention_tree", fn, dim3(a.rows, a.n_heads), dim3(kThreads), 0, a);
}

}  // namespace

extern "C" int cw_attention_tree(cw_ctx *ctx, const cw_kv_pages *kv, const cw_batch *b,
                                 const float *q, size_t q_stride, int n_heads, float *out,
                                 size_t out_stride) {
    CW_CHECK_ARG(ctx && kv && b && q && out, "cw_attention_tree: null argument");
    PageMap map;
    CW_TRY(check_pages("cw_attention_tree", kv, b, true, &map));
    CW_CHECK_ARG(b->first_row, "cw_attention_tree: first_row is needed");
    CW_CHECK_ARG(b->rows > 0 && b->rows <= kMaxRows, "cw_attention_tree: rows=%d (1 .. 2^23)",
                 b->rows);
    CW_CHECK_ARG(!b->mask || b->mask_words > 0, "cw_attention_tree: mask_words=%d", b->mask_words);
    CW_CHECK_ARG(n_heads > 0 && n_heads <= 4096 && n_heads % kv->n_kv_heads == 0,
                 "cw_attention_tree: n_heads=%d must be a multiple of n_kv_heads=%d (at most 4096)",
                 n_heads, kv->n_kv_heads);
    const size_t width = (size_t)n_heads * kv->head_dim;
    CW_CHECK_ARG(q_stride >= width && out_stride >= width && q_stride < (1u << 31) &&
                     out_stride < (1u << 31) && q_stride % 4 == 0 && out_stride % 4 == 0,
                 "cw_attention_tree: strides %zu and %zu of rows of %zu floats (multiples of 4)",
                 q_stride, out_stride, width);
    CW_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                 "cw_attention_tree: q and out must be 16-byte aligned");
    CW_CHECK_ARG(rows_apart(b->rows, q, q_stride, width, out, out_stride, width),
                 "cw_attention_tree: rows of q and out overlap");
    CW_HIP(hipSetDevice(ctx->device));
    TreeArgs a{q, q_stride, out, out_stride, kv->k, kv->v, map, b->first_row, b->cached, b->n_seq,
               b->rows, b->mask, b->mask_words, n_heads, kv->n_kv_heads,
               (float)(1.4426950408889634 / std::sqrt((double)kv->head_dim))};
    return kv->kv_dtype == CW_F16 ? launch_rows<_Float16>(ctx, a, kv->head_dim)
                                  : launch_rows<float>(ctx, a, kv->head_dim);
}
