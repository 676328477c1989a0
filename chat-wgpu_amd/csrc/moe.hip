// A mixture-of-experts layer over split Q4_0 experts, the whole of it for the rows
// (tokens) of a step: y = [residual +] sum_e p_e Wd_e (silu(Wg_e x) * (Wu_e x))
// over the top_k experts of a row.
//
// The products run on the matrix cores like q4_gemm.hip's, x as f16 pairs hi + lo
// under a power of two a row (22 bits), W as its nibbles (exact), a block's scale
// after its 32 products.  Few rows meet an expert, so one 16x16x32 MFMA has eight
// rows' hi halves and the same rows' lo halves as its 16 rows; the two sums of a
// row meet at the end.
//
// W goes from memory to registers without LDS: a lane of the 16 x 4 (W row, k
// group) loads whole blocks, block 4 s + g of its row, and four lane groups hand
// each other their words (two swaps of lane halves, two of rows of 16: one
// instruction a block), so that group g has bytes 4 g .. 4 g + 3 of each of the
// four blocks, which is the fragment that nibbles() takes.  The x image lies as the
// fragments are read and stays in the L2s.

#include "prompt_device.hpp"

namespace {

using namespace cwi;

constexpr int kMaxExperts = 512, kMaxTop = 32;
constexpr int kTile = 8;       // rows of one MFMA
constexpr int kFew = kTile;    // rows that need no lists: every expert has one tile at most
constexpr int kChunk = 1024;   // rows that go through the layer together, at most
constexpr size_t kChunkBytes = (size_t)1 << 30;  // of workspace, unless kFew rows need more

struct MoeArgs {
    cw_moe m;
    const float *x, *residual;
    const int *positions;
    int rows;
    float *y;
    int *experts;     // the caller's, or null
    float *weights;
    double *score;    // [rows][n_experts]
    int *ids;         // [rows][top_k]; -1: a padding row's
    float *p;         // [rows][top_k]
    uint8_t *ximg, *himg;    // images of x and of h: [row][block][hi | lo][group] x 16 B
    float *xscale, *hscale;
    float *h;         // [rows][top_k][hidden]
    float *z;         // [rows][top_k][dim]
    // more than kFew rows: (row, choice) pairs by expert, and tiles of them
    int *list;        // [rows * top_k]
    int4 *tiles;      // expert, first of the list, count
    int *n_tiles;
};

__device__ __forceinline__ bool live(const MoeArgs &a, int r) {
    return !a.positions || a.positions[r] >= 0;
}

// ---------------------------------------------------------------- images

// 8 elements of a block under scale sc, as the fragment's 16 bytes of hi and of lo
// (the order in which nibbles() yields the weights; the first four times 16)
__device__ __forceinline__ void split8(float4 ve, float4 vf, float sc, u32x4 *hi, u32x4 *lo) {
    const float v[8] = {ve.x, ve.z, vf.x, vf.z, ve.y, ve.w, vf.y, vf.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float f = (k & 1) ? sc : 16.0f * sc;
        const float t0 = v[2 * k] * f, t1 = v[2 * k + 1] * f;  // exact: powers of two
        const f16x2 h = {(_Float16)t0, (_Float16)t1};
        const f16x2 l = {(_Float16)(t0 - (float)h.x), (_Float16)(t1 - (float)h.y)};
        (*hi)[k] = __builtin_bit_cast(uint32_t, h);
        (*lo)[k] = __builtin_bit_cast(uint32_t, l);
    }
}

__device__ __forceinline__ float max8(float4 a, float4 b) {
    return fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                 fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w))));
}

// The exponent that brings mx into [2^10, 2^11); an infinity gives one whose
// products are NaN.
__device__ __forceinline__ int split_exponent(float mx) {
    return mx > 0.0f ? max(ilogbf(mx) - 10, -126) : 0;
}

// The image of a row of K elements and its scale, by a workgroup of NT threads.
template <int NT>
__device__ void split_row(const float *x, int K, uint8_t *img, float *scale) {
    __shared__ float red[NT / 64];
    const int tid = threadIdx.x;
    auto at = [](int c) { return (c >> 2) * 32 + 4 * (c & 3); };
    float mx = 0.0f;
    for (int c = tid; c < K / 8; c += NT)
        mx = fmaxf(mx, max8(*reinterpret_cast<const float4 *>(x + at(c)),
                            *reinterpret_cast<const float4 *>(x + at(c) + 16)));
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) mx = fmaxf(mx, red[w]);
    const int e = split_exponent(mx);
    const float sc = ldexpf(1.0f, -e);
    if (tid == 0) *scale = ldexpf(1.0f, e);
    for (int c = tid; c < K / 8; c += NT) {
        u32x4 hi, lo;
        split8(*reinterpret_cast<const float4 *>(x + at(c)),
               *reinterpret_cast<const float4 *>(x + at(c) + 16), sc, &hi, &lo);
        uint8_t *o = img + (size_t)(c >> 2) * 128 + (c & 3) * 16;
        *reinterpret_cast<u32x4 *>(o) = hi;
        *reinterpret_cast<u32x4 *>(o + 64) = lo;
    }
}

// ---------------------------------------------------------------- routing

__device__ __forceinline__ bool ahead(double a, int i, double b, int j) {
    return a > b || (a == b && i < j);
}

// Scores are kept without NaN, which would be ahead of nothing and behind nothing:
// as -inf they are chosen last.
__device__ __forceinline__ double ranked(double s) { return s >= -INFINITY ? s : -INFINITY; }

// Scores of at most R rows, a workgroup an expert (f64 products of f32 values are
// exact, their sums are off by 2^-53 of the terms); the workgroups behind the
// experts make the rows' images.
template <int R>
__global__ __launch_bounds__(256) void moe_score_few_kernel(MoeArgs a) {
    __shared__ double red[4][R];
    const int tid = threadIdx.x, dim = a.m.dim, E = a.m.n_experts;
    const int e = blockIdx.x;
    if (e >= E) {
        const int r = e - E;
        split_row<256>(a.x + (size_t)r * dim, dim, a.ximg + (size_t)r * dim * 4, a.xscale + r);
        return;
    }
    double s[R] = {};
    const float *w = a.m.router + (size_t)e * dim;
    for (int i = tid * 4; i < dim; i += 1024) {
        const float4 v = *reinterpret_cast<const float4 *>(w + i);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float4 x = *reinterpret_cast<const float4 *>(a.x + (size_t)min(r, a.rows - 1) * dim + i);
            s[r] = fma((double)x.x, (double)v.x, s[r]);
            s[r] = fma((double)x.y, (double)v.y, s[r]);
            s[r] = fma((double)x.z, (double)v.z, s[r]);
            s[r] = fma((double)x.w, (double)v.w, s[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) s[r] += __shfl_xor(s[r], d);
        if ((tid & 63) == 0) red[tid >> 6][r] = s[r];
    }
    __syncthreads();
    if (tid < a.rows)
        a.score[(size_t)tid * E + e] = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
}

// Scores of 16 rows and 16 experts a workgroup, on the f64 matrix cores, whose 16
// waves split the sum; then the rows' images.
typedef double f64x4 __attribute__((ext_vector_type(4)));
__global__ __launch_bounds__(1024) void moe_score_kernel(MoeArgs a) {
    __shared__ double red[16][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int dim = a.m.dim, E = a.m.n_experts;
    const int et = (E + 15) / 16, rt = (a.rows + 15) / 16;
    if ((int)blockIdx.x >= et * rt) {
        const int r = blockIdx.x - et * rt;
        split_row<1024>(a.x + (size_t)r * dim, dim, a.ximg + (size_t)r * dim * 4, a.xscale + r);
        return;
    }
    const int e0 = blockIdx.x % et * 16, r0 = blockIdx.x / et * 16;
    const int li = lane & 15, lg = lane >> 4;
    const float *x = a.x + (size_t)min(r0 + li, a.rows - 1) * dim + 4 * lg;
    const float *w = a.m.router + (size_t)min(e0 + li, E - 1) * dim + 4 * lg;
    f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (int i = wave * 16; i < dim; i += 256) {
        const float4 u = *reinterpret_cast<const float4 *>(x + i);
        const float4 v = *reinterpret_cast<const float4 *>(w + i);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u.x, (double)v.x, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u.y, (double)v.y, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u.z, (double)v.z, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u.w, (double)v.w, acc, 0, 0, 0);
    }
    // D[4 r + lane / 16][lane % 16] in element r
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][(4 * r + lg) * 16 + li] = acc[r];
    __syncthreads();
    if (tid >= 256) return;
    double s = 0.0;
#pragma unroll
    for (int w16 = 0; w16 < 16; ++w16) s += red[w16][tid];
    const int r = r0 + (tid >> 4), e = e0 + (tid & 15);
    if (r < a.rows && e < E) a.score[(size_t)r * E + e] = s;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_max(double v) {
    const int2 o = __builtin_bit_cast(int2, v);
    const int2 s = {__builtin_amdgcn_update_dpp(o.x, o.x, CTRL, ROWS, 0xf, false),
                    __builtin_amdgcn_update_dpp(o.y, o.y, CTRL, ROWS, 0xf, false)};
    return fmax(v, __builtin_bit_cast(double, s));
}

// The largest of the lanes' values, in every lane.
__device__ __forceinline__ double wave_max(double v) {
    v = dpp_max<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v = dpp_max<0x112, 0xf>(v);
    v = dpp_max<0x114, 0xf>(v);
    v = dpp_max<0x118, 0xf>(v);
    v = dpp_max<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v = dpp_max<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    const int2 o = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, int2{__builtin_amdgcn_readlane(o.x, 63),
                                           __builtin_amdgcn_readlane(o.y, 63)});
}

// The choice of row r by one wave: ids, p and the caller's copies.
__device__ void choose(const MoeArgs &a, int r) {
    constexpr int N = kMaxExperts / 64;
    const int lane = threadIdx.x & 63, E = a.m.n_experts, K = a.m.top_k;
    if (!live(a, r)) {
        if (lane < K) a.ids[r * K + lane] = -1;
        return;
    }
    const int n = (E + 63) / 64;
    double v[N], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int e = lane + 64 * j;
        v[j] = j < n && e < E ? a.score[(size_t)r * E + e] : 0.0;
        if (j < n && e < E) most = fmax(most, v[j]);
    }
    most = wave_max(most);
    double all = 0.0, sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (j >= n) break;
        if (lane + 64 * j < E) all += exp(v[j] - most);
        v[j] = ranked(v[j]);
    }
    for (int d = 32; d >= 1; d >>= 1) all += __shfl_xor(all, d);
    unsigned taken = 0;
    double mine = 0.0;
    int id = 0;
    for (int k = 0; k < K; ++k) {
        double best = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n && lane + 64 * j < E && !(taken >> j & 1)) best = fmax(best, v[j]);
        best = wave_max(best);
        int at = E;
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
            if (j >= n) continue;
            const uint64_t m = __ballot(lane + 64 * j < E && !(taken >> j & 1) && v[j] == best);
            if (m) at = 64 * j + __builtin_ctzll(m);
        }
        if (lane == (at & 63)) taken |= 1u << (at >> 6);
        if (lane == k) {
            mine = exp(best - most);
            id = at;
        }
    }
    for (int k = 0; k < K; ++k) sum += __shfl(mine, k);
    if (lane >= K) return;
    const float p = (float)(mine / (a.m.normalise ? sum : all));
    a.ids[r * K + lane] = id;
    a.p[r * K + lane] = p;
    if (a.experts) a.experts[r * K + lane] = id;
    if (a.weights) a.weights[r * K + lane] = p;
}

// The pairs (row * top_k + choice) by expert and their tiles of `tile` pairs, by
// one workgroup.  Which row of its tile a pair gets hangs on the order of LDS
// atomics; its result does not.
__device__ void sort_pairs(const MoeArgs &a, int tile) {
    __shared__ int count[kMaxExperts], first[kMaxExperts];
    const int tid = threadIdx.x, E = a.m.n_experts, P = a.rows * a.m.top_k;
    for (int e = tid; e < E; e += blockDim.x) count[e] = 0;
    __syncthreads();
    for (int i = tid; i < P; i += blockDim.x)
        if (a.ids[i] >= 0) atomicAdd(&count[a.ids[i]], 1);
    __syncthreads();
    if (tid < 64) {
        constexpr int N = kMaxExperts / 64;
        int pairs = 0, tiles = 0;
        for (int j = 0; j < N; ++j) {
            const int e = tid * N + j, c = e < E ? count[e] : 0;
            pairs += c;
            tiles += (c + tile - 1) / tile;
        }
        int p = pairs, t = tiles;
        for (int d = 1; d < 64; d <<= 1) {
            const int op = __shfl_up(p, d), ot = __shfl_up(t, d);
            if (tid >= d) {
                p += op;
                t += ot;
            }
        }
        if (tid == 63) a.n_tiles[0] = t;
        p -= pairs;
        t -= tiles;
        for (int j = 0; j < N; ++j) {
            const int e = tid * N + j, c = e < E ? count[e] : 0;
            if (e < E) first[e] = p;
            for (int i = 0; i < c; i += tile) a.tiles[t++] = make_int4(e, p + i, min(tile, c - i), 0);
            p += c;
        }
    }
    __syncthreads();
    for (int i = tid; i < P; i += blockDim.x)
        if (a.ids[i] >= 0) a.list[atomicAdd(&first[a.ids[i]], 1)] = i;
}

__global__ __launch_bounds__(1024) void moe_choose_kernel(MoeArgs a, int tile, int sort) {
    for (int r = blockIdx.x * 16 + (threadIdx.x >> 6); r < a.rows; r += gridDim.x * 16) choose(a, r);
    if (!sort) return;
    __syncthreads();
    sort_pairs(a, tile);
}

__global__ __launch_bounds__(1024) void moe_sort_kernel(MoeArgs a, int tile) { sort_pairs(a, tile); }

// ---------------------------------------------------------------- products

// What a wave holds of one step of four blocks: CT tiles of 16 W rows, MT tiles of
// eight x rows.
template <int MT, int CT>
struct Step {
    u32x4 q[CT], x[MT][4];
    uint2 d[CT];
};

// A wave's operands: uniform bases and the lane's offsets into them.
template <int MT, int CT>
struct Operands {
    const uint8_t *q[CT];   // the tile's first W row
    const uint16_t *d[CT];
    const uint8_t *x;
    uint32_t row;           // the lane's W row of a tile
    size_t xo[MT];
    int nb, lg;
};

// WHOLE: rows are whole steps, and their scales 8-byte aligned.  Else blocks past
// the row's end re-read its last under a scale of 0.
template <int MT, int CT, bool WHOLE>
__device__ __forceinline__ void load_step(const Operands<MT, CT> &o, int s, Step<MT, CT> &f) {
    const int b = WHOLE ? 4 * s + o.lg : min(4 * s + o.lg, o.nb - 1);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        f.q[c] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4 *>(o.q[c] + (o.row * o.nb + b) * 16u));
        const uint16_t *d = o.d[c] + o.row * o.nb + 4 * s;
        if constexpr (WHOLE) {
            f.d[c] = *reinterpret_cast<const uint2 *>(d);
        } else {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = 4 * s + i < o.nb ? d[i] : 0;
            f.d[c] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f.x[m][i] = *reinterpret_cast<const u32x4 *>(
                o.x + o.xo[m] + (size_t)(WHOLE ? 4 * s + i : min(4 * s + i, o.nb - 1)) * 128);
}

// Word w of the lane groups' blocks -> block i of word `group`.
__device__ __forceinline__ u32x4 exchange(u32x4 q) {
    const auto a = __builtin_amdgcn_permlane16_swap(q[0], q[1], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(q[2], q[3], false, false);
    const auto c = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    return u32x4{c[0], d[0], c[1], d[1]};
}

template <int MT, int CT>
__device__ __forceinline__ void multiply(const Step<MT, CT> &f, f32x4 (&acc)[MT][CT]) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const u32x4 w = exchange(f.q[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x8 b = nibbles(w[i]);
            const f16x2 d2 = __builtin_bit_cast(f16x2, i < 2 ? f.d[c].x : f.d[c].y);
            const float d = (float)d2[i & 1];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const f32x4 t = mfma16(__builtin_bit_cast(f16x8, f.x[m][i]), b, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][c][r] = __builtin_fmaf(d, t[r], acc[m][c][r]);
            }
        }
    }
}

// acc += the products of steps s, s + by, ... of the row's n: two steps' loads in
// flight.
template <int MT, int CT, bool WHOLE>
__device__ __forceinline__ void products(const Operands<MT, CT> &o, int s, int by, int n,
                                         f32x4 (&acc)[MT][CT]) {
    if (s >= n) return;
    Step<MT, CT> f[2];
    load_step<MT, CT, WHOLE>(o, s, f[0]);
    for (;; s += 2 * by) {
        load_step<MT, CT, WHOLE>(o, min(s + by, n - 1), f[1]);
        multiply<MT, CT>(f[0], acc);
        if (s + by >= n) break;
        load_step<MT, CT, WHOLE>(o, min(s + 2 * by, n - 1), f[0]);
        multiply<MT, CT>(f[1], acc);
        if (s + 2 * by >= n) break;
    }
}

// ---------------------------------------------------------------- few rows
//
// Three launches and no lists.  A workgroup of the first product has one choice
// (row, rank) and 16 columns of h; it finds the expert from the scores, and whether
// another row chose it too: the first such row's workgroups compute all of them.

constexpr int kFewThreads = 512, kFewWaves = kFewThreads / 64;

template <bool WHOLE>
__global__ __launch_bounds__(kFewThreads) void moe_up_few_kernel(MoeArgs a) {
    extern __shared__ double score[];  // [rows][n_experts]
    __shared__ f32x4 red[kFewWaves][2][64];
    __shared__ int chosen, rank_of[kFew];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int E = a.m.n_experts, K = a.m.top_k, hidden = a.m.hidden;
    if ((int)blockIdx.x < a.rows) {
        if (wave == 0) choose(a, blockIdx.x);
        return;
    }
    const int cols = hidden / 16, slot = (blockIdx.x - a.rows) / cols;
    const int col = (blockIdx.x - a.rows) % cols * 16;
    const int row = slot / K, k = slot % K;
    if (!live(a, row)) return;
    for (int i = tid; i < a.rows * E; i += kFewThreads) score[i] = ranked(a.score[i]);
    __syncthreads();
    // the expert of rank k: `per` lanes count those ahead of one
    int per = 1;
    while (per < 64 && 2 * per * E <= kFewThreads) per *= 2;
    {
        const double *s = score + row * E;
        const int e = tid / per;
        const double mine = e < E ? s[e] : 0.0;
        int n = 0;
        for (int i = tid % per; i < E; i += per) n += ahead(s[i], i, mine, e);
        for (int d = 1; d < per; d <<= 1) n += __shfl_xor(n, d);
        if (e < E && n == k) chosen = e;
    }
    __syncthreads();
    const int e = chosen;
    if (wave < kFew) {
        int n = K;
        if (wave < a.rows && live(a, wave)) {
            const double *s = score + wave * E, mine = s[e];
            n = 0;
            for (int i = 0; i < E; i += 64)
                n += __popcll(__ballot(i + lane < E && ahead(s[min(i + lane, E - 1)], i + lane, mine, e)));
        }
        if (lane == 0) rank_of[wave] = n;
    }
    __syncthreads();
    for (int r = 0; r < row; ++r)
        if (rank_of[r] < K) return;
    const int li = lane & 15, lg = lane >> 4, nb = a.m.dim / 32;
    const size_t w0 = ((size_t)e * hidden + col) * nb;
    Operands<1, 2> o;
    o.q[0] = a.m.gate_quants + w0 * 16;
    o.q[1] = a.m.up_quants + w0 * 16;
    o.d[0] = a.m.gate_scales + w0;
    o.d[1] = a.m.up_scales + w0;
    o.x = a.ximg;
    o.row = li;
    const int xr = rank_of[li & 7] < K ? li & 7 : row;
    o.xo[0] = (size_t)xr * nb * 128 + (li >> 3) * 64 + lg * 16;
    o.nb = nb;
    o.lg = lg;
    f32x4 acc[1][2] = {};
    products<1, 2, WHOLE>(o, wave, kFewWaves, (nb + 3) / 4, acc);
    red[wave][0][lane] = acc[0][0];
    red[wave][1][lane] = acc[0][1];
    __syncthreads();
    // row m of x, column n: element m % 4 of lanes 16 (m / 4) + n (hi) and 32 more (lo)
    const int m = tid >> 4, n = tid & 15;
    if (m >= a.rows || rank_of[m] >= K) return;
    const int from = (m >> 2) * 16 + n;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
        g += red[w][0][from][m & 3] + red[w][0][from + 32][m & 3];
        u += red[w][1][from][m & 3] + red[w][1][from + 32][m & 3];
    }
    const float sc = kUnscale * a.xscale[m];
    a.h[((size_t)m * K + rank_of[m]) * hidden + col + n] = silu_mul(g * sc, u * sc);
}

// A workgroup has 16 columns of a row's y; its waves share the experts out, or
// parts of them where there are fewer.  A wave splits its stretch of h itself, 32
// blocks at a time under their own power of two, while their W is on its way.
template <bool WHOLE>
__global__ __launch_bounds__(kFewThreads) void moe_down_few_kernel(MoeArgs a) {
    constexpr int S = 8;  // steps at a time
    __shared__ u32x4 img[kFewWaves][S * 4 * 8];
    __shared__ float red[kMaxTop][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int K = a.m.top_k, hidden = a.m.hidden, dim = a.m.dim, nb = hidden / 32;
    const int r = blockIdx.y, col = blockIdx.x * 16;
    if (!live(a, r)) return;
    const int parts = K < kFewWaves ? kFewWaves / K : 1, steps = (nb + 3) / 4;
    const int per = (steps + parts - 1) / parts;
    for (int u = wave; u < K * parts; u += kFewWaves) {
        const int j = u / parts, s0 = u % parts * per, s1 = min(steps, s0 + per);
        const int pair = r * K + j, e = a.ids[pair];
        const float *h = a.h + (size_t)pair * hidden;
        const size_t w0 = ((size_t)e * dim + col) * nb;
        float total = 0.0f;
        for (int s = s0; s < s1; s += S) {
            u32x4 q[S];
            uint2 d[S];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const int st = min(s + i, s1 - 1), b = min(4 * st + lg, nb - 1);
                q[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(
                    a.m.down_quants + (w0 + (uint32_t)(li * nb + b)) * 16));
                const uint16_t *p = a.m.down_scales + w0 + (uint32_t)(li * nb + 4 * st);
                if constexpr (WHOLE) {
                    d[i] = *reinterpret_cast<const uint2 *>(p);
                } else {
                    uint32_t v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) v[t] = 4 * st + t < nb ? p[t] : 0;
                    d[i] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
                }
            }
            float4 ve[2], vf[2];
            float mx = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int c = lane + 64 * t, b = min(4 * s + (c >> 2), nb - 1);
                const float *x = h + 32 * b + 4 * (c & 3);
                ve[t] = *reinterpret_cast<const float4 *>(x);
                vf[t] = *reinterpret_cast<const float4 *>(x + 16);
                mx = fmaxf(mx, max8(ve[t], vf[t]));
            }
#pragma unroll
            for (int dd = 32; dd >= 1; dd >>= 1) mx = fmaxf(mx, __shfl_xor(mx, dd));
            const int ex = split_exponent(mx);
            const float sc = ldexpf(1.0f, -ex);
            __builtin_amdgcn_wave_barrier();  // the reads of the last stretch
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int c = lane + 64 * t;
                u32x4 hi, lo;
                split8(ve[t], vf[t], sc, &hi, &lo);
                img[wave][(c >> 2) * 8 + (c & 3)] = hi;
                img[wave][(c >> 2) * 8 + 4 + (c & 3)] = lo;
            }
            __builtin_amdgcn_wave_barrier();
            float acc = 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                if (s + i < s1) {
                    const u32x4 w = exchange(q[i]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        // rows 0 .. 7 of the fragment are h's hi, 8 .. 15 its lo
                        const u32x4 x = img[wave][(4 * i + t) * 8 + (li >> 3) * 4 + lg];
                        const f32x4 v = mfma16(__builtin_bit_cast(f16x8, x), nibbles(w[t]),
                                               f32x4{0.f, 0.f, 0.f, 0.f});
                        const f16x2 d2 = __builtin_bit_cast(f16x2, t < 2 ? d[i].x : d[i].y);
                        acc = __builtin_fmaf((float)d2[t & 1], v[0], acc);
                    }
                }
            }
            total = __builtin_fmaf(kUnscale * ldexpf(1.0f, ex), acc, total);
        }
        total += __shfl_xor(total, 32);
        if (lane < 16) red[u][li] = a.p[pair] * total;
    }
    __syncthreads();
    if (tid >= 16) return;
    float y = 0.0f;
    for (int u = 0; u < K * parts; ++u) y += red[u][tid];
    const size_t at = (size_t)r * dim + col + tid;
    a.y[at] = a.residual ? a.residual[at] + y : y;
}

// ---------------------------------------------------------------- more rows

constexpr int kTileThreads = 256, kTileWaves = 4;

// The lane's x rows of a tile: pairs of the list, the last one again past its end.
__device__ __forceinline__ int pair_of(const MoeArgs &a, int4 tile, int i) {
    return a.list[tile.y + min(i, tile.z - 1)];
}

// 32 columns of h of a tile of pairs; the waves split dim.
template <int MT, bool WHOLE>
__global__ __launch_bounds__(kTileThreads) void moe_up_tile_kernel(MoeArgs a) {
    __shared__ f32x4 red[kTileWaves][4][64];
    if ((int)blockIdx.y >= a.n_tiles[0]) return;
    const int4 tile = a.tiles[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int hidden = a.m.hidden, nb = a.m.dim / 32, col = blockIdx.x * 32;
    const int e = __builtin_amdgcn_readfirstlane(tile.x);
    Operands<MT, 4> o;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const size_t w0 = ((size_t)e * hidden + col + (c & 1) * 16) * nb;
        o.q[c] = (c < 2 ? a.m.gate_quants : a.m.up_quants) + w0 * 16;
        o.d[c] = (c < 2 ? a.m.gate_scales : a.m.up_scales) + w0;
    }
    o.x = a.ximg;
    o.row = li;
    o.nb = nb;
    o.lg = lg;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = pair_of(a, tile, 8 * m + (li & 7)) / a.m.top_k;
        o.xo[m] = (size_t)r * nb * 128 + (li >> 3) * 64 + lg * 16;
    }
    f32x4 acc[MT][4] = {};
    products<MT, 4, WHOLE>(o, wave, kTileWaves, (nb + 3) / 4, acc);
    const int i = tid >> 5, n = tid & 31, from = (i >> 2) * 16 + (n & 15);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m) __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) red[wave][c][lane] = acc[m][c];
        __syncthreads();
        if (8 * m + i < tile.z) {
            float g = 0.0f, u = 0.0f;
#pragma unroll
            for (int w = 0; w < kTileWaves; ++w) {
                g += red[w][n >> 4][from][i & 3] + red[w][n >> 4][from + 32][i & 3];
                u += red[w][2 + (n >> 4)][from][i & 3] + red[w][2 + (n >> 4)][from + 32][i & 3];
            }
            const int pair = pair_of(a, tile, 8 * m + i);
            const float sc = kUnscale * a.xscale[pair / a.m.top_k];
            a.h[(size_t)pair * hidden + col + n] = silu_mul(g * sc, u * sc);
        }
    }
}

__global__ __launch_bounds__(256) void moe_split_kernel(MoeArgs a) {
    const size_t pair = blockIdx.x;
    if (a.ids[pair] < 0) return;
    split_row<256>(a.h + pair * a.m.hidden, a.m.hidden, a.himg + pair * a.m.hidden * 4,
                   a.hscale + pair);
}

// Columns of z of a tile of pairs, 64 a wave; ks waves split hidden.
template <int MT, bool WHOLE>
__global__ __launch_bounds__(kTileThreads) void moe_down_tile_kernel(MoeArgs a, int ks) {
    __shared__ f32x4 red[kTileWaves][4][64];
    if ((int)blockIdx.y >= a.n_tiles[0]) return;
    const int4 tile = a.tiles[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int dim = a.m.dim, nb = a.m.hidden / 32;
    const int cols = 64 * (kTileWaves / ks), col0 = blockIdx.x * cols;
    const int e = __builtin_amdgcn_readfirstlane(tile.x);
    Operands<MT, 4> o;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int col = min(col0 + wave / ks * 64 + 16 * c, dim - 16);
        const size_t w0 = ((size_t)e * dim + col) * nb;
        o.q[c] = a.m.down_quants + w0 * 16;
        o.d[c] = a.m.down_scales + w0;
    }
    o.x = a.himg;
    o.row = li;
    o.nb = nb;
    o.lg = lg;
#pragma unroll
    for (int m = 0; m < MT; ++m)
        o.xo[m] = (size_t)pair_of(a, tile, 8 * m + (li & 7)) * nb * 128 + (li >> 3) * 64 + lg * 16;
    f32x4 acc[MT][4] = {};
    products<MT, 4, WHOLE>(o, wave % ks, ks, (nb + 3) / 4, acc);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m) __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) red[wave][c][lane] = acc[m][c];
        __syncthreads();
        for (int t = tid; t < 8 * cols; t += kTileThreads) {
            const int i = t / cols, n = t % cols, from = (i >> 2) * 16 + (n & 15);
            if (8 * m + i >= tile.z || col0 + n >= dim) continue;
            float v = 0.0f;
            for (int w = 0; w < ks; ++w) {
                const f32x4 *p = red[n / 64 * ks + w][n / 16 % 4];
                v += p[from][i & 3] + p[from + 32][i & 3];
            }
            const int pair = pair_of(a, tile, 8 * m + i);
            a.z[(size_t)pair * dim + col0 + n] = a.p[pair] * (kUnscale * a.hscale[pair] * v);
        }
    }
}

// y = [residual +] the sum of a row's experts in order of their rank
__global__ __launch_bounds__(256) void moe_sum_kernel(MoeArgs a) {
    const int r = blockIdx.y, K = a.m.top_k, dim = a.m.dim;
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= dim || !live(a, r)) return;
    const float *z = a.z + (size_t)r * K * dim + n;
    const float4 v = sum_parts(K, [&](int k) {
        return *reinterpret_cast<const float4 *>(z + (size_t)k * dim);
    });
    const float s[4] = {v.x, v.y, v.z, v.w};
    const size_t at = (size_t)r * dim + n;
#pragma unroll
    for (int j = 0; j < 4; ++j) a.y[at + j] = a.residual ? a.residual[at + j] + s[j] : s[j];
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

bool whole_steps(int in_f, const uint16_t *s) {
    return in_f % 128 == 0 && ((uintptr_t)s & 7) == 0;
}

// Places of the workspace, each 256-byte aligned; with base null their size.
size_t lay_out(const cw_moe &m, int rows, char *base, MoeArgs *a) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *p = base + at;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t K = m.top_k, pairs = (size_t)rows * K;
    const bool lists = rows > kFew;
    a->score = reinterpret_cast<double *>(take((size_t)rows * m.n_experts * 8));
    a->ids = reinterpret_cast<int *>(take(pairs * 4));
    a->p = reinterpret_cast<float *>(take(pairs * 4));
    a->ximg = reinterpret_cast<uint8_t *>(take((size_t)rows * m.dim * 4));
    a->xscale = reinterpret_cast<float *>(take((size_t)rows * 4));
    a->h = reinterpret_cast<float *>(take(pairs * m.hidden * 4));
    if (lists) {
        a->himg = reinterpret_cast<uint8_t *>(take(pairs * m.hidden * 4));
        a->hscale = reinterpret_cast<float *>(take(pairs * 4));
        a->z = reinterpret_cast<float *>(take(pairs * m.dim * 4));
        a->list = reinterpret_cast<int *>(take(pairs * 4));
        a->tiles = reinterpret_cast<int4 *>(take((pairs / kTile + m.n_experts) * 16));
        a->n_tiles = reinterpret_cast<int *>(take(4));
    }
    return at;
}

int run_few(cw_ctx *ctx, const MoeArgs &a) {
    const int E = a.m.n_experts, K = a.m.top_k;
    auto score = a.rows == 1 ? moe_score_few_kernel<1> : a.rows <= 4 ? moe_score_few_kernel<4>
                                                                     : moe_score_few_kernel<kFew>;
    CW_TRY(launch(ctx, "moe_score", score, dim3(E + a.rows), dim3(256), 0, a));
    const bool gw = whole_steps(a.m.dim, a.m.gate_scales) && whole_steps(a.m.dim, a.m.up_scales);
    CW_TRY(launch(ctx, "moe_up", gw ? moe_up_few_kernel<true> : moe_up_few_kernel<false>,
                  dim3(a.rows + a.rows * K * (a.m.hidden / 16)), dim3(kFewThreads), a.rows * E * 8, a));
    const bool dw = whole_steps(a.m.hidden, a.m.down_scales);
    return launch(ctx, "moe_down", dw ? moe_down_few_kernel<true> : moe_down_few_kernel<false>,
                  dim3(a.m.dim / 16, a.rows), dim3(kFewThreads), 0, a);
}

int run_tiles(cw_ctx *ctx, const MoeArgs &a) {
    const int E = a.m.n_experts, K = a.m.top_k, pairs = a.rows * K;
    const int mean = (pairs + E - 1) / E;
    const int mt = mean <= 4 ? 1 : mean <= 12 ? 2 : 4, tile = kTile * mt;
    const int score = (E + 15) / 16 * ((a.rows + 15) / 16);
    CW_TRY(launch(ctx, "moe_score", moe_score_kernel, dim3(score + a.rows), dim3(1024), 0, a));
    const bool one = a.rows <= 64;
    CW_TRY(launch(ctx, "moe_choose", moe_choose_kernel, dim3(one ? 1 : (a.rows + 15) / 16), dim3(1024),
                  0, a, tile, one ? 1 : 0));
    if (!one) CW_TRY(launch(ctx, "moe_sort", moe_sort_kernel, dim3(1), dim3(1024), 0, a, tile));
    const int most = std::min(pairs, E + pairs / tile);
    const bool gw = whole_steps(a.m.dim, a.m.gate_scales) && whole_steps(a.m.dim, a.m.up_scales);
    auto up = mt == 1 ? (gw ? moe_up_tile_kernel<1, true> : moe_up_tile_kernel<1, false>)
              : mt == 2 ? (gw ? moe_up_tile_kernel<2, true> : moe_up_tile_kernel<2, false>)
                        : (gw ? moe_up_tile_kernel<4, true> : moe_up_tile_kernel<4, false>);
    CW_TRY(launch(ctx, "moe_up", up, dim3(a.m.hidden / 32, most), dim3(kTileThreads), 0, a));
    CW_TRY(launch(ctx, "moe_split", moe_split_kernel, dim3(pairs), dim3(256), 0, a));
    const bool dw = whole_steps(a.m.hidden, a.m.down_scales);
    auto down = mt == 1 ? (dw ? moe_down_tile_kernel<1, true> : moe_down_tile_kernel<1, false>)
                : mt == 2 ? (dw ? moe_down_tile_kernel<2, true> : moe_down_tile_kernel<2, false>)
                          : (dw ? moe_down_tile_kernel<4, true> : moe_down_tile_kernel<4, false>);
    const int steps = (a.m.hidden / 32 + 3) / 4, ks = steps >= 16 ? 4 : steps >= 4 ? 2 : 1;
    const int cols = 64 * (kTileWaves / ks);
    CW_TRY(launch(ctx, "moe_down", down, dim3((a.m.dim + cols - 1) / cols, most), dim3(kTileThreads),
                  0, a, ks));
    return launch(ctx, "moe_sum", moe_sum_kernel, dim3((a.m.dim + 1023) / 1024, a.rows), dim3(256), 0, a);
}

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
    MoeArgs a{};
    int chunk = std::min(rows, kChunk);
    while (chunk > kFew && lay_out(m, chunk, nullptr, &a) > kChunkBytes) chunk = std::max(kFew, chunk / 2);
    void *scratch = nullptr;
    CW_TRY(ctx_scratch(ctx, lay_out(m, chunk, nullptr, &a), &scratch));
    for (int r0 = 0; r0 < rows; r0 += chunk) {
        a.m = m;
        a.rows = std::min(chunk, rows - r0);
        (void)lay_out(m, a.rows, static_cast<char *>(scratch), &a);
        a.x = x + (size_t)r0 * m.dim;
        a.residual = residual ? residual + (size_t)r0 * m.dim : nullptr;
        a.positions = positions ? positions + r0 : nullptr;
        a.y = y + (size_t)r0 * m.dim;
        a.experts = experts ? experts + (size_t)r0 * m.top_k : nullptr;
        a.weights = weights ? weights + (size_t)r0 * m.top_k : nullptr;
        CW_TRY(a.rows <= kFew ? run_few(ctx, a) : run_tiles(ctx, a));
    }
    return CW_OK;
}
