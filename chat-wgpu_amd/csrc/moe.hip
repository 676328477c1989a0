// A mixture-of-experts layer over split Q4_0 experts, the whole of it for the rows
// (tokens) of a step: y = [residual +] sum_e p_e Wd_e (silu(Wg_e x) * (Wu_e x))
// over the top_k experts of a row.
//
// The choice hangs on the scores, so they are sums in f64 (products of f32 values are
// exact there), and their ranks are counted, not sorted.  Rows that chose an expert
// form its list; tiles of 8 or 16 of a list go through its matrices.
//
// The products run on the matrix cores like q4_gemm.hip's, x as f16 pairs hi + lo
// under a power of two a row (22 bits), W as its nibbles (exact), a block's scale
// after its 32 products.  Few rows meet an expert: eight rows' hi halves and the same
// rows' lo halves are the 16 rows of one 16x16x32 MFMA, and the two sums of a row
// meet at the end; 16 rows take two of them one after the other.  x stays in
// registers; W, which is read once, goes through a ring in LDS of each wave's own.
//
// What bounds it: the experts' weights from memory (128 of 2,048 x 768 are 340 MB with
// their scales), which reading alone brings in at 6.3 TB/s.  Microseconds of the launches,
// 8 of these 128 experts a row:
//   1 row     scores 2.3, choice and up 9.0, down 8.2: launches' beginnings and ends
//   48 rows   scores 5, choice 6, up 48 (44 at best), split 5, down 28, sum 5: up and
//             down read at 4.3 TB/s (loads without products 40 and 23.5), the vector
//             units, which decode and scale, 0.6 to 0.7 busy
//   500 rows  scores 13, choice 7, up 129 to 138, split 8, down 94 to 101, sum 9: tiles of
//             one expert decode its weights again; vector units 0.65, matrix cores 0.24 busy
// More than kChunk rows go through in pieces that each read and decode every expert: 4,000
// are four of 390 us.

#include "prompt_device.hpp"

namespace {

using namespace cwi;

constexpr int kMaxExperts = 512, kMaxTop = 32;
constexpr int kTile = 8;       // rows of one MFMA
// Counts lie a few words apart: atomics on one line follow one another (the choice of 500
// rows 11 us side by side, 8.6, 7.0 and 6.6 with 2, 4 and 8; tiles read more lines).
constexpr int kApart = 4;
constexpr int kMaxSplits = 8;  // workgroups that share a score's sum
constexpr int kChunk = 1024;   // rows that go through the layer together, at most
constexpr size_t kChunkBytes = (size_t)1 << 30;  // of workspace, unless kTile rows need more

struct MoeArgs {
    cw_moe m;
    const float *x, *residual;
    const int *positions;
    int rows;
    float *y;
    int *experts;     // the caller's, or null
    float *weights;
    double *score;    // [splits][rows][n_experts]
    int splits;
    int *ids;         // [rows][top_k]; -1: a padding row's
    float *p;         // [rows][top_k]
    uint8_t *ximg, *himg;    // images of x and of h: [row][block][group][hi | lo] x 16 B
    float *xscale, *hscale;
    float *h;         // [rows][top_k][hidden]
    float *z;         // [rows][top_k][dim]
    int *count;       // [n_experts], kApart words apart: pairs (row, choice) of each, and
    int *list;        // [n_experts][rows]: those pairs, row * top_k + choice
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
        // (sc first: it goes up to 2^126, and 16 sc would be infinite)
        float t0 = v[2 * k] * sc, t1 = v[2 * k + 1] * sc;
        if (!(k & 1)) {
            t0 *= 16.0f;
            t1 *= 16.0f;
        }
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
        u32x4 *o = reinterpret_cast<u32x4 *>(img + (size_t)c * 32);
        o[0] = hi;
        o[1] = lo;
    }
}

// ---------------------------------------------------------------- routing

__device__ __forceinline__ bool ahead(double a, int i, double b, int j) {
    return a > b || (a == b && i < j);
}

// Scores are kept without NaN, which would be ahead of nothing and behind nothing:
// as -inf they are chosen last.
__device__ __forceinline__ double ranked(double s) { return s >= -INFINITY ? s : -INFINITY; }

// The scores of one row, a workgroup an expert (f64 products of f32 values are
// exact, their sums are off by 2^-53 of the terms); the last workgroup makes the
// row's image.  128 scores of 2,048: 2.7 us, where the matrix cores' 8 workgroups
// would wait for 128 KB each.
__global__ __launch_bounds__(256) void moe_score_row_kernel(MoeArgs a) {
    __shared__ double red[4];
    const int tid = threadIdx.x, dim = a.m.dim, e = blockIdx.x;
    if (e == a.m.n_experts) {
        split_row<256>(a.x, dim, a.ximg, a.xscale);
        return;
    }
    double s = 0.0;
    const float *w = a.m.router + (size_t)e * dim;
#pragma unroll 2
    for (int i = tid * 4; i < dim; i += 1024) {
        const float4 v = *reinterpret_cast<const float4 *>(w + i);
        const float4 x = *reinterpret_cast<const float4 *>(a.x + i);
        s = fma((double)x.x, (double)v.x, s);
        s = fma((double)x.y, (double)v.y, s);
        s = fma((double)x.z, (double)v.z, s);
        s = fma((double)x.w, (double)v.w, s);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) a.score[e] = (red[0] + red[1]) + (red[2] + red[3]);
}

// A part of the sum of the scores of 16 rows and 16 experts a workgroup, on the f64
// matrix cores, the waves sharing it out; then the rows' images.  The first clears
// the experts' counts.
typedef double f64x4 __attribute__((ext_vector_type(4)));
__global__ __launch_bounds__(256, 2) void moe_score_kernel(MoeArgs a) {
    __shared__ double red[4][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int dim = a.m.dim, E = a.m.n_experts;
    const int et = (E + 15) / 16, rt = (a.rows + 15) / 16, tiles = et * rt;
    int b = blockIdx.x;
    if (b == 0)
        for (int e = tid; e < E; e += 256) a.count[e * kApart] = 0;
    if (b >= tiles * a.splits) {
        const int r = b - tiles * a.splits;
        split_row<256>(a.x + (size_t)r * dim, dim, a.ximg + (size_t)r * dim * 4, a.xscale + r);
        return;
    }
    const int part = b / tiles;
    b %= tiles;
    const int e0 = b % et * 16, r0 = b / et * 16;
    const int li = lane & 15, lg = lane >> 4;
    const float *x = a.x + (size_t)min(r0 + li, a.rows - 1) * dim + 4 * lg;
    const float *w = a.m.router + (size_t)min(e0 + li, E - 1) * dim + 4 * lg;
    f64x4 acc = {0.0, 0.0, 0.0, 0.0};
    const int by = a.splits * 64;
    constexpr int D = 8;  // loads in flight
    for (int i0 = (part * 4 + wave) * 16; i0 < dim; i0 += D * by) {
        float4 u[D], v[D];
#pragma unroll
        for (int k = 0; k < D; ++k) {
            const int i = i0 + k * by < dim ? i0 + k * by : i0;
            u[k] = *reinterpret_cast<const float4 *>(x + i);
            v[k] = *reinterpret_cast<const float4 *>(w + i);
        }
        __builtin_amdgcn_sched_barrier(0);  // (all of them, before the first is waited for)
#pragma unroll
        for (int k = 0; k < D; ++k) {
            if (i0 + k * by >= dim) break;
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[k].x, (double)v[k].x, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[k].y, (double)v[k].y, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[k].z, (double)v[k].z, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[k].w, (double)v[k].w, acc, 0, 0, 0);
        }
    }
    // D[4 r + lane / 16][lane % 16] in element r
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][(4 * r + lg) * 16 + li] = acc[r];
    __syncthreads();
    const int r = r0 + (tid >> 4), e = e0 + (tid & 15);
    if (r < a.rows && e < E)
        a.score[((size_t)part * a.rows + r) * E + e] =
            (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
}

// Lanes to an expert when NT threads rank E of them, and the scores that they go
// through, in whole runs of 8 (those behind E, -inf, are ahead of nothing).
constexpr int kRun = 8, kRanked = kMaxExperts + 64 * kRun;
__device__ __forceinline__ int rank_lanes(int NT, int E) {
    int per = 1;
    while (per < 64 && 2 * per * E <= NT) per *= 2;
    return per;
}

// score[e] = row r's scores, by a workgroup of NT threads (not yet synchronised).
template <int NT>
__device__ __forceinline__ void load_scores(const MoeArgs &a, int r, double *score) {
    const int E = a.m.n_experts, run = rank_lanes(NT, E) * kRun;
    for (int e = threadIdx.x; e < (E + run - 1) / run * run; e += NT) {
        double v[kMaxSplits];
#pragma unroll
        for (int i = 0; i < kMaxSplits; ++i)
            v[i] = e < E && i < a.splits ? a.score[((size_t)i * a.rows + r) * E + e] : 0.0;
        double s = v[0];
#pragma unroll
        for (int i = 1; i < kMaxSplits; ++i) s += v[i];
        score[e] = e < E ? ranked(s) : -INFINITY;
    }
}

// f(expert, rank) for every expert, by `per` lanes each that count those ahead of
// it (8 rounds of finding the largest of 128 took 10 us a row).
template <int NT, typename F>
__device__ __forceinline__ void ranks(const double *score, int E, F f) {
    const int per = rank_lanes(NT, E), part = threadIdx.x % per;
    for (int e0 = 0; e0 < E; e0 += NT / per) {
        const int e = e0 + threadIdx.x / per;
        const double mine = score[min(e, E - 1)];
        int n = 0;
        for (int i0 = part; i0 < E; i0 += per * kRun) {
            double v[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k) v[k] = score[i0 + k * per];
#pragma unroll
            for (int k = 0; k < kRun; ++k) n += ahead(v[k], i0 + k * per, mine, e);
        }
        for (int d = 1; d < per; d <<= 1) n += __shfl_xor(n, d);
        if (part == 0 && e < E) f(e, n);
    }
}

// The choice of row r by a workgroup of NT threads: ids, p, the caller's copies,
// and (LISTS) the experts' lists, whose order hangs on the atomics: which of a
// tile's rows a pair becomes does not show in its result.
template <int NT, bool LISTS>
__device__ void choose(const MoeArgs &a, int r) {
    __shared__ double score[kRanked], term[kMaxTop], part[NT / 64];
    __shared__ int id[kMaxTop];
    const int tid = threadIdx.x, E = a.m.n_experts, K = a.m.top_k;
    if (!live(a, r)) {
        if (tid < K) a.ids[r * K + tid] = -1;
        return;
    }
    load_scores<NT>(a, r, score);
    __syncthreads();
    ranks<NT>(score, E, [&](int e, int n) {
        if (n < K) id[n] = e;
    });
    __syncthreads();
    const double most = score[id[0]];
    if (tid < K) term[tid] = exp(score[id[tid]] - most);
    if (!a.m.normalise) {
        double s = 0.0;
        for (int e = tid; e < E; e += NT) s += exp(score[e] - most);
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
        if ((tid & 63) == 0) part[tid >> 6] = s;
    }
    __syncthreads();
    if (tid >= K) return;
    double sum = 0.0;
    if (a.m.normalise)
        for (int k = 0; k < K; ++k) sum += term[k];
    else
        for (int w = 0; w < NT / 64; ++w) sum += part[w];
    const int i = r * K + tid, e = id[tid];
    const float p = (float)(term[tid] / sum);
    a.ids[i] = e;
    a.p[i] = p;
    if (a.experts) a.experts[i] = e;
    if (a.weights) a.weights[i] = p;
    if constexpr (LISTS) a.list[(size_t)e * a.rows + atomicAdd(&a.count[e * kApart], 1)] = i;
}

// A workgroup a row: 6 us for 48 rows of 128 experts, 7 for 500 (5.3 without the lists'
// atomics; with 512 or 256 threads a row the same).
__global__ __launch_bounds__(1024) void moe_choose_kernel(MoeArgs a) { choose<1024, true>(a, blockIdx.x); }

// ---------------------------------------------------------------- products
//
// A stage is 16 W rows of J groups of four blocks, brought into LDS by the wave that
// takes it and by no other, so nothing but a wave's own wait count orders it.  Loads
// straight into registers ask for 16 bytes of another row with every lane, and the
// L1s, which take 64 bytes of neighbouring lanes a cycle, then bound everything (48
// rows of 128 experts: 30 million accesses, 49 of 70 us).  In LDS quants lie as
// [row][slot] x 16 B, two groups (a line of a row of W) or four blocks at a time, with
// block b in slot b ^ row / 2 & 7 or b ^ row / 4 & 3, so that the reads of a word, four
// bytes of each row's block, touch every bank once; then scales [row][2 J words].
template <int J>
struct Stage {
    static constexpr int Q = J * 1024, BYTES = Q + (J > 2 ? 512 : 256);
    static constexpr int DMAS = J + (J > 2 ? 2 : 1);
    static constexpr int LINE = J % 2 ? 4 : 8;  // blocks of a row that lie together
};

// A lane's offsets: its rows and blocks of the DMAs, its words of the scales', and of
// LDS the words of the blocks that it multiplies.
template <int J>
struct StageLane {
    uint32_t q[2], s[2], at[Stage<J>::LINE], scale;
    int block[2], word[2];
};
template <int J>
__device__ __forceinline__ StageLane<J> stage_lane(int lane, int nb) {
    constexpr int L = Stage<J>::LINE;
    StageLane<J> l;
    const int li = lane & 15, lg = lane >> 4;
    // L = 8: DMAs of rows 0 .. 7 and 8 .. 15; 4: of all 16 rows, the second two unused
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int row = L == 8 ? 8 * k + (lane >> 3) : lane >> 2;
        l.q[k] = (uint32_t)row * nb * 16;
        l.block[k] = L == 8 ? (lane ^ row >> 1) & 7 : (lane ^ row >> 2) & 3;
        const int i = min(lane + 64 * k, 32 * J - 1);
        l.word[k] = i % (2 * J);
        l.s[k] = (uint32_t)(i / (2 * J)) * nb * 2;
    }
#pragma unroll
    for (int i = 0; i < L; ++i)
        l.at[i] = li * (16 * L) + (L == 8 ? (i ^ li >> 1) & 7 : (i ^ li >> 2) & 3) * 16 + lg * 4;
    l.scale = Stage<J>::Q + li * 8 * J;
    return l;
}

// Asks for a stage: q and s point at the first row's first block, of which [0, n) exist
// (for those behind the last one is read again).
template <int J>
__device__ __forceinline__ void issue_stage(const StageLane<J> &l, const uint8_t *q, const uint16_t *s,
                                            int n, uint32_t buf) {
    constexpr int L = Stage<J>::LINE;
    const bool whole = n == 4 * J;  // (but for a row's last stage)
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int k = L == 8 ? j & 1 : 0, first = L == 8 ? j / 2 * 8 : j * 4;  // the line's first block
        uint32_t off = l.q[k] + 16 * l.block[k];
        if (!whole) off = l.q[k] + 16 * min(l.block[k], n - 1 - min(first, n - 1));
        dma16u(q + 16 * (whole ? first : min(first, n - 1)), off, buf + j * 1024);
    }
#pragma unroll
    for (int t = 0; t < (J > 2 ? 2 : 1); ++t) {
        uint32_t off = l.s[t] + 4 * l.word[t];
        if (!whole) off = l.s[t] + 4 * min(l.word[t], (n - 1) / 2);
        dma4u(s, off, buf + Stage<J>::Q + 256 * t);
    }
}

// acc += the stage times the x fragments x(half, block), which are 0 for blocks that do
// not exist.  Eight rows: their hi and lo halves are the fragment's 16 rows (H = 1);
// 16 rows: two fragments one after the other (H = 2), so that a block's scale meets the
// sum of both.  A block's products are scaled and added while the next
// one's run and its weights are decoded; a group's words are read a group ahead.
template <int J, int H, typename X>
__device__ __forceinline__ void multiply_stage(const StageLane<J> &l, const unsigned char *buf, X x,
                                               f32x4 &acc) {
    constexpr int L = Stage<J>::LINE;
    uint32_t w[2][4];
    uint2 d4[2];
    auto read = [&](int j) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[j & 1][i] = *reinterpret_cast<const uint32_t *>(
                buf + (L == 8 ? l.at[4 * (j & 1) + i] + j / 2 * 2048 : l.at[i] + j * 1024));
        d4[j & 1] = *reinterpret_cast<const uint2 *>(buf + l.scale + 8 * j);
    };
    f32x4 t[2];
    auto add = [&](int k) {
        const uint2 s = d4[k / 4 & 1];
        const f16x2 d2 = __builtin_bit_cast(f16x2, k & 2 ? s.y : s.x);
        const float d = (float)d2[k & 1];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(d, t[k & 1][r], acc[r]);
    };
    f16x8 b[2];
    read(0);
    b[0] = nibbles(w[0][0]);
#pragma unroll
    for (int k = 0; k < 4 * J; ++k) {
        t[k & 1] = mfma16(x(0, k), b[k & 1], f32x4{0.f, 0.f, 0.f, 0.f});
        if constexpr (H == 2) t[k & 1] = mfma16(x(1, k), b[k & 1], t[k & 1]);
        if (k + 1 < 4 * J) b[k + 1 & 1] = nibbles(w[(k + 1) / 4 & 1][(k + 1) & 3]);
        if (k > 0) add(k - 1);
        // (behind the last use of the scales that it replaces)
        if (k % 4 == 0 && k / 4 + 1 < J) read(k / 4 + 1);
        // (else all products come first, each in registers of its own)
        __builtin_amdgcn_sched_group_barrier(0x008, H, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 13, 0);
    }
    add(4 * J - 1);
    // the sums are wanted here (the compiler would put them off to the next stage, and
    // keep every product until then)
    asm volatile("" : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]));
}

// Rows of an odd number of blocks, or whose scales are not 4-byte aligned: a lane of the
// 16 x 4 (W row, k group) loads block 4 s + group of its row, and the lane groups hand
// each other their words (two swaps of lane halves, two of rows of 16).
struct Step {
    u32x4 q[4], x[4];
    uint2 d[4];
};
struct Operands {
    const uint8_t *q[4];   // the column tiles' first W rows
    const uint16_t *d[4];
};

// xo: where the lane's fragment begins in a block's image
__device__ __forceinline__ void load_step(const Operands &o, const uint8_t *img, size_t xo,
                                          int nb, int s, Step &f) {
    const int lane = threadIdx.x & 63, row = lane & 15, lg = lane >> 4;
    const int b = min(4 * s + lg, nb - 1);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        f.q[c] = *reinterpret_cast<const u32x4 *>(o.q[c] + (uint32_t)(row * nb + b) * 16);
        const uint16_t *d = o.d[c] + row * nb + 4 * s;
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = 4 * s + i < nb ? d[i] : 0;
        f.d[c] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f.x[i] = *reinterpret_cast<const u32x4 *>(img + xo + (size_t)min(4 * s + i, nb - 1) * 128);
}

// Word w of the lane groups' blocks -> block i of word `group`.
__device__ __forceinline__ u32x4 exchange(u32x4 q) {
    const auto a = __builtin_amdgcn_permlane16_swap(q[0], q[1], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(q[2], q[3], false, false);
    const auto c = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    return u32x4{c[0], d[0], c[1], d[1]};
}

__device__ __forceinline__ void multiply_step(const Step &f, f32x4 (&acc)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const u32x4 w = exchange(f.q[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x8 b = nibbles(w[i]);
            const f16x2 d2 = __builtin_bit_cast(f16x2, i < 2 ? f.d[c].x : f.d[c].y);
            const float d = (float)d2[i & 1];
            const f32x4 t = mfma16(__builtin_bit_cast(f16x8, f.x[i]), b, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[c][r] = __builtin_fmaf(d, t[r], acc[c][r]);
        }
    }
}

// acc += the products of steps s, s + by, ...: two steps' loads in flight.
__device__ __forceinline__ void multiply_steps(const Operands &o, const uint8_t *img,
                                               size_t xo, int nb, int s, int by,
                                               f32x4 (&acc)[4]) {
    const int n = (nb + 3) / 4;
    if (s >= n) return;
    Step f[2];
    load_step(o, img, xo, nb, s, f[0]);
    for (;; s += 2 * by) {
        load_step(o, img, xo, nb, min(s + by, n - 1), f[1]);
        multiply_step(f[0], acc);
        if (s + by >= n) break;
        load_step(o, img, xo, nb, min(s + 2 * by, n - 1), f[0]);
        multiply_step(f[1], acc);
        if (s + 2 * by >= n) break;
    }
}

// ---------------------------------------------------------------- tiles of pairs

// Tile b of `tile` pairs of one expert, counted over the experts: every wave finds
// it from the counts (lane i has experts i * per ..), which costs it a load and a
// scan instead of a launch that lists the tiles.  n = 0: there are fewer.
struct Tile {
    int e, n;
    const int *list;
};
__device__ __forceinline__ Tile find_tile(const MoeArgs &a, int tile, int b) {
    constexpr int N = kMaxExperts / 64;
    const int lane = threadIdx.x & 63, E = a.m.n_experts, per = (E + 63) / 64;
    int c[N], mine = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        c[j] = j < per && lane * per + j < E ? a.count[(lane * per + j) * kApart] : 0;
        mine += (c[j] + tile - 1) / tile;
    }
    int to = mine;
#define CW_SCAN_STEP(ctrl, rows) to += __builtin_amdgcn_update_dpp(0, to, ctrl, rows, 0xf, true)
    CW_SCAN_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
    CW_SCAN_STEP(0x112, 0xf);
    CW_SCAN_STEP(0x114, 0xf);
    CW_SCAN_STEP(0x118, 0xf);
    CW_SCAN_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    CW_SCAN_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef CW_SCAN_STEP
    const uint64_t has = __ballot(to > b);
    if (!has) return Tile{0, 0, nullptr};
    const int owner = __builtin_ctzll(has);
    int e = lane * per, left = b - (to - mine), n = 0;  // (of the owner's lane)
    bool found = false;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int t = (c[j] + tile - 1) / tile;
        if (!found && left < t) {
            found = true;
            e = lane * per + j;
            n = c[j];
        } else if (!found) {
            left -= t;
        }
    }
    e = __builtin_amdgcn_readlane(e, owner);
    left = __builtin_amdgcn_readlane(left, owner);
    n = __builtin_amdgcn_readlane(n, owner);
    return Tile{e, min(tile, n - left * tile), a.list + (size_t)e * a.rows + left * tile};
}

// A tile's pair i, its last again past the end
__device__ __forceinline__ int pair_of(const Tile &t, int i) { return t.list[min(i, t.n - 1)]; }

// How a tile kernel of 8 H rows and J groups of blocks of x in a wave's registers (0:
// through registers, any row length) is laid out.  16 rows decode W half as often, but
// have 128 B of x for 64: eight waves share a sum where four do.  At four waves a SIMD the
// products take 125 and 126 registers of 128, without scratch.
template <int H, int J>
struct TileShape {
    static constexpr int ROWS = kTile * H, WAVES = 4 * H;  // WAVES at most
    // stages of SJ groups, SUBS of them a slice of x, R in LDS for each wave
    static constexpr int SJ = J == 3 ? 3 : 2, SUBS = J / SJ, R = J == 4 ? 3 : 2;
    static constexpr int RING = J ? WAVES * R * Stage<SJ>::BYTES : 16;
};

// A tile of pairs times stretches of its expert's columns: of h (UP: 32 gate and the
// same 32 up columns a set) or of z (64 columns a set).  ks waves split the sum, others
// take other sets; W goes through each wave's ring of stages, x stays in registers
// where a wave's slice of it is all it has, for `groups` sets one after the other.
// (Eight rows take one set: with two or three the next one's W is asked for ahead, but
// 48 rows still take 45.7 and 47.1 us, 46.4 with one.)
template <bool UP, int H, int J>
__global__ __launch_bounds__((TileShape<H, J>::WAVES * 64))
__attribute__((amdgpu_waves_per_eu(4, 4)))
void moe_tile_kernel(MoeArgs a, int ks, int groups) {
    using T = TileShape<H, J>;
    constexpr int SJ = T::SJ, SUBS = T::SUBS, R = T::R;
    constexpr int SET = UP ? 32 : 64;  // columns
    using S = Stage<SJ>;
    __shared__ __attribute__((aligned(1024))) unsigned char ring[T::RING];
    __shared__ f32x4 red[T::WAVES][4][32 * H];
    // the tile's pairs, the scales of their rows and (down) the experts' shares in them
    __shared__ int pairs[64];
    __shared__ float scales[64], shares[UP ? 1 : 64];
    const Tile tile = find_tile(a, T::ROWS, blockIdx.y);
    if (tile.n == 0) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int K = a.m.top_k, N = UP ? a.m.hidden : a.m.dim, nb = (UP ? a.m.dim : a.m.hidden) / 32;
    const int cs = (int)blockDim.x / 64 / ks, sets = (N + SET - 1) / SET;
    const int set0 = blockIdx.x * groups * cs;
    const int n_groups = H == 1 ? 1 : min(groups, (sets - set0 + cs - 1) / cs);
    const uint8_t *const img = UP ? a.ximg : a.himg;

    // the first column of the wave's set of a group (past the last set the last again, not
    // stored), and the W row of its column tile c from there
    auto first_col = [&](int g) { return min(set0 + g * cs + wave / ks, sets - 1) * SET; };
    auto tile_row = [&](int col, int c) { return UP ? (c & 1) * 16 : min(c * 16, N - 16 - col); };

    // x rows of the lane's fragments, hi or lo of row li / 2 or both of row li (rows past
    // the tile's end read nothing)
    const int row = H == 1 ? li >> 1 : li, row_pair = pair_of(tile, row);
    const size_t xo = (size_t)(UP ? row_pair / K : row_pair) * nb * 128 + lg * 32 +
                      (H == 1 ? (li & 1) * 16 : 0);
    // (by DMA: values of its own to be stored once x is there would cost every thread
    // registers through the products)
    if (wave == 0) {
        const int pair = pair_of(tile, lane);
        auto at = [](void *p) { return lds_off(static_cast<unsigned char *>(p)); };
        dma4u(tile.list, min(lane, tile.n - 1) * 4, at(pairs));
        dma4u(UP ? a.xscale : a.hscale, (UP ? pair / K : pair) * 4, at(scales));
        if constexpr (!UP) dma4u(a.p, pair * 4, at(shares));
    }

    // A group's sums from the waves that share them, to h or z.  Eight rows: a lane's
    // elements are hi and lo of rows 2 lg and 2 lg + 1, of 16 rows 4 lg to 4 lg + 3.
    auto store = [&](int g, const f32x4 (&acc)[4]) {
        lds_barrier();  // the last reads of red
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if constexpr (H == 1)
                reinterpret_cast<float2 *>(red[wave][c])[lane] =
                    make_float2(acc[c][0] + acc[c][1], acc[c][2] + acc[c][3]);
            else
                red[wave][c][lane] = acc[c];
        lds_barrier();
        // a thread: P rows of one column, which one lane of each wave holds (lanes along
        // the columns: reads of P floats each, side by side)
        constexpr int P = H == 1 ? 2 : 4;
        using Rows = __attribute__((ext_vector_type(P))) float;
        const int width = SET * cs;
        for (int t = tid; t < T::ROWS / P * width; t += (int)blockDim.x) {
            const int i = t / width * P, s = t % width / SET, n0 = t % SET;
            const int col = (set0 + g * cs + s) * SET + n0;
            if (i >= tile.n) break;
            if (col >= N) continue;
            const int from = i / P * 16 + (n0 & 15);
            auto sum = [&](int c) {
                Rows v = 0.0f;
                for (int w = 0; w < ks; ++w)
                    v += reinterpret_cast<const Rows *>(red[s * ks + w][c])[from];
                return v;
            };
            const Rows v = sum(n0 >> 4), u = UP ? sum(2 + (n0 >> 4)) : v;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                if (i + e >= tile.n) break;
                const size_t at = (size_t)pairs[i + e] * N + col;
                const float scale = kUnscale * scales[i + e];
                if constexpr (UP) a.h[at] = silu_mul(v[e] * scale, u[e] * scale);
                // (the scale last: p times a small one would be below f32's normal range)
                else a.z[at] = v[e] * shares[i + e] * scale;
            }
        }
    };

    if constexpr (J == 0) {
        static_assert(H == 1);
        const int col = first_col(0);
        Operands o;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const size_t w0 = ((size_t)tile.e * N + col + tile_row(col, c)) * nb;
            o.q[c] = (!UP ? a.m.down_quants : c < 2 ? a.m.gate_quants : a.m.up_quants) + w0 * 16;
            o.d[c] = (!UP ? a.m.down_scales : c < 2 ? a.m.gate_scales : a.m.up_scales) + w0;
        }
        f32x4 acc[4] = {};
        multiply_steps(o, img, xo, nb, wave % ks, ks, acc);
        wait_vm<0>();  // the scales
        store(0, acc);
    } else {
        unsigned char *const mine = ring + wave * R * S::BYTES;
        const StageLane<SJ> l = stage_lane<SJ>(lane, nb);
        const int slices = (nb + 4 * J - 1) / (4 * J), rounds = (slices + ks - 1) / ks;
        // the wave's first group of blocks in a round (a wave without any goes through
        // the row's last ones with no x)
        auto first = [&](int t) { return min(t * ks + wave % ks, slices - 1) * J; };
        // Stages are asked for R - 1 ahead, tile c = k / SUBS and sub = k % SUBS of a round,
        // k a constant where it is called: what changes with the round alone is kept.
        const uint32_t lds = lds_off(mine);
        const uint8_t *q0, *q1 = nullptr;
        const uint16_t *d0, *d1 = nullptr;
        int ig = 0, it = 0, icol = 0, ib = 0, ibuf = 0;  // of the next stage to ask for
        auto begin = [&] {
            icol = first_col(ig);
            ib = first(it);
            const size_t w0 = ((size_t)tile.e * N + icol) * nb + 4 * ib;
            q0 = (UP ? a.m.gate_quants : a.m.down_quants) + w0 * 16;
            d0 = (UP ? a.m.gate_scales : a.m.down_scales) + w0;
            if constexpr (UP) {
                q1 = a.m.up_quants + w0 * 16;
                d1 = a.m.up_scales + w0;
            }
        };
        auto issue = [&](int k) {
            if (k == 4 * SUBS) {
                if (++it == rounds) {
                    it = 0;
                    ++ig;
                }
                begin();
            }
            const int c = k / SUBS % 4, sub = k % SUBS;
            // (past the row's end its last group again)
            const int skip = min(sub * SJ, (nb + 3) / 4 - 1 - ib), n = min(4 * SJ, nb - 4 * (ib + skip));
            const uint32_t at = tile_row(icol, c) * nb + 4 * skip;
            issue_stage<SJ>(l, (UP && c >= 2 ? q1 : q0) + 16 * (size_t)at, (UP && c >= 2 ? d1 : d0) + at, n,
                            lds + ibuf * S::BYTES);
            ibuf = ibuf + 1 == R ? 0 : ibuf + 1;
        };
        const int total = n_groups * rounds * 4 * SUBS;
        int left = total, buf = 0;
        u32x4 x[H][4 * J];
        for (int g = 0; g < n_groups; ++g) {
            f32x4 acc[4] = {};
            for (int t = 0; t < rounds; ++t) {
                if (g == 0 || rounds > 1) {
                    const int b = first(t) * 4, n = t * ks + wave % ks < slices ? min(4 * J, nb - b) : 0;
#pragma unroll
                    for (int i = 0; i < 4 * J; ++i)
#pragma unroll
                        for (int h = 0; h < H; ++h) x[h][i] = u32x4{0, 0, 0, 0};
                    if (row < tile.n) {
                        const uint8_t *p = img + xo + (size_t)b * 128;
#pragma unroll
                        for (int i = 0; i < 4 * J; ++i)
                            if (i < n)
#pragma unroll
                                for (int h = 0; h < H; ++h)
                                    x[h][i] = *reinterpret_cast<const u32x4 *>(p + 128 * i + 16 * h);
                    }
                    // (x ahead of the first stages: behind them it comes last, 48 rows
                    // 46 -> 55 us)
                    if (g + t == 0) {
                        begin();
#pragma unroll
                        for (int k = 0; k < R - 1; ++k) issue(k);
                    }
                    // here, or the compiler waits for x, and so for every stage that is on
                    // its way, before each stage (and for the scales)
                    wait_vm<0>();
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub) {
                        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): reads of the buffer asked for next
                        if (left >= R) {
                            issue(c * SUBS + sub + R - 1);
                            wait_vm<(R - 1) * S::DMAS>();
                        } else if (R == 3 && left == 2) {
                            wait_vm<S::DMAS>();
                        } else {
                            wait_vm<0>();
                        }
                        multiply_stage<SJ, H>(
                            l, mine + buf * S::BYTES,
                            [&](int h, int i) { return __builtin_bit_cast(f16x8, x[h][4 * SJ * sub + i]); },
                            acc[c]);
                        --left;
                        buf = buf + 1 == R ? 0 : buf + 1;
                    }
            }
            store(g, acc);
        }
    }
}

// h's images: every workgroup of the down product reads a row's, so its largest value
// is found and it is split once.  5 us for 48 rows of 8 experts, 8 for 500 (23 MB).
__global__ __launch_bounds__(256) void moe_split_kernel(MoeArgs a) {
    const size_t pair = blockIdx.x;
    if (a.ids[pair] < 0) return;
    split_row<256>(a.h + pair * a.m.hidden, a.m.hidden, a.himg + pair * a.m.hidden * 4,
                   a.hscale + pair);
}

// ---------------------------------------------------------------- few rows
//
// One row needs no lists and no launch for the choice: a workgroup has one rank of
// the choice and 16 columns of h, and finds the expert of that rank itself.  The
// first workgroup writes the choice down for the second product.

constexpr int kRowThreads = 512, kRowWaves = kRowThreads / 64;

// DMA: rows of an even number of blocks, scales 4-byte aligned
template <bool DMA>
__global__ __launch_bounds__(kRowThreads) void moe_up_row_kernel(MoeArgs a) {
    constexpr int J = 2, R = 2;  // (with 4 one workgroup fits a CU: 12.6 us for 384 of them)
    using S = Stage<J>;
    __shared__ __attribute__((aligned(1024))) unsigned char ring[DMA ? kRowWaves * R * S::BYTES : 16];
    __shared__ double score[kRanked];
    __shared__ float red[kRowWaves][2][16];
    __shared__ int chosen;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int E = a.m.n_experts, hidden = a.m.hidden;
    if (blockIdx.x == 0) {
        choose<kRowThreads, false>(a, 0);
        return;
    }
    if (!live(a, 0)) return;
    const int cols = hidden / 16, rank = (blockIdx.x - 1) / cols, col = (blockIdx.x - 1) % cols * 16;
    load_scores<kRowThreads>(a, 0, score);
    __syncthreads();
    ranks<kRowThreads>(score, E, [&](int e, int n) {
        if (n == rank) chosen = e;
    });
    __syncthreads();
    const int e = __builtin_amdgcn_readfirstlane(chosen);
    const int li = lane & 15, lg = lane >> 4, nb = a.m.dim / 32;
    const size_t w0 = ((size_t)e * hidden + col) * nb;
    const uint8_t *const img = a.ximg + lg * 32 + (li & 1) * 16;
    f32x4 acc[4] = {};
    if constexpr (DMA) {
        unsigned char *const mine = ring + wave * R * S::BYTES;
        const StageLane<J> l = stage_lane<J>(lane, nb);
        const int slices = (nb + 4 * J - 1) / (4 * J);
        const int total = wave < slices ? ((slices - 1 - wave) / kRowWaves + 1) * 2 : 0;
        const uint32_t lds = lds_off(mine);
        auto issue = [&](int k) {  // gate, up of the wave's k / 2th slice
            const int b = (wave + k / 2 * kRowWaves) * 4 * J;
            issue_stage<J>(l, (k & 1 ? a.m.up_quants : a.m.gate_quants) + (w0 + b) * 16,
                           (k & 1 ? a.m.up_scales : a.m.gate_scales) + w0 + b, min(4 * J, nb - b),
                           lds + k % R * S::BYTES);
        };
        for (int k = 0; k < R && k < total; ++k) issue(k);
        for (int k = 0; k < total; k += 2) {
            const int b = (wave + k / 2 * kRowWaves) * 4 * J;
            u32x4 x[4 * J];
#pragma unroll
            for (int i = 0; i < 4 * J; ++i) {
                x[i] = u32x4{0, 0, 0, 0};
                if (b + i < nb) x[i] = *reinterpret_cast<const u32x4 *>(img + (size_t)(b + i) * 128);
            }
            // (x was asked for behind them)
            wait_vm<0>();
#pragma unroll
            for (int c = 0; c < 2; ++c)
                multiply_stage<J, 1>(l, mine + (k + c) % R * S::BYTES,
                                     [&](int, int i) { return __builtin_bit_cast(f16x8, x[i]); }, acc[c]);
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
            for (int c = 0; c < 2; ++c)
                if (k + c + R < total) issue(k + c + R);
        }
    } else {
        Operands o;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            o.q[c] = (c & 1 ? a.m.up_quants : a.m.gate_quants) + w0 * 16;
            o.d[c] = (c & 1 ? a.m.up_scales : a.m.gate_scales) + w0;
        }
        const size_t xo = lg * 32 + (li & 1) * 16;
        multiply_steps(o, a.ximg, xo, nb, wave, kRowWaves, acc);
    }
    // every two rows are the row's hi and lo
    if (lane < 16) {
        red[wave][0][lane] = acc[0][0] + acc[0][1];
        red[wave][1][lane] = acc[1][0] + acc[1][1];
    }
    __syncthreads();
    if (tid >= 16) return;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) {
        g += red[w][0][tid];
        u += red[w][1][tid];
    }
    const float sc = kUnscale * a.xscale[0];
    a.h[(size_t)rank * hidden + col + tid] = silu_mul(g * sc, u * sc);
}

// A workgroup has 16 columns of a row's y; its waves share the experts out, or parts of
// them where there are fewer.  A stage is the columns' rows of W, 8 blocks of each, and
// that stretch of h, which the wave splits itself under a power of two of the stretch.
template <bool DMA>
__global__ __launch_bounds__(kRowThreads) void moe_down_row_kernel(MoeArgs a) {
    constexpr int W = kRowWaves, J = 2;
    constexpr int R = 2;  // (with 3 one workgroup fits a CU: one row 8.6 us for 8.1, six 18.6 for 17.2)
    using S = Stage<J>;
    constexpr int BYTES = S::BYTES + 1024;  // h behind W
    __shared__ __attribute__((aligned(1024))) unsigned char ring[W * R * BYTES];
    __shared__ u32x4 img[W][4 * J * 8];
    __shared__ float red[kMaxTop][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int K = a.m.top_k, hidden = a.m.hidden, dim = a.m.dim, nb = hidden / 32;
    const int r = blockIdx.y, col = blockIdx.x * 16;
    if (!live(a, r)) return;
    const int my_id = a.ids[r * K + min(lane, K - 1)];
    const float my_p = a.p[r * K + min(lane, K - 1)];
    const int parts = K < W ? W / K : 1, steps = (nb + 3) / 4;
    const int per = (steps + parts - 1) / parts;
    unsigned char *const mine = ring + wave * R * BYTES;
    const uint32_t lds = lds_off(mine);
    const StageLane<J> l = stage_lane<J>(lane, nb);
    // unit u: part u % parts of expert u / parts, steps [s0, s1)
    auto begin = [&](int u) { return u % parts * per; };
    auto end = [&](int u) { return min(steps, u % parts * per + per); };
    int iu = wave, is = begin(wave), ibuf = 0;  // the next stage to ask for
    auto blocks = [&](int u, int s) { return min(4 * min(J, end(u) - s), nb - 4 * s); };  // of a stage
    auto skip = [&](int &u, int &s) {  // to the next unit that has steps
        while (u < K * parts && s >= end(u)) {
            u += W;
            s = begin(u);
        }
    };
    skip(iu, is);
    auto issue = [&] {
        const int j = iu / parts, e = __builtin_amdgcn_readlane(my_id, j);
        const size_t w0 = ((size_t)e * dim + col) * nb + 4 * is;
        const uint32_t buf = lds + ibuf * BYTES;
        const int n = blocks(iu, is);
        if constexpr (DMA) {
            issue_stage<J>(l, a.m.down_quants + w0 * 16, a.m.down_scales + w0, n, buf);
            const float *h = a.h + ((size_t)r * K + j) * hidden + 128 * is;
            // lane: chunk lane % 32 (block, group), its first or its second four elements
            dma16u(h, (32 * min(lane >> 2 & 7, n - 1) + 4 * (lane & 3) + (lane >> 5) * 16) * 4,
                   buf + S::BYTES);
        }
        ibuf = ibuf + 1 == R ? 0 : ibuf + 1;
        is += J;
        skip(iu, is);
    };
    int asked = 0, buf = 0;
    if constexpr (DMA)
        for (; asked < R - 1 && iu < K * parts; ++asked) issue();
    int u = wave, s = begin(wave);
    float total = 0.0f;
    skip(u, s);
    if (lane < 16)
        for (int k = wave; k < K * parts; k += W) red[k][lane] = 0.0f;
    while (u < K * parts) {
        const int j = u / parts, s1 = end(u), jn = min(J, s1 - s);
        float4 ve, vf;
        u32x4 q[J];
        uint2 d[J];
        const unsigned char *const at = mine + buf * BYTES;
        if constexpr (DMA) {
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): reads of the buffer asked for next
            if (iu < K * parts) {
                issue();
                ++asked;
            }
            // the stage behind this one may still be on its way
            if (asked == 2) wait_vm<S::DMAS + 1>();
            else wait_vm<0>();
            --asked;
            ve = *reinterpret_cast<const float4 *>(at + S::BYTES + (lane & 31) * 16);
            vf = *reinterpret_cast<const float4 *>(at + S::BYTES + 512 + (lane & 31) * 16);
            if ((lane & 31) >= 4 * blocks(u, s)) ve = vf = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
            const int e = __builtin_amdgcn_readlane(my_id, j);
            const size_t w0 = ((size_t)e * dim + col + li) * nb;
#pragma unroll
            for (int i = 0; i < J; ++i) {
                const int st = min(s + i, s1 - 1);
                q[i] = *reinterpret_cast<const u32x4 *>(a.m.down_quants + (w0 + min(4 * st + lg, nb - 1)) * 16);
                uint32_t v[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) v[t] = 4 * st + t < nb ? a.m.down_scales[w0 + 4 * st + t] : 0;
                d[i] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
            }
            const float *h = a.h + ((size_t)r * K + j) * hidden +
                             32 * min(4 * s + (lane >> 2 & 7), nb - 1) + 4 * (lane & 3);
            ve = *reinterpret_cast<const float4 *>(h);
            vf = *reinterpret_cast<const float4 *>(h + 16);
        }
        float mx = max8(ve, vf);
#pragma unroll
        for (int dd = 32; dd >= 1; dd >>= 1) mx = fmaxf(mx, __shfl_xor(mx, dd));
        const int ex = split_exponent(mx);
        u32x4 hi, lo;
        split8(ve, vf, ldexpf(1.0f, -ex), &hi, &lo);
        __builtin_amdgcn_wave_barrier();  // the reads of the last stretch
        // (both halves of the wave have the same chunks: one stores hi, the other lo)
        img[wave][(lane & 31) * 2 + (lane >> 5)] = lane < 32 ? hi : lo;
        __builtin_amdgcn_wave_barrier();
        // every two rows of the fragment are h's hi and lo
        const u32x4 *const x = &img[wave][lg * 2 + (li & 1)];
        f32x4 acc = {};
        if constexpr (DMA) {
            multiply_stage<J, 1>(l, at,
                                 [&](int, int i) { return __builtin_bit_cast(f16x8, x[8 * i]); }, acc);
        } else {
#pragma unroll
            for (int i = 0; i < J; ++i) {
                if (i >= jn) break;
                const u32x4 w = exchange(q[i]);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const f32x4 v = mfma16(__builtin_bit_cast(f16x8, x[8 * (4 * i + t)]), nibbles(w[t]),
                                           f32x4{0.f, 0.f, 0.f, 0.f});
                    const f16x2 d2 = __builtin_bit_cast(f16x2, t < 2 ? d[i].x : d[i].y);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[k] = __builtin_fmaf((float)d2[t & 1], v[k], acc[k]);
                }
            }
        }
        total = __builtin_fmaf(kUnscale * ldexpf(1.0f, ex), acc[0] + acc[1], total);
        buf = buf + 1 == R ? 0 : buf + 1;
        s += J;
        if (s >= s1) {
            const float p = __builtin_bit_cast(
                float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_p), j));
            if (lane < 16) red[u][lane] = p * total;
            total = 0.0f;
        }
        skip(u, s);
    }
    __syncthreads();
    if (tid >= 16) return;
    float y = 0.0f;
    for (int k = 0; k < K * parts; ++k) y += red[k][tid];
    const size_t o = (size_t)r * dim + col + tid;
    a.y[o] = a.residual ? a.residual[o] + y : y;
}

// y = [residual +] the sum of a row's experts in order of their rank: 5 us for 48 rows of 8
// (a launch), 9 for 500 (37 MB)
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

// Rows whose scales a DMA takes two at a time: an even number of blocks, 4-byte aligned
// (2112 x 832, 4 of 64 experts: 20 rows' up and down 29 + 15 us through the stages, 55 +
// 26 through registers; 500 rows 154 + 58, 216 + 125).
bool in_stages(int in_f, const uint16_t *s) { return in_f % 64 == 0 && ((uintptr_t)s & 3) == 0; }

// Workgroups that share a score's sum, 64 elements a wave at least
int score_splits(const cw_moe &m, int rows) {
    return rows == 1 ? 1 : std::min(kMaxSplits, std::max(1, m.dim / 512));
}

// Whether the second product goes row by row, reading an expert again for each row
// that chose it: that saves two launches and the passes over h and z, and pays while
// few rows meet (us by rows and by tiles; 8 of 128 experts, 2048 x 768: 2 rows 29, 36;
// 8 rows 53, 53; 16 rows 78, 68; 2 of 8, 4096 x 12288: 2 rows 95, 98; 4 rows 131, 126).
bool down_by_rows(const cw_moe &m, int rows) {
    return rows == 1 || 2 * rows * m.top_k <= m.n_experts;
}

// Places of the workspace, each 256-byte aligned; with base null their size.
size_t lay_out(const cw_moe &m, int rows, char *base, MoeArgs *a) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *p = base + at;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t pairs = (size_t)rows * m.top_k;
    a->splits = score_splits(m, rows);
    a->score = reinterpret_cast<double *>(take((size_t)a->splits * rows * m.n_experts * 8));
    a->ids = reinterpret_cast<int *>(take(pairs * 4));
    a->p = reinterpret_cast<float *>(take(pairs * 4));
    a->ximg = reinterpret_cast<uint8_t *>(take((size_t)rows * m.dim * 4));
    a->xscale = reinterpret_cast<float *>(take((size_t)rows * 4));
    a->h = reinterpret_cast<float *>(take(pairs * m.hidden * 4));
    a->count = reinterpret_cast<int *>(take((size_t)m.n_experts * kApart * 4));
    a->list = reinterpret_cast<int *>(take((size_t)m.n_experts * rows * 4));
    if (!down_by_rows(m, rows)) {
        a->himg = reinterpret_cast<uint8_t *>(take(pairs * m.hidden * 4));
        a->hscale = reinterpret_cast<float *>(take(pairs * 4));
        a->z = reinterpret_cast<float *>(take(pairs * m.dim * 4));
    }
    return at;
}

int run_down_rows(cw_ctx *ctx, const MoeArgs &a) {
    const bool dma = in_stages(a.m.hidden, a.m.down_scales);
    return launch(ctx, "moe_down", dma ? moe_down_row_kernel<true> : moe_down_row_kernel<false>,
                  dim3(a.m.dim / 16, a.rows), dim3(kRowThreads), 0, a);
}

// How the waves of a workgroup divide a product: J groups of blocks of x each (0:
// through registers), ks waves to a sum, cs sets at a time, `groups` of those.
struct TilePlan {
    int J, ks, cs, groups, grid;
};
template <int H>
TilePlan tile_plan(const cw_ctx *ctx, bool up, const cw_moe &m, bool dma, int tiles) {
    constexpr int W = 4 * H;
    const int nb = (up ? m.dim : m.hidden) / 32, sets = up ? m.hidden / 32 : (m.dim + 63) / 64;
    TilePlan p{0, nb >= 64 ? 4 : nb >= 8 ? 2 : 1, 1, 1, 0};
    int rounds = 1;
    if (dma) {
        // 16 rows: x of all of the sum if that fits; then the most of the waves' and the
        // stages' blocks that exist, and the fewest rounds
        int best = -1;
        for (int J = H == 1 ? 4 : 2; J >= 2; --J)
            for (int ks = W; ks >= 1; --ks) {
                const int r = ((nb + 4 * J - 1) / (4 * J) + ks - 1) / ks;
                const int used = nb * 1000 / (r * ks * 4 * J) * (W / ks * ks) / W;
                const int score = (H == 2 && r == 1 ? 1 << 20 : 0) + used * 64 - std::min(r, 63);
                if (score > best) {
                    best = score;
                    p.J = J;
                    p.ks = ks;
                    rounds = r;
                }
            }
    }
    p.cs = std::max(1, std::min(W / p.ks, sets));
    const int units = (sets + p.cs - 1) / p.cs;
    // 16 rows' x is read again for every workgroup: no more of them than fill the chip's
    // places (two a CU) twice (500 rows, 8 of 128 experts: once 271 us, twice 260, four
    // times 293, one set each 495 at 800 rows for 355)
    if (H == 2 && rounds == 1) p.groups = std::min(std::max(1, tiles * units / (4 * ctx->n_cu)), units);
    p.grid = (units + p.groups - 1) / p.groups;
    return p;
}

// Tiles of eight rows up to ten an expert, else of 16 (us with 8 and with 16; 8 of 128
// experts, 2048 x 768: 7 rows an expert 113, 119; 10: 136, 138; 15: 171, 160; 31: 294,
// 260; 2 of 8, 4096 x 12288: 8 rows 200, 212; 12: 258, 253; 40: 588, 564).  W that goes
// through registers takes eight (with 16 of 31 an expert, 2080 x 800, up and down 214 +
// 129 us for 197 + 116: two waves a SIMD instead of four).
template <bool UP>
int launch_product(cw_ctx *ctx, const MoeArgs &a) {
    const int E = a.m.n_experts, pairs = a.rows * a.m.top_k;
    const bool dma = UP ? in_stages(a.m.dim, a.m.gate_scales) && in_stages(a.m.dim, a.m.up_scales)
                        : in_stages(a.m.hidden, a.m.down_scales);
    const bool wide = dma && (pairs + E - 1) / E > 10;
    // tiles at most, and how many to expect of rows that choose evenly
    const int tile = wide ? 2 * kTile : kTile, most = std::min(pairs, E + pairs / tile);
    const int tiles = std::min(pairs, std::max(E, pairs / tile));
    const TilePlan p = wide ? tile_plan<2>(ctx, UP, a.m, dma, tiles) : tile_plan<1>(ctx, UP, a.m, dma, tiles);
    return launch(ctx, UP ? "moe_up" : "moe_down",
                  wide       ? moe_tile_kernel<UP, 2, 2>
                  : p.J == 0 ? moe_tile_kernel<UP, 1, 0>
                  : p.J == 2 ? moe_tile_kernel<UP, 1, 2>
                  : p.J == 3 ? moe_tile_kernel<UP, 1, 3>
                             : moe_tile_kernel<UP, 1, 4>,
                  dim3(p.grid, most), dim3(64 * p.ks * p.cs), 0, a, p.ks, p.groups);
}

int run(cw_ctx *ctx, const MoeArgs &a) {
    const int E = a.m.n_experts, K = a.m.top_k, pairs = a.rows * K;
    if (a.rows == 1) {
        const bool dma = in_stages(a.m.dim, a.m.gate_scales) && in_stages(a.m.dim, a.m.up_scales);
        CW_TRY(launch(ctx, "moe_score", moe_score_row_kernel, dim3(E + 1), dim3(256), 0, a));
        CW_TRY(launch(ctx, "moe_up", dma ? moe_up_row_kernel<true> : moe_up_row_kernel<false>,
                      dim3(1 + K * (a.m.hidden / 16)), dim3(kRowThreads), 0, a));
        return run_down_rows(ctx, a);
    }
    const int score = (E + 15) / 16 * ((a.rows + 15) / 16) * a.splits;
    CW_TRY(launch(ctx, "moe_score", moe_score_kernel, dim3(score + a.rows), dim3(256), 0, a));
    CW_TRY(launch(ctx, "moe_choose", moe_choose_kernel, dim3(a.rows), dim3(1024), 0, a));
    CW_TRY(launch_product<true>(ctx, a));
    if (down_by_rows(a.m, a.rows)) return run_down_rows(ctx, a);
    CW_TRY(launch(ctx, "moe_split", moe_split_kernel, dim3(pairs), dim3(256), 0, a));
    CW_TRY(launch_product<false>(ctx, a));
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
    CW_CHECK_ARG(!residual || residual == y || residual + n <= y || y + n <= residual,
                 "cw_moe_rows: residual and y overlap");
    CW_HIP(hipSetDevice(ctx->device));
    MoeArgs a{};
    int chunk = std::min(rows, kChunk);
    while (chunk > kTile && lay_out(m, chunk, nullptr, &a) > kChunkBytes) chunk = std::max(kTile, chunk / 2);
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
        CW_TRY(run(ctx, a));
    }
    return CW_OK;
}
