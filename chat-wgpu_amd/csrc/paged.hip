// Several requests in one paged KV cache: rotary rows with and without the norm
// of each head and the cache write, block tables from request lengths, the move of
// accepted rows.  The attention over that cache is tree_attention.hip's.

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "paged_device.hpp"

namespace {

using namespace cwi;

constexpr int kThreads = 256;

// ---------------------------------------------------------------- rotary rows
//
// y_a = g (x_a cos - x_b sin), y_b = g (x_b cos + x_a sin) for each pair (a, b),
// at the angle pos * f.  The table holds f / 2 pi in f64 (turns per position):
// its rounding and the product's are 2^-53 of the turns each, of which a position
// has 0.16 at most: 3.6e-11 of a turn in all at a million positions, 7.6e-8 at
// 2^31, so far positions cost next to no accuracy; in f32 a position of a million
// would leave 0.06 of a radian.  The rest, at most pi / 4, is x + lo in f32.

// cos and sin of 2 pi t by their Taylor series at the nearest quarter turn
// (|x| <= pi / 4: the first term left out is 2e-9), lo by the first two terms of
// the angles' sum: half a step and a little in all, as a rounding of the exact ones;
// times a gain of 48 bits
__device__ __forceinline__ float2 turn(double t, float gain, float gain_lo) {
    t -= rint(t);
    const double q = rint(4.0 * t);
    const double rest = (t - 0.25 * q) * 6.283185307179586;
    const float x = (float)rest, lo = (float)(rest - x);
    const float z = x * x;
    const float s = x + (x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880)))) +
                         (lo - 0.5f * z * lo));
    const float c = 1.0f + (z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 - z * (1.0f / 3628800))))) -
                            x * lo);
    const int k = (int)q & 3;
    const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
    const float gc = __builtin_fmaf(cc, gain, cc * gain_lo), gs = __builtin_fmaf(ss, gain, ss * gain_lo);
    return make_float2(k == 1 || k == 2 ? -gc : gc, k >= 2 ? -gs : gs);
}

struct RopeArgs {
    const double *turns;  // [rot / 2]
    float gain, gain_lo;
    int rot, pairs;       // rotated elements of a head; CW_ROPE_PAIRS
    const float *x;
    size_t x_stride;
    const int *positions, *slots;
    int rows, heads, kv_heads, hd;  // heads rotated into y, then (cache form) kv_heads of k and of v
    float *y;
    size_t y_stride;
    int copy;  // elements behind rot are copied to y (not in place)
    void *kc, *vc;
    int n_slots;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A unit that is read once (non-temporal: 4,100 rows with the cache write 36.7
// -> 32.4 us)
template <int V>
__device__ __forceinline__ void read_once(float *to, const float *from) {
    if constexpr (V == 4)
        *reinterpret_cast<f32x4 *>(to) = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(from));
    else
        *to = *from;
}
template <int V, bool STREAM>
__device__ __forceinline__ void put_unit(float *to, const float *from) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(*reinterpret_cast<const f32x4 *>(from), reinterpret_cast<f32x4 *>(to));
    else
        *reinterpret_cast<Vec<float, V> *>(to) = *reinterpret_cast<const Vec<float, V> *>(from);
}

// Workgroup (row, `par` of the heads).  A unit is V pairs (a thread reads V
// elements from either half, or 2 V in a row) or V copied elements; U units make
// a head, and a thread has one unit of one head.  V = 4 where rows are 16-byte
// aligned, 1 where not.  STREAM: y is written past the caches.  Bound by memory:
// 6,000 rows of 40 heads 43 us, 5.6 TB/s read and written; few rows by the
// launch, 4 us.
template <typename KVT, int V, bool PAIRS, bool CACHE, bool STREAM = false>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(RopeArgs a, int U, int par) {
    const int r = blockIdx.x, pos = a.positions[r];
    if (pos < 0) return;
    const int tid = threadIdx.x;
    if (tid >= U * par) return;
    const int u = tid % U, rot_units = a.rot / (2 * V);
    const bool rotates = u < rot_units;
    // elements i0 .. i0 + V - 1 (and, of a pair unit, i1 .. i1 + V - 1) of a head
    const int i0 = !rotates ? a.rot + (u - rot_units) * V : PAIRS ? 2 * V * u : V * u;
    const int i1 = PAIRS ? i0 + V : i0 + a.rot / 2;
    float2 cs[V];
    if (rotates) {
#pragma unroll
        for (int j = 0; j < V; ++j) cs[j] = turn((double)pos * a.turns[V * u + j], a.gain, a.gain_lo);
    }
    const int slot = CACHE ? a.slots[r] : -1;
    const bool write = CACHE && (unsigned)slot < (unsigned)a.n_slots;
    const int heads = write ? a.heads + 2 * a.kv_heads : a.heads;
    const float *row = a.x + (size_t)r * a.x_stride;
    const int h = blockIdx.y * par + tid / U;
    if (h >= heads) return;
    const bool q = h < a.heads, k = h < a.heads + a.kv_heads;
    if (q && !rotates && !a.copy) return;
    const float *src = row + (size_t)h * a.hd;
    Vec<float, 2 * V> x;
    read_once<V>(x.v, src + i0);
    if (rotates) {
        read_once<V>(x.v + V, src + i1);
        if (k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float &xa = x.v[PAIRS ? 2 * j : j], &xb = x.v[PAIRS ? 2 * j + 1 : V + j];
                const float ya = __builtin_fmaf(xa, cs[j].x, -(xb * cs[j].y));
                xb = __builtin_fmaf(xb, cs[j].x, xa * cs[j].y);
                xa = ya;
            }
        }
    }
    if (q) {
        float *dst = a.y + (size_t)r * a.y_stride + (size_t)h * a.hd;
        put_unit<V, STREAM>(dst + i0, x.v);
        if (rotates) put_unit<V, STREAM>(dst + i1, x.v + V);
    } else if constexpr (CACHE) {
        const int g = h - a.heads - (k ? 0 : a.kv_heads);
        KVT *dst = static_cast<KVT *>(k ? a.kc : a.vc) +
                   ((size_t)slot * a.kv_heads + g) * a.hd;
        Vec<KVT, 2 * V> o;
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) o.v[j] = (KVT)x.v[j];  // f16: to nearest even
        using O = Vec<KVT, V>;
        *reinterpret_cast<O *>(dst + i0) = *reinterpret_cast<O *>(o.v);
        if (rotates) *reinterpret_cast<O *>(dst + i1) = *reinterpret_cast<O *>(o.v + V);
    }
}

template <typename KVT, bool CACHE>
int launch_rope(cw_ctx *ctx, const char *label, const RopeArgs &a, bool wide, bool stream = false) {
    const int V = wide ? 4 : 1;
    const bool tail = a.copy || (CACHE && a.hd > a.rot);
    const int U = a.rot / (2 * V) + (tail ? (a.hd - a.rot) / V : 0);
    const int par = kThreads / U;  // U <= 256: head_dim is at most that
    const int heads = a.heads + (CACHE ? 2 * a.kv_heads : 0);
    const dim3 grid(a.rows, (heads + par - 1) / par);
    auto fn = wide ? (a.pairs ? rope_rows_kernel<KVT, 4, true, CACHE>
                              : rope_rows_kernel<KVT, 4, false, CACHE>)
                   : (a.pairs ? rope_rows_kernel<KVT, 1, true, CACHE>
                              : rope_rows_kernel<KVT, 1, false, CACHE>);
    if constexpr (!CACHE)
        if (wide && stream)
            fn = a.pairs ? rope_rows_kernel<KVT, 4, true, false, true>
                         : rope_rows_kernel<KVT, 4, false, false, true>;
    return launch(ctx, label, fn, grid, dim3(kThreads), 0, a, U, par);
}

// ---------------------------------------------------------------- normalised heads
//
// y = rotation of x / sqrt(sum(x^2) / hd + eps) * gain for each head: the norm's
// factor is the head's, so a head's G lanes (a power of two, one for every eight
// elements) hold it whole, add its squares up among themselves and rotate what
// they hold.  A lane has four pairs (4 elements of either half, or 8 in a row), or
// 8 elements behind rot, of one head; every head of a row makes the row's angles anew.
//
// What bounds it: memory, each value read and written once, and the vector units beside
// it.  6,000 rows of 24 heads of 128 (147 MB) take 26 to 30 us, 4.9 to 5.6 TB/s, with
// the vector units busy throughout (angles in f64, norm, rotation); 4,100 rows of 32 + 2 x
// 8 with the write into an f16 cache 34 us (185 MB, 5.4 TB/s), into an f32 one 37 to 39
// (202 MB, 5.2 to 5.5 TB/s); 32 to 48 rows one launch, 3.7 us.

struct NormArgs {
    const float *q_gain, *k_gain;  // [hd]
    float eps;
    int q_heads;  // heads under q_gain; those behind them are keys
};

// Whether a sum of squares whose mean (with eps) this is has lost nothing to f32's ends:
// heads of values past 2^60, or far below 1 without an eps to speak of, go through f64.
__device__ __forceinline__ bool in_range(float mean) { return mean >= 0x1p-100f && mean <= 0x1p120f; }

// y and the cache rows of head h: 8 elements, 4 from i0 on and 4 from i1
template <typename KVT, bool CACHE, bool WIDE, bool STREAM>
__device__ __forceinline__ void put_head(const RopeArgs &a, int r, int slot, int h, int i0, int i1,
                                         const float *x) {
    if (h < a.heads) {
        float *dst = a.y + (size_t)r * a.y_stride + (size_t)h * a.hd;
        if constexpr (WIDE) {
            put_unit<4, STREAM>(dst + i0, x);
            put_unit<4, STREAM>(dst + i1, x + 4);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                dst[i0 + j] = x[j];
                dst[i1 + j] = x[4 + j];
            }
        }
    } else if constexpr (CACHE) {
        const bool k = h < a.heads + a.kv_heads;
        const int g = h - a.heads - (k ? 0 : a.kv_heads);
        KVT *dst = static_cast<KVT *>(k ? a.kc : a.vc) + ((size_t)slot * a.kv_heads + g) * a.hd;
        Vec<KVT, 8> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = (KVT)x[j];  // f16: to nearest even
        using O = Vec<KVT, 4>;
        *reinterpret_cast<O *>(dst + i0) = *reinterpret_cast<O *>(o.v);
        *reinterpret_cast<O *>(dst + i1) = *reinterpret_cast<O *>(o.v + 4);
    }
}

// Workgroup (row, part of the heads).  WIDE: rows and gains are 16-byte aligned;
// STREAM as above.
template <typename KVT, bool PAIRS, bool CACHE, bool WIDE, bool STREAM = false>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(RopeArgs a, NormArgs n, int G) {
    const int r = blockIdx.x, pos = a.positions[r];
    if (pos < 0) return;
    const int tid = threadIdx.x, par = kThreads / G;
    const int u = tid & (G - 1), rot_units = a.rot / 8;
    const bool on = u < a.hd / 8, rotates = u < rot_units;
    const int i0 = !on ? 0 : !rotates || PAIRS ? 8 * u : 4 * u;
    const int i1 = rotates && !PAIRS ? i0 + a.rot / 2 : i0 + 4;
    float2 cs[4];
    if (rotates) {
#pragma unroll
        for (int j = 0; j < 4; ++j) cs[j] = turn((double)pos * a.turns[4 * u + j], a.gain, a.gain_lo);
    }
    const int slot = CACHE ? a.slots[r] : -1;
    const bool write = CACHE && (unsigned)slot < (unsigned)a.n_slots;
    const int heads = write ? a.heads + 2 * a.kv_heads : a.heads;
    const float *row = a.x + (size_t)r * a.x_stride;
    const int h = blockIdx.y * par + tid / G;
    if (h >= heads) return;
    const float *src = row + (size_t)h * a.hd;
    Vec<float, 8> x;
    if constexpr (WIDE) {
        read_once<4>(x.v, src + i0);
        read_once<4>(x.v + 4, src + i1);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.v[j] = src[i0 + j];
            x.v[4 + j] = src[i1 + j];
        }
    }
    if (h < a.heads + (CACHE ? a.kv_heads : 0)) {  // (values stay as they are)
        const float *gain = h < n.q_heads ? n.q_gain : n.k_gain;
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(x.v[j], x.v[j], ss);
        if (!on) ss = 0.0f;
        for (int d = 1; d < G; d <<= 1) ss += __shfl_xor(ss, d);
        const float mean = ss / (float)a.hd + n.eps;
        if (in_range(mean)) {
            const float inv = 1.0f / sqrtf(mean);
#pragma unroll
            for (int j = 0; j < 8; ++j) x.v[j] *= inv;
        } else {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fma((double)x.v[j], (double)x.v[j], sum);
            if (!on) sum = 0.0;
            for (int d = 1; d < G; d <<= 1) sum += __shfl_xor(sum, d);
            const double inv = 1.0 / sqrt(sum / a.hd + n.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) x.v[j] = (float)(x.v[j] * inv);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.v[j] *= gain[i0 + j];
            x.v[4 + j] *= gain[i1 + j];
        }
        if (rotates) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float &xa = x.v[PAIRS ? 2 * j : j], &xb = x.v[PAIRS ? 2 * j + 1 : 4 + j];
                const float ya = __builtin_fmaf(xa, cs[j].x, -(xb * cs[j].y));
                xb = __builtin_fmaf(xb, cs[j].x, xa * cs[j].y);
                xa = ya;
            }
        }
    }
    if (on) put_head<KVT, CACHE, WIDE, STREAM>(a, r, slot, h, i0, i1, x.v);
}

// Heads or rotated parts that are no whole eighths: a wave a head, an element or a
// pair a lane.
template <typename KVT, bool CACHE>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_any_kernel(RopeArgs a, NormArgs n) {
    const int r = blockIdx.x, pos = a.positions[r], lane = threadIdx.x & 63;
    if (pos < 0) return;
    const int slot = CACHE ? a.slots[r] : -1;
    const bool write = CACHE && (unsigned)slot < (unsigned)a.n_slots;
    const int h = blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6);
    if (h >= (write ? a.heads + 2 * a.kv_heads : a.heads)) return;
    const float *src = a.x + (size_t)r * a.x_stride + (size_t)h * a.hd;
    const bool normed = h < a.heads + (CACHE ? a.kv_heads : 0);
    const float *gain = h < n.q_heads ? n.q_gain : n.k_gain;
    float ss = 0.0f;
    for (int i = lane; i < a.hd; i += 64) ss = __builtin_fmaf(src[i], src[i], ss);
    for (int d = 1; d < 64; d <<= 1) ss += __shfl_xor(ss, d);
    const float mean = ss / (float)a.hd + n.eps;
    const bool fine = in_range(mean);
    const float inv = 1.0f / sqrtf(mean);
    double inv64 = 0.0;
    if (!fine) {
        double sum = 0.0;
        for (int i = lane; i < a.hd; i += 64) sum = fma((double)src[i], (double)src[i], sum);
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        inv64 = 1.0 / sqrt(sum / a.hd + n.eps);
    }
    auto get = [&](int i) {
        return !normed ? src[i] : (fine ? src[i] * inv : (float)(src[i] * inv64)) * gain[i];
    };
    auto put = [&](int i, float v) {
        if (h < a.heads) {
            a.y[(size_t)r * a.y_stride + (size_t)h * a.hd + i] = v;
        } else if constexpr (CACHE) {
            const bool k = h < a.heads + a.kv_heads;
            const int g = h - a.heads - (k ? 0 : a.kv_heads);
            static_cast<KVT *>(k ? a.kc : a.vc)[((size_t)slot * a.kv_heads + g) * a.hd + i] = (KVT)v;
        }
    };
    const int rot = normed ? a.rot : 0;
    for (int p = lane; p < rot / 2; p += 64) {
        const float2 cs = turn((double)pos * a.turns[p], a.gain, a.gain_lo);
        const int ia = a.pairs ? 2 * p : p, ib = a.pairs ? ia + 1 : p + rot / 2;
        const float xa = get(ia), xb = get(ib);
        put(ia, __builtin_fmaf(xa, cs.x, -(xb * cs.y)));
        put(ib, __builtin_fmaf(xb, cs.x, xa * cs.y));
    }
    for (int i = rot + lane; i < a.hd; i += 64) put(i, get(i));
}

template <typename KVT, bool CACHE>
int launch_qk_norm(cw_ctx *ctx, const char *label, const RopeArgs &a, const NormArgs &n, bool wide,
                   bool stream = false) {
    const int heads = a.heads + (CACHE ? 2 * a.kv_heads : 0);
    if (a.hd % 8 || a.rot % 8) {
        constexpr int kHeads = kThreads / 64;
        return launch(ctx, label, qk_norm_rope_any_kernel<KVT, CACHE>,
                      dim3(a.rows, (heads + kHeads - 1) / kHeads), dim3(kThreads), 0, a, n);
    }
    int G = 1;
    while (G < a.hd / 8) G <<= 1;
    const int par = kThreads / G;
    auto fn = wide ? (a.pairs ? qk_norm_rope_kernel<KVT, true, CACHE, true>
                              : qk_norm_rope_kernel<KVT, false, CACHE, true>)
                   : (a.pairs ? qk_norm_rope_kernel<KVT, true, CACHE, false>
                              : qk_norm_rope_kernel<KVT, false, CACHE, false>);
    if constexpr (!CACHE)
        if (wide && stream)
            fn = a.pairs ? qk_norm_rope_kernel<KVT, true, false, true, true>
                         : qk_norm_rope_kernel<KVT, false, false, true, true>;
    return launch(ctx, label, fn, dim3(a.rows, (heads + par - 1) / par), dim3(kThreads), 0, a, n, G);
}

// ---------------------------------------------------------------- block tables

constexpr int kScan = 1024;     // threads of the one workgroup that sums lengths
constexpr int kLdsSeqs = 4095;  // requests whose offsets are searched in LDS

// Where each request's rows, new blocks and returned blocks begin; [n_seq + 1] each.
struct Offsets {
    int *first, *need, *give;
};

struct TableArgs {
    const int *cached, *fresh, *held, *n_free;
    int n_seq, rows, page, shift, n_blocks, max_blocks;
    const uint32_t *mask;
    int mask_words;
    int *tables, *held_out, *free_list, *n_free_out, *first_row, *positions, *slots, *status;
    Offsets off;
};

// The last b with first[b] <= i
__device__ __forceinline__ int owner(const int *first, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (first[m] <= i) lo = m;
        else hi = m;
    }
    return lo;
}

// Positions and slots of rows item, item + step, ...; table entries of new
// blocks likewise.  top: free blocks once the returned ones are back.
__device__ void fill_tables(const TableArgs &a, const int *first, const int *need, int item, int step,
                            int live, int top) {
    const int n = a.n_seq, R = first[n], D = need[n];
    for (int i = item; live && i < D; i += step) {
        const int b = owner(need, n, i), k = i - need[b];
        const int had = a.held_out[b] - (need[b + 1] - need[b]);
        a.tables[(size_t)b * a.max_blocks + had + k] = a.free_list[top - 1 - i];
    }
    for (int r = item; r < a.rows; r += step) {
        int pos = -1, slot = -1;
        if (live && r < R) {
            const int b = owner(first, n, r), i = r - first[b], c = a.cached[b];
            const int e = (c + i) >> a.shift;
            const int had = a.held_out[b] - (need[b + 1] - need[b]);
            const int id = e < had ? a.tables[(size_t)b * a.max_blocks + e]
                                   : a.free_list[top - 1 - (need[b] + e - had)];
            if ((unsigned)id < (unsigned)a.n_blocks)
                slot = (id << a.shift) + ((c + i) & (a.page - 1));
            int depth = i;
            if (a.mask) {  // the bits of the request's own nodes
                const int nodes = first[b + 1] - first[b];
                depth = -1;
                for (int w = 0; w < a.mask_words && 32 * w < nodes; ++w) {
                    const uint32_t own = nodes - 32 * w >= 32 ? ~0u : (1u << (nodes - 32 * w)) - 1;
                    depth += __popc(a.mask[(size_t)r * a.mask_words + w] & own);
                }
                depth = max(depth, 0);
            }
            pos = c + depth;
        }
        a.positions[r] = pos;
        a.slots[r] = slot;
    }
}

// One workgroup: thread t sums the lengths of a run of requests, a scan over
// the threads gives each its offsets, and a second walk writes them; then the
// returned blocks.  FILL: the rows and tables too, offsets in LDS (few of
// either; at most kLdsSeqs requests).  Bound by its chain of loads: lengths,
// then table and free list: 48 requests of a row each 5.0 us.
template <bool FILL>
__global__ __launch_bounds__(kScan) void block_scan_kernel(TableArgs a) {
    __shared__ long long part[3][kScan / 64];
    __shared__ int flags, bad;
    __shared__ int s_first[FILL ? kLdsSeqs + 1 : 1], s_need[FILL ? kLdsSeqs + 1 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n_seq;
    int *const first = FILL ? s_first : a.off.first, *const need_at = FILL ? s_need : a.off.need;
    if (tid == 0) flags = bad = 0;
    const int per = (n + kScan - 1) / kScan, b0 = min(n, tid * per), b1 = min(n, b0 + per);
    const int n_free = *a.n_free;
    struct Lengths {
        int rows, need, give, held;
        bool ok;
    };
    auto lengths = [&](int b) {
        const int c = a.cached[b], f = a.fresh[b], held = a.held[b];
        const long long len = f < 0 ? 0 : (long long)c + f;
        const long long blocks = (len + a.page - 1) >> a.shift;  // at most 2^28 each
        return Lengths{max(f, 0), f < 0 || blocks < held ? 0 : (int)(blocks - held), f < 0 ? held : 0,
                       held, c >= 0 && held >= 0 && held <= a.max_blocks && len <= 0x7fffffff};
    };
    Lengths mine{};  // of the first request, kept for the second walk
    long long sum[3] = {0, 0, 0};
    int over = 0, wrong = 0;
    for (int b = b0; b < b1; ++b) {
        const Lengths x = lengths(b);
        if (b == b0) mine = x;
        if (!x.ok) {
            wrong = 1;
            continue;
        }
        over |= x.held + x.need > a.max_blocks;
        sum[0] += x.rows;
        sum[1] += x.need;
        sum[2] += x.give;
    }
    __syncthreads();
    if (over) flags = CW_BLOCKS_TABLE;  // (every writer writes the same)
    if (wrong) bad = 1;
    long long inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        inc[k] = wave_scan(sum[k], lane);
        if (lane == 63) part[k][wave] = inc[k];
    }
    __syncthreads();
    long long total[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long before = 0, all = 0;
        for (int w = 0; w < kScan / 64; ++w) {
            const long long p = part[k][w];
            if (w < wave) before += p;
            all += p;
        }
        inc[k] += before - sum[k];  // what the requests before this thread's add up to
        total[k] = all;
    }
    const long long back = n_free + total[2];
    int st = flags;
    if (bad || n_free < 0 || back > a.n_blocks) {
        st = CW_BLOCKS_BAD;
    } else {
        if (total[0] > a.rows) st |= CW_BLOCKS_ROWS;
        if (total[1] > back) st |= CW_BLOCKS_FREE;
    }
    const int live = st == 0, top = (int)back;
    const bool gives = live && total[2] > 0;
    for (int b = b0; b < b1; ++b) {
        const Lengths x = b == b0 ? mine : lengths(b);
        first[b] = a.first_row[b] = live ? (int)inc[0] : 0;
        need_at[b] = live ? (int)inc[1] : 0;
        if (gives) a.off.give[b] = (int)inc[2];
        a.held_out[b] = live ? x.held + x.need - x.give : x.held;
        inc[0] += x.rows;
        inc[1] += x.need;
        inc[2] += x.give;
    }
    if (tid == 0) {
        first[n] = a.first_row[n] = live ? (int)total[0] : 0;
        need_at[n] = live ? (int)total[1] : 0;
        if (gives) a.off.give[n] = (int)total[2];
        a.n_free_out[0] = live ? top - (int)total[1] : n_free;
        a.status[0] = st;
    }
    __syncthreads();
    if (gives) {  // returned blocks
        for (int j = tid; j < (int)total[2]; j += kScan) {
            const int b = owner(a.off.give, n, j);
            a.free_list[n_free + j] = a.tables[(size_t)b * a.max_blocks + j - a.off.give[b]];
        }
        __syncthreads();
    }
    if (FILL) fill_tables(a, first, need_at, tid, kScan, live, top);
}

// Rows and table entries, over the chip, behind block_scan_kernel<false> (600
// requests of up to 400 rows: 5 us each).
__global__ __launch_bounds__(kThreads) void block_fill_kernel(TableArgs a) {
    __shared__ int s_first[kLdsSeqs + 1], s_need[kLdsSeqs + 1];
    const int n = a.n_seq, live = a.status[0] == 0;
    const int top = a.n_free_out[0] + a.off.need[n];
    const int *first = a.off.first, *need = a.off.need;
    if (n <= kLdsSeqs) {
        for (int b = threadIdx.x; b <= n; b += kThreads) {
            s_first[b] = first[b];
            s_need[b] = need[b];
        }
        __syncthreads();
        first = s_first;
        need = s_need;
    }
    fill_tables(a, first, need, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads, live, top);
}

// ---------------------------------------------------------------- accepted rows
//
// Row cached + i takes row cached + path[i], path increasing, so path[i] >= i
// and no row is read after an earlier move wrote it: a thread that moves its 16
// bytes of a row in order of i needs no copy of the rows, and has the loads of
// eight moves in flight (a load's row is never among the rows stored before it).
// Lane i of each wave looks up move i.  A launch and three dependent loads: 3.4 us
// for 48 requests of six moves.
__global__ __launch_bounds__(kThreads) void accept_kernel(PageMap m, u32x4 *k, u32x4 *v,
                                                          int row_u4, const int *cached,
                                                          const int *path, int max_path,
                                                          const int *path_len, int *cached_out) {
    constexpr int D = 8;
    const int b = blockIdx.y, lane = threadIdx.x & 63, c = cached[b];
    const int n = min(max(path_len[b], 0), max_path);
    const int u = blockIdx.x * kThreads + threadIdx.x;
    if (u == 0 && cached_out) cached_out[b] = c + n;
    if (c < 0) return;
    const bool on = u < 2 * row_u4;
    u32x4 *const base = u < row_u4 ? k + u : v + (on ? u - row_u4 : 0);
    for (int i0 = 0; i0 < n; i0 += 64) {
        int src = -1, dst = -1;
        if (i0 + lane < n) {
            const int node = path[(size_t)b * max_path + i0 + lane];
            // (no position is past 2^31 - 1)
            if (node >= 0 && node != i0 + lane && max(node, i0 + lane) <= 0x7fffffff - c) {
                src = slot_of(m, b, c + node);
                dst = slot_of(m, b, c + i0 + lane);
            }
            if (src < 0 || dst < 0) src = dst = -1;
        }
        for (int i = 0; i < min(n - i0, 64); i += D) {
            u32x4 w[D];
#pragma unroll
            for (int d = 0; d < D; ++d) {
                // (without a move: slot 0, not stored)
                w[d] = base[(size_t)max(__builtin_amdgcn_readlane(src, i + d), 0) * row_u4];
            }
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int t = __builtin_amdgcn_readlane(dst, i + d);
                if (on && t >= 0) base[(size_t)t * row_u4] = w[d];
            }
        }
    }
}

bool same_spec(const cw_rope_spec &a, const cw_rope_spec &b) {
    return a.rot_dim == b.rot_dim && a.scaling == b.scaling && a.trained == b.trained &&
           a.theta == b.theta && a.factor == b.factor && a.beta_fast == b.beta_fast &&
           a.beta_slow == b.beta_slow && a.low_turns == b.low_turns &&
           a.high_turns == b.high_turns;
}

int check_spec(const char *what, const cw_rope_spec &s, int head_dim) {
    CW_CHECK_ARG(s.rot_dim > 0 && s.rot_dim % 2 == 0 && s.rot_dim <= head_dim,
                 "%s: rot_dim=%d must be even and at most head_dim=%d", what, s.rot_dim, head_dim);
    CW_CHECK_ARG(s.layout == CW_ROPE_HALVES || s.layout == CW_ROPE_PAIRS, "%s: layout=%d", what,
                 s.layout);
    CW_CHECK_ARG(std::isfinite(s.theta) && s.theta > 1.0, "%s: theta=%g must be above 1", what,
                 s.theta);
    if (s.scaling == CW_ROPE_PLAIN) return CW_OK;
    CW_CHECK_ARG(s.scaling == CW_ROPE_LINEAR || s.scaling == CW_ROPE_YARN ||
                     s.scaling == CW_ROPE_BANDS,
                 "%s: scaling=%d", what, s.scaling);
    CW_CHECK_ARG(std::isfinite(s.factor) && s.factor >= 1.0, "%s: factor=%g must be 1 or more",
                 what, s.factor);
    if (s.scaling == CW_ROPE_LINEAR) return CW_OK;
    CW_CHECK_ARG(s.trained > 0, "%s: trained=%d must be positive", what, s.trained);
    if (s.scaling == CW_ROPE_YARN) {
        CW_CHECK_ARG(std::isfinite(s.beta_fast) && s.beta_slow > 0.0 && s.beta_fast >= s.beta_slow,
                     "%s: beta_fast=%g must be at least beta_slow=%g, both positive", what,
                     s.beta_fast, s.beta_slow);
        CW_CHECK_ARG(std::isfinite(s.gain) && s.gain >= 0.0, "%s: gain=%g", what, s.gain);
        return CW_OK;
    }
    CW_CHECK_ARG(std::isfinite(s.high_turns) && s.low_turns > 0.0 && s.high_turns > s.low_turns,
                 "%s: high_turns=%g must be above low_turns=%g, both positive", what, s.high_turns,
                 s.low_turns);
    return CW_OK;
}

// Turns per position of each pair, in f64.
void rope_turns_host(const cw_rope_spec &s, double *turns) {
    constexpr double two_pi = 6.283185307179586;
    const int half = s.rot_dim / 2;
    double lo = 0.0, hi = 1.0;
    if (s.scaling == CW_ROPE_YARN) {
        // the (fractional) pair that turns `beta` times over the trained length
        auto pair = [&](double beta) {
            return s.rot_dim * std::log(s.trained / (beta * two_pi)) / (2.0 * std::log(s.theta));
        };
        lo = std::max(std::floor(pair(s.beta_fast)), 0.0);
        hi = std::min(std::ceil(pair(s.beta_slow)), (double)(s.rot_dim - 1));
        if (hi <= lo) hi = lo + 1e-3;
    }
    for (int i = 0; i < half; ++i) {
        const double f = std::pow(s.theta, -2.0 * i / s.rot_dim);
        double keep = 1.0;  // share of the unscaled frequency
        if (s.scaling == CW_ROPE_LINEAR) keep = 0.0;
        if (s.scaling == CW_ROPE_YARN)
            keep = 1.0 - std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0);
        if (s.scaling == CW_ROPE_BANDS)
            keep = std::min(std::max((s.trained * f / two_pi - s.low_turns) /
                                         (s.high_turns - s.low_turns), 0.0), 1.0);
        turns[i] = (s.scaling == CW_ROPE_PLAIN ? f : f * keep + f / s.factor * (1.0 - keep)) / two_pi;
    }
}

// Tables of specs that no recording names: a base or factor that follows the
// context's length makes a new one every step, so the oldest one's memory is taken
// for the next.  (A recorded kernel may read its table until the context ends.)
constexpr int kRopeTurns = 64;

// The device table of a spec's turns: made on first use, kept by the context.
int ctx_rope_turns(cw_ctx *ctx, const char *what, cw_rope_spec s, const double **out) {
    s.layout = 0;
    s.gain = 0.0;
    if (s.scaling == CW_ROPE_PLAIN) s.factor = 1.0;
    if (s.scaling != CW_ROPE_YARN) s.beta_fast = s.beta_slow = 0.0;
    if (s.scaling != CW_ROPE_BANDS) s.low_turns = s.high_turns = 0.0;
    if (s.scaling == CW_ROPE_PLAIN || s.scaling == CW_ROPE_LINEAR) s.trained = 0;
    for (auto &t : ctx->rope_turns)
        if (same_spec(t.spec, s)) {
            t.recorded |= ctx->capturing;
            *out = t.turns;
            return CW_OK;
        }
    CW_TRY(refuse_while_capturing(ctx, "a table of frequencies must be built"));
    constexpr int kMost = 128;  // pairs of a head
    double host[kMost];
    rope_turns_host(s, host);
    const size_t bytes = (size_t)(s.rot_dim / 2) * sizeof(double);
    int kept = 0;
    for (const auto &t : ctx->rope_turns) kept += !t.recorded;
    void *p = nullptr;
    if (kept >= kRopeTurns) {
        const auto old = std::find_if(ctx->rope_turns.begin(), ctx->rope_turns.end(),
                                      [](const auto &t) { return !t.recorded; });
        p = old->turns;
        // (out of the list first: after an error below nothing names a half table)
        ctx->rope_turns.erase(old);
        // launches that read it are done
        hipError_t e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) {
            (void)hipFree(p);
            return hip_fail(e, "ctx_rope_turns: reusing a table of frequencies", __FILE__, __LINE__);
        }
    } else {
        CW_HIP(hipMalloc(&p, kMost * sizeof(double)));
    }
    hipError_t e = hipMemcpy(p, host, bytes, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(p);
        return hip_fail(e, "the copy of a table of frequencies", __FILE__, __LINE__);
    }
    try {
        ctx->rope_turns.push_back({s, static_cast<double *>(p), false});
    } catch (const std::bad_alloc &) {
        (void)hipFree(p);
        set_error("%s: out of host memory", what);
        return CW_ERR_OOM;
    }
    *out = static_cast<double *>(p);
    return CW_OK;
}

void spec_gain(const cw_rope_spec &s, RopeArgs *a) {
    const double g = s.scaling != CW_ROPE_YARN ? 1.0 : s.gain > 0.0 ? s.gain : 0.1 * std::log(s.factor) + 1.0;
    a->gain = (float)g;
    a->gain_lo = (float)(g - a->gain);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_norm(const char *what, const float *q_gain, int n_heads, const float *k_gain,
               int n_kv_heads, float eps) {
    CW_CHECK_ARG((q_gain || n_heads == 0) && (k_gain || n_kv_heads == 0),
                 "%s: null gain of %d query and %d key heads", what, n_heads, n_kv_heads);
    CW_CHECK_ARG(std::isfinite(eps) && eps >= 0.0f, "%s: eps=%g", what, (double)eps);
    return CW_OK;
}

// Checks of rows of [q | k | v] that go to q_out and the cache; *a but for the
// frequencies, and whether q's rows are 16-byte aligned.
int check_kv_rows(const char *what, const cw_rope_spec *spec, const cw_kv_pages *kv,
                  const float *qkv, size_t stride, const int *positions, const int *slots, int rows,
                  int n_heads, float *q_out, size_t q_stride, RopeArgs *a, bool *wide) {
    CW_CHECK_ARG(rows > 0 && rows <= kMaxRows && n_heads >= 0 && n_heads <= 4096,
                 "%s: rows=%d (at most 2^23) n_heads=%d (4096)", what, rows, n_heads);
    CW_CHECK_ARG((n_heads > 0) == (q_out != nullptr), "%s: q_out goes with n_heads=%d", what,
                 n_heads);
    PageMap map;
    CW_TRY(check_pages(what, kv, nullptr, true, &map));
    CW_TRY(check_spec(what, *spec, kv->head_dim));
    const size_t q_width = (size_t)n_heads * kv->head_dim;
    const size_t width = q_width + 2 * (size_t)kv->n_kv_heads * kv->head_dim;
    CW_CHECK_ARG(stride >= width && stride < (1u << 31), "%s: stride %zu of rows of %zu floats",
                 what, stride, width);
    CW_CHECK_ARG(!n_heads || (q_stride >= q_width && q_stride < (1u << 31)),
                 "%s: q_stride %zu of rows of %zu floats", what, q_stride, q_width);
    const bool in_place = n_heads && q_out == qkv && q_stride == stride;
    CW_CHECK_ARG(!n_heads || in_place ||
                     rows_apart(rows, qkv, stride, width, q_out, q_stride, q_width),
                 "%s: rows of qkv and q_out overlap", what);
    spec_gain(*spec, a);
    a->rot = spec->rot_dim;
    a->pairs = spec->layout == CW_ROPE_PAIRS;
    a->x = qkv;
    a->x_stride = stride;
    a->positions = positions;
    a->slots = slots;
    a->rows = rows;
    a->heads = n_heads;
    a->kv_heads = kv->n_kv_heads;
    a->hd = kv->head_dim;
    a->y = q_out;
    a->y_stride = q_stride;
    a->copy = !in_place && kv->head_dim > spec->rot_dim;
    a->kc = kv->k;
    a->vc = kv->v;
    a->n_slots = kv->page * kv->n_blocks;
    *wide = aligned16(qkv) && stride % 4 == 0 &&
            (!n_heads || (aligned16(q_out) && q_stride % 4 == 0));
    return CW_OK;
}

}  // namespace

namespace cwi {

bool rows_apart(int rows, const float *a, size_t sa, size_t wa, const float *b, size_t sb,
                size_t wb) {
    if (a > b) {
        std::swap(a, b);
        std::swap(sa, sb);
        std::swap(wa, wb);
    }
    const size_t d = (size_t)((uintptr_t)b - (uintptr_t)a);
    if (d >= ((size_t)(rows - 1) * sa + wa) * sizeof(float)) return true;
    if (sa != sb || d % sizeof(float)) return false;
    // rows of b begin at column c of a's
    const size_t c = d / sizeof(float) % sa;
    return c >= wa && c + wb <= sa;
}

int check_pages(const char *what, const cw_kv_pages *kv, const cw_batch *b, bool need_kv,
                PageMap *map) {
    CW_CHECK_ARG(kv->page > 0 && kv->n_blocks > 0, "%s: page=%d n_blocks=%d must be positive", what,
                 kv->page, kv->n_blocks);
    CW_CHECK_ARG((long long)kv->page * kv->n_blocks <= 0x7fffffffLL,
                 "%s: %d blocks of %d positions are more than 2^31 - 1 slots", what, kv->n_blocks,
                 kv->page);
    if (need_kv) {
        CW_CHECK_ARG(kv->k && kv->v, "%s: null cache", what);
        CW_CHECK_ARG(aligned16(kv->k) && aligned16(kv->v), "%s: caches must be 16-byte aligned",
                     what);
        CW_CHECK_ARG(kv->kv_dtype == CW_F32 || kv->kv_dtype == CW_F16, "%s: kv_dtype=%d", what,
                     kv->kv_dtype);
        CW_CHECK_ARG(kv->n_kv_heads > 0 && kv->n_kv_heads <= 1024, "%s: n_kv_heads=%d", what,
                     kv->n_kv_heads);
        const int hd = kv->head_dim;
        CW_CHECK_ARG(hd == 16 || hd == 32 || hd == 64 || hd == 128 || hd == 256,
                     "%s: head_dim=%d (16, 32, 64, 128 or 256)", what, hd);
    }
    *map = PageMap{nullptr, 0, kv->page, 0, kv->n_blocks};
    if (!b) return CW_OK;
    CW_CHECK_ARG(b->cached && b->n_seq > 0 && b->n_seq <= 65535,
                 "%s: n_seq=%d (1 .. 65535) with their cached counts", what, b->n_seq);
    if (!b->tables) {
        CW_CHECK_ARG(b->n_seq <= kv->n_blocks, "%s: %d requests, and %d blocks without tables",
                     what, b->n_seq, kv->n_blocks);
        return CW_OK;
    }
    CW_CHECK_ARG(b->max_blocks > 0, "%s: max_blocks=%d", what, b->max_blocks);
    CW_CHECK_ARG(kv->page >= 16 && (kv->page & (kv->page - 1)) == 0,
                 "%s: page=%d must be a power of two from 16 on", what, kv->page);
    map->tables = b->tables;
    map->max_blocks = b->max_blocks;
    map->shift = __builtin_ctz((unsigned)kv->page);
    return CW_OK;
}

}  // namespace cwi

extern "C" {

int cw_rope_rows(cw_ctx *ctx, const cw_rope_spec *spec, const float *x, size_t x_stride,
                 const int *positions, int rows, int heads, int head_dim, float *y,
                 size_t y_stride) {
    CW_CHECK_ARG(ctx && spec && x && positions && y, "cw_rope_rows: null argument");
    CW_CHECK_ARG(rows > 0 && rows <= kMaxRows && heads > 0 && heads <= 4096 && head_dim > 0 &&
                     head_dim <= 256,
                 "cw_rope_rows: rows=%d (at most 2^23) heads=%d (4096) head_dim=%d (256)", rows,
                 heads, head_dim);
    CW_TRY(check_spec("cw_rope_rows", *spec, head_dim));
    const size_t width = (size_t)heads * head_dim;
    CW_CHECK_ARG(x_stride >= width && y_stride >= width && x_stride < (1u << 31) &&
                     y_stride < (1u << 31),
                 "cw_rope_rows: strides %zu and %zu of rows of %zu floats", x_stride, y_stride,
                 width);
    const bool in_place = x == y && x_stride == y_stride;
    CW_CHECK_ARG(in_place || rows_apart(rows, x, x_stride, width, y, y_stride, width),
                 "cw_rope_rows: rows of x and y overlap");
    CW_HIP(hipSetDevice(ctx->device));
    RopeArgs a{};
    CW_TRY(ctx_rope_turns(ctx, "cw_rope_rows", *spec, &a.turns));
    spec_gain(*spec, &a);
    a.rot = spec->rot_dim;
    a.pairs = spec->layout == CW_ROPE_PAIRS;
    a.x = x;
    a.x_stride = x_stride;
    a.positions = positions;
    a.rows = rows;
    a.heads = heads;
    a.hd = head_dim;
    a.y = y;
    a.y_stride = y_stride;
    a.copy = !in_place && head_dim > spec->rot_dim;
    const bool wide = aligned16(x) && aligned16(y) && x_stride % 4 == 0 && y_stride % 4 == 0 &&
                      head_dim % 4 == 0 && a.rot % 8 == 0;
    // Past 32 MB (the eight L2s) whoever reads y next finds it in none of them;
    // written past them 6,000 rows of 40 heads take 43.2 us, else 49.2.  With the
    // cache write below, whose rows end in two places, it gains nothing (32.4
    // against 35.2 us for 4,100 rows).
    const bool stream = (size_t)rows * width * sizeof(float) > (size_t)32 << 20;
    return launch_rope<float, false>(ctx, "rope_rows", a, wide, stream);
}

int cw_rope_kv_rows(cw_ctx *ctx, const cw_rope_spec *spec, const cw_kv_pages *kv,
                    const float *qkv, size_t stride, const int *positions, const int *slots,
                    int rows, int n_heads, float *q_out, size_t q_stride) {
    CW_CHECK_ARG(ctx && spec && kv && qkv && positions && slots, "cw_rope_kv_rows: null argument");
    RopeArgs a{};
    bool wide = false;
    CW_TRY(check_kv_rows("cw_rope_kv_rows", spec, kv, qkv, stride, positions, slots, rows, n_heads,
                         q_out, q_stride, &a, &wide));
    CW_HIP(hipSetDevice(ctx->device));
    CW_TRY(ctx_rope_turns(ctx, "cw_rope_kv_rows", *spec, &a.turns));
    wide = wide && a.rot % 8 == 0;
    if (kv->kv_dtype == CW_F16) return launch_rope<_Float16, true>(ctx, "rope_kv_rows", a, wide);
    return launch_rope<float, true>(ctx, "rope_kv_rows", a, wide);
}

int cw_qk_norm_rope_rows(cw_ctx *ctx, const cw_rope_spec *spec, const float *x, size_t x_stride,
                         const float *q_gain, const float *k_gain, float eps, const int *positions,
                         int rows, int n_heads, int n_kv_heads, int head_dim, float *y,
                         size_t y_stride) {
    CW_CHECK_ARG(ctx && spec && x && positions && y, "cw_qk_norm_rope_rows: null argument");
    CW_CHECK_ARG(rows > 0 && rows <= kMaxRows && n_heads >= 0 && n_heads <= 4096 &&
                     n_kv_heads >= 0 && n_kv_heads <= 4096 && n_heads + n_kv_heads > 0 &&
                     head_dim > 0 && head_dim <= 256,
                 "cw_qk_norm_rope_rows: rows=%d (at most 2^23) n_heads=%d n_kv_heads=%d (4096) "
                 "head_dim=%d (256)",
                 rows, n_heads, n_kv_heads, head_dim);
    CW_TRY(check_norm("cw_qk_norm_rope_rows", q_gain, n_heads, k_gain, n_kv_heads, eps));
    CW_TRY(check_spec("cw_qk_norm_rope_rows", *spec, head_dim));
    const size_t width = (size_t)(n_heads + n_kv_heads) * head_dim;
    CW_CHECK_ARG(x_stride >= width && y_stride >= width && x_stride < (1u << 31) &&
                     y_stride < (1u << 31),
                 "cw_qk_norm_rope_rows: strides %zu and %zu of rows of %zu floats", x_stride,
                 y_stride, width);
    const bool in_place = x == y && x_stride == y_stride;
    CW_CHECK_ARG(in_place || rows_apart(rows, x, x_stride, width, y, y_stride, width),
                 "cw_qk_norm_rope_rows: rows of x and y overlap");
    CW_HIP(hipSetDevice(ctx->device));
    RopeArgs a{};
    CW_TRY(ctx_rope_turns(ctx, "cw_qk_norm_rope_rows", *spec, &a.turns));
    spec_gain(*spec, &a);
    a.rot = spec->rot_dim;
    a.pairs = spec->layout == CW_ROPE_PAIRS;
    a.x = x;
    a.x_stride = x_stride;
    a.positions = positions;
    a.rows = rows;
    a.heads = n_heads + n_kv_heads;
    a.hd = head_dim;
    a.y = y;
    a.y_stride = y_stride;
    const bool wide = aligned16(x) && aligned16(y) && x_stride % 4 == 0 && y_stride % 4 == 0 &&
                      aligned16(q_gain) && aligned16(k_gain);
    // as in cw_rope_rows
    const bool stream = (size_t)rows * width * sizeof(float) > (size_t)32 << 20;
    return launch_qk_norm<float, false>(ctx, "qk_norm_rope_rows", a,
                                        NormArgs{q_gain, k_gain, eps, n_heads}, wide, stream);
}

int cw_qk_norm_rope_kv_rows(cw_ctx *ctx, const cw_rope_spec *spec, const cw_kv_pages *kv,
                            const float *qkv, size_t stride, const float *q_gain,
                            const float *k_gain, float eps, const int *positions,
                            const int *slots, int rows, int n_heads, float *q_out,
                            size_t q_stride) {
    CW_CHECK_ARG(ctx && spec && kv && qkv && positions && slots,
                 "cw_qk_norm_rope_kv_rows: null argument");
    RopeArgs a{};
    bool wide = false;
    CW_TRY(check_kv_rows("cw_qk_norm_rope_kv_rows", spec, kv, qkv, stride, positions, slots, rows,
                         n_heads, q_out, q_stride, &a, &wide));
    CW_TRY(check_norm("cw_qk_norm_rope_kv_rows", q_gain, n_heads, k_gain, kv->n_kv_heads, eps));
    CW_HIP(hipSetDevice(ctx->device));
    CW_TRY(ctx_rope_turns(ctx, "cw_qk_norm_rope_kv_rows", *spec, &a.turns));
    wide = wide && aligned16(q_gain) && aligned16(k_gain);
    const NormArgs n{q_gain, k_gain, eps, n_heads};
    if (kv->kv_dtype == CW_F16)
        return launch_qk_norm<_Float16, true>(ctx, "qk_norm_rope_kv_rows", a, n, wide);
    return launch_qk_norm<float, true>(ctx, "qk_norm_rope_kv_rows", a, n, wide);
}

int cw_block_tables(cw_ctx *ctx, const cw_kv_pages *kv, const cw_batch *b, const int *fresh,
                    const int *held, int *held_out, int *free_list, const int *n_free,
                    int *n_free_out, int *positions, int *slots, int *status) {
    CW_CHECK_ARG(ctx && kv && b && fresh && held && held_out && free_list && n_free &&
                     n_free_out && positions && slots && status,
                 "cw_block_tables: null argument");
    CW_CHECK_ARG(b->tables && b->first_row, "cw_block_tables: tables and first_row are needed");
    PageMap map;
    CW_TRY(check_pages("cw_block_tables", kv, b, false, &map));
    CW_CHECK_ARG(b->rows > 0 && b->rows <= kMaxRows, "cw_block_tables: rows=%d (1 .. 2^23)", b->rows);
    CW_CHECK_ARG(!b->mask || b->mask_words > 0, "cw_block_tables: mask_words=%d", b->mask_words);
    CW_HIP(hipSetDevice(ctx->device));
    const size_t n = (size_t)b->n_seq + 1;
    void *scratch = nullptr;
    CW_TRY(ctx_scratch(ctx, 3 * n * sizeof(int), &scratch));
    int *const s = static_cast<int *>(scratch);
    TableArgs a{b->cached, fresh, held, n_free, b->n_seq, b->rows, kv->page, map.shift,
                kv->n_blocks, b->max_blocks, b->mask, b->mask_words, b->tables, held_out,
                free_list, n_free_out, b->first_row, positions, slots, status,
                Offsets{s, s + n, s + 2 * n}};
    if (b->rows <= 2 * kScan && b->n_seq <= kLdsSeqs)
        return launch(ctx, "block_tables", block_scan_kernel<true>, dim3(1), dim3(kScan), 0, a);
    CW_TRY(launch(ctx, "block_tables", block_scan_kernel<false>, dim3(1), dim3(kScan), 0, a));
    const int blocks = std::min((b->rows + kThreads - 1) / kThreads, 4 * ctx->n_cu);
    return launch(ctx, "block_tables", block_fill_kernel, dim3(blocks), dim3(kThreads), 0, a);
}

int cw_kv_accept(cw_ctx *ctx, const cw_kv_pages *kv, const cw_batch *b, const int *path,
                 int max_path, const int *path_len, int *cached_out) {
    CW_CHECK_ARG(ctx && kv && b && path && path_len, "cw_kv_accept: null argument");
    CW_CHECK_ARG(max_path > 0 && max_path <= 1 << 30,
                 "cw_kv_accept: max_path=%d must be positive and at most 2^30", max_path);
    PageMap map;
    CW_TRY(check_pages("cw_kv_accept", kv, b, true, &map));
    CW_CHECK_ARG(cached_out != b->cached, "cw_kv_accept: cached_out is cached");
    CW_HIP(hipSetDevice(ctx->device));
    const int row_u4 = kv->n_kv_heads * kv->head_dim * (kv->kv_dtype == CW_F16 ? 2 : 4) / 16;
    const dim3 grid((2 * row_u4 + kThreads - 1) / kThreads, b->n_seq);
    return launch(ctx, "kv_accept", accept_kernel, grid, dim3(kThreads), 0, map,
                  static_cast<u32x4 *>(kv->k), static_cast<u32x4 *>(kv->v), row_u4, b->cached, path,
                  max_path, path_len, cached_out);
}

}  // extern "C"
