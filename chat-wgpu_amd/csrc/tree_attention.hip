// Attention of many rows over a paged cache of several requests: decode steps,
// pieces of prompts and trees of drafted tokens in one call.
//
// o_h = sum_p softmax_p(q_h . k_p / sqrt(hd)) v_p over the positions that a row
// sees: its request's cached ones, and of the request's own rows (nodes) those
// its mask shows.

#include <cmath>
#include <type_traits>

#include "paged_device.hpp"
#include "prompt_device.hpp"

namespace {

using namespace cwi;

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
    int wgs;      // workgroups that share the units (tree_kernel)
    float *part;  // [wgs][2][row block][hd] partial o (part_at), then
    float *ml;    // [wgs][2][row block][2] their (max log2 e, sum)
};

// Whether positions of the request lie behind its table, or its slots
__device__ __forceinline__ bool lost_length(const TreeArgs &a, const SeqRows &s) {
    const int last = s.cached + s.n - 1;
    return a.map.tables ? (last >> a.map.shift) >= a.map.max_blocks : last >= a.map.page;
}

// Whether node i of a request sees its node j (row: the node's row of the mask)
__device__ __forceinline__ bool sees(const TreeArgs &a, int row, int i, int j) {
    if (!a.mask) return j <= i;
    return (j >> 5) < a.mask_words &&
           (a.mask[(size_t)row * a.mask_words + (j >> 5)] >> (j & 31) & 1);
}

// Bit k: node i of a request of n nodes sees node j + k; nodes below 0 (cached
// positions) are seen.  j is the same for all lanes.  Three words of the mask,
// requested together.
__device__ __forceinline__ uint64_t sees64(const TreeArgs &a, int row, int i, int n, int j) {
    auto low = [](int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; };
    uint64_t m;
    if (a.mask) {
        const uint32_t *words = a.mask + (size_t)row * a.mask_words;
        const int w = j >> 5, s = j & 31;
        uint32_t x[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) x[k] = words[min(max(w + k, 0), a.mask_words - 1)];
#pragma unroll
        for (int k = 0; k < 3; ++k) x[k] = w + k < 0 ? ~0u : w + k < a.mask_words ? x[k] : 0u;
        m = ((uint64_t)x[1] << 32 | x[0]) >> s | ((uint64_t)x[2] << 32) << (32 - s);
    } else {
        m = low(i - j + 1);
    }
    return m & low(n - j);
}

// Over f32 the weights carry 2^-bits, the bits of the request's length: the sum of
// all its weights times V is then no larger than the largest V, so any V that f32
// holds has its mean.  (Sums of f16 V cannot get past f32.)  The factor is the same
// for every segment of a request and cancels in o / sum.  It costs V below 2^bits
// times f32's smallest normal value the bits that subnormal sums lack: at 3,000
// positions none of 1e-35, 5e-6 of 1e-37.
template <typename KVT>
__device__ __forceinline__ float unit_of(const SeqRows &s) {
    return sizeof(KVT) == 4 ? ldexpf(1.0f, __builtin_clz((unsigned)(s.cached + s.n)) - 32) : 1.0f;
}

// head_dim 16, for which the tiles below (K fragments and o of 32 elements and
// more) are not laid out: one (row, head) a workgroup, 16 lanes a position, four positions at once; the groups' (max, sum, o)
// meet in LDS.  Bound by the loads' latency and the caches, which have K and V for
// every head of a row again.
template <typename KVT, int THREADS>
__global__ __launch_bounds__(THREADS) void tree_row_kernel(TreeArgs a) {
    constexpr int HD = 16, G = THREADS / HD, U = 4;
    __shared__ float so[G][HD], sm[G], sl[G];
    const int r = blockIdx.x, h = blockIdx.y, g = h / (a.n_heads / a.n_kv);
    const int e = threadIdx.x % HD, mine = threadIdx.x / HD;
    // the request whose rows hold r
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (a.first_row[m] <= r) lo = m;
        else hi = m;
    }
    SeqRows s = seq_rows(a.first_row, a.cached, a.rows, lo);
    auto has = [&](const SeqRows &t) { return r >= t.r0 && r < t.r0 + t.n; };
    // a row range that is out of order leads the search astray: look at all
    for (int c = 0; !has(s) && c < a.n_seq; c += 64) {
        const int b = min(c + (int)(threadIdx.x & 63), a.n_seq - 1);
        const unsigned long long hit = __ballot(has(seq_rows(a.first_row, a.cached, a.rows, b)));
        if (hit) {
            lo = c + __ffsll((long long)hit) - 1;
            s = seq_rows(a.first_row, a.cached, a.rows, lo);
        }
    }
    if (!has(s)) return;
    const int i = r - s.r0;
    const float q = a.q[(size_t)r * a.q_stride + (size_t)h * HD + e], unit = unit_of<KVT>(s);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    bool lost = lost_length(a, s);  // or a position without a block
    const int end = lost ? 0 : s.cached + s.n;
    const KVT *kc = static_cast<const KVT *>(a.kc), *vc = static_cast<const KVT *>(a.vc);
    for (int p0 = mine; p0 < end; p0 += G * U) {
        float k[U], v[U], d[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + u * G, slot = p < end ? slot_of(a.map, lo, p) : 0;
            lost |= slot < 0;
            on[u] = p < end && slot >= 0 && (p < s.cached || sees(a, r, i, p - s.cached));
            const size_t at = ((size_t)max(slot, 0) * a.n_kv + g) * HD + e;
            k[u] = on[u] ? (float)kc[at] : 0.0f;
            v[u] = on[u] ? (float)vc[at] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            d[u] = q * k[u];
#pragma unroll
            for (int off = HD / 2; off >= 1; off >>= 1) d[u] += __shfl_xor(d[u], off);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            const float x = d[u] * a.scale;
            const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(x - ref) * unit;
            m = mn;
            l = __builtin_fmaf(l, f, w);
            o = __builtin_fmaf(o, f, w * v[u]);
        }
    }
    so[mine][e] = o;
    if (e == 0) sm[mine] = m, sl[mine] = lost ? NAN : l;
    __syncthreads();
    if (mine > 0) return;
    float M = -INFINITY, L = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < G; ++w) M = fmaxf(M, sm[w]);
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < G; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w] - ref);
        L += sl[w] * f;
        y += so[w][e] * f;
    }
    a.out[(size_t)r * a.out_stride + (size_t)h * HD + e] = L == 0.0f ? 0.0f : y / L;
}

// ---------------------------------------------------------------- tiles on the matrix cores

// v_mfma layouts (lane l: li = l % 16, lg = l / 16): 16x16x32 f16 holds
// A[li][8 lg + j], B[8 lg + j][li]; 16x16x16 f16 A[li][4 lg + j], B[4 lg + j][li];
// 16x16x4 f32 A[li][lg], B[lg][li]; all D[4 lg + r][li].

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ SeqRows uniform(SeqRows s) {
    return SeqRows{uniform(s.r0), uniform(s.n), uniform(s.cached)};
}

template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
    __builtin_amdgcn_sched_barrier(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// LDS operations of this wave are done
__device__ __forceinline__ void wait_lds() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// Workgroup barrier for LDS data; loads in flight stay in flight
__device__ __forceinline__ void lds_barrier() {
    wait_lds();
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Over the lanes li, li + 16, li + 32, li + 48: a row of the transposed products.
// (Elements of a vector are copied before a bit cast: of the element itself it
// would take the vector's first.)
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
    const uint32_t v0 = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(v0, v0, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    const uint32_t v1 = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b = __builtin_amdgcn_permlane32_swap(v1, v1, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    v = f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
    // keeps the swaps here: moved into a branch that fewer lanes take they
    // would swap with none
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ float group_max(float v) {
    return over_groups(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float group_sum(float v) {
    return over_groups(v, [](float x, float y) { return x + y; });
}

// v = hi + lo, N values in f16 (22 bits), rounded to nearest even: two values
// take two conversions and two mixed subtractions
template <int N, typename H>
__device__ __forceinline__ void split_f16(const float (&v)[N], H &hi, H &lo) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    uint32_t h[N / 2], l[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * j], v[2 * j + 1]}), f16x2));
        float a, b;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(h[j]), "v"(v[2 * j]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
            : "=v"(b) : "v"(h[j]), "v"(v[2 * j + 1]));
        l[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    }
    __builtin_memcpy(&hi, h, sizeof(hi));
    __builtin_memcpy(&lo, l, sizeof(lo));
}

// ---- who does what.  A tile is kt positions for one block of rt rows (a row: a
// node and one of its query heads) of one kv head; the tiles of a request are
// ordered (kv head, row block, position).  A row block costs kOpen tiles to begin
// (its queries, the first tile's way from memory) and the positions that its rows
// can see, of which without a mask later blocks have more; all of it is dealt to
// the workgroups in equal runs, so that requests of any lengths share the chip
// evenly, and a tile belongs to the run that its first position is in.  A run's
// piece of a row block is a segment; what no workgroup has whole is joined by
// tree_merge_kernel.  (Where every block of a prompt counts and takes the tiles of
// the last, 2,000 rows of 16 heads take 85 us instead of 58, eight prompts of 345
// over f32 55 instead of 44.)
// (kOpen 0, 2, 3, 4 and 8, us with the join: 48 single rows at 100 .. 8,000 positions
// 83, 71.2, 70.9, 71.0 and 73; 61 nodes at 4,100 30.8, 28.5, 28.1, 27.9 and 28.1;
// four pieces of 80 to 300 rows over f32 97, 91.3, 91.5, 92.1 and 96.5.  Workgroups of one CU and the XCDs are served unevenly, equal runs end
// up to 1.5 times apart; short runs fetched by whoever is free gain nothing,
// as the rest of the chip then has the memory to itself: 164 us either way for
// 64 requests of 4,000 positions.)

constexpr int kOpen = 3;

struct Work {
    int blocks;     // of rows
    int len, grow;  // block i: len + (i + 1) grow units
    int c, n, group, kt, rt;
    bool causal;
    // units before block i of a kv head; begin(blocks): of all
    __device__ __forceinline__ long long begin(int i) const {
        return (long long)((uint64_t)(uint32_t)i * (2u * len + (uint32_t)(i + 1) * grow) >> 1);
    }
    __device__ __forceinline__ int size(int i) const { return len + (i + 1) * grow; }
    __device__ __forceinline__ long long first_tile(int i) const { return begin(i) + kOpen * kt; }
    __device__ __forceinline__ int tiles(int i) const {
        const int seen = causal ? min(n, ((i + 1) * rt - 1) / group + 1) : n;
        return (c + seen + kt - 1) / kt;
    }
    // the block that unit x of a kv head is in
    __device__ __forceinline__ int block(long long x) const {
        int lo = 0, hi = blocks;
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if (begin(m) <= x) lo = m;
            else hi = m;
        }
        return lo;
    }
};
__device__ __forceinline__ Work work_of(const TreeArgs &a, const SeqRows &s, int group, int kt, int rt) {
    // without a mask block i sees at most 1 + (i + 1) rt / group nodes; a tile that is
    // begun counts whole; of a request that is lost nothing is read
    const bool lost = lost_length(a, s);
    const int blocks = (int)(((long long)s.n * group + rt - 1) / rt), c = lost ? 0 : s.cached;
    const int n = lost ? 1 : s.n;
    const bool causal = !a.mask && blocks > 1 && !lost;
    const int see = causal ? c + kt : (c + n + kt - 1) / kt * kt;
    Work w{blocks, kOpen * kt + see, causal ? (rt + group - 1) / group : 0, c, n, group, kt, rt, causal};
    // sums over 2^16 requests and 2^10 heads stay below 2^62, whatever the device
    // arrays hold
    if (w.begin(blocks) >> 36) w.blocks = 0;
    return w;
}

__device__ __forceinline__ long long from_lane(long long v, int l) {
    return (long long)(uint32_t)__builtin_amdgcn_readlane((int)v, l) |
           (long long)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32;
}

// n / d of no negative numbers, in 32 bits where they fit
__device__ __forceinline__ long long divide(long long n, long long d) {
    if ((n | d) >> 31 == 0) return (long long)((uint32_t)n / (uint32_t)d);
    return n / d;
}

// Runs of q or q + 1 tiles' units, none shorter than a tile: so a run inside a row
// block has a tile's first
struct Deal {
    long long q, units;
    int rem, kt;
    __device__ Deal(long long u, int wgs, int kt) : units(u), kt(kt) {
        const long long t = (u + kt - 1) / kt;
        q = divide(t, wgs);
        rem = (int)(t - q * wgs);
    }
    __device__ long long start(int w) const {
        const long long u = (q * w + min(w, rem)) * kt;
        return u < units ? u : units;
    }
    __device__ int owner(long long u) const {
        const long long t = u / kt, big = (q + 1) * rem;
        return t < big ? (int)divide(t, q + 1) : rem + (int)divide(t - big, q);
    }
};

// A segment, and where the next one begins
struct Seg {
    SeqRows s;
    int b, h, rb, t0, t1, nrows, last, part;  // part: its place among the partials
    bool whole, lost;                         // lost: positions that no table entry covers
    bool once;                                // the request's only row block
    bool rest;                                // its last tile is the row block's, and positions follow
};
struct Cursor {
    long long u, end, base;  // next unit, end of the run, first unit of request b
    int b;
};

// The requests' rows: a lane each of the first 64, the others from memory
struct Requests {
    SeqRows s;
    __device__ __forceinline__ SeqRows at(const TreeArgs &a, int b) const {
        if (b < 64)
            return SeqRows{__builtin_amdgcn_readlane(s.r0, b), __builtin_amdgcn_readlane(s.n, b),
                           __builtin_amdgcn_readlane(s.cached, b)};
        return uniform(seq_rows(a.first_row, a.cached, a.rows, b));
    }
};

// The workgroup's run
template <int KT, int RT>
__device__ __forceinline__ Cursor first_unit(const TreeArgs &a, int group, int lane, Requests &req) {
    auto rows = [&](int b) {
        return b < a.n_seq ? seq_rows(a.first_row, a.cached, a.rows, b) : SeqRows{0, 0, 0};
    };
    auto units = [&](const SeqRows &s) {
        const Work w = work_of(a, s, group, KT, RT);
        return a.n_kv * w.begin(w.blocks);
    };
    req.s = rows(lane);
    const long long v0 = units(req.s), inc0 = wave_scan(v0, lane);
    long long total = from_lane(inc0, 63);
    for (int c = 64; c < a.n_seq; c += 64) total += from_lane(wave_scan(units(rows(c + lane)), lane), 63);
    const Deal deal(total, a.wgs, KT);
    Cursor cur{deal.start(blockIdx.x), deal.start(blockIdx.x + 1), 0, 0};
    if (cur.u >= cur.end) return cur;
    long long v = v0, inc = inc0;
    for (int c = 0;;) {
        const unsigned long long hit = __ballot(inc > cur.u);
        if (hit) {
            const int at = __ffsll((long long)hit) - 1;
            cur.b = c + at;
            cur.base = from_lane(inc - v, at);
            return cur;
        }
        const long long before = from_lane(inc, 63);
        c += 64;
        if (c >= a.n_seq) break;
        v = units(rows(c + lane));
        inc = wave_scan(v, lane) + before;
    }
    cur.end = cur.u;  // (not reached: u is below the total)
    return cur;
}

template <int KT, int RT>
__device__ __forceinline__ bool next_segment(const TreeArgs &a, int group, const Requests &req,
                                             Cursor &cur, Seg &g) {
    while (cur.u < cur.end && cur.b < a.n_seq) {
        g.s = req.at(a, cur.b);
        const Work wk = work_of(a, g.s, group, KT, RT);
        const long long per = wk.begin(wk.blocks);  // of a kv head
        if (cur.u >= cur.base + a.n_kv * per) {
            cur.base += a.n_kv * per;
            ++cur.b;
            continue;
        }
        const long long local = cur.u - cur.base;
        g.h = uniform((int)divide(local, per));
        const long long x = local - g.h * per;
        g.rb = uniform(wk.block(x));
        // of the block's units, less than 2^31: the run's
        const int from = uniform((int)(x - wk.begin(g.rb))), left = wk.size(g.rb) - from;
        const int take = cur.end - cur.u < left ? (int)(cur.end - cur.u) : left;
        cur.u += take;
        const int tiles = wk.tiles(g.rb), open = kOpen * KT;
        g.t0 = uniform((unsigned)max(from - open + KT - 1, 0) / KT);
        g.t1 = uniform(min(tiles, (int)((unsigned)max(from + take - open + KT - 1, 0) / KT)));
        if (g.t0 >= g.t1) continue;  // no tile begins in it
        g.b = cur.b;
        g.nrows = g.s.n * group;
        g.last = g.s.cached + g.s.n - 1;
        g.once = wk.blocks == 1;
        g.whole = g.t0 == 0 && g.t1 == tiles;
        g.rest = g.t1 == tiles && tiles * KT <= g.last;
        g.part = blockIdx.x * 2 + (g.t0 > 0 ? 0 : 1);
        g.lost = lost_length(a, g.s);
        return true;
    }
    return false;
}

// The block of the 16 positions of group gi of the request (a block holds all 16),
// and their first slot; -1 where the table names no block
__device__ __forceinline__ int block16(const TreeArgs &a, const Seg &g, int gi) {
    const int p0 = min(gi, g.last >> 4) << 4;
    return a.map.tables ? a.map.tables[(size_t)g.b * a.map.max_blocks + (p0 >> a.map.shift)] : 0;
}
__device__ __forceinline__ int slot16(const TreeArgs &a, const Seg &g, int gi, int id) {
    const int p0 = min(gi, g.last >> 4) << 4;
    if (!a.map.tables) return g.b * a.map.page + p0;
    return (unsigned)id < (unsigned)a.map.n_blocks ? (id << a.map.shift) + (p0 & (a.map.page - 1)) : -1;
}

// Whether the table names no block for one of the positions behind the row block's
// last tile (which no row of it sees)
template <int KT>
__device__ __forceinline__ bool rest_lost(const TreeArgs &a, const Seg &g, int lane) {
    if (!g.rest || g.lost) return false;
    int bad = 0;
    for (int gi = g.t1 * (KT / 16) + lane; gi <= g.last >> 4; gi += 64) bad |= slot16(a, g, gi, block16(a, g, gi)) < 0;
    return __any(bad);
}

// Where elements col .. col + 3 (col % 4 = 0) of a row of a partial o lie: as the
// products leave 16 rows in a wave's lanes, so that it stores, and the join loads,
// 1 KB in a piece; for few rows (the split kernel's) one after the other
template <int HD, int RT>
__device__ __forceinline__ size_t part_at(size_t row, int col) {
    if (RT == 16) return row * HD + col;
    return (row / 16 * (HD / 16) + col / 16) * 256 + (size_t)((col / 4 % 4) * 16 + (int)(row % 16)) * 4;
}

// Where a row's elements 16 n + 4 c4 .. + 3 go: the output where the segment has
// every tile (over the row's sum l), else a partial
struct Dest {
    float *p;
    int step;  // from one n to the next
    float l;   // what they are divided by; 1 for a partial
    __device__ __forceinline__ void put(int n, f32x4 v) const {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = l == 0.0f ? 0.0f : v[e] * f;
        *reinterpret_cast<f32x4 *>(p + n * step) = v;
    }
};
template <int HD, int RT>
__device__ __forceinline__ Dest dest(const TreeArgs &a, const Seg &g, int group, int row, int c4,
                                     float m, float l) {
    if (g.whole) {
        const int rr = g.rb * RT + row, node = rr / group;
        return Dest{a.out + (size_t)(g.s.r0 + node) * a.out_stride +
                        (size_t)(g.h * group + rr - node * group) * HD + c4 * 4, 16, l};
    }
    const size_t at = (size_t)g.part * RT + row;
    if (c4 == 0) *reinterpret_cast<float2 *>(a.ml + at * 2) = make_float2(m, l);
    return Dest{a.part + part_at<HD, RT>(at, c4 * 4), 256, 1.0f};
}

// A segment whose nodes have a V that is no finite number: as 0 * V it would
// reach rows that do not see it, so the products are taken one by one, a wave a
// row, a lane HD / 64 elements.  Every block of the segment is in the cache.  (The
// weights carry 2^up, where the tiles' do, and `unit`.)
template <typename KVT, int HD, int RT>
__device__ void one_by_one(const TreeArgs &a, const Seg &g, int group, int kt, float up, float unit) {
    constexpr int E = HD < 64 ? 1 : HD / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool on = lane * E < HD;  // (all, from head_dim 64 on)
    const KVT *kc = static_cast<const KVT *>(a.kc), *vc = static_cast<const KVT *>(a.vc);
    for (int row = wave; row < RT && g.rb * RT + row < g.nrows; row += blockDim.x >> 6) {
        const int rr = g.rb * RT + row, node = rr / group;
        const size_t head = (size_t)(g.h * group + rr - node * group) * HD + lane * E;
        float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = on ? a.q[(size_t)(g.s.r0 + node) * a.q_stride + head + e] : 0.0f;
        for (int p = g.t0 * kt; p < min(g.t1 * kt, g.last + 1); ++p) {
            const int slot = slot_of(a.map, g.b, p);
            const int j = p - g.s.cached;
            if (j >= 0 && !sees(a, g.s.r0 + node, node, j)) continue;
            const size_t at = ((size_t)max(slot, 0) * a.n_kv + g.h) * HD + (on ? lane * E : 0);
            float d = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) d = __builtin_fmaf(q[e], (float)kc[at + e], d);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) d += __shfl_xor(d, off);
            d *= a.scale;
            const float mn = fmaxf(m, d), ref = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(d - ref + up) * unit;
            m = mn;
            l = __builtin_fmaf(l, f, w);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(o[e], f, w * (float)vc[at + e]);
        }
        const size_t part = (size_t)g.part * RT + row;
#pragma unroll
        for (int e = 0; e < E && on; ++e) {
            if (g.whole)
                a.out[(size_t)(g.s.r0 + node) * a.out_stride + head + e] = l == 0.0f ? 0.0f : o[e] / l;
            else
                a.part[part_at<HD, RT>(part, lane * E & ~3) + (lane * E + e) % 4] = o[e];
        }
        if (!g.whole && lane == 0) *reinterpret_cast<float2 *>(a.ml + part * 2) = make_float2(m, l);
    }
}

// Instructions other than vector and scalar arithmetic stay on their side
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x6); }

// whether one of the register's f16 pair, or its f32, is no finite number
template <bool F16>
__device__ __forceinline__ int not_finite(uint32_t w) {
    constexpr uint32_t E = F16 ? 0x7c00u : 0x7f800000u;
    return (int)((w & E) == E) | (int)(F16 && (w >> 16 & E) == E);
}

// ---- operands that both kernels read: rows of one kv head in LDS, 16-byte
// chunk c of row r at slot c ^ (r & SWZ) of its row, so that the fragment reads
// spread over the banks
template <typename KVT, int HD_>
struct Tile {
    static constexpr int HD = HD_, ES = (int)sizeof(KVT);
    static constexpr bool F16 = ES == 2;
    static constexpr int ROWB = HD * ES, CPR = ROWB / 16;
    static constexpr int SWZ = CPR < 16 ? CPR - 1 : 15;
    static constexpr int GROUPB = 16 * ROWB;  // 16 positions
    static constexpr int NU = ROWB / 64;      // DMAs of them
    static constexpr int DT = HD / 16;        // 16 x 16 tiles of o^T
    static constexpr int KS = F16 ? HD / 32 : HD / 16;  // 16-byte reads of a K fragment
    // weights carry 2^UP (it cancels in o / sum), so that small ones keep their
    // bits as f16 hi + lo: 22 bits down to 2^-18 of the largest
    static constexpr float UP = F16 ? 15.0f : 0.0f;
    typedef typename std::conditional<F16, f16x8, f32x4>::type frag;
};

// dma16 of lines that nobody reads again (non-temporal: 64 single rows at 4,000
// positions 182 -> 165 us; where a second row block reads them it costs a tenth), with
// dma16's wait state
__device__ __forceinline__ void dma16_once(const void *base, uint32_t off, unsigned char *lds_dst) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(off), "s"(base), "{m0}"(lds_off(lds_dst))
                 : "memory");
}

// 16 positions of a kv head from slot `slot` on into LDS, 1 KB a DMA; rows
// behind `rows` repeat it.  off: this lane's offsets where all 16 are there.
template <typename T>
__device__ __forceinline__ void dma_offsets(uint32_t (&off)[T::NU], uint32_t row_b, int lane) {
#pragma unroll
    for (int n = 0; n < T::NU; ++n) {
        const int r = n * (64 / T::CPR) + lane / T::CPR;
        off[n] = r * row_b + (((lane % T::CPR) ^ (r & T::SWZ)) << 4);
    }
}
template <typename T>
__device__ __forceinline__ void dma_group(const char *src, unsigned char *dst, int rows,
                                          const uint32_t (&off)[T::NU], uint32_t row_b, int lane,
                                          bool once) {
    if (rows >= 15 && once) {
#pragma unroll
        for (int n = 0; n < T::NU; ++n) dma16_once(src, off[n], dst + n * 1024);
    } else if (rows >= 15) {
#pragma unroll
        for (int n = 0; n < T::NU; ++n) dma16(src, off[n], dst + n * 1024);
    } else {
#pragma unroll
        for (int n = 0; n < T::NU; ++n) {
            const int r = n * (64 / T::CPR) + lane / T::CPR;
            dma16(src, off[n] - (uint32_t)max(r - rows, 0) * row_b, dst + n * 1024);
        }
    }
}

// q of QT tiles of 16 rows (B operands): f16 as hi + lo of q times the power of
// two that brings the row's largest to 2^14 .. 2^15, qs the scores' factor
template <typename T, int QT>
struct Query {
    f16x8 hi[T::F16 ? QT : 1][T::F16 ? T::HD / 32 : 1], lo[T::F16 ? QT : 1][T::F16 ? T::HD / 32 : 1];
    f32x4 f[T::F16 ? 1 : QT][T::F16 ? 1 : T::HD / 16];
    float qs[QT];
    int node[QT];

    f32x4 raw[T::F16 ? QT : 1][T::F16 ? T::HD / 16 : 1];

    // requests the rows; convert() once other requests are out
    __device__ __forceinline__ void load(const TreeArgs &a, const Seg &g, int group, int w_row,
                                         int li, int lg) {
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            const int rr = min(w_row + i * 16 + li, g.nrows - 1);
            node[i] = rr / group;
            const float *qr = a.q + (size_t)(g.s.r0 + node[i]) * a.q_stride +
                              (size_t)(g.h * group + rr - node[i] * group) * T::HD;
#pragma unroll
            for (int x = 0; x < T::HD / 16; ++x) {
                if constexpr (T::F16)
                    raw[i][x] = *reinterpret_cast<const f32x4 *>(qr + 32 * (x / 2) + 8 * lg + 4 * (x % 2));
                else
                    f[i][x] = *reinterpret_cast<const f32x4 *>(qr + 16 * x + 4 * lg);
            }
        }
    }
    __device__ __forceinline__ void convert(float scale) {
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            qs[i] = scale;
            if constexpr (T::F16) {
                float mx = 0.0f;
#pragma unroll
                for (int x = 0; x < T::HD / 16; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fabsf(raw[i][x][j]));
                mx = group_max(mx);
                const int e = max(__builtin_amdgcn_frexp_expf(mx), -110);  // mx in [2^(e-1), 2^e)
                const bool fin = mx > 0.0f && mx < INFINITY;
                const float up = fin ? ldexpf(1.0f, 15 - e) : 1.0f;
                qs[i] = fin ? ldexpf(scale, e - 15) : scale;
#pragma unroll
                for (int ks = 0; ks < T::HD / 32; ++ks) {
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = raw[i][2 * ks + j / 4][j % 4] * up;
                    split_f16(w, hi[i][ks], lo[i][ks]);
                }
            }
        }
    }
};

// K fragment x of the 16 rows at Ks
template <typename T>
__device__ __forceinline__ typename T::frag k_frag(const unsigned char *Ks, int x, int li, int lg) {
    return *reinterpret_cast<const typename T::frag *>(Ks + li * T::ROWB + (((4 * x + lg) ^ (li & T::SWZ)) << 4));
}

// s^T = K q^T of 16 positions, K's fragments in registers
template <typename T>
__device__ __forceinline__ f32x4 scores(const typename T::frag (&kf)[T::KS], const Query<T, 1> &q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f}, t = s;  // two chains
    if constexpr (T::F16) {
#pragma unroll
        for (int x = 0; x < T::KS; ++x) {
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[x], q.hi[0][x], s, 0, 0, 0);
            t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[x], q.lo[0][x], t, 0, 0, 0);
        }
    } else {
#pragma unroll
        for (int x = 0; x < T::KS; ++x) {
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x][0], q.f[0][x][0], s, 0, 0, 0);
            t = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x][1], q.f[0][x][1], t, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x][2], q.f[0][x][2], s, 0, 0, 0);
            t = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x][3], q.f[0][x][3], t, 0, 0, 0);
        }
    }
    return s + t;
}

// Running softmax of one row (this lane's: li) over N tiles of 16 scores, each
// with a (positive) factor, which become the weights (times 2^up and `unit`);
// returns the factor of what was summed before.
template <int N>
__device__ __forceinline__ float soften(f32x4 (&s)[N], const float (&f)[N], float up, float unit, float &m, float &l) {
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n)
        mx = fmaxf(mx, fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3])) * f[n]);
    const float mnew = fmaxf(m, group_max(mx));
    // a row that has seen nothing keeps -inf: its weights are 2^-inf = 0
    const float ref = mnew == -INFINITY ? 0.0f : mnew;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mnew;
    float ls = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], f[n], up - ref)) * unit;
            ls += s[n][r];
        }
    l = l * alpha + ls;
    return alpha;
}

// Element 4 col .. 4 col + 3 of row li of o^T, in registers as the products
// leave it: f16 tile d has elements 16 d + 4 lg + r; f32 tile 4 c + e has
// elements 64 c + 16 lg + 4 r + e (its V fragments are four elements wide)
template <typename T>
__device__ __forceinline__ f32x4 o_quad(const f32x4 (&o)[T::DT], int n) {
    if constexpr (T::F16) return o[n];
    const int c = n / 4 * 4, r = n % 4;
    return f32x4{o[c][r], o[c + 1][r], o[c + 2][r], o[c + 3][r]};
}
template <typename T>
__device__ __forceinline__ int o_col(int n, int lg) {
    return T::F16 ? 16 * n + 4 * lg : n / 4 * 64 + 16 * lg + n % 4 * 4;
}

// ---- few rows of a kv head (at most 16): a workgroup's four waves share them
// and take 16 of a tile's 64 positions each, through LDS of their own, so
// nothing waits for another wave before the end of a segment.  Bound by memory: 48
// single rows at 100 .. 8,000 positions (366 MB) 64.5 us, 5.7 TB/s.
template <typename KVT, int HD>
struct SplitCfg : Tile<KVT, HD> {
    typedef Tile<KVT, HD> T;
    static constexpr int NW = 4, KT = 64, RT = 16;
    static constexpr int STAGE = 2 * T::GROUPB;  // K and V of a wave's 16 positions
    static constexpr int LDS = 4 * 2 * STAGE;
    static constexpr int PER_CU = LDS <= 72 * 1024 ? 2 : 1;
    static_assert(4 * RT * HD * 4 <= LDS, "the waves' o must fit the stages");
    static_assert(LDS + 4096 <= 160 * 1024, "stages must fit a CU");
};

template <typename KVT, int HD>
__global__ __launch_bounds__(256, (SplitCfg<KVT, HD>::PER_CU)) void tree_split_kernel(TreeArgs a) {
    using C = SplitCfg<KVT, HD>;
    using T = Tile<KVT, HD>;
    constexpr int KT = C::KT, RT = C::RT, DT = T::DT;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
    __shared__ float w_ml[4][RT][2];
    __shared__ int w_odd[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int group = a.n_heads / a.n_kv;
    const uint32_t row_b = (uint32_t)a.n_kv * T::ROWB;
    unsigned char *const mine = lds + wave * 2 * C::STAGE;
    uint32_t off[T::NU];
    dma_offsets<T>(off, row_b, lane);
    Requests req;
    Cursor cur = first_unit<KT, RT>(a, group, lane, req);
    Seg g;
    while (next_segment<KT, RT>(a, group, req, cur, g)) {
        lds_barrier();  // the last segment's reads of LDS are done
        const char *const kc = static_cast<const char *>(a.kc) + (size_t)g.h * T::ROWB;
        const char *const vc = static_cast<const char *>(a.vc) + (size_t)g.h * T::ROWB;
        bool bad = g.lost, odd = false;
        int slots = 0, tb = g.t0;  // of this wave's positions of tile tb + lane
        auto ids = [&]() { return block16(a, g, (tb + lane) * 4 + wave); };
        auto look_up = [&](int id) {
            slots = slot16(a, g, (tb + lane) * 4 + wave, id);
            bad |= __any(slots < 0 && tb + lane < g.t1);
            slots = max(slots, 0);  // a block has 16 positions: in the cache, and the row is lost
        };
        auto load = [&](int t) {
            const size_t at = (size_t)(uint32_t)__builtin_amdgcn_readlane(slots, t - tb) * row_b;
            const int rows = g.last - (min(t * 4 + wave, g.last >> 4) << 4);
            unsigned char *const dst = mine + (t & 1) * C::STAGE;
            dma_group<T>(kc + at, dst, rows, off, row_b, lane, g.once);
            dma_group<T>(vc + at, dst + T::GROUPB, rows, off, row_b, lane, g.once);
        };
        const int t1 = g.lost ? g.t0 : g.t1;
        const int first_ids = g.t0 < t1 ? ids() : 0;  // requested before the queries
        Query<T, 1> q;
        q.load(a, g, group, g.rb * RT, li, lg);
        if (g.t0 < t1) {
            look_up(first_ids);
            load(g.t0);
        }
        q.convert(a.scale);
        const float unit = unit_of<KVT>(g.s);
        f32x4 o[DT];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int t = g.t0; t < t1; ++t) {
            if (t + 1 < t1) {
                if (t + 1 - tb == 64) {
                    tb += 64;
                    look_up(ids());
                }
                wait_lds();  // reads of the tile before, whose place this takes
                load(t + 1);
                wait_vm<2 * T::NU>();
            } else {
                wait_vm<0>();
            }
            const unsigned char *const Ks = mine + (t & 1) * C::STAGE, *const Vs = Ks + T::GROUPB;
            // every fragment is requested before the first is used
            typename T::frag kf[T::KS];
#pragma unroll
            for (int x = 0; x < T::KS; ++x) kf[x] = k_frag<T>(Ks, x, li, lg);
            f16x4 vh[T::F16 ? DT : 1];
            f32x4 vf[T::F16 ? 1 : 4][T::F16 ? 1 : HD / 64];
            if constexpr (T::F16) {
                // V^T: within 16 lanes, lane i receives element i % 4 of the 8
                // bytes at lane 4 j + i / 4's address: element 16 d + i of rows 4 lg + j
                const int row = 4 * lg + (li >> 2), c = (li & 3) >> 1;
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    vh[d] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(
                        Vs + row * T::ROWB + (((2 * d + c) ^ (row & T::SWZ)) << 4) + (li & 1) * 8)));
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) {
                        const int row = 4 * lg + r;
                        vf[r][c] = *reinterpret_cast<const f32x4 *>(
                            Vs + row * T::ROWB + (((16 * c + li) ^ (row & T::SWZ)) << 4));
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x4 s[1] = {scores<T>(kf, q)};
            const int k0 = t * KT + wave * 16;
            if (k0 + 16 > g.s.cached) {  // nodes: by the mask
                const uint64_t vis = sees64(a, g.s.r0 + q.node[0], q.node[0], g.s.n, k0 - g.s.cached) >> 4 * lg;
#pragma unroll
                for (int r = 0; r < 4; ++r) s[0][r] = vis >> r & 1 ? s[0][r] : -INFINITY;
                int x = 0;
                if constexpr (T::F16) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const uint2 w = __builtin_bit_cast(uint2, vh[d]);
                        x |= not_finite<true>(w.x) | not_finite<true>(w.y);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float w = vf[r][c][e];
                                x |= not_finite<false>(__builtin_bit_cast(uint32_t, w));
                            }
                }
                odd |= __any(x);
            }
            const float before = m, f[1] = {q.qs[0]};
            const float alpha = soften<1>(s, f, T::UP, unit, m, l);
            if (__any(m > before)) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] *= alpha;
            }
            if constexpr (T::F16) {
                const float w[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
                f16x4 ph, pl;
                split_f16(w, ph, pl);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vh[d], ph, o[d], 0, 0, 0);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vh[d], pl, o[d], 0, 0, 0);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
                        o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[r][d / 4][d % 4], s[0][r], o[d], 0, 0, 0);
            }
        }
        // join the waves
        bad |= rest_lost<KT>(a, g, lane);
        l = group_sum(l);
        if (lg == 0) {
            w_ml[wave][li][0] = m;
            w_ml[wave][li][1] = bad ? NAN : l;
        }
        if (lane == 0) w_odd[wave] = (int)odd | (int)bad << 1;
        lds_barrier();  // and every wave is done with its stages
        // (a request that has lost a block gets NaN below: its tiles may hold
        // anything, and nothing of them is an answer)
        if (uniform(w_odd[0] | w_odd[1] | w_odd[2] | w_odd[3]) == 1) {
            one_by_one<KVT, HD, RT>(a, g, group, KT, T::UP, unit);
            continue;
        }
        constexpr int OS = HD / 4 < 16 ? HD / 4 - 1 : 15;
        f32x4 *const ow = reinterpret_cast<f32x4 *>(lds);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, w_ml[w][li][0]);
        const float down = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
#pragma unroll
        for (int n = 0; n < DT; ++n) {
            f32x4 v = o_quad<T>(o, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= down;
            ow[(wave * RT + li) * (HD / 4) + ((o_col<T>(n, lg) / 4) ^ (li & OS))] = v;
        }
        lds_barrier();
        for (int x = tid; x < RT * (HD / 4); x += 256) {
            const int row = x / (HD / 4), c4 = x % (HD / 4);
            if (g.rb * RT + row >= g.nrows) continue;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, w_ml[w][row][0]);
            const float ref = M == -INFINITY ? 0.0f : M;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                L += w_ml[w][row][1] * __builtin_amdgcn_exp2f(w_ml[w][row][0] - ref);
                v += ow[(w * RT + row) * (HD / 4) + (c4 ^ (row & OS))];
            }
            dest<HD, RT>(a, g, group, row, c4, M, L).put(0, v);
        }
    }
}

// ---- more rows over an f16 cache: the four waves take 16 QT rows each, and share
// the tile's positions in LDS.  Of many rows the products bound it: 128 nodes of
// each of 8 requests at 4,000 positions, 32 heads, 147 us, 910 TFLOP/s of them; of
// few the chain of lengths, block ids, first tile and four tiles a workgroup: 61
// nodes at 4,100 positions 22 us.  (Tiles of 32 positions, two workgroups a CU with
// three tiles on their way each: 25.7 us for 61 nodes at 4,100 positions, against
// 21.6; one workgroup of eight waves, with tiles of 64 positions: 44 us for twelve
// requests of 4 to 16 nodes, against 36.)
template <int HD_, int QT>
struct TileCfg : Tile<_Float16, HD_> {
    typedef Tile<_Float16, HD_> T;
    static constexpr int NW = 4, KT = T::ROWB <= 256 ? 64 : 32, RT = 64 * QT;
    static constexpr int ST = KT / 16;
    static constexpr int TILE = KT * T::ROWB;
    static constexpr int LDS = 4 * TILE;  // two buffers of K and V
    static constexpr int PER_CU = LDS <= 72 * 1024 ? 2 : 1;
    static constexpr int GPW = KT / 32;   // groups of 16 rows that a wave loads a tile
    static_assert(LDS + 4096 <= 160 * 1024, "tiles must fit a CU");
};

template <int HD, int QT>
__global__ __launch_bounds__(256, (TileCfg<HD, QT>::PER_CU)) void tree_tile_kernel(TreeArgs a) {
    using C = TileCfg<HD, QT>;
    using T = Tile<_Float16, HD>;
    constexpr int KT = C::KT, RT = C::RT, DT = T::DT, ST = C::ST;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
    __shared__ int bad_seg, odd_seg;  // the last segment without a block, with a V that is not finite
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int group = a.n_heads / a.n_kv;
    const uint32_t row_b = (uint32_t)a.n_kv * T::ROWB;
    // a wave's groups of a tile: K and V of group `wave`, or (32 positions)
    // group wave % 2 of K or V
    const int my_group = C::GPW == 2 ? wave : wave & 1;
    uint32_t off[T::NU];
    dma_offsets<T>(off, row_b, lane);
    Requests req;
    Cursor cur = first_unit<KT, RT>(a, group, lane, req);
    if (tid == 0) bad_seg = odd_seg = 0;
    int seg = 0;
    Seg g;
    while (next_segment<KT, RT>(a, group, req, cur, g)) {
        ++seg;
        lds_barrier();  // the last segment's reads of LDS are done, bad_seg is set up
        const char *const kc = static_cast<const char *>(a.kc) + (size_t)g.h * T::ROWB;
        const char *const vc = static_cast<const char *>(a.vc) + (size_t)g.h * T::ROWB;
        int slots = 0, tb = g.t0;
        auto ids = [&]() { return block16(a, g, (tb + lane) * (KT / 16) + my_group); };
        auto look_up = [&](int id) {
            slots = slot16(a, g, (tb + lane) * (KT / 16) + my_group, id);
            if (__any(slots < 0 && tb + lane < g.t1)) bad_seg = seg;
            slots = max(slots, 0);  // a block has 16 positions: in the cache, and the row is lost
        };
        auto load = [&](int t) {
            const size_t at = (size_t)(uint32_t)__builtin_amdgcn_readlane(slots, t - tb) * row_b;
            const int rows = g.last - (min(t * (KT / 16) + my_group, g.last >> 4) << 4);
            unsigned char *const dst = lds + (t & 1) * 2 * C::TILE + my_group * T::GROUPB;
            if (C::GPW == 2 || wave < 2) dma_group<T>(kc + at, dst, rows, off, row_b, lane, g.once);
            if (C::GPW == 2 || wave >= 2) dma_group<T>(vc + at, dst + C::TILE, rows, off, row_b, lane, g.once);
        };
        const int t1 = g.lost ? g.t0 : g.t1;
        const int w_row = g.rb * RT + wave * 16 * QT;
        const int first_ids = g.t0 < t1 ? ids() : 0;  // requested before the queries
        Query<T, QT> q;
        q.load(a, g, group, w_row, li, lg);
        if (g.t0 < t1) {
            look_up(first_ids);
            load(g.t0);
        }
        q.convert(a.scale);
        f32x4 o[QT][DT];
        float m[QT], l[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int t = g.t0; t < t1; ++t) {
            wait_vm<0>();
            lds_barrier();  // tile t is there, the other buffer free
            if (t + 1 < t1) {
                if (t + 1 - tb == 64) {
                    tb += 64;
                    look_up(ids());
                }
                load(t + 1);
            }
            const int k0 = t * KT;
            const unsigned char *const Ks = lds + (t & 1) * 2 * C::TILE, *const Vs = Ks + C::TILE;
            const bool tail = k0 + KT > g.s.cached;
            if (tail && (C::GPW == 2 || wave >= 2)) {  // the V rows that this wave loaded
                int x = 0;
#pragma unroll
                for (int n = 0; n < T::NU; ++n) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(Vs + my_group * T::GROUPB + n * 1024 + lane * 16);
                    x |= not_finite<true>(w.x) | not_finite<true>(w.y) | not_finite<true>(w.z) |
                         not_finite<true>(w.w);
                }
                if (__any(x)) odd_seg = seg;
            }
            if (w_row >= g.nrows) continue;
            uint64_t vis[QT];
            if (tail) {
#pragma unroll
                for (int i = 0; i < QT; ++i)
                    vis[i] = sees64(a, g.s.r0 + q.node[i], q.node[i], g.s.n, k0 - g.s.cached) >> 4 * lg;
            }
            // Fragments are requested some steps before their products.  A product
            // waits for the one before it of the same sum, so steps are of two
            // sums: two tiles of rows, or two fragments for one.
            constexpr int P = QT == 1 ? 2 : 1;
            f32x4 s[QT][ST];
            constexpr int KN = ST * T::KS, KA = KN < 4 ? KN : 4;
            f16x8 kf[KA + P];
            auto k_n = [](int e) { return e / (P * T::KS) * P + e % P; };  // 16 positions, and
            auto k_x = [](int e) { return e / P % T::KS; };                // part of their rows
            auto k_at = [&](int e) { return k_frag<T>(Ks + k_n(e) * T::GROUPB, k_x(e), li, lg); };
#pragma unroll
            for (int e = 0; e < KA; ++e) kf[e] = k_at(e);
#pragma unroll
            for (int e0 = 0; e0 < KN; e0 += P) {
#pragma unroll
                for (int e = e0; e < e0 + P; ++e)
                    if (e + KA < KN) kf[(e + KA) % (KA + P)] = k_at(e + KA);
                keep_order();
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = e0; e < e0 + P; ++e)
#pragma unroll
                        for (int i = 0; i < QT; ++i) {
                            f32x4 &d = s[i][k_n(e)];
                            if (half == 0 && k_x(e) == 0) d = f32x4{0.f, 0.f, 0.f, 0.f};
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                kf[e % (KA + P)], half ? q.lo[i][k_x(e)] : q.hi[i][k_x(e)], d, 0, 0, 0);
                        }
                keep_order();
            }
            if (tail) {  // nodes: by the mask
#pragma unroll
                for (int i = 0; i < QT; ++i)
#pragma unroll
                    for (int n = 0; n < ST; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[i][n][r] = vis[i] >> (n * 16 + r) & 1 ? s[i][n][r] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                const float before = m[i];
                float f[ST];
#pragma unroll
                for (int n = 0; n < ST; ++n) f[n] = q.qs[i];
                const float alpha = soften<ST>(s[i], f, T::UP, 1.0f, m[i], l[i]);
                if (__any(m[i] > before)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[i][d][r] *= alpha;
                }
            }
            f16x8 ph[ST / 2][QT], pl[ST / 2][QT];
#pragma unroll
            for (int kk = 0; kk < ST / 2; ++kk)
#pragma unroll
                for (int i = 0; i < QT; ++i) {
                    float w[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) w[r] = s[i][2 * kk + r / 4][r % 4];
                    split_f16(w, ph[kk][i], pl[kk][i]);
                }
            const int row = 4 * lg + (li >> 2), c = (li & 3) >> 1;
            auto v_at = [&](int e) {
                // the k order of the fragments: rows 4 lg + j of both groups of 16
                const int d = e % DT;
                const unsigned char *p = Vs + e / DT * 2 * T::GROUPB + row * T::ROWB +
                                         (((2 * d + c) ^ (row & T::SWZ)) << 4) + (li & 1) * 8;
                const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
                const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + T::GROUPB)));
                return __builtin_bit_cast(f16x8, make_uint4(x.x, x.y, y.x, y.y));
            };
            constexpr int VA = 4, VN = DT * (ST / 2);
            f16x8 vf[VA + P];
#pragma unroll
            for (int e = 0; e < VA; ++e) vf[e] = v_at(e);
#pragma unroll
            for (int e0 = 0; e0 < VN; e0 += P) {
#pragma unroll
                for (int e = e0; e < e0 + P; ++e)
                    if (e + VA < VN) vf[(e + VA) % (VA + P)] = v_at(e + VA);
                keep_order();
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = e0; e < e0 + P; ++e)
#pragma unroll
                        for (int i = 0; i < QT; ++i)
                            o[i][e % DT] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                vf[e % (VA + P)], half ? pl[e / DT][i] : ph[e / DT][i], o[i][e % DT], 0, 0, 0);
                keep_order();
            }
        }
        // the last tile's odd_seg, or (no tile) bad_seg, known to all
        if (g.t0 == t1 || t1 * KT > g.s.cached) lds_barrier();
        const bool bad = g.lost || uniform(bad_seg) == seg || rest_lost<KT>(a, g, lane);
        if (!bad && uniform(odd_seg) == seg) {
            one_by_one<_Float16, HD, RT>(a, g, group, KT, T::UP, 1.0f);
            continue;
        }
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            l[i] = group_sum(l[i]);
            int at = lane;
            asm volatile("" : "+v"(at));  // (addresses of its own, not kept through the tiles)
            const int row = wave * 16 * QT + i * 16 + (at & 15);
            if (g.rb * RT + row >= g.nrows) continue;
            const Dest to = dest<HD, RT>(a, g, group, row, at >> 4, m[i], bad ? NAN : l[i]);
#pragma unroll
            for (int n = 0; n < DT; ++n) to.put(n, o[i][n]);
        }
    }
}

// ---- more rows over an f32 cache.  The f32 products of the matrix cores run
// at a sixteenth of the f16 rate, so K and V are split as q and the weights are
// (hi + lo in f16, 22 bits) and take three products instead of one: hi hi, hi lo
// and lo hi.  A wave loads its share of a tile into registers, scales it by the
// power of two that brings its largest value to 2^14 .. 2^15, and leaves hi and
// lo in LDS with that exponent: K's is undone in the scores' factor, V's in the
// weights, against the largest exponent so far (which o follows as it does the
// running maximum).  Every wave of a workgroup has 16 rows and a share of each
// tile; with eight waves the same conversions serve twice the rows (one workgroup
// a CU, tiles of 64 positions): 256 rows of each of 8 requests at 4,000 positions
// 154 us instead of 215, 64 rows 62 either way.  A position is so kept to 22 bits
// down to 2^-17 of its neighbours' largest, and to 2^-40 of that below: of the same
// order as the weights.  Nodes that a row does not see must not cost its others
// their bits, so where a node is further from its neighbours the segment is taken
// one by one.
template <int HD_, int NW_>
struct WideCfg : Tile<_Float16, HD_> {
    typedef Tile<_Float16, HD_> T;
    static constexpr int NW = NW_;
    static constexpr int KT = NW == 4 ? (HD_ <= 64 ? 64 : 32) : (HD_ == 256 ? 32 : 64), RT = 16 * NW, ST = KT / 16;
    static constexpr int PW = KT / NW;               // positions of a wave
    static constexpr int LPR = HD_ / 4;              // lanes of a row
    static constexpr int NL = PW * LPR / 64;         // loads of its K
    static constexpr int HALF = KT * T::ROWB;        // hi or lo of a tile's K or V
    static constexpr int LDS = 2 * 4 * HALF;
    static constexpr int PER_CU = NW == 4 && LDS <= 72 * 1024 ? 2 : 1;
};

template <int HD, int NW>
__global__ __launch_bounds__(64 * NW, (WideCfg<HD, NW>::PER_CU * NW / 4)) void tree_wide_kernel(TreeArgs a) {
    using C = WideCfg<HD, NW>;
    using T = Tile<_Float16, HD>;
    constexpr int KT = C::KT, RT = C::RT, DT = T::DT, ST = C::ST, PW = C::PW, NL = C::NL;
    constexpr int kNone = -10000;  // exponent of nothing but zeros
    constexpr int kFar = 16;       // exponents so far apart cost bits
    __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
    __shared__ int w_exp[2][2][NW];   // exponents of a tile's K and V, a wave each
    __shared__ int bad_seg, odd_seg;  // the last segment without a block, with a value that is not finite
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int group = a.n_heads / a.n_kv;
    const size_t row_f = (size_t)a.n_kv * HD;
    const int my_group = wave * PW / 16, my_row = wave * PW % 16 + lane / C::LPR;  // of 16 positions
    Requests req;
    Cursor cur = first_unit<KT, RT>(a, group, lane, req);
    if (tid == 0) bad_seg = odd_seg = 0;
    int seg = 0;
    Seg g;
    while (next_segment<KT, RT>(a, group, req, cur, g)) {
        ++seg;
        lds_barrier();  // the last segment's reads of LDS are done, bad_seg is set up
        const float *const kc = static_cast<const float *>(a.kc) + (size_t)g.h * HD + lane % C::LPR * 4;
        const float *const vc = static_cast<const float *>(a.vc) + (size_t)g.h * HD + lane % C::LPR * 4;
        int slots = 0, tb = g.t0;
        auto ids = [&]() { return block16(a, g, (tb + lane) * ST + my_group); };
        auto look_up = [&](int id) {
            slots = slot16(a, g, (tb + lane) * ST + my_group, id);
            if (__any(slots < 0 && tb + lane < g.t1)) bad_seg = seg;
            slots = max(slots, 0);  // a block has 16 positions: in the cache, and the row is lost
        };
        f32x4 rk[NL], rv[NL];
        auto load = [&](int t) {
            if (t - tb == 64) {
                tb += 64;
                look_up(ids());
            }
            const int slot = __builtin_amdgcn_readlane(slots, t - tb);
            const int rows = g.last - (min(t * ST + my_group, g.last >> 4) << 4);
#pragma unroll
            for (int n = 0; n < NL; ++n) {
                const size_t at = (size_t)(slot + min(my_row + n * (64 / C::LPR), rows)) * row_f;
                rk[n] = *reinterpret_cast<const f32x4 *>(kc + at);
                rv[n] = *reinterpret_cast<const f32x4 *>(vc + at);
            }
        };
        // the loaded rows, scaled and split, into LDS
        auto store = [&](int t) {
            unsigned char *const buf = lds + (t & 1) * 4 * C::HALF;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f32x4(&r)[NL] = x ? rv : rk;
                // the largest magnitude's bits (ordered as the values, then inf and
                // NaN): as signed bits of the positive, as unsigned of the negative
                uint32_t un = 0;
                int sn = 0;
#pragma unroll
                for (int n = 0; n < NL; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float w = r[n][e];
                        un = max(un, __builtin_bit_cast(uint32_t, w));
                        sn = max(sn, __builtin_bit_cast(int, w));
                    }
                uint32_t top = max((uint32_t)sn, un >> 31 ? un & 0x7fffffffu : 0u);
#define CW_MAX_STEP(ctrl, rows) top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, ctrl, rows, 0xf, true))
                CW_MAX_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
                CW_MAX_STEP(0x112, 0xf);
                CW_MAX_STEP(0x114, 0xf);
                CW_MAX_STEP(0x118, 0xf);
                CW_MAX_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
                CW_MAX_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef CW_MAX_STEP
                top = (uint32_t)__builtin_amdgcn_readlane((int)top, 63);
                if (top >= 0x7f800000u) odd_seg = seg;
                const int e = max((int)(top >> 23) - 126, -100);  // all below 2^e
                const float up = __builtin_bit_cast(float, (uint32_t)(15 - min(e, 128) + 127) << 23);
                w_exp[t & 1][x][wave] = x && !top ? kNone : e;
                if (t * KT + KT > g.s.cached) {  // some nodes' values: are they far apart?
                    const float near = ldexpf(1.0f, e - 14);
                    float mx[NL];
                    bool far = false;
#pragma unroll
                    for (int n = 0; n < NL; ++n) {
                        mx[n] = fmaxf(fmaxf(fabsf(r[n][0]), fabsf(r[n][1])), fmaxf(fabsf(r[n][2]), fabsf(r[n][3])));
                        far |= mx[n] < near;
                    }
                    if (__any(far)) {
                        far = false;
#pragma unroll
                        for (int n = 0; n < NL; ++n) {
#pragma unroll
                            for (int off = 1; off < C::LPR; off <<= 1) mx[n] = fmaxf(mx[n], __shfl_xor(mx[n], off));
                            far |= mx[n] > 0.0f && mx[n] < near;
                        }
                        if (__any(far)) odd_seg = seg;
                    }
                }
#pragma unroll
                for (int n = 0; n < NL; ++n) {
                    const float w[4] = {r[n][0] * up, r[n][1] * up, r[n][2] * up, r[n][3] * up};
                    f16x4 hi, lo;
                    split_f16(w, hi, lo);
                    const int row = wave * PW + lane / C::LPR + n * (64 / C::LPR), c = lane % C::LPR;
                    unsigned char *const p = buf + x * 2 * C::HALF + row * T::ROWB +
                                             (((c >> 1) ^ (row & T::SWZ)) << 4) + (c & 1) * 8;
                    *reinterpret_cast<f16x4 *>(p) = hi;
                    *reinterpret_cast<f16x4 *>(p + C::HALF) = lo;
                }
            }
        };
        const int t1 = g.lost ? g.t0 : g.t1;
        const int w_row = g.rb * RT + wave * 16;
        const int first_ids = g.t0 < t1 ? ids() : 0;  // requested before the queries
        Query<T, 1> q;
        q.load(a, g, group, w_row, li, lg);
        if (g.t0 < t1) {
            look_up(first_ids);
            load(g.t0);
        }
        q.convert(a.scale);
        if (g.t0 < t1) {
            store(g.t0);
            if (g.t0 + 1 < t1) load(g.t0 + 1);
        }
        f32x4 o[DT];
        float m = -INFINITY, l = 0.0f;
        int E = kNone;  // V counts 2^(E - 15) in o
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int t = g.t0; t < t1; ++t) {
            lds_barrier();  // tile t is there, the other buffer free
            const int k0 = t * KT;
            const unsigned char *const Ks = lds + (t & 1) * 4 * C::HALF, *const Vs = Ks + 2 * C::HALF;
            // Of a SIMD's two waves one prepares the next tile before its products
            // and one behind them, so that conversions run beside products (128
            // rows of eight requests 162 -> 155 us; at head_dim 256, where it
            // costs registers, 183 -> 192)
            constexpr bool EARLY = NW == 8 && HD <= 128;
            auto next = [&]() {
                if (t + 1 < t1) {
                    store(t + 1);
                    if (t + 2 < t1) load(t + 2);
                }
            };
            if (EARLY && wave >= 4) next();
            if (w_row < g.nrows) {
                uint64_t vis = 0;
                const bool tail = k0 + KT > g.s.cached;
                if (tail) vis = sees64(a, g.s.r0 + q.node[0], q.node[0], g.s.n, k0 - g.s.cached) >> 4 * lg;
                constexpr int P = 2;  // sums in flight, as above
                f32x4 s[ST];
                constexpr int KN = ST * T::KS, KA = 2;
                typename T::frag kh[KA + P], kl[KA + P];
                auto k_n = [](int e) { return e / (P * T::KS) * P + e % P; };
                auto k_x = [](int e) { return e / P % T::KS; };
                auto k_get = [&](int e) {
                    kh[e % (KA + P)] = k_frag<T>(Ks + k_n(e) * T::GROUPB, k_x(e), li, lg);
                    kl[e % (KA + P)] = k_frag<T>(Ks + C::HALF + k_n(e) * T::GROUPB, k_x(e), li, lg);
                };
#pragma unroll
                for (int e = 0; e < KA; ++e) k_get(e);
#pragma unroll
                for (int e0 = 0; e0 < KN; e0 += P) {
#pragma unroll
                    for (int e = e0; e < e0 + P; ++e)
                        if (e + KA < KN) k_get(e + KA);
                    keep_order();
#pragma unroll
                    for (int part = 0; part < 3; ++part)
#pragma unroll
                        for (int e = e0; e < e0 + P; ++e) {
                            f32x4 &d = s[k_n(e)];
                            if (part == 0 && k_x(e) == 0) d = f32x4{0.f, 0.f, 0.f, 0.f};
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                part == 2 ? kl[e % (KA + P)] : kh[e % (KA + P)],
                                part == 1 ? q.lo[0][k_x(e)] : q.hi[0][k_x(e)], d, 0, 0, 0);
                        }
                    keep_order();
                }
                // the tile's exponents: K's of this lane's positions, V's against all so far
                float kf[ST], vf_[ST];
                int top = E, least = 1000;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const int e = w_exp[t & 1][1][w];
                    top = max(top, e);
                    least = e == kNone ? least : min(least, e);
                }
                if (tail && (least < top - kFar || (E != kNone && E < top - kFar))) odd_seg = seg;
#pragma unroll
                for (int n = 0; n < ST; ++n) {
                    const int w = (16 * n + 4 * lg) / PW;
                    kf[n] = ldexpf(1.0f, w_exp[t & 1][0][w] - 15);
                    vf_[n] = ldexpf(1.0f, w_exp[t & 1][1][w] - top);
                }
                const float down = ldexpf(1.0f, E - top);
                const bool grown = uniform(top) > uniform(E);
                E = top;
                if (tail) {
#pragma unroll
                    for (int n = 0; n < ST; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[n][r] = vis >> (n * 16 + r) & 1 ? s[n][r] : -INFINITY;
                }
                float f[ST];
#pragma unroll
                for (int n = 0; n < ST; ++n) f[n] = fmaxf(q.qs[0] * kf[n], 1e-37f);  // (-inf keeps its sign)
                const float before = m;
                const float alpha = soften<ST>(s, f, T::UP, 1.0f, m, l) * down;
                if (grown || __any(m > before)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[d][r] *= alpha;
                }
                f16x8 ph[ST / 2], pl[ST / 2];
#pragma unroll
                for (int kk = 0; kk < ST / 2; ++kk) {
                    float w[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) w[r] = s[2 * kk + r / 4][r % 4] * vf_[2 * kk + r / 4];
                    split_f16(w, ph[kk], pl[kk]);
                }
                const int row = 4 * lg + (li >> 2), c = (li & 3) >> 1;
                auto v_at = [&](const unsigned char *base, int e) {
                    const unsigned char *p = base + e / DT * 2 * T::GROUPB + row * T::ROWB +
                                             (((2 * (e % DT) + c) ^ (row & T::SWZ)) << 4) + (li & 1) * 8;
                    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
                    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + T::GROUPB)));
                    return __builtin_bit_cast(f16x8, make_uint4(x.x, x.y, y.x, y.y));
                };
                constexpr int VA = 2, VN = DT * (ST / 2);
                f16x8 vh[VA + P], vl[VA + P];
                auto v_get = [&](int e) {
                    vh[e % (VA + P)] = v_at(Vs, e);
                    vl[e % (VA + P)] = v_at(Vs + C::HALF, e);
                };
#pragma unroll
                for (int e = 0; e < VA; ++e) v_get(e);
#pragma unroll
                for (int e0 = 0; e0 < VN; e0 += P) {
#pragma unroll
                    for (int e = e0; e < e0 + P; ++e)
                        if (e + VA < VN) v_get(e + VA);
                    keep_order();
#pragma unroll
                    for (int part = 0; part < 3; ++part)
#pragma unroll
                        for (int e = e0; e < e0 + P; ++e)
                            o[e % DT] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                part == 2 ? vl[e % (VA + P)] : vh[e % (VA + P)],
                                part == 1 ? pl[e / DT] : ph[e / DT], o[e % DT], 0, 0, 0);
                    keep_order();
                }
            }
            if (!EARLY || wave < 4) next();
        }
        lds_barrier();  // bad_seg and odd_seg are known to all
        const bool bad = g.lost || uniform(bad_seg) == seg || rest_lost<KT>(a, g, lane);
        // o counts 2^(E - 30), the weights 2^-15, until here: no sum of them gets far
        const float unit = unit_of<float>(g.s), per_l = ldexpf(unit, -15), per_o = ldexpf(1.0f, max(E, -200) - 30);
        if (!bad && uniform(odd_seg) == seg) {
            one_by_one<float, HD, RT>(a, g, group, KT, T::UP, per_l);
            continue;
        }
        l = group_sum(l) * per_l;
        int at = lane;
        asm volatile("" : "+v"(at));  // (addresses of its own, not kept through the tiles)
        const int row = wave * 16 + (at & 15);
        if (g.rb * RT + row < g.nrows) {
            const Dest to = dest<HD, RT>(a, g, group, row, at >> 4, m, bad ? NAN : l);
#pragma unroll
            for (int n = 0; n < DT; ++n) {
                f32x4 v = o[n];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = v[r] * unit * per_o;
                to.put(n, v);
            }
        }
    }
}

// Joins the partials of the rows whose units were dealt to several workgroups,
// in the order of the positions.  16 rows of a request and kv head, 16 elements of
// them, are one wave's registers as the products left them; a lane has its row's
// maximum and sum beside them.  A workgroup has four such pieces of 16 elements,
// or (SPLIT) one, whose partials its waves share: four times the workgroups, for
// few rows of many partials, which wait for what a CU can have on its way (up to
// 46 rows at 9,390 positions at head_dim 256, 85 partials each: 13 us, 35 without;
// twelve requests of 4 to 16 rows, with more workgroups than CUs: 9.0, 6.7
// without).  A wave a row and head instead took 26 us for 1,024 rows of 32 heads,
// this 16: lengths and owners are looked up once for 16 rows.
template <typename C, bool SPLIT>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr int HD = C::HD, kt = C::KT, rt = C::RT;
    constexpr int D = SPLIT ? 8 : 4;  // partials in flight
    __shared__ float s_m[SPLIT ? 4 : 1][16], s_l[SPLIT ? 4 : 1][16];
    __shared__ f32x4 s_y[SPLIT ? 4 : 1][SPLIT ? 64 : 1];
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = uniform((int)(threadIdx.x >> 6));
    const int h = blockIdx.y, n = SPLIT ? blockIdx.z : blockIdx.z * 4 + wave;
    const int group = a.n_heads / a.n_kv;
    long long total = 0, base = -1, tiles = 0;
    int tile = 0;
    SeqRows mine{0, 0, 0};
    for (int c = 0; c < a.n_seq; c += 64) {
        SeqRows s{0, 0, 0};
        if (c + lane < a.n_seq) s = seq_rows(a.first_row, a.cached, a.rows, c + lane);
        const Work w = work_of(a, s, group, kt, rt);
        const long long v = a.n_kv * w.begin(w.blocks), inc = wave_scan(v, lane);
        const long long t = ((long long)s.n * group + 15) / 16, upto = wave_scan(t, lane) + tiles;
        const unsigned long long hit = __ballot(upto > blockIdx.x);
        if (hit && base < 0) {
            const int at = __ffsll((long long)hit) - 1;
            base = total + from_lane(inc - v, at);
            tile = (int)(blockIdx.x - from_lane(upto - t, at));
            mine = Requests{s}.at(a, at);
        }
        total += from_lane(inc, 63);
        tiles = from_lane(upto, 63);
    }
    if (base < 0) return;
    const Work wk = work_of(a, mine, group, kt, rt);
    if (!wk.blocks) return;
    const Deal deal(total, a.wgs, kt);
    const int rb = tile * 16 / rt, row = tile * 16 - rb * rt;  // of the row block
    const long long u0 = base + h * wk.begin(wk.blocks) + wk.first_tile(rb);
    const int first = uniform(deal.owner(u0)), last = uniform(deal.owner(u0 + (long long)(wk.tiles(rb) - 1) * kt));
    if (first == last) return;  // one workgroup had them all, and wrote the output
    if (!SPLIT && n * 16 >= HD) return;
    const int lr = min(li, mine.n * group - 1 - tile * 16);  // (rows behind the last: not loaded)
    const int each = SPLIT ? (last - first + 4) / 4 : last - first + 1;
    const int w0 = SPLIT ? first + wave * each : first, w1 = min(w0 + each, last + 1);
    float M = -INFINITY, L = 0.0f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int c = w0; c < w1; c += D) {
        float2 ml[D];
        f32x4 v[D];
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int w = min(c + d, w1 - 1);
            const size_t at = (size_t)(w * 2 + (w == first ? 1 : 0)) * rt + row;
            ml[d] = *reinterpret_cast<const float2 *>(a.ml + (at + lr) * 2);
            v[d] = *reinterpret_cast<const f32x4 *>(a.part + at * HD + n * 256 + lg * 64 + lr * 4);
        }
        __builtin_amdgcn_sched_barrier(0);  // all of them requested
        float Mn = M;
#pragma unroll
        for (int d = 0; d < D; ++d) Mn = fmaxf(Mn, ml[d].x);
        const float ref = Mn == -INFINITY ? 0.0f : Mn, old = __builtin_amdgcn_exp2f(M - ref);
        M = Mn;
        L *= old;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= old;
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const bool has = c + d < w1;  // (else the last one again)
            const float f = __builtin_amdgcn_exp2f(ml[d].x - ref);
            L = has ? __builtin_fmaf(f, ml[d].y, L) : L;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = has ? __builtin_fmaf(f, v[d][e], y[e]) : y[e];
        }
    }
    if constexpr (SPLIT) {
        if (lg == 0) {
            s_m[wave][li] = M;
            s_l[wave][li] = L;
        }
        s_y[wave][lane] = y;
        __syncthreads();
        if (wave > 0) return;
        for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][li]);
        const float ref = M == -INFINITY ? 0.0f : M;
        L = 0.0f;
        y = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][li] - ref);
            L = __builtin_fmaf(f, s_l[w][li], L);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(f, s_y[w][lane][e], y[e]);
        }
    }
    const int rr = tile * 16 + li, node = rr / group;
    if (node >= mine.n) return;
    const float f = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = L == 0.0f ? 0.0f : y[e] * f;
    *reinterpret_cast<f32x4 *>(a.out + (size_t)(mine.r0 + node) * a.out_stride +
                               (size_t)(h * group + rr - node * group) * HD + n * 16 + lg * 4) = y;
}

// The same for few rows a request (the split kernel's): a wave every so many
// heads of a row, the lanes four elements of every 256 / HD-th partial.  (48
// single rows of 4 query heads a kv head 4.5 us; in tiles of 16 rows 6.9.)
template <typename C>
__global__ __launch_bounds__(256) void tree_merge_rows_kernel(TreeArgs a) {
    constexpr int HD = C::HD, kt = C::KT, rt = C::RT;
    constexpr int CL = HD / 4, SL = 64 / CL;
    const int r = blockIdx.x, lane = threadIdx.x & 63;
    const int group = a.n_heads / a.n_kv;
    long long total = 0, base = -1;
    SeqRows mine{0, 0, 0};
    for (int c = 0; c < a.n_seq; c += 64) {
        SeqRows s{0, 0, 0};
        if (c + lane < a.n_seq) s = seq_rows(a.first_row, a.cached, a.rows, c + lane);
        const Work w = work_of(a, s, group, kt, rt);
        const long long v = a.n_kv * w.begin(w.blocks), inc = wave_scan(v, lane);
        const unsigned long long hit = __ballot(r >= s.r0 && r < s.r0 + s.n);
        if (hit && base < 0) {
            const int at = __ffsll((long long)hit) - 1;
            base = total + from_lane(inc - v, at);
            mine = Requests{s}.at(a, at);
        }
        total += from_lane(inc, 63);
    }
    if (base < 0) return;
    const Work wk = work_of(a, mine, group, kt, rt);
    if (!wk.blocks) return;
    const Deal deal(total, a.wgs, kt);
    const int col = lane % CL * 4, sl = lane / CL;
    for (int head = uniform((int)(blockIdx.y * 4 + (threadIdx.x >> 6))); head < a.n_heads; head += gridDim.y * 4) {
        const int h = head / group, rr = (r - mine.r0) * group + head - h * group;
        const int rb = rr / rt;
        const long long u0 = base + h * wk.begin(wk.blocks) + wk.first_tile(rb);
        const int w0 = uniform(deal.owner(u0)), w1 = uniform(deal.owner(u0 + (long long)(wk.tiles(rb) - 1) * kt));
        if (w0 == w1) continue;  // one workgroup had them all, and wrote the output
        auto at = [&](int w) { return (size_t)(w * 2 + (w == w0 ? 1 : 0)) * rt + rr % rt; };
        float M = -INFINITY, L = 0.0f;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        for (int c = w0; c <= w1; c += 64) {
            const int n = min(64, w1 + 1 - c);
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (lane < n) ml = *reinterpret_cast<const float2 *>(a.ml + at(c + lane) * 2);
            constexpr int D = 8;  // partials in flight
            f32x4 v[D];
            auto fetch = [&](int p0) {
#pragma unroll
                for (int d = 0; d < D; ++d)
                    v[d] = *reinterpret_cast<const f32x4 *>(a.part + at(c + min(p0 + d * SL + sl, n - 1)) * HD + col);
            };
            fetch(0);
            float mx = ml.x;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            const float Mn = fmaxf(M, mx), ref = Mn == -INFINITY ? 0.0f : Mn;
            const float old = __builtin_amdgcn_exp2f(M - ref), f = __builtin_amdgcn_exp2f(ml.x - ref);
            M = Mn;
            float ls = lane < n ? f * ml.y : 0.0f;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) ls += __shfl_xor(ls, o);
            L = L * old + ls;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] *= old;
            for (int p0 = 0;;) {
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    const int p = p0 + d * SL + sl;
                    const float w = __shfl(f, p & 63);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        y[e] = p < n ? __builtin_fmaf(w, v[d][e], y[e]) : y[e];
                }
                p0 += D * SL;
                if (p0 >= n) break;
                fetch(p0);
            }
        }
#pragma unroll
        for (int o = CL; o < 64; o <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], o);
        const float f = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = L == 0.0f ? 0.0f : y[e] * f;
        if (sl == 0) *reinterpret_cast<f32x4 *>(a.out + (size_t)r * a.out_stride + (size_t)head * HD + col) = y;
    }
}

template <typename C>
int launch_tiles(cw_ctx *ctx, TreeArgs a, void (*fn)(TreeArgs)) {
    a.wgs = ctx->n_cu * C::PER_CU;
    const size_t rows = (size_t)a.wgs * 2 * C::RT;
    void *scratch = nullptr;
    CW_TRY(ctx_scratch(ctx, rows * (C::HD + 2) * sizeof(float), &scratch));
    a.part = static_cast<float *>(scratch);
    a.ml = a.part + rows * C::HD;
    CW_TRY(launch(ctx, "attention_tree", fn, dim3(a.wgs), dim3(C::NW * 64), 0, a));
    if constexpr (C::RT == 16) {
        // four heads a workgroup while that is about what the chip holds at once, more
        // for more rows, which also share the look at the lengths
        const int by_chip = (8 * ctx->n_cu + a.rows - 1) / a.rows;
        return launch(ctx, "attention_tree_merge", tree_merge_rows_kernel<C>,
                      dim3(a.rows, std::min((a.n_heads + 3) / 4, by_chip)), dim3(256), 0, a);
    } else {
        // tiles of 16 rows that the requests have at most
        const unsigned tiles = (unsigned)((long long)a.rows * (a.n_heads / a.n_kv) / 16) + a.n_seq;
        if ((long long)tiles * a.n_kv * ((C::HD + 63) / 64) <= ctx->n_cu)
            return launch(ctx, "attention_tree_merge", tree_merge_kernel<C, true>,
                          dim3(tiles, a.n_kv, C::HD / 16), dim3(256), 0, a);
        return launch(ctx, "attention_tree_merge", tree_merge_kernel<C, false>,
                      dim3(tiles, a.n_kv, (C::HD + 63) / 64), dim3(256), 0, a);
    }
}
template <typename KVT, int HD>
int launch_split(cw_ctx *ctx, const TreeArgs &a) {
    return launch_tiles<SplitCfg<KVT, HD>>(ctx, a, tree_split_kernel<KVT, HD>);
}
template <int HD, int QT>
int launch_tile(cw_ctx *ctx, const TreeArgs &a) {
    return launch_tiles<TileCfg<HD, QT>>(ctx, a, tree_tile_kernel<HD, QT>);
}
template <int HD, int NW>
int launch_wide(cw_ctx *ctx, const TreeArgs &a) {
    return launch_tiles<WideCfg<HD, NW>>(ctx, a, tree_wide_kernel<HD, NW>);
}

// By the rows of a (request, kv head) on average; us at head_dim 128, 8 requests
// of 4,000 positions unless said otherwise:
//   f16, 4 / 16 / 32 rows: split 26.4 / 28.5 / 34.2 (of two tiles of rows), tiles
//   27.1 / 27.4 / 30.3; one request of 4 rows: 8.7 and 10.3; tiles of 64 and of
//   128 rows: 54 and 51 for 128 rows with joins of 10 and 12, 159 and 153 for 512,
//   28.6 and 34 for 244 of a single request;
//   f32, 8 / 16 / 32 rows: split 46 / 48 / 71, wide 54 / 55 / 58.
// Over f32 eight waves: 64 and 256 rows 35 / 39 and 113 / 93 (four / eight waves)
// at head_dim 64, 2,000 positions at head_dim 256 49 / 56 for 64 and 265 / 183
// for 512; at head_dim 128 they are no slower from 32 rows on.
// head_dim 256: the split kernel's registers leave a CU one workgroup, 27.9 us for
// 4 rows over f16; tiles 27.3.
template <typename KVT, int HD>
int launch_by_rows(cw_ctx *ctx, const TreeArgs &a) {
    const long long rows = ((long long)a.rows + a.n_seq - 1) / a.n_seq * (a.n_heads / a.n_kv);
    if constexpr (HD <= 128 && (HD > 32 || sizeof(KVT) == 2))  // (its V reads of f32 are 64 elements wide)
        if (rows <= (sizeof(KVT) == 2 ? 8 : 16)) return launch_split<KVT, HD>(ctx, a);
    if constexpr (sizeof(KVT) == 4) {
        if constexpr (HD != 128)
            if (rows <= 64) return launch_wide<HD, 4>(ctx, a);
        return launch_wide<HD, 8>(ctx, a);
    } else {
        if constexpr (HD <= 128)
            if (rows > 256) return launch_tile<HD, 2>(ctx, a);
        return launch_tile<HD, 1>(ctx, a);
    }
}

template <typename KVT>
int launch_by_size(cw_ctx *ctx, const TreeArgs &a, int hd) {
    if (hd == 32) return launch_by_rows<KVT, 32>(ctx, a);
    if (hd == 64) return launch_by_rows<KVT, 64>(ctx, a);
    if (hd == 128) return launch_by_rows<KVT, 128>(ctx, a);
    if (hd == 256) return launch_by_rows<KVT, 256>(ctx, a);
    // 1,024 threads for what would leave a CU two workgroups (4,000 positions: 8 and
    // 512 (row, head)s 34 and 89 us, with 256 threads 124 and 212), else 256 (4,096
    // of them over f32: 362 us, 610 with 1,024)
    const bool few = (long long)a.rows * a.n_heads <= 2 * ctx->n_cu;
    return few ? launch(ctx, "attention_tree", tree_row_kernel<KVT, 1024>, dim3(a.rows, a.n_heads), dim3(1024), 0, a)
               : launch(ctx, "attention_tree", tree_row_kernel<KVT, 256>, dim3(a.rows, a.n_heads), dim3(256), 0, a);
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
    CW_CHECK_ARG((long long)b->rows * (n_heads / kv->n_kv_heads) <= 1 << 27,
                 "cw_attention_tree: %d rows of %d query heads a kv head are more than 2^27", b->rows,
                 n_heads / kv->n_kv_heads);
    CW_CHECK_ARG((long long)b->rows * n_heads <= 1LL << 33,
                 "cw_attention_tree: %d rows of %d query heads are more than 2^33", b->rows, n_heads);
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
               (float)(1.4426950408889634 / std::sqrt((double)kv->head_dim)), 0, nullptr, nullptr};
    return kv->kv_dtype == CW_F16 ? launch_by_size<_Float16>(ctx, a, kv->head_dim)
                                  : launch_by_size<float>(ctx, a, kv->head_dim);
}
