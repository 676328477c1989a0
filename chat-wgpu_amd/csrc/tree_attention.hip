// Attention of many rows over a paged cache of several requests: decode steps,
// pieces of prompts and trees of drafted tokens in one call.
//
// o_h = sum_p softmax_p(q_h . k_p / sqrt(hd)) v_p over the positions that a row
// sees: its request's cached ones, and of the request's own rows (nodes) those
// its mask shows.

#include <cmath>

#include "paged_device.hpp"
#include "prompt_device.hpp"

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
    int wgs;      // workgroups that share the units (tree_kernel)
    float *part;  // [wgs][2][row block][hd] partial o, then
    float *ml;    // [wgs][2][row block][2] their (max log2 e, sum)
};

// Whether node i of a request sees its node j (row: the node's row of the mask)
__device__ __forceinline__ bool sees(const TreeArgs &a, int row, int i, int j) {
    if (!a.mask) return j <= i;
    return (j >> 5) < a.mask_words &&
           (a.mask[(size_t)row * a.mask_words + (j >> 5)] >> (j & 31) & 1);
}

// The lowest n of 32 bits (none below 0, all from 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
}

// Bit r: node i of a request of n nodes sees node j + r, r < 4; nodes below 0
// (cached positions) are seen.  Without branches for the lanes.
__device__ __forceinline__ uint32_t sees4(const TreeArgs &a, int row, int i, int n, int j) {
    uint32_t m;
    if (a.mask) {
        const uint32_t *words = a.mask + (size_t)row * a.mask_words;
        const int w = j >> 5;
        uint32_t lo = words[min(max(w, 0), a.mask_words - 1)];
        uint32_t hi = words[min(max(w + 1, 0), a.mask_words - 1)];
        lo = w < 0 ? ~0u : w < a.mask_words ? lo : 0u;
        hi = w + 1 < 0 ? ~0u : w + 1 < a.mask_words ? hi : 0u;
        m = (uint32_t)(((uint64_t)hi << 32 | lo) >> (j & 31));
    } else {
        m = low_bits(i - j + 1);
    }
    return m & low_bits(n - j);
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

// ---------------------------------------------------------------- tiles on the matrix cores

// v_mfma layouts (lane l: li = l % 16, lg = l / 16): 16x16x32 f16 holds
// A[li][8 lg + j], B[8 lg + j][li]; 16x16x16 f16 A[li][4 lg + j], B[4 lg + j][li];
// 16x16x4 f32 A[li][lg], B[lg][li]; all D[4 lg + r][li].

// KT positions a tile, QT tiles of 16 rows a wave.  SPLIT: the four waves share
// the rows and take 16 of the tile's 64 positions each; else they share the
// positions and take 16 QT rows each.
template <typename KVT, int HD_, int QT_, bool SPLIT_>
struct TC {
    static constexpr int HD = HD_, QT = QT_, ES = (int)sizeof(KVT);
    static constexpr bool SPLIT = SPLIT_, F16 = ES == 2;
    static constexpr int ROWB = HD * ES;    // bytes of a row of one kv head
    static constexpr int CPR = ROWB / 16;   // 16-byte chunks of it
    static constexpr int SWZ = CPR < 16 ? CPR - 1 : 15;
    static constexpr int KT = SPLIT || ROWB <= 256 ? 64 : 32;
    static constexpr int TILE = KT * ROWB;  // bytes of a K (or V) tile
    static constexpr int GROUPB = 16 * ROWB;
    static constexpr int ST = SPLIT ? 1 : KT / 16;       // score tiles of a wave
    static constexpr int RT = 16 * QT * (SPLIT ? 1 : 4); // rows of a workgroup
    static constexpr int NU = ROWB / 64;                 // DMAs of 16 rows
    static constexpr int GPW = 2 * KT / 64;              // groups of 16 rows a wave loads a tile
    static constexpr int NLD = GPW * NU;                 // DMAs a wave issues a tile
    static constexpr int LDS = 4 * TILE;                 // two buffers of K and V
    static constexpr float UP = F16 ? 15.0f : 0.0f;
    static_assert(!SPLIT || 4 * RT * HD * 4 <= LDS, "the waves' o must fit the tiles");
    static_assert(LDS + 4096 <= 160 * 1024, "tiles must fit a CU");
};

// The units of a request: a unit is one tile of positions for one row block of
// one kv head; a request's are ordered (kv head, row block, tile).
struct Work {
    int tiles, blocks;
    long long units;
};
__device__ __forceinline__ Work work_of(const SeqRows &s, int group, int n_kv, int kt, int rt) {
    if (!s.n) return Work{0, 0, 0};
    const int t = (s.cached + s.n + kt - 1) / kt, rb = (int)(((long long)s.n * group + rt - 1) / rt);
    return Work{t, rb, (long long)n_kv * rb * t};
}

__device__ __forceinline__ long long wave_scan(long long v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// All units are dealt to `wgs` workgroups in runs of q or q + 1.
struct Deal {
    long long q;
    int rem;
    __device__ Deal(long long units, int wgs) {
        q = units / wgs;
        rem = (int)(units - q * wgs);
    }
    __device__ long long start(int w) const { return q * w + min(w, rem); }
    __device__ int owner(long long u) const {
        const long long big = (q + 1) * rem;
        return u < big ? (int)(u / (q + 1)) : rem + (int)((u - big) / q);
    }
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long uniform(long long v) {
    return (long long)(uint32_t)uniform((int)v) | (long long)uniform((int)(v >> 32)) << 32;
}

__device__ __forceinline__ SeqRows uniform(SeqRows s) {
    return SeqRows{uniform(s.r0), uniform(s.n), uniform(s.cached)};
}

typedef const __attribute__((address_space(4))) int *const_i32;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

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

// v = hi + lo in f16 (22 bits)
__device__ __forceinline__ void split_f16(float v, _Float16 &hi, _Float16 &lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

template <typename KVT, int HD, int QT, bool SPLIT>
__global__ __launch_bounds__(256, (TC<KVT, HD, QT, SPLIT>::LDS <= 72 * 1024 ? 2 : 1)) void tree_kernel(TreeArgs a) {
    using C = TC<KVT, HD, QT, SPLIT>;
    constexpr int KT = C::KT, ST = C::ST, RT = C::RT, ROWB = C::ROWB, DT = HD / 16;
    constexpr bool F16 = C::F16;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
    __shared__ float w_ml[SPLIT ? 4 : 1][SPLIT ? RT : 1][2];
    __shared__ int bad_seg;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int group = a.n_heads / a.n_kv;
    const size_t row_b = (size_t)a.n_kv * ROWB;

    // the units of all requests, and the request where this workgroup begins
    auto lane_units = [&](int b) {
        return b < a.n_seq ? work_of(seq_rows(a.first_row, a.cached, a.rows, b), group, a.n_kv, KT,
                                     RT).units : 0;
    };
    long long total = 0;
    for (int b = 0; b < a.n_seq; b += 64) total += __shfl(wave_scan(lane_units(b + lane), lane), 63);
    total = uniform(total);
    const Deal deal(total, a.wgs);
    const long long u_end = deal.start(blockIdx.x + 1);
    long long u = deal.start(blockIdx.x);
    if (u >= u_end) return;
    int b = 0;
    long long base = 0;
    for (int c = 0; c < a.n_seq; c += 64) {
        const long long v = lane_units(c + lane), inc = wave_scan(v, lane) + base;
        const unsigned long long hit = __ballot(inc > u);
        if (hit) {
            const int at = __ffsll((long long)hit) - 1;
            b = uniform(c + at);
            base = uniform(__shfl(inc - v, at));
            break;
        }
        base = uniform(__shfl(inc, 63));
    }

    if (tid == 0) bad_seg = 0;
    int seg = 0;
    while (u < u_end && b < a.n_seq) {
        const SeqRows s = uniform(seq_rows(a.first_row, a.cached, a.rows, b));
        const Work wk = work_of(s, group, a.n_kv, KT, RT);
        if (u >= base + wk.units) {  // (requests without rows have no units)
            base += wk.units;
            ++b;
            continue;
        }
        ++seg;
        const long long local = u - base;
        const int hr = uniform((int)(local / wk.tiles)), t0 = uniform((int)(local - (long long)hr * wk.tiles));
        const int t1 = (int)min((long long)wk.tiles, t0 + (u_end - u));
        const int h = uniform(hr / wk.blocks), rb = hr - h * wk.blocks;
        const bool whole = t0 == 0 && t1 == wk.tiles;
        const int slot_part = blockIdx.x * 2 + (t0 > 0 ? 0 : 1);
        u += t1 - t0;
        const int last = s.cached + s.n - 1, nrows = s.n * group;
        const char *const kc = static_cast<const char *>(a.kc) + (size_t)h * ROWB;
        const char *const vc = static_cast<const char *>(a.vc) + (size_t)h * ROWB;
        lds_barrier();  // the last segment's reads of LDS are done, bad_seg is set up

        // first slot of the 16 positions of group gi; -1: they have no block
        auto slot16 = [&](int gi) -> int {
            const int p0 = min(gi, last >> 4) << 4;
            bool bad;
            int slot;
            if (a.map.tables) {
                const int e = p0 >> a.map.shift;
                const const_i32 tab = (const_i32)(uintptr_t)(a.map.tables + (size_t)b * a.map.max_blocks);
                const int id = tab[uniform(min(e, a.map.max_blocks - 1))];
                bad = e >= a.map.max_blocks || (unsigned)id >= (unsigned)a.map.n_blocks;
                slot = bad ? -1 : (id << a.map.shift) + (p0 & (a.map.page - 1));
            } else {
                bad = min(p0 + 15, last) >= a.map.page;
                slot = bad ? -1 : b * a.map.page + p0;
            }
            if (bad && lane == 0) bad_seg = seg;
            return uniform(slot);
        };
        // a wave's groups of a tile: K and V of group `wave`, or (32 positions)
        // group wave % 2 of K or V
        const int my_group = C::GPW == 2 ? wave : wave & 1;
        auto load = [&](int t, int slot, unsigned char *buf) {
            const int p0 = min(t * (KT / 16) + my_group, last >> 4) << 4;
            const int rows = slot < 0 ? 0 : last - p0;  // (without a block: slot 0, results are NaN)
            slot = max(slot, 0);
#pragma unroll
            for (int x = 0; x < C::GPW; ++x) {
                const bool is_v = C::GPW == 2 ? x == 1 : wave >= 2;
                const char *src = (is_v ? vc : kc) + (size_t)slot * row_b;
                unsigned char *dst = buf + (is_v ? C::TILE : 0) + my_group * C::GROUPB;
#pragma unroll
                for (int n = 0; n < C::NU; ++n) {
                    // chunk c of row r lies at slot c ^ (r & SWZ) of its row, so that
                    // the fragment reads spread over the banks; rows behind the
                    // last position repeat it
                    const int r = n * (64 / C::CPR) + lane / C::CPR;
                    const int c = (lane % C::CPR) ^ (r & C::SWZ);
                    dma16(src, (uint32_t)min(r, rows) * (uint32_t)row_b + c * 16, dst + n * 1024);
                }
            }
        };
        const int per_tile = KT / 16;
        int slot = slot16(t0 * per_tile + my_group);
        load(t0, slot, lds);
        slot = slot16((t0 + 1) * per_tile + my_group);

        // q of this lane's rows (B operands), as two f16 of q times a power of
        // two that brings the row's largest below 2^15
        const int w_row = rb * RT + (SPLIT ? 0 : wave * 16 * QT);
        int node[QT], head[QT];
        f16x8 qh[F16 ? QT : 1][HD / 32], ql[F16 ? QT : 1][HD / 32];
        f32x4 qf[F16 ? 1 : QT][HD / 16];
        float qs[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            const int rr = min(w_row + i * 16 + li, nrows - 1);
            node[i] = rr / group;
            head[i] = h * group + rr % group;
            const float *qr = a.q + (size_t)(s.r0 + node[i]) * a.q_stride + (size_t)head[i] * HD;
            qs[i] = a.scale;
            if constexpr (F16) {
                f32x4 v[HD / 32][2];
                float mx = 0.0f;
#pragma unroll
                for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        v[ks][x] = *reinterpret_cast<const f32x4 *>(qr + 32 * ks + 8 * lg + 4 * x);
#pragma unroll
                        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fabsf(v[ks][x][j]));
                    }
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                // mx in [2^(e-1), 2^e)
                const int e = max(__builtin_amdgcn_frexp_expf(mx), -110);
                const bool fin = mx > 0.0f && mx < INFINITY;
                const float up = fin ? ldexpf(1.0f, 15 - e) : 1.0f;
                qs[i] = fin ? ldexpf(a.scale, e - 15) : a.scale;
#pragma unroll
                for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        _Float16 hi, lo;
                        split_f16(v[ks][j / 4][j % 4] * up, hi, lo);
                        qh[i][ks][j] = hi;
                        ql[i][ks][j] = lo;
                    }
            } else {
#pragma unroll
                for (int x = 0; x < HD / 16; ++x)
                    qf[i][x] = *reinterpret_cast<const f32x4 *>(qr + 16 * x + 4 * lg);
            }
        }

        f32x4 o[QT][DT];  // o^T: dims 16 d + 4 lg + r of row li
        float mrow[QT], lsum[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            mrow[i] = -INFINITY;
            lsum[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const int ka = li * ROWB + ((lg ^ (li & C::SWZ)) << 4);
        const int vrow = 4 * lg + (li >> 2);
        const int va = vrow * ROWB + ((((li & 3) >> 1) ^ (vrow & C::SWZ)) << 4) + (li & 1) * 8;

        for (int t = t0; t < t1; ++t) {
            unsigned char *const buf = lds + ((t - t0) & 1) * 2 * C::TILE;
            unsigned char *const next = lds + ((t - t0 + 1) & 1) * 2 * C::TILE;
            if constexpr (SPLIT) {
                // each wave reads only what it loaded: no barrier
                if (t + 1 < t1) {
                    wait_lds();  // of the tile before, whose place this takes
                    load(t + 1, slot, next);
                    slot = slot16((t + 2) * per_tile + my_group);
                    wait_vm<C::NLD>();
                } else {
                    wait_vm<0>();
                }
            } else {
                wait_vm<0>();
                lds_barrier();  // tile t is there, the other buffer free
                if (t + 1 < t1) {
                    load(t + 1, slot, next);
                    slot = slot16((t + 2) * per_tile + my_group);
                }
                if (w_row >= nrows) continue;
            }
            const int k0 = t * KT + (SPLIT ? wave * 16 : 0);  // this wave's first position
            const unsigned char *const Ks = buf + (SPLIT ? wave * C::GROUPB : 0);
            const unsigned char *const Vs = Ks + C::TILE;

            f32x4 sc[QT][ST];
#pragma unroll
            for (int kt = 0; kt < ST; ++kt) {
#pragma unroll
                for (int i = 0; i < QT; ++i) sc[i][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (F16) {
#pragma unroll
                    for (int ks = 0; ks < HD / 32; ++ks) {
                        const f16x8 kf = *reinterpret_cast<const f16x8 *>(Ks + ((ka ^ (ks << 6)) + kt * C::GROUPB));
#pragma unroll
                        for (int i = 0; i < QT; ++i)
                            sc[i][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[i][ks], sc[i][kt], 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < QT; ++i)
                            sc[i][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[i][ks], sc[i][kt], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < HD / 16; ++x) {
                        const f32x4 kf = *reinterpret_cast<const f32x4 *>(Ks + ((ka ^ (x << 6)) + kt * C::GROUPB));
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int i = 0; i < QT; ++i)
                                sc[i][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[r], qf[i][x][r], sc[i][kt], 0, 0, 0);
                    }
                }
            }
            // what a row sees: every cached position; of the nodes by the mask
            const bool tail = k0 + 16 * ST > s.cached;
            if (tail) {
#pragma unroll
                for (int i = 0; i < QT; ++i)
#pragma unroll
                    for (int kt = 0; kt < ST; ++kt) {
                        const uint32_t vis = sees4(a, s.r0 + node[i], node[i], s.n,
                                                   k0 + kt * 16 + 4 * lg - s.cached);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            sc[i][kt][r] = vis >> r & 1 ? sc[i][kt][r] : -INFINITY;
                    }
            }
            float alpha[QT];
            bool grew = false;
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                float mx = sc[i][0][0];
#pragma unroll
                for (int kt = 0; kt < ST; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[i][kt][r]);
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float mnew = fmaxf(mrow[i], mx * qs[i]);
                const float ref = mnew == -INFINITY ? 0.0f : mnew;
                alpha[i] = __builtin_amdgcn_exp2f(mrow[i] - ref);
                grew |= mnew > mrow[i];
                mrow[i] = mnew;
                float ls = 0.0f;
#pragma unroll
                for (int kt = 0; kt < ST; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][kt][r], qs[i], C::UP - ref));
                        sc[i][kt][r] = p;
                        ls += p;
                    }
                lsum[i] = lsum[i] * alpha[i] + ls;
            }
            if (__any(grew)) {
#pragma unroll
                for (int i = 0; i < QT; ++i)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[i][d][r] *= alpha[i];
            }
            // a V that is no finite number would reach rows that do not see it
            // as 0 * V: such a tile's products are taken one by one
            bool odd = false;
            if (tail) {
#pragma unroll
                for (int n = 0; n < 16 * ST * C::CPR / 64; ++n) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(Vs + n * 1024 + lane * 16);
                    constexpr uint32_t E = F16 ? 0x7c00u : 0x7f800000u;
                    for (uint32_t x : {w.x, w.y, w.z, w.w})
                        odd |= (x & E) == E || (F16 && (x >> 16 & E) == E);
                }
            }
            if (__any(odd)) {
#pragma unroll 1
                for (int key = 0; key < 16 * ST; ++key) {
                    const int kt = key >> 4, r = key & 3, from = li + 4 * (key & 12);
#pragma unroll
                    for (int i = 0; i < QT; ++i) {
                        float p = 0.0f;
#pragma unroll
                        for (int x = 0; x < ST; ++x)
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                if (x == kt && y == r) p = sc[i][x][y];
                        p = __shfl(p, from);
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const int e = 16 * d + 4 * lg + y;
                                const int c = e * C::ES / 16;
                                const float v = (float)*reinterpret_cast<const KVT *>(
                                    Vs + key * ROWB + ((c ^ (key & C::SWZ)) << 4) + e * C::ES % 16);
                                if (p != 0.0f) o[i][d][y] = __builtin_fmaf(p, v, o[i][d][y]);
                            }
                    }
                }
            } else if constexpr (F16 && ST == 1) {
                f16x4 ph[QT], pl[QT];
#pragma unroll
                for (int i = 0; i < QT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        _Float16 hi, lo;
                        split_f16(sc[i][0][r], hi, lo);
                        ph[i][r] = hi;
                        pl[i][r] = lo;
                    }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    // V^T: within 16 lanes, lane i receives element i % 4 of the 8
                    // bytes at lane 4 j + i / 4's address: dim 16 d + i of keys 4 lg + j
                    const f16x4 vf = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4 *)(Vs + (va ^ (d << 5)))));
#pragma unroll
                    for (int i = 0; i < QT; ++i)
                        o[i][d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vf, ph[i], o[i][d], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < QT; ++i)
                        o[i][d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vf, pl[i], o[i][d], 0, 0, 0);
                }
            } else if constexpr (F16) {
#pragma unroll
                for (int kk = 0; kk < ST / 2; ++kk) {
                    f16x8 ph[QT], pl[QT];
#pragma unroll
                    for (int i = 0; i < QT; ++i)
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            _Float16 hi, lo;
                            split_f16(sc[i][2 * kk + r / 4][r % 4], hi, lo);
                            ph[i][r] = hi;
                            pl[i][r] = lo;
                        }
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const unsigned char *p = Vs + ((va ^ (d << 5)) + kk * 2 * C::GROUPB);
                        const uint2 r0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
                        const uint2 r1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + C::GROUPB)));
                        const f16x8 vf = __builtin_bit_cast(f16x8, make_uint4(r0.x, r0.y, r1.x, r1.y));
#pragma unroll
                        for (int i = 0; i < QT; ++i)
                            o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[i], o[i][d], 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < QT; ++i)
                            o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[i], o[i][d], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int kt = 0; kt < ST; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 4 * lg + r;
                        const int vb = row * ROWB + (((li >> 2) ^ (row & C::SWZ)) << 4) + (li & 3) * 4;
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            const float vf = *reinterpret_cast<const float *>(Vs + ((vb ^ (d << 6)) + kt * C::GROUPB));
#pragma unroll
                            for (int i = 0; i < QT; ++i)
                                o[i][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, sc[i][kt][r], o[i][d], 0, 0, 0);
                        }
                    }
            }
        }

        // the segment's result: the output where it has every tile, else a partial
        auto put = [&](int row_in, int nd, int hd_, int col, f32x4 v, float m, float l) {
            if (whole) {
                const float f = l == 0.0f ? 0.0f : 1.0f / l;
                f32x4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = l == 0.0f ? 0.0f : v[r] * f;
                *reinterpret_cast<f32x4 *>(a.out + (size_t)(s.r0 + nd) * a.out_stride + (size_t)hd_ * HD + col) = y;
            } else {
                const size_t at = (size_t)slot_part * RT + row_in;
                *reinterpret_cast<f32x4 *>(a.part + at * HD + col) = v;
                if (col == 0) *reinterpret_cast<float2 *>(a.ml + at * 2) = make_float2(m, l);
            }
        };
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            lsum[i] += __shfl_xor(lsum[i], 16);
            lsum[i] += __shfl_xor(lsum[i], 32);
        }
        if constexpr (SPLIT) {
            if (lg == 0)
#pragma unroll
                for (int i = 0; i < QT; ++i) {
                    w_ml[wave][i * 16 + li][0] = mrow[i];
                    w_ml[wave][i * 16 + li][1] = lsum[i];
                }
            lds_barrier();  // and every wave is done with its tiles
            f32x4 *const ow = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                const int row = i * 16 + li;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < 4; ++w) M = fmaxf(M, w_ml[w][row][0]);
                const float f = __builtin_amdgcn_exp2f(mrow[i] - (M == -INFINITY ? 0.0f : M));
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    f32x4 v = o[i][d];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] *= f;
                    ow[(wave * RT + row) * (HD / 4) + ((4 * d + lg) ^ (row & (HD / 4 < 16 ? HD / 4 - 1 : 15)))] = v;
                }
            }
            lds_barrier();
            const bool bad = bad_seg == seg;
            for (int x = tid; x < RT * (HD / 4); x += 256) {
                const int row = x / (HD / 4), c4 = x % (HD / 4), rr = rb * RT + row;
                if (rr >= nrows) continue;
                float M = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) M = fmaxf(M, w_ml[w][row][0]);
                const float ref = M == -INFINITY ? 0.0f : M;
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    l += w_ml[w][row][1] * __builtin_amdgcn_exp2f(w_ml[w][row][0] - ref);
                    v += ow[(w * RT + row) * (HD / 4) + (c4 ^ (row & (HD / 4 < 16 ? HD / 4 - 1 : 15)))];
                }
                put(row, rr / group, h * group + rr % group, 4 * c4, v, M, bad ? NAN : l);
            }
        } else {
            const bool bad = bad_seg == seg;  // (set before the last tile's barrier)
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                if (w_row + i * 16 + li >= nrows) continue;
                const int row = (SPLIT ? 0 : wave * 16 * QT) + i * 16 + li;
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    put(row, node[i], head[i], 16 * d + 4 * lg, o[i][d], mrow[i], bad ? NAN : lsum[i]);
            }
        }
    }
}

// Joins the partials of every row whose units went to more than one workgroup:
// one workgroup a row, a thread four elements of a head.
template <int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int kt, int rt) {
    const int r = blockIdx.x, lane = threadIdx.x & 63;
    const int group = a.n_heads / a.n_kv;
    long long total = 0, base = -1;
    SeqRows mine{0, 0, 0};
    for (int c = 0; c < a.n_seq; c += 64) {
        SeqRows s{0, 0, 0};
        if (c + lane < a.n_seq) s = seq_rows(a.first_row, a.cached, a.rows, c + lane);
        const long long v = work_of(s, group, a.n_kv, kt, rt).units, inc = wave_scan(v, lane);
        const unsigned long long hit = __ballot(r >= s.r0 && r < s.r0 + s.n);
        if (hit && base < 0) {
            const int at = __ffsll((long long)hit) - 1;
            base = total + __shfl(inc - v, at);
            mine = SeqRows{__shfl(s.r0, at), __shfl(s.n, at), __shfl(s.cached, at)};
        }
        total += __shfl(inc, 63);
    }
    if (base < 0) return;
    const Work wk = work_of(mine, group, a.n_kv, kt, rt);
    const Deal deal(total, a.wgs);
    for (int x = threadIdx.x; x < a.n_heads * (HD / 4); x += 256) {
        const int head = x / (HD / 4), col = x % (HD / 4) * 4;
        const int h = head / group, rr = (r - mine.r0) * group + head % group;
        const long long u0 = base + ((long long)h * wk.blocks + rr / rt) * wk.tiles;
        const int w0 = deal.owner(u0), w1 = deal.owner(u0 + wk.tiles - 1);
        if (w0 == w1) continue;  // one workgroup had them all, and wrote the output
        auto at = [&](int w) { return (size_t)(w * 2 + (w == w0 ? 1 : 0)) * rt + rr % rt; };
        float M = -INFINITY, L = 0.0f;
        for (int w = w0; w <= w1; ++w) M = fmaxf(M, a.ml[at(w) * 2]);
        const float ref = M == -INFINITY ? 0.0f : M;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        for (int w = w0; w <= w1; ++w) {
            const float2 ml = *reinterpret_cast<const float2 *>(a.ml + at(w) * 2);
            const float f = __builtin_amdgcn_exp2f(ml.x - ref);
            L = __builtin_fmaf(f, ml.y, L);
            const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part + at(w) * HD + col);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(f, v[e], y[e]);
        }
        const float f = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = L == 0.0f ? 0.0f : y[e] * f;
        *reinterpret_cast<f32x4 *>(a.out + (size_t)r * a.out_stride + (size_t)head * HD + col) = y;
    }
}

template <typename KVT, int HD, int QT, bool SPLIT>
int launch_tiles(cw_ctx *ctx, TreeArgs a) {
    using C = TC<KVT, HD, QT, SPLIT>;
    a.wgs = ctx->n_cu * (C::LDS <= 72 * 1024 ? 2 : 1);
    const size_t rows = (size_t)a.wgs * 2 * C::RT;
    void *scratch = nullptr;
    CW_TRY(ctx_scratch(ctx, rows * (HD + 2) * sizeof(float), &scratch));
    a.part = static_cast<float *>(scratch);
    a.ml = a.part + rows * HD;
    CW_TRY(launch(ctx, "attention_tree", tree_kernel<KVT, HD, QT, SPLIT>, dim3(a.wgs), dim3(256), 0, a));
    return launch(ctx, "attention_tree_merge", tree_merge_kernel<HD>, dim3(a.rows), dim3(256), 0, a,
                  C::KT, C::RT);
}

// By the rows of a (request, kv head) on average.
template <typename KVT, int HD>
int launch_by_rows(cw_ctx *ctx, const TreeArgs &a) {
    const long long rows = ((long long)a.rows + a.n_seq - 1) / a.n_seq * (a.n_heads / a.n_kv);
    if constexpr (HD * sizeof(KVT) <= 512) {
        if (rows <= 16) return launch_tiles<KVT, HD, 1, true>(ctx, a);
        if (rows <= 32) return launch_tiles<KVT, HD, 2, true>(ctx, a);
    }
    if constexpr (HD <= 128 && sizeof(KVT) == 2)
        if (rows > 64) return launch_tiles<KVT, HD, 2, false>(ctx, a);
    return launch_tiles<KVT, HD, 1, false>(ctx, a);
}

template <typename KVT>
int launch_by_size(cw_ctx *ctx, const TreeArgs &a, int hd) {
    if (hd == 64) return launch_by_rows<KVT, 64>(ctx, a);
    if (hd == 128) return launch_by_rows<KVT, 128>(ctx, a);
    if (hd == 256) return launch_by_rows<KVT, 256>(ctx, a);
    auto fn = hd == 16 ? tree_row_kernel<KVT, 16> : tree_row_kernel<KVT, 32>;
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
               (float)(1.4426950408889634 / std::sqrt((double)kv->head_dim)), 0, nullptr, nullptr};
    return kv->kv_dtype == CW_F16 ? launch_by_size<_Float16>(ctx, a, kv->head_dim)
                                  : launch_by_size<float>(ctx, a, kv->head_dim);
}
