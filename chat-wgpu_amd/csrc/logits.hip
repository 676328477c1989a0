// Rows of logits under a server's rules: penalties for repeated tokens, biases,
// grammar masks; the likeliest token and its log softmax.
//
// With c_v the times that token v was generated and seen_v whether it occurs at
// all (tokens of the request, nodes that the row sees):
//   l_v = x_v; seen_v: l_v > 0 ? l_v / repeat : l_v * repeat;
//   l_v -= frequency c_v + presence [c_v > 0]; l_v += bias_v; not allowed: -inf.
// The token is t = argmax l, its log softmax -log(1 + s), s = sum of exp(l_v -
// l_t) over v != t.  s is kept without the token's own 1, which for a likely
// token would take all of s's digits.
//
// One pass over the logits.  A workgroup has a slice of a row's vocabulary, whose
// logits its threads ask for first and keep in registers.  It counts the slice's tokens
// in LDS: it reads the request's whole history, eight tokens a thread in flight, and
// keeps what falls into its slice, so no count goes through memory.  Counts are whole
// numbers and a bias is chosen by its place in the list, so the order of the LDS
// atomics does not show.  Each wave then has its largest logit, and one exponential for
// each other.  (max, s, index) of the slices are joined by a second launch in a fixed
// order.
//
// What bounds it, at 151936 tokens: for one row the latencies of two launches, one behind
// the other (5.3 + 2.8 us).  61 rows after 4100 tokens take 19 to 20 us for 37 MB: vector
// units 0.70 busy, the counts 8 us of the whole (each of the 38 slices reads the history).
// 48 rows with masks, biases and out take 20.7 us for 59 MB.

#include "paged_device.hpp"
#include "prompt_device.hpp"

namespace {

using namespace cwi;

constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;  // a token's count: seen, though not generated

struct LogitArgs {
    cw_logit_rules r;
    const int *first_row;
    int n_seq, batch_rows;
    const uint32_t *mask;
    int mask_words;
    const int *at;
    const float *x;
    size_t stride;
    int vocab;
    float *out;
    size_t out_stride;
    int parts;         // workgroups a row
    struct Top *part;  // [rows][parts]; null: no token is wanted
    uint32_t *token;
    float *logprob;
};

constexpr int kNone = -1, kPadding = -2;

// The largest of some logits, its index (kNone: all are -inf or NaN), and the sum
// of exp(l - m) over the others.
struct Top {
    float m, s;
    int i;
};

__device__ __forceinline__ Top join(Top a, Top b) {
    if (b.i >= 0 && (a.i < 0 || b.m > a.m || (b.m == a.m && b.i < a.i))) {
        const Top t = a;
        a = b;
        b = t;
    }
    if (b.i >= 0) a.s += (1.0f + b.s) * expf(b.m - a.m);
    else a.s += b.s;  // 0 or NaN
    return a;
}

template <typename V>
__device__ __forceinline__ V rule(const V *p, int b, V none) {
    return p ? p[b] : none;
}

// Requests from b0 on, one a lane (past the last one the last again).
struct Owners {
    int r0, r1;
};
__device__ __forceinline__ Owners owners(const LogitArgs &a, int b0) {
    const int b = min(b0 + (int)(threadIdx.x & 63), a.n_seq - 1);
    return Owners{a.first_row[b], a.first_row[b + 1]};
}

// The request whose rows the batch row is among, n_seq if none; by every wave.  Of more
// than 64 the 64 are looked at whose first begins at or before the row and the next 64's
// behind it; where first_row does not ascend, all of them in turn.
__device__ __forceinline__ int owner_of(const LogitArgs &a, Owners o, int br) {
    auto among = [&](int b0) {
        const uint64_t has = __ballot(o.r0 >= 0 && o.r0 <= br && br < o.r1 && o.r1 <= a.batch_rows);
        return has ? min(b0 + __builtin_ctzll(has), a.n_seq - 1) : a.n_seq;
    };
    int b = among(0);
    if (b < a.n_seq || a.n_seq <= 64) return b;
    const int lane = threadIdx.x & 63, runs = (a.n_seq + 63) / 64;
    int run = -1;
    for (int i = 0; i < runs; i += 64)
        run += __builtin_popcountll(
            __ballot(i + lane < runs && a.first_row[64 * min(i + lane, runs - 1)] <= br));
    if (run > 0) {
        o = owners(a, 64 * run);
        b = among(64 * run);
        if (b < a.n_seq) return b;
    }
    for (int b0 = 64; b0 < a.n_seq; b0 += 64) {
        o = owners(a, b0);
        b = among(b0);
        if (b < a.n_seq) return b;
    }
    return a.n_seq;
}

// IT runs of V logits a thread, V = 4 where rows are 16-byte aligned and whole fours.
template <int V, int IT>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitArgs a) {
    constexpr int N = V * IT, kSlice = kThreads * N;
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ Top tops[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.y;
    const int lo = blockIdx.x * kSlice, n = min(kSlice, a.vocab - lo);
    const bool counts = a.r.tokens || a.r.node_token, biased = a.r.bias;
    uint32_t *const count = lds, *const last = lds + (counts ? kSlice : 0);

    // What is to come from memory is asked for in the order of its use.
    const Owners first = owners(a, 0);
    const int br = a.at ? a.at[row] : (int)row;
    // the thread's logits: V from at(0), V from at(1), ...
    auto at = [&](int it) { return (it * kThreads + tid) * V; };
    const float *x = a.x + row * a.stride + lo;
    float l[N];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
#pragma unroll
        for (int j = 0; j < V; ++j) l[it * V + j] = -INFINITY;
        if (at(it) < n) {
            if constexpr (V == 4) {
                const float4 q = *reinterpret_cast<const float4 *>(x + at(it));
                l[4 * it] = q.x;
                l[4 * it + 1] = q.y;
                l[4 * it + 2] = q.z;
                l[4 * it + 3] = q.w;
            } else {
                l[it] = x[at(it)];
            }
        }
    }
    uint32_t bits[IT];
    const uint32_t *allowed = nullptr;
    if (a.r.allowed) {
        const int k = a.r.allowed_row ? a.r.allowed_row[row] : (int)row;
        if ((unsigned)k < (unsigned)a.r.n_allowed) allowed = a.r.allowed + (size_t)k * a.r.allowed_words;
    }
#pragma unroll
    for (int it = 0; it < IT; ++it)
        bits[it] = allowed && at(it) < n ? allowed[(lo + at(it)) >> 5] : ~0u;

    const int tables = counts + biased;
    for (int v = tid; v < tables * kSlice / 4; v += kThreads)
        reinterpret_cast<uint4 *>(lds)[v] = make_uint4(0, 0, 0, 0);
    const int b = owner_of(a, first, br);
    if (b == a.n_seq) {
        if (a.part && tid == 0) a.part[row * a.parts + blockIdx.x].i = kPadding;
        return;
    }
    const float given = rule(a.r.repeat, b, 1.0f);
    const float presence = rule(a.r.presence, b, 0.0f), frequency = rule(a.r.frequency, b, 0.0f);
    const bool penal = given != 1.0f || presence != 0.0f || frequency != 0.0f;
    const int len = a.r.tokens && penal ? min(max(a.r.length[b], 0), a.r.max_len) : 0;
    const int prompt = rule(a.r.prompt, b, 0);
    const int r0 = a.first_row[b], nodes = a.first_row[b + 1] - r0, self = br - r0;
    const int e0 = biased ? a.r.bias_first[b] : 0, e1 = biased ? a.r.bias_first[b + 1] : 0;
    if (tables) {
        lds_barrier();
        auto add = [&](int v, bool made) {
            if ((unsigned)(v - lo) < (unsigned)n) {
                if (made) atomicAdd(&count[v - lo], 1u);
                else atomicOr(&count[v - lo], kPrompt);
            }
        };
        constexpr int U = 8;
        const int *t = a.r.tokens + (size_t)b * a.r.max_len;
        for (int i = tid; i < len; i += U * kThreads) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = t[min(i + u * kThreads, len - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * kThreads < len) add(v[u], i + u * kThreads >= prompt);
        }
        if (a.r.node_token && penal)
            for (int j = tid; j < nodes; j += kThreads) {
                const bool sees =
                    !a.mask ? j <= self
                            : j < 32 * a.mask_words &&
                                  (a.mask[(size_t)br * a.mask_words + (j >> 5)] >> (j & 31) & 1);
                const int v = a.r.node_token[r0 + j];
                if (sees) add(v, true);
            }
        if (biased && e0 >= 0 && e1 <= a.r.n_bias)
            for (int e = e0 + tid; e < e1; e += kThreads) {
                const int v = a.r.bias_token[e];
                if ((unsigned)(v - lo) < (unsigned)n) atomicMax(&last[v - lo], (uint32_t)e + 1);
            }
        lds_barrier();
    }

    // Where a wave has tokens that were seen, all its logits go through their rules: under
    // a branch each, waves with some would take it for nearly every logit.  With inv the
    // nearest to 1 / repeat, v inv and one step after it are v / repeat to its last bit, as
    // long as the remainder, 2^-24 of v, is in f32's normal range (infinities and zeros have
    // no step; of a quotient within two steps of f32's largest v inv may be infinite).
    // 1 / repeat is finite from 2^-126 on (compared as whole numbers, by the scalar units;
    // dividing where it is not, or waiting for repeat further up, cost every call 1 %).
    const float repeat = __builtin_bit_cast(float, max(__builtin_bit_cast(int, given), 0x00800000));
    const float inv = 1.0f / repeat;
    float m = -INFINITY;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        if (counts) {
            uint32_t c[V], any = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) any |= c[j] = count[at(it) + j];
            if (__any(any)) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const uint32_t made = c[j] & ~kPrompt;
                    float v = l[it * V + j];
                    const float q = v * inv, step = __builtin_fmaf(__builtin_fmaf(-q, repeat, v), inv, q);
                    const float less = step == step ? step : q;
                    v = c[j] ? (v > 0.0f ? less : v * repeat) : v;
                    // (0 added would make a -0 that no rule is for 0)
                    l[it * V + j] = __builtin_fmaf(made ? -frequency : -0.0f, (float)made, v) -
                                    (made ? presence : 0.0f);
                }
            }
        }
        if (biased) {
            uint32_t e[V], any = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) any |= e[j] = last[at(it) + j];
            if (__any(any)) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e[j]) l[it * V + j] += a.r.bias[e[j] - 1];
            }
        }
        if (allowed) {
            const uint32_t allow = bits[it] >> ((lo + at(it)) & 31);
#pragma unroll
            for (int j = 0; j < V; ++j) l[it * V + j] = allow >> j & 1 ? l[it * V + j] : -INFINITY;
        }
        if (a.out && at(it) < n) {
            float *o = a.out + row * a.out_stride + lo + at(it);
            if constexpr (V == 4)
                *reinterpret_cast<float4 *>(o) =
                    make_float4(l[4 * it], l[4 * it + 1], l[4 * it + 2], l[4 * it + 3]);
            else
                o[0] = l[it];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, l[it * V + j]);
    }
    if (!a.part) return;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    // the wave's largest: the first of those that equal it, the others among the rest
    Top top{m, 0.0f, kNone};
    int same = 0;
    if (m > -INFINITY)
#pragma unroll
        for (int it = IT - 1; it >= 0; --it) {
            uint64_t is[V], any = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                is[j] = __ballot(l[it * V + j] == m);
                any |= is[j];
                same += __builtin_popcountll(is[j]);
            }
            if (any) {
                const int from = __builtin_ctzll(any);
                int j = V - 1;
#pragma unroll
                for (int k = V - 2; k >= 0; --k) j = is[k] >> from & 1 ? k : j;
                top.i = lo + (it * kThreads + wave * 64 + from) * V + j;
            }
        }
    // exp(d) = (2^(d log2(e) / 2))^2, so that small ones keep their bits; log2(e) / 2 in
    // two parts, for one rounding of the product
    constexpr float kHi = 0x1.715476p-1f, kLo = 0x1.4ae0cp-27f;
    const float below = top.i >= 0 ? m : 0.0f;  // (-inf - -inf)
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float d = l[k] - below;
        float e = __builtin_amdgcn_exp2f(__builtin_fmaf(d, kHi, d * kLo));
        e = l[k] == m ? 0.0f : e;  // (of two infinities e is NaN)
        s = __builtin_fmaf(e, e, s);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if (lane == 0) {
        // (m - m: of two infinities the difference is NaN, here as in join)
        top.s = same > 1 ? s + ((float)(same - 1) + (m - m)) : s;
        tops[wave] = top;
    }
    __syncthreads();
    if (tid == 0) {
        top = tops[0];
        for (int w = 1; w < kThreads / 64; ++w) top = join(top, tops[w]);
        a.part[row * a.parts + blockIdx.x] = top;
    }
}

// A wave a row: each lane joins slices 64 apart, then the lanes' largest is found and
// their sums, under it, are added: 2.8 us for 149 slices of one row (4.5 with the lanes
// joined in pairs, an exponential each time).
__global__ __launch_bounds__(64) void logits_join_kernel(LogitArgs a) {
    constexpr int U = 4;  // slices in flight
    const size_t row = blockIdx.x;
    const Top *p = a.part + row * a.parts;
    const int first = p[0].i;
    Top top{-INFINITY, 0.0f, kNone};
    for (int i = threadIdx.x; i < a.parts; i += 64 * U) {
        Top t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) t[u] = p[min(i + 64 * u, a.parts - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + 64 * u < a.parts) top = join(top, t[u]);
    }
    if (first == kPadding) return;  // (every slice of a padding row says so)
    float m = top.m;
    int best = top.i >= 0 ? top.i : INT_MAX;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float om = __shfl_xor(m, d);
        const int oi = __shfl_xor(best, d);
        if (oi != INT_MAX && (best == INT_MAX || om > m || (om == m && oi < best))) {
            m = om;
            best = oi;
        }
    }
    float s = top.i < 0 || top.i == best ? top.s : (1.0f + top.s) * expf(top.m - m);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if (threadIdx.x == 0) {
        if (a.token) a.token[row] = best != INT_MAX ? (uint32_t)best : CW_NO_TOKEN;
        if (a.logprob) a.logprob[row] = best != INT_MAX ? -log1pf(s) : -INFINITY;
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

using namespace cwi;

extern "C" int cw_logits_rows(cw_ctx *ctx, const cw_logit_rules *rules, const cw_batch *b,
                              const int *at, const float *logits, size_t stride, int rows,
                              int vocab, float *out, size_t out_stride, uint32_t *token,
                              float *logprob) {
    CW_CHECK_ARG(ctx && rules && b && logits, "cw_logits_rows: null argument");
    CW_CHECK_ARG(out || token || logprob, "cw_logits_rows: no output");
    CW_CHECK_ARG(rows > 0 && rows <= 65535 && vocab > 0 && vocab <= 1 << 24,
                 "cw_logits_rows: rows=%d (at most 65535) vocab=%d (2^24)", rows, vocab);
    CW_CHECK_ARG(b->first_row && b->n_seq > 0 && b->n_seq <= 65535 && b->rows > 0 &&
                     b->rows <= kMaxRows,
                 "cw_logits_rows: a batch of n_seq=%d (1 .. 65535) and rows=%d (1 .. 2^23) with first_row",
                 b->n_seq, b->rows);
    CW_CHECK_ARG(!b->mask || b->mask_words > 0, "cw_logits_rows: mask_words=%d", b->mask_words);
    CW_CHECK_ARG(stride >= (size_t)vocab && stride < (1u << 31),
                 "cw_logits_rows: stride %zu of rows of %d logits", stride, vocab);
    if (out) {
        CW_CHECK_ARG(out_stride >= (size_t)vocab && out_stride < (1u << 31),
                     "cw_logits_rows: out_stride %zu of rows of %d logits", out_stride, vocab);
        CW_CHECK_ARG((out == logits && out_stride == stride) ||
                         rows_apart(rows, logits, stride, vocab, out, out_stride, vocab),
                     "cw_logits_rows: rows of logits and out overlap");
    }
    const cw_logit_rules &r = *rules;
    CW_CHECK_ARG(!r.tokens || (r.length && r.max_len > 0),
                 "cw_logits_rows: tokens need their length and max_len=%d", r.max_len);
    CW_CHECK_ARG(!r.bias || (r.bias_first && r.bias_token && r.n_bias > 0),
                 "cw_logits_rows: biases need bias_first, bias_token and n_bias=%d", r.n_bias);
    CW_CHECK_ARG(!r.allowed || (r.n_allowed > 0 && r.allowed_words >= (vocab + 31) / 32),
                 "cw_logits_rows: n_allowed=%d masks of allowed_words=%d for %d tokens",
                 r.n_allowed, r.allowed_words, vocab);
    CW_HIP(hipSetDevice(ctx->device));
    LogitArgs a{};
    a.r = r;
    a.first_row = b->first_row;
    a.n_seq = b->n_seq;
    a.batch_rows = b->rows;
    a.mask = b->mask;
    a.mask_words = b->mask_words;
    a.at = at;
    a.x = logits;
    a.stride = stride;
    a.vocab = vocab;
    a.out = out;
    a.out_stride = out_stride;
    a.token = token;
    a.logprob = logprob;
    const bool wide = aligned16(logits) && stride % 4 == 0 && vocab % 4 == 0 &&
                      (!out || (aligned16(out) && out_stride % 4 == 0));
    // Slices of 4096 tokens where they fill the chip twice, else of 1024 (one row of 151936
    // after 900 tokens 5.4 us, 7.1 with 4096; 61 rows after 4100 19.9 us, 22.8 with 2048).
    const bool few = (long)rows * ((vocab + 4095) / 4096) < 2 * ctx->n_cu;
    const int slice = few ? 1024 : 4096;
    a.parts = (vocab + slice - 1) / slice;
    if (token || logprob) {
        void *scratch = nullptr;
        CW_TRY(ctx_scratch(ctx, (size_t)rows * a.parts * sizeof(Top), &scratch));
        a.part = static_cast<Top *>(scratch);
    }
    const int tables = (r.tokens || r.node_token ? 1 : 0) + (r.bias ? 1 : 0);
    CW_TRY(launch(ctx, "logits_rows",
                  wide ? few ? logits_kernel<4, 1> : logits_kernel<4, 4>
                       : few ? logits_kernel<1, 4> : logits_kernel<1, 16>,
                  dim3(a.parts, rows), dim3(kThreads), tables * slice * 4, a));
    if (!a.part) return CW_OK;
    return launch(ctx, "logits_join", logits_join_kernel, dim3(rows), dim3(64), 0, a);
}
