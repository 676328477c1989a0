// Shared by the operators of several requests in one paged cache (paged.hip,
// tree_attention.hip): where a request's position lies in the cache.

#pragma once

#include "cw_internal.hpp"

namespace cwi {

// Slots of request b: through its table row (page a power of two, 1 << shift),
// or slots b*page .. b*page + page - 1 of its own where there are no tables.
struct PageMap {
    const int *tables;
    int max_blocks, page, shift, n_blocks;
};

// The slot of position p of request b; -1 where no block of the cache holds it.
__device__ __forceinline__ int slot_of(const PageMap &m, int b, int p) {
    if (!m.tables) return p >= 0 && p < m.page ? b * m.page + p : -1;
    const int e = p >> m.shift;
    if ((unsigned)e >= (unsigned)m.max_blocks) return -1;
    const int id = m.tables[(size_t)b * m.max_blocks + e];
    return (unsigned)id < (unsigned)m.n_blocks ? (id << m.shift) + (p & (m.page - 1)) : -1;
}

constexpr int kMaxRows = 1 << 23;  // of a call: a launch takes under 2^32 threads

// Checks of cw_kv_pages and of the tables of a cw_batch; *map on success.
int check_pages(const char *what, const cw_kv_pages *kv, const cw_batch *b, bool need_kv,
                PageMap *map);

// Sums over the lanes up to this one, of no negative values; those under 2^24
// are added in 32 bits along the lanes.
__device__ __forceinline__ long long wave_scan(long long v, int lane) {
    if (!__any(v >> 24 != 0)) {
        int x = (int)v;
#define CW_SCAN_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, true)
        CW_SCAN_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
        CW_SCAN_STEP(0x112, 0xf);
        CW_SCAN_STEP(0x114, 0xf);
        CW_SCAN_STEP(0x118, 0xf);
        CW_SCAN_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
        CW_SCAN_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef CW_SCAN_STEP
        return x;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Whether `rows` rows of wa floats, sa apart from a on, and of wb floats, sb
// apart from b on, share no float.  Rows of different strides that lie within
// each other's range count as sharing one.
bool rows_apart(int rows, const float *a, size_t sa, size_t wa, const float *b, size_t sb,
                size_t wb);

// The rows r0 .. r0 + n - 1 of request b and its cached positions; n = 0 where
// the device arrays hold something else than a range of rows.
struct SeqRows {
    int r0, n, cached;
};
__device__ __forceinline__ SeqRows seq_rows(const int *first_row, const int *cached, int rows,
                                            int b) {
    const int r0 = first_row[b], r1 = first_row[b + 1], c = cached[b];
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= rows && c >= 0 && c <= (1 << 30) - (r1 - r0);
    return SeqRows{ok ? r0 : 0, ok ? r1 - r0 : 0, ok ? c : 0};
}

}  // namespace cwi
