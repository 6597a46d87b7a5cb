// Index arithmetic of the operators over a paged key/value cache (kv_append.hip,
// attention_paged.hip), shared by kernels, host code and host tests.
//
// A cache holds num_pages pages; K and V of one page are [kv_heads][page_size]
// [head_dim], so one head's slots of a page are contiguous.  A batch holds
// sequences of new rows: sequence s owns rows [row_start[s], row_start[s + 1])
// (row s alone when row_start is null), holds kv_len[s] positions with them, and
// position t lives in slot t % page_size of page table[s][t / page_size].
// Everything read from device memory is clamped before it is used as an index.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define MVLM_HD __host__ __device__ __forceinline__
#else
#define MVLM_HD inline
#endif

namespace mvlm {

constexpr int PAGED_MAX_POSITIONS = 1 << 30;

// n / d for 0 <= n < 2^31 by one multiplication: m = ceil(2^(31 + L) / d) with
// 2^(L - 1) < d <= 2^L is below 2^32 + 1, and its excess m d - 2^(31 + L) < d <= 2^L
// moves n m / 2^(31 + L) by less than 1 / d.
struct FastDiv {
    uint64_t mul;
    int shift;
    int div;
    MVLM_HD int quotient(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};
inline FastDiv fast_div(int d) {
    int L = 0;
    while (((int64_t)1 << L) < d) ++L;
    return FastDiv{((((uint64_t)1 << (31 + L)) + (uint64_t)d - 1) / (uint64_t)d), 31 + L, d};
}

struct PagedKv {
    uint16_t* k;
    uint16_t* v;
    int dtype;
    int num_pages, kv_heads, D;
    FastDiv page;              // by page_size
    // slot of (page, kv head, offset within the page) in units of head_dim
    // elements; below 2^31 (checked on the host)
    MVLM_HD int slot(int page_id, int head, int offset) const {
        return (page_id * kv_heads + head) * page.div + offset;
    }
};

struct PagedSeqs {
    int seqs, rows;
    const int* row_start;      // null: one row per sequence
    const int* kv_len;
    const int* table;
    int width;                 // table entries per sequence
    int positions;             // width * page_size: positions a table can hold
};

// One sequence's share of the batch: rows [row0, row0 + n), `held` positions with
// them, of which `len` have a place in its table.
struct PagedSpan {
    int row0, n, held, len;
    // position of new row j (negative: it has none) and the keys below it that exist
    MVLM_HD int position(int j) const { return held - n + j; }
    MVLM_HD int visible(int j) const {
        const int p = position(j) + 1;
        return p < 0 ? 0 : p < len ? p : len;
    }
};
MVLM_HD int paged_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
// start, stop: row_start[s], row_start[s + 1]; held: kv_len[s]
MVLM_HD PagedSpan paged_span(int start, int stop, int held, int rows, int positions) {
    PagedSpan p;
    p.row0 = paged_clamp(start, 0, rows);
    p.n = paged_clamp(stop, p.row0, rows) - p.row0;
    p.held = paged_clamp(held, 0, PAGED_MAX_POSITIONS);
    p.len = p.held < positions ? p.held : positions;
    return p;
}

}  // namespace mvlm
