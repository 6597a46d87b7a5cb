// Arguments of the kernels over a paged cache, and what their wavefronts share:
// finding a row's sequence, and dividing the attention's work.
#pragma once

#include "common.h"
#include "paged.h"

namespace mvlm {

struct KvAppendArgs {
    PagedSeqs batch;
    PagedKv kv;
    const void* qkv;
    int x_dtype;
    int64_t ld;
    int heads;
    FastDiv chunk;                 // by head_dim / 8
    const float* rope;             // [rope_positions][rot / 2][2] cos, sin
    int rope_positions, rot, interleaved;
    uint16_t* q_out;               // [rows][heads][D], the cache's type (bf16 for an 8-bit cache)
    const float* q_weight;         // [D] norms of q and k heads; null: none
    const float* k_weight;
    float eps, per_dim;            // per_dim: 1 / head_dim
};

struct KvReadArgs {
    PagedSeqs batch;
    PagedKv kv;
    FastDiv chunk;                 // by head_dim / 8
    void* k_out;                   // [rows][kv_heads][D], rows ld elements apart; null: not wanted
    void* v_out;
    int dtype;
    int64_t ld;
};

// How one kernel's share of a batch is cut into blocks.
struct PagedDivision {
    int tile;                      // f-rows per tile; 0: there is no such share
    int64_t blocks_per_head;       // blocks wanted per kv head
    int unit_min, unit_step;       // least keys per block, and what a block's keys are a multiple of
    int items;                     // upper bound of the items per kv head
    int records;                   // room in the workspace, in tiles per kv head
    float* ws;                     // partial results of split tiles
    uint32_t* arrived;             // [records][kv_heads] splits that are done, zero between launches
};
// f-rows up to which a sequence next to ones of many stays with tiles of 32 (2048 rows and 8 times
// n on 500 .. 3000 positions, 32 heads of 64: n = 48 179 us and 201 in tiles of 256, 100 198 and
// 203, 200 240 and 217)
constexpr int PAGED_FEW = 128;
constexpr int PAGED_QUEUES = 8;        // one per XCD: their blocks share an L2
constexpr int PAGED_MAX_KV_HEADS = 1024;

struct PagedAttnArgs {
    PagedSeqs batch;
    PagedKv kv;
    const uint16_t* q;             // [rows][heads][D], the cache's type (bf16 for an 8-bit cache)
    void* o;                       // [rows][heads][D]
    int o_dtype, heads, group;     // group: heads per kv head
    float scale_log2;              // scale * log2(e)
    // division of the work (attention_paged.hip): of all sequences, or, where tiles of 256
    // rows are made (many.tile != 0 and the lengths are worth it), of those with
    // few new rows, f = n group <= PAGED_FEW, and of those with more
    PagedDivision few, many;
    uint32_t* made;                // written by the kernel for many rows: whether it made the batch
    int many_least;                // tiles per kv head, times what their keys can be split, that are worth the second kernel
};

hipError_t launch_kv_append(hipStream_t s, const KvAppendArgs& a);
hipError_t launch_kv_read(hipStream_t s, const KvReadArgs& a);
// Fills a's division of the work for a device, all but its memory.
void plan_attention_paged(PagedAttnArgs* a, int num_cus);
// Bytes of partial results and words of counters of a share; placing them.
size_t paged_ws_bytes(const PagedAttnArgs& a, const PagedDivision& d);
size_t paged_words(const PagedAttnArgs& a, const PagedDivision& d);
hipError_t launch_attention_paged(hipStream_t s, const PagedAttnArgs& a, int num_cus);

#if defined(__HIPCC__)

// Sequence of a row of the batch and its span, the same in all lanes; -1 for a
// row of no sequence.  Starts are counted 64 at a time (they do not decrease, so
// the count of those <= row, less one, is the last sequence that starts there,
// and the sequences before it that start there too are empty).
__device__ __forceinline__ int paged_seq_of_row(const PagedSeqs& b, int row, PagedSpan* span) {
    if (!b.row_start) {
        *span = paged_span(row, row + 1, b.kv_len[row], b.rows, b.positions);
        return row;
    }
    const int lane = (int)(threadIdx.x & 63);
    int count = 0;
    for (int base = 0; base < b.seqs; base += 64) {
        const bool before = base + lane < b.seqs && b.row_start[base + lane] <= row;
        count += __popcll(__builtin_amdgcn_ballot_w64(before));
    }
    const int seq = count - 1;
    if (seq < 0) return -1;
    *span = paged_span(b.row_start[seq], b.row_start[seq + 1], b.kv_len[seq], b.rows, b.positions);
    return row >= span->row0 && row < span->row0 + span->n ? seq : -1;
}

// v plus the values of the lanes before (inclusive scan over 64 lanes)
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

// Tiles of the attention.  The new rows of a sequence and the heads of a group
// are one axis, f = j group + g (j: new row, g: head in the group), cut into
// tiles of R; the keys of a tile are cut into splits of `unit` keys, the same
// number for every tile of a sequence.  An item is one (tile, split).
struct PagedItem {
    int seq;
    PagedSpan span;
    int tile, split;
    int unit;
    int record;                    // of split 0 of this tile; -1: the tile is not split
};

template <int R, bool MANY>
__device__ __forceinline__ int paged_tiles(const PagedSpan& p, int group, int few) {
    const int64_t f = (int64_t)p.n * group;
    return (f > few) == MANY ? (int)((f + R - 1) / R) : 0;
}

// Keys per block: total work (tiles x keys) over the blocks wanted, at least
// unit_min, rounded up to unit_step.
__device__ __forceinline__ int paged_unit(const PagedDivision& a, int64_t total) {
    int64_t u = (total + a.blocks_per_head - 1) / a.blocks_per_head;
    u = u < a.unit_min ? a.unit_min : u;
    u = (u + a.unit_step - 1) / a.unit_step * a.unit_step;
    return (int)(u > PAGED_MAX_POSITIONS ? PAGED_MAX_POSITIONS : u);
}

__device__ __forceinline__ PagedSpan paged_lane_span(const PagedSeqs& b, int s) {
    if (s >= b.seqs) return PagedSpan{0, 0, 0, 0};
    return b.row_start ? paged_span(b.row_start[s], b.row_start[s + 1], b.kv_len[s], b.rows, b.positions)
                       : paged_span(s, s + 1, b.kv_len[s], b.rows, b.positions);
}

// A share's keys per block and its items per kv head, the same in all lanes.
struct PagedShare {
    int unit, items, few_rows;
    PagedSpan first;               // of the lane-th sequence
};
__device__ __forceinline__ int paged_splits(int len, int unit) { return len > unit ? (len + unit - 1) / unit : 1; }

// few_rows: the f-rows up to which a sequence belongs to the share of few
template <int R, bool MANY>
__device__ __forceinline__ PagedShare paged_share(const PagedAttnArgs& a, const PagedSpan& sp, int few_rows) {
    const PagedSeqs& b = a.batch;
    const PagedDivision& div = MANY ? a.many : a.few;
    const int lane = (int)(threadIdx.x & 63);
    PagedShare sh;
    sh.first = sp;
    sh.few_rows = few_rows;
    int64_t total = 0;
    for (int base = 0; base < b.seqs; base += 64) {
        const PagedSpan p = base ? paged_lane_span(b, base + lane) : sp;
        total += (int64_t)paged_tiles<R, MANY>(p, a.group, few_rows) * p.len;
    }
    // summed over the lanes as two numbers of 24 and 30 bits; read from one lane, so that
    // no branch on it is taken as divergent
    const int64_t lo = __builtin_amdgcn_readlane(wave_scan((int)(total & 0xFFFFFF)), 63);
    const int64_t hi = __builtin_amdgcn_readlane(wave_scan((int)(total >> 24)), 63);
    sh.unit = paged_unit(div, (hi << 24) + lo);
    // A batch whose starts do not decrease makes no more items than were planned for
    // (paged_divide).  One that makes more is not begun at all, so that no counter of
    // splits is left in mid-count; the sum stops short of 2^31.
    constexpr int MOST = 1 << 24;
    int items = 0;
    for (int base = 0; base < b.seqs; base += 64) {
        const PagedSpan p = base ? paged_lane_span(b, base + lane) : sp;
        const int64_t more = (int64_t)paged_tiles<R, MANY>(p, a.group, few_rows) * paged_splits(p.len, sh.unit);
        items += (int)(more < MOST - items ? more : MOST - items);
    }
    sh.items = __builtin_amdgcn_readlane(wave_scan(items), 63);
    if (sh.items > div.items) sh.items = 0;
    return sh;
}

// The index-th item of a share, below its items, the same in all lanes; false if there is none.
template <int R, bool MANY>
__device__ __forceinline__ bool paged_locate(const PagedAttnArgs& a, const PagedShare& share, int index, PagedItem* out) {
    const PagedSeqs& b = a.batch;
    const PagedDivision& div = MANY ? a.many : a.few;
    const int lane = (int)(threadIdx.x & 63);
    int first = 0, record = 0;                             // items and records before these 64 sequences
    for (int base = 0; base < b.seqs; base += 64) {
        const PagedSpan sp = base ? paged_lane_span(b, base + lane) : share.first;
        const int tiles = paged_tiles<R, MANY>(sp, a.group, share.few_rows), splits = paged_splits(sp.len, share.unit);
        const int items = tiles * splits, records = splits > 1 ? tiles * splits : 0;
        const int end = first + wave_scan(items), rec_end = record + wave_scan(records);
        const uint64_t mine = __builtin_amdgcn_ballot_w64(index >= end - items && index < end);
        if (mine) {
            const int l = __builtin_ctzll(mine);
            auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            out->seq = base + l;
            out->span = PagedSpan{at(sp.row0), at(sp.n), at(sp.held), at(sp.len)};
            out->unit = share.unit;
            const int ns = at(splits), r = index - at(end - items);
            const int nth = r / ns;
            out->tile = at(tiles) - 1 - nth;               // the last tile sees the most keys: it starts first
            out->split = r - nth * ns;
            out->record = ns > 1 ? at(rec_end - records) + nth * ns : -1;
            // no batch has more records than planned for (paged_divide); a tile's splits agree on it
            return ns == 1 || out->record <= div.records - ns;
        }
        first = __builtin_amdgcn_readlane(end, 63);
        record = __builtin_amdgcn_readlane(rec_end, 63);
    }
    return false;
}

#endif

}  // namespace mvlm
