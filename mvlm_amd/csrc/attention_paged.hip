// Attention of new rows over their sequences' pages:
//   O[r][h] = sum_t softmax_t(scale q[r][h] . K[t][h / group]) V[t][h / group]
// over the positions t <= the row's own that lie on a page (paged.h).  Q, K, V
// fp16 or bf16, fp32 scores and softmax, O fp32 or the cache's type; a row
// that sees no key is 0.
//
// Few rows read many keys, so the keys' bytes bound it (many rows, whose products
// do, are attention_paged_chunk.hip's).  The new rows of a sequence times the heads
// that share a kv head are one axis, cut into tiles of R = 16 (single tokens) or 32:
// the group's heads read each key once.  The keys of a tile are cut into splits so
// that the batch as a whole, whatever its lengths, makes about the wanted number of
// equal blocks (paged_share, found by every block from the lengths in device memory,
// so that one captured launch serves every step); each wave of a block takes every
// NW-th tile of 32 keys with an online softmax of its own, the block merges its waves
// through LDS, and the block of a tile that ends last merges the splits (paged_merge),
// always in their order.
//
//  * S^T = K Q^T, v_mfma_f32_16x16x32 or 32x32x16: A = R keys straight from memory in
//    the operand's layout (lane l: key l % R, 8 dims from 8 (l / R) on), B = Q.  Lane
//    l's results are row l % R and every (64 / R)-th four keys from 4 (l / R) on, so a
//    row's statistics are per lane.
//  * O^T = V^T P^T: the S^T results of a tile are its B operand as they stand when V^T
//    is read in the same key order, which ds_read_b64_tr_b16 gives from V rows in LDS
//    (lane 4k + i of 16 reads dims 4i .. of key k and receives dim lane % 16 of 4 keys).
//  * K and V of the next tile are asked for while this one is computed, the page of the
//    one behind it before them: a wave has about 12 KB (head_dim 64) in flight.
//  * P is rounded to the cache's type for a 16-bit O, as the rounding of O
//    itself is of that size (bf16 single tokens: kept to 16 bits); for an fp32 O
//    it is kept to 22 bits and more, as the sum of two fp16 or three bf16 parts,
//    one product each (PagedP).
//  * the running maximum moves only when a score exceeds it by more than SLACK
//    (PagedP), so most tiles rescale nothing.
//  * hidden keys may hold anything: their scores are replaced, not added to,
//    and their V rows are staged as zeros.
//
// Measured (fp16 unless said): 16 sequences of 30 .. 2047 positions, 32 heads of 64,
// 132 MB: 31.5 us, 4.2 TB/s (a large copy reaches 5.1); 64 sequences of 1000 .. 1500:
// 121 us, 5.4 TB/s; 4 of 20000 .. 32768, bf16, 32 heads of 128 over 8, 448 MB: 84 us,
// 5.3 TB/s; one of 512: 7.35 us, the launch and a chain of loads (lengths, table, keys).
// Each block walks the lengths of all sequences three times: beyond some 500 that is
// felt (1024 sequences of 200 .. 400, 32 heads of 128 over 8: 373 us, 3.4 TB/s).
#include "attention_paged.h"

#include <algorithm>
#include <climits>

namespace mvlm {

// NW: waves per block
template <int R, int KS, bool BF, int PP, int NW>
__global__ __launch_bounds__(64 * NW, KS <= 2 && NW == 4 ? 3 : 2) void paged_attention_kernel(const PagedAttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int index = (int)(blockIdx.x / (uint32_t)a.kv.kv_heads), h = (int)blockIdx.x - index * a.kv.kv_heads;
    if constexpr (R == 32 && NW == 4)
        if (a.many.tile && *a.made) return;                    // by the kernel for many rows, which ran before
    const PagedShare share = paged_share<R, false>(a, paged_lane_span(a.batch, (int)(threadIdx.x & 63)), INT_MAX);
    if (index < share.items) paged_few_item<R, KS, BF, PP, NW>(a, share, index, h, lds);
}

// Division of a share of the sequences (those of at most PAGED_FEW f-rows or all, or
// those of more) for `blocks` blocks.  The sum of ceil(len / unit) over tiles is at most total / unit
// + tiles, and a tile is split when len > unit, so split tiles make at most
// 2 total / unit records.
static PagedDivision paged_divide(const PagedAttnArgs& a, int tile, int64_t blocks, int64_t tiles, int unit_min,
                                  int unit_step) {
    PagedDivision d{};
    d.tile = tile;
    d.unit_step = unit_step;
    d.unit_min = unit_min;
    d.blocks_per_head = (blocks + a.kv.kv_heads - 1) / a.kv.kv_heads;
    d.items = (int)(d.blocks_per_head + tiles);
    d.records = (int)(2 * d.blocks_per_head);
    return d;
}

void plan_attention_paged(PagedAttnArgs* a, int num_cus) {
    const PagedSeqs& b = a->batch;
    const int64_t f = (int64_t)b.rows * a->group;
    a->few = a->many = PagedDivision{};
    // Tiles of 256 rows pay once they give every CU a block, alone or with their keys split;
    // below that tiles of 32 make more of the chip (768 rows of 32 heads: 12 us, 32 in tiles
    // of 256).  Where what the tables can hold would be enough, both kernels are launched, and
    // the first decides by what is held; the one that has nothing to do costs about 2.5 us (768 rows in a
    // table of 768 positions 13.5 us, of 32768 16.1; 2048 bf16 rows on 8192 303 us without the second launch, 306).
    const bool single = !b.row_start;                          // every sequence has `group` f-rows
    const int64_t tiles256 = (single ? (int64_t)b.seqs * (a->group / CHUNK_R) : f / CHUNK_R) * a->kv.kv_heads;
    const bool many = tiles256 * std::max(1, b.positions / CHUNK_UNIT) >= num_cus;
    a->many_least = (num_cus + a->kv.kv_heads - 1) / a->kv.kv_heads;
    if (many) {
        // a sequence with more than PAGED_FEW f-rows ends in one tile that is not full
        const int64_t tiles = f / CHUNK_R + std::min<int64_t>(b.seqs, f / PAGED_FEW + 1);
        a->many = paged_divide(*a, CHUNK_R, num_cus, tiles, CHUNK_UNIT, CHUNK_KEYS);
    }
    // Tiles of 16 rows where no sequence has more; half of a tile of 32 would be empty (4 of 32768,
    // D = 128: 84 us and 128; 16 of 2047 34.3 and 34.8; one of 512 7.2 and 8.9)
    const int R = single && a->group <= 16 && !many ? 16 : 32;
    const int64_t tiles = single ? (int64_t)b.seqs * ((a->group + R - 1) / R) : f / R + b.seqs;
    // blocks wanted per CU, measured at 1.. 6: 16 rows 2 (16 sequences up to 2047: 30.6 us, 33.3 at
    // 3, 34.0 at 4; 4 of 32768, D = 128: 84.9, 94.7, 88.4), 32 rows 1 (256 rows and 11 single tokens:
    // 28.5 us, 29.7 at 2; 256 and 7 of 8 heads of 128 52.9 and 62.1)
    // Tiles that leave most CUs idle, over tables that do not hold more than 512 keys for
    // each CU, take eight waves instead of four: their splits are few or none (one sequence of
    // 512: 8.4 -> 7.4 us, also where its table has room for more than this rule takes; 4 of 32768 would take
    // 88.4 us instead of 84.8, one of 8192 22.7 instead of 18.8).
    const int64_t heads_tiles = tiles * a->kv.kv_heads;
    const int waves = R == 16 && 2 * heads_tiles <= num_cus && heads_tiles * b.positions <= 512 * (int64_t)num_cus ? 8 : 4;
    a->few = paged_divide(*a, R, (R == 16 ? 2 : 1) * (int64_t)num_cus, tiles, (waves == 8 ? 2 : 1) * PAGED_KEYS * waves,
                          PAGED_KEYS * waves);
}

size_t paged_ws_bytes(const PagedAttnArgs& a, const PagedDivision& d) {
    return (size_t)d.records * a.kv.kv_heads * d.tile * (a.kv.D + 2) * sizeof(float);
}
size_t paged_words(const PagedAttnArgs& a, const PagedDivision& d) { return (size_t)d.records * a.kv.kv_heads; }

template <int R, int KS, bool BF, int PP, int NW>
static hipError_t launch_waves(hipStream_t s, const PagedAttnArgs& a) {
    constexpr int bytes = NW * PagedLayout<R, KS>::REGION + 16;
    if constexpr (bytes > 65536)
        if (const hipError_t e = allow_dynamic_lds<paged_attention_kernel<R, KS, BF, PP, NW>>(bytes); e != hipSuccess) return e;
    const dim3 grid((unsigned)(a.kv.kv_heads * a.few.items));
    if (a.many.tile) launch_kernel_part(LaunchPart::Last, paged_attention_kernel<R, KS, BF, PP, NW>, grid, dim3(64 * NW), (uint32_t)bytes, s, a);
    else launch_kernel(paged_attention_kernel<R, KS, BF, PP, NW>, grid, dim3(64 * NW), (uint32_t)bytes, s, a);
    return hipGetLastError();
}

template <int R, int KS, bool BF, int PP>
static hipError_t launch_few(hipStream_t s, const PagedAttnArgs& a) {
    if constexpr (R == 16)
        if (a.few.unit_step == 8 * PAGED_KEYS) return launch_waves<R, KS, BF, PP, 8>(s, a);
    return launch_waves<R, KS, BF, PP, 4>(s, a);
}

template <int R, int KS>
static hipError_t launch_few_dims(hipStream_t s, const PagedAttnArgs& a) {
    const bool wide = a.o_dtype == MVLM_F32;
    // bf16 single tokens have two parts for a bf16 O as well, as their products cost next to nothing (4 of
    // 32768 85.4 us with one and with two, 64 of 500 .. 1500 18.5 and 18.8, one of 512 7.1 and 7.3; fp16, whose
    // one part is 8 times as fine and whose second is summed apart, 18.5 and 19.1, 7.2 and 7.5)
    if (a.kv.dtype == MVLM_F16) return wide ? launch_few<R, KS, false, 2>(s, a) : launch_few<R, KS, false, 1>(s, a);
    return wide ? launch_few<R, KS, true, 3>(s, a) : launch_few<R, KS, true, R == 16 ? 2 : 1>(s, a);
}

template <int R>
static hipError_t launch_few_rows(hipStream_t s, const PagedAttnArgs& a) {
    if (a.kv.D <= 32) return launch_few_dims<R, 1>(s, a);
    if (a.kv.D <= 64) return launch_few_dims<R, 2>(s, a);
    if (a.kv.D <= 96) return launch_few_dims<R, 3>(s, a);
    return launch_few_dims<R, 4>(s, a);
}

hipError_t launch_attention_paged(hipStream_t s, const PagedAttnArgs& a, int num_cus) {
    if (a.many.tile)
        if (const hipError_t e = launch_attention_paged_chunk(s, a, num_cus); e != hipSuccess) return e;
    return a.few.tile == 16 ? launch_few_rows<16>(s, a) : launch_few_rows<32>(s, a);
}

}  // namespace mvlm
