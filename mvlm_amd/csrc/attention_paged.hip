// Attention of new rows over their sequences' pages:
//   O[r][h] = sum_t softmax_t(scale q[r][h] . K[t][h / group]) V[t][h / group]
// over the positions t <= the row's own that lie on a page (paged.h).  Q, K, V
// fp16 or bf16, fp32 scores and softmax, O fp32 or the cache's type; a row
// that sees no key is 0.
//
// Few rows read many keys, so the keys' bytes bound it.  The new rows of a
// sequence times the heads that share a kv head are one axis, cut into tiles of
// 16: the group's heads read each key once.  The keys of a tile are cut into
// splits so that the batch as a whole, whatever its lengths, makes about the
// wanted number of equal blocks (paged_find); each wave of a block takes every
// NW-th tile of 32 keys with an online softmax of its own, the block merges
// its waves through LDS, and a second kernel merges the splits.
//
//  * S^T = K Q^T, v_mfma_f32_16x16x32: A = 16 keys straight from memory in the
//    operand's layout (lane l: key l % 16, dims 8 (l / 16) .. +7), B = Q.  Lane
//    l's results are row l % 16 and keys 4 (l / 16) .. +3, so a row's
//    statistics are per lane.
//  * O^T = V^T P^T: the two S^T results of a tile are its B operand as they
//    stand when V^T is read in the same key order, keys 4g .. 4g+3 and
//    16+4g .. +3 for g = l / 16, which ds_read_b64_tr_b16 gives from V rows in
//    LDS (lane 4k + i of 16 reads dims 4i .. of key k and receives dim
//    lane % 16 of 4 keys).
//  * P is rounded to the cache's type for a 16-bit O, as the rounding of O
//    itself is of that size; for an fp32 O it is kept to 22 bits and more, as
//    the sum of two fp16 or three bf16 parts, one product each.
//  * the running maximum moves only when a score exceeds it by more than 8 (in
//    the exp2 domain), so P stays below 2^8 and most tiles rescale nothing.
//  * hidden keys may hold anything: their scores are replaced, not added to,
//    and their V rows are staged as zeros.
#include "attention_paged.h"

#include <algorithm>

namespace mvlm {

constexpr int PAGED_R = 16;        // rows per tile
constexpr int PAGED_KEYS = 32;     // keys per wave and step
constexpr int PAGED_NW = 4;        // waves per block

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// LDS of a wave: 32 V rows while it runs, 16 rows of output and their statistics
// when it merges.  V's pitch is 32 mod 64 bytes, so that the 8 rows of 32 bytes
// that half a transposed read touches lie in different banks.
template <int KS>
struct PagedLayout {
    static constexpr int DP = 32 * KS;                         // padded head_dim
    static constexpr int VP = DP + 16;                         // halfs
    static constexpr int OP = DP + 4;                          // floats
    static constexpr int STAGE = PAGED_KEYS * VP * 2;
    static constexpr int MERGE = PAGED_R * OP * 4 + 2 * PAGED_R * 4;
    static constexpr int REGION = ((STAGE > MERGE ? STAGE : MERGE) + 15) / 16 * 16;
};

// KS: head_dim <= 32 KS; BF: bf16 cache; PP: parts of P
template <int KS, bool BF, int PP>
__global__ __launch_bounds__(64 * PAGED_NW) void paged_attention_kernel(const PagedAttnArgs a) {
    using L = PagedLayout<KS>;
    constexpr int DT = 2 * KS, VI = 2 * KS, NW = PAGED_NW;
    __shared__ __attribute__((aligned(16))) uint8_t lds[NW * L::REGION];
    const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int D = a.kv.D, index = (int)(blockIdx.x / (uint32_t)a.kv.kv_heads);
    const int h = (int)blockIdx.x - index * a.kv.kv_heads;
    PagedItem it;
    if (!paged_find<PAGED_R, false, false>(a, index, &it)) return;
    const PagedSpan sp = it.span;

    // this lane's row of the tile
    const int f = it.tile * PAGED_R + c16, rows_f = sp.n * a.group;
    const int j = f / a.group, gh = f - j * a.group;
    const int last = f < rows_f ? sp.visible(j) : 0;           // keys below it are visible
    const int first_row = it.tile * PAGED_R / a.group, last_row = min(it.tile * PAGED_R + PAGED_R - 1, rows_f - 1) / a.group;
    const int open_end = sp.visible(first_row);                // keys below it are visible to every row
    const int k_begin = it.split * it.unit, k_end = min(k_begin + it.unit, sp.visible(last_row));
    if (it.split > 0 && k_begin >= k_end) return;              // the combine knows (paged_combine_kernel)

    u32x4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = 32 * s + 8 * g4;
        qf[s] = u32x4{0u, 0u, 0u, 0u};
        if (f < rows_f && d < D)
            qf[s] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(sp.row0 + j) * a.heads + h * a.group + gh) * D + d);
    }

    uint16_t* vt = (uint16_t*)(lds + wave * L::REGION);        // [32 keys][VP]
    const int cpr = D / 8;
    int vkey[VI], vdim[VI];                                    // V chunk c = lane + 64 i: key c / cpr, dims 8 (c % cpr)
#pragma unroll
    for (int i = 0; i < VI; ++i) {
        const int c = lane + 64 * i;
        vkey[i] = c / cpr;
        vdim[i] = 8 * (c - vkey[i] * cpr);
    }
    const int* table = a.batch.table + (int64_t)it.seq * a.batch.width;
    // slot of key kv0 + lane % 32, -1 where there is none
    auto find_slot = [&](int kv0) {
        const int key = kv0 + (lane & 31);
        if (key >= k_end) return -1;
        const int pi = a.kv.page.quotient(key), page = table[pi];
        return page >= 0 && page < a.kv.num_pages ? a.kv.slot(page, h, key - pi * a.kv.page.div) : -1;
    };

    float mrun = -INFINITY, lrun = 0.0f;                       // lrun: this lane's keys only
    f32x4 oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) oacc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // K fragments and V chunks of a tile are asked for while the tile before is
    // computed: K's registers are free once its scores are, V's once it is in LDS.
    u32x4 kf[2][KS], vf[VI];
    auto load_k = [&](int slot) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int sl = max(__shfl(slot, 16 * u + c16, 64), 0);   // a hidden key's score is replaced below
            const uint16_t* row = a.kv.k + (int64_t)sl * D;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 32 * s + 8 * g4;
                kf[u][s] = *reinterpret_cast<const u32x4*>(row + (d < D ? d : 0));
            }
        }
    };
    auto load_v = [&](int slot) {
#pragma unroll
        for (int i = 0; i < VI; ++i) {
            const int sl = max(__shfl(slot, vkey[i] & 31, 64), 0);
            vf[i] = *reinterpret_cast<const u32x4*>(a.kv.v + (int64_t)sl * D + vdim[i]);
        }
    };
    int kv0 = k_begin + PAGED_KEYS * wave;
    int slot = find_slot(kv0);
    load_k(slot);
    load_v(slot);
    int slot_next = find_slot(kv0 + PAGED_KEYS * NW);
    for (; kv0 < k_end; kv0 += PAGED_KEYS * NW) {
        const uint32_t gone = (uint32_t)__builtin_amdgcn_ballot_w64(slot < 0);
#pragma unroll
        for (int i = 0; i < VI; ++i)
            if (vkey[i] < PAGED_KEYS) {
                if (gone && ((gone >> vkey[i]) & 1u)) vf[i] = u32x4{0u, 0u, 0u, 0u};
                *reinterpret_cast<u32x4*>(vt + vkey[i] * L::VP + vdim[i]) = vf[i];
            }
        slot = slot_next;
        load_v(slot);
        asm volatile("" ::: "memory");                         // this wave's LDS: its reads follow its stores

        float p[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                // dims past head_dim: K's registers hold other dims there
                if (32 * k + 32 > D && 32 * k + 8 * g4 >= D) kf[u][k] = u32x4{0u, 0u, 0u, 0u};
                s = mfma16<BF>(kf[u][k], qf[k], s);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) p[4 * u + r] = s[r];
        }
        load_k(slot);
        slot_next = find_slot(kv0 + 2 * PAGED_KEYS * NW);
        if (gone || kv0 + PAGED_KEYS > open_end) {
            asm volatile("");                                  // a branch: few tiles need this
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = 16 * (e >> 2) + 4 * g4 + (e & 3);
                if (kv0 + i >= last || ((gone >> i) & 1u)) p[e] = -INFINITY;
            }
        }
        float tmax = p[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) tmax = fmaxf(tmax, p[e]);
        tmax *= a.scale_log2;
        if (__builtin_amdgcn_ballot_w64(tmax > mrun + 8.0f)) {
            tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
            tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
            const float mnew = fmaxf(mrun, tmax);
            const float factor = mnew == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mrun - mnew);
            lrun *= factor;
#pragma unroll
            for (int t = 0; t < DT; ++t) oacc[t] *= factor;
            mrun = mnew;
        }
        const float msafe = mrun == -INFINITY ? 0.0f : mrun;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[e], a.scale_log2, -msafe));
            lrun += p[e];
        }
        u32x4 pb[PP];
#pragma unroll
        for (int w = 0; w < PP; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) pb[w][e] = round2<BF, true>(p[2 * e], p[2 * e + 1]);
        const uint16_t* vg = vt + (4 * g4 + (c16 >> 2)) * L::VP + 4 * (c16 & 3);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            lds_i16x4* p0 = (lds_i16x4*)(uintptr_t)lds_offset(vg + 16 * t);
            lds_i16x4* p1 = (lds_i16x4*)(uintptr_t)lds_offset(vg + 16 * t + 16 * L::VP);
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p0));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p1));
#pragma unroll
            for (int w = 0; w < PP; ++w) oacc[t] = mfma16<BF>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pb[w], oacc[t]);
        }
        asm volatile("" ::: "memory");
    }
    lrun += __shfl_xor(lrun, 16, 64);
    lrun += __shfl_xor(lrun, 32, 64);

    // merge the waves: each parks its rows, then the block combines them
    float* om = (float*)(lds + wave * L::REGION);              // [16][OP]
    float* ml = om + PAGED_R * L::OP;                          // max[16], sum[16]
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(om + c16 * L::OP + 16 * t + 4 * g4) = oacc[t];
    if (g4 == 0) {
        ml[c16] = mrun;
        ml[PAGED_R + c16] = lrun;
    }
    __syncthreads();
    const int d4 = D / 4;
    for (int i = (int)threadIdx.x; i < PAGED_R * d4; i += 64 * NW) {
        const int r = i / d4, d = 4 * (i - r * d4);
        if (it.tile * PAGED_R + r >= rows_f) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) mx = fmaxf(mx, ((const float*)(lds + w * L::REGION))[PAGED_R * L::OP + r]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float* rw = (const float*)(lds + w * L::REGION);
            const float e = __builtin_amdgcn_exp2f(rw[PAGED_R * L::OP + r] - ref);
            sum += e * rw[PAGED_R * L::OP + PAGED_R + r];
            o += e * *reinterpret_cast<const f32x4*>(rw + r * L::OP + d);
        }
        if (it.record >= 0) {
            *reinterpret_cast<f32x4*>(paged_ws_out<PAGED_R>(a, it.record + it.split, h) + r * D + d) = o;
            if (d == 0) paged_ws_ml<PAGED_R, false>(a, it.record + it.split, h)[r] = f32x2{mx, sum};
            continue;
        }
        paged_store4<BF>(a, sp, h, it.tile * PAGED_R + r, d, sum == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * (1.0f / sum));
    }
}

// Division of the sequences of at most (or of more than) PAGED_FEW f-rows: `blocks`
// blocks are wanted.  The sum of ceil(len / unit) over tiles is at most total / unit
// + tiles, and a tile is split when len > unit, so split tiles make at most
// 2 total / unit records.
static PagedDivision paged_divide(const PagedAttnArgs& a, int tile, int64_t blocks, int64_t tiles, int unit_step) {
    PagedDivision d{};
    d.tile = tile;
    d.unit_step = unit_step;
    d.unit_min = unit_step;
    d.blocks_per_head = (blocks + a.kv.kv_heads - 1) / a.kv.kv_heads;
    d.tiles = (int)tiles;
    d.items = (int)(d.blocks_per_head + tiles);
    d.records = (int)(2 * d.blocks_per_head);
    return d;
}

size_t plan_attention_paged(PagedAttnArgs* a, int num_cus) {
    const PagedSeqs& b = a->batch;
    const int64_t f = (int64_t)b.rows * a->group;
    const bool single = !b.row_start;                          // every sequence has `group` f-rows
    a->few = a->many = PagedDivision{};
    if (!single || a->group <= PAGED_FEW) {
        const int64_t few = single ? (int64_t)b.seqs * ((a->group + PAGED_R - 1) / PAGED_R) : f / PAGED_R + b.seqs;
        a->few = paged_divide(*a, PAGED_R, 4 * (int64_t)num_cus, few, PAGED_KEYS * PAGED_NW);
    }
    if (single ? a->group > PAGED_FEW : f > PAGED_FEW) {
        const int rw = 1;
        // at most one sequence in PAGED_FEW f-rows has more of them
        a->many = paged_divide(*a, 128 * rw, (int64_t)num_cus * (rw == 1 ? 2 : 1), f / (128 * rw) + std::min<int64_t>(b.seqs, f / PAGED_FEW + 1),
                               256);
    }
    size_t bytes = 0;
    for (const PagedDivision* d : {&a->few, &a->many})
        bytes = std::max(bytes, (size_t)d->records * a->kv.kv_heads * d->tile * (a->kv.D + 2) * sizeof(float));
    return bytes;
}

template <int KS, bool BF, int PP>
static void launch_few(PagedLaunch& go) {
    go(paged_attention_kernel<KS, BF, PP>, go.a.few.items);
    go(paged_combine_kernel<BF, PAGED_R, false>, go.a.few.tiles);
}

template <int KS>
static void launch_few_dims(PagedLaunch& go) {
    const bool wide = go.a.o_dtype == MVLM_F32;
    if (go.a.kv.dtype == MVLM_F16) {
        if (wide) launch_few<KS, false, 2>(go);
        else launch_few<KS, false, 1>(go);
    } else {
        if (wide) launch_few<KS, true, 3>(go);
        else launch_few<KS, true, 1>(go);
    }
}

hipError_t launch_attention_paged(hipStream_t s, const PagedAttnArgs& a) {
    PagedLaunch go{s, a, (a.few.tile ? 2 : 0) + (a.many.tile ? 2 : 0)};
    if (a.many.tile) launch_attention_paged_chunk(go);
    if (a.few.tile) {
        if (a.kv.D <= 32) launch_few_dims<1>(go);
        else if (a.kv.D <= 64) launch_few_dims<2>(go);
        else if (a.kv.D <= 96) launch_few_dims<3>(go);
        else launch_few_dims<4>(go);
    }
    return hipGetLastError();
}

}  // namespace mvlm
