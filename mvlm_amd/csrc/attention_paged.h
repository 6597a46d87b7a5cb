// What the kernels of the attention over a paged cache share (attention_paged.hip for
// few new rows, attention_paged_chunk.hip for many).
#pragma once

#include "common.h"
#include "device_math.h"
#include "paged_ops.h"

namespace mvlm {

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

// (lo, hi) rounded to nearest even, packed; with REST, lo and hi become what was lost
template <bool BF, bool REST>
__device__ __forceinline__ uint32_t round2(float& lo, float& hi) {
    if constexpr (BF) {
        const bf16x2v h = __builtin_convertvector(f32x2{lo, hi}, bf16x2v);
        if constexpr (REST) lo -= (float)h[0], hi -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    } else {
        const f16x2v h = __builtin_convertvector(f32x2{lo, hi}, f16x2v);
        if constexpr (REST) lo -= (float)h[0], hi -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    }
}

// Probabilities are kept relative to a reference that follows a row's maximum: it moves
// when a score exceeds the maximum it was taken from by more than SLACK (in the exp2
// domain), and lies BIAS below that, so they stay up to 2^(SLACK + BIAS).  Numerators
// and sums carry the same factor.  bf16 has fp32's range and rescales seldom.  An fp16 part
// is a multiple of 2^-24, so with the row's largest at 2^12 or above it is off by 2^-37 of
// that at most, and has its 11 bits down to 2^-26 of it (with the largest at 1: to 2^-14, and thousands
// of keys ten nats and more below one lost the same bits).  A second part is rounded 2^11
// times as large and summed apart: both together hold 22 bits down to 2^-26 of the largest
// and are off by 2^-48 of it at most below.
// SLACK 3 costs 1% and less (2048 fp16 rows on 8192, 32 heads of 128 over 8: 326 -> 328 us, 32 heads of 64
// 209 -> 212; SLACK 1 334 and 220), the second sum 3 .. 10% where the matrix cores bound
// (fp32 O: 433 -> 470 us, 312 -> 331; 768 rows 14.0 -> 14.4) and nothing for single tokens.
template <bool BF>
struct PagedP {
    static constexpr float SLACK = BF ? 8.0f : 3.0f, BIAS = BF ? 0.0f : 12.0f;
    static constexpr float REST = BF ? 1.0f : 2048.0f;
};

// Partial results of a split tile: per record (one split of one tile of one kv
// head) its R rows of D floats of unnormalized output, then, behind all records, R
// (max, sum) pairs each.  They cross workgroups, so they move with device-scope
// stores and loads (sc1), and a workgroup's are complete before it counts itself in.
constexpr int SC1 = 16;                // cache policy of a raw buffer access

template <int R>
struct PagedParts {
    __amdgpu_buffer_rsrc_t out, ml;
    int D, kv_heads, h;
    __device__ __forceinline__ PagedParts(const PagedAttnArgs& a, const PagedDivision& d, int head)
        : D(a.kv.D), kv_heads(a.kv.kv_heads), h(head) {
        const int64_t n = (int64_t)d.records * kv_heads * R;
        out = __builtin_amdgcn_make_buffer_rsrc(d.ws, 0, (int)(n * D * 4), 0x00020000);
        ml = __builtin_amdgcn_make_buffer_rsrc(d.ws + n * D, 0, (int)(n * 8), 0x00020000);
    }
    __device__ __forceinline__ int row(int record, int r) const { return (record * kv_heads + h) * R + r; }
    __device__ __forceinline__ void store_out(int record, int r, int d, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), out, (row(record, r) * D + d) * 4, 0, SC1);
    }
    __device__ __forceinline__ void store_ml(int record, int r, float m, float l) const {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{m, l}), ml, row(record, r) * 8, 0, SC1);
    }
    __device__ __forceinline__ f32x4 load_out(int record, int r, int d) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(out, (row(record, r) * D + d) * 4, 0, SC1));
    }
    __device__ __forceinline__ f32x2 load_ml(int record, int r) const {
        return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(ml, row(record, r) * 8, 0, SC1));
    }
};

// four outputs of row f of a tile's sequence, from dim d on
template <bool BF>
__device__ __forceinline__ void paged_store4(const PagedAttnArgs& a, const PagedSpan& sp, int h, int f, int d, f32x4 v) {
    const int j = f / a.group, g = f - j * a.group;
    const int64_t at = ((int64_t)(sp.row0 + j) * a.heads + h * a.group + g) * a.kv.D + d;
    if (a.o_dtype == MVLM_F32)
        *reinterpret_cast<f32x4*>((float*)a.o + at) = v;
    else {
        float e[4] = {v[0], v[1], v[2], v[3]};
        *reinterpret_cast<u32x2*>((uint16_t*)a.o + at) = u32x2{round2<BF, false>(e[0], e[1]), round2<BF, false>(e[2], e[3])};
    }
}

// Ends an item of a split tile, called by all THREADS threads of the block once
// their parts are stored: the block that arrives last of the tile's splits merges
// them, in their order, and leaves the counter at zero.  No block waits for another.
template <bool BF, int R, int THREADS>
__device__ __forceinline__ void paged_merge(const PagedAttnArgs& a, const PagedDivision& div, const PagedItem& it, int h,
                                            uint32_t* lds_word) {
    const PagedSpan sp = it.span;
    const int rows = min(R, sp.n * a.group - it.tile * R), D = a.kv.D;
    // the splits that have keys; those behind them ended at once
    const int splits = max(1, (sp.visible((it.tile * R + rows - 1) / a.group) + it.unit - 1) / it.unit);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t* word = div.arrived + it.record * a.kv.kv_heads + h;
        const uint32_t before = __hip_atomic_fetch_add(word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == (uint32_t)splits - 1) __hip_atomic_store(word, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *lds_word = before;
    }
    __syncthreads();
    if (*lds_word != (uint32_t)splits - 1) return;
    const PagedParts<R> parts(a, div, h);
    const int d4 = D / 4;
    // a thread's share, ITEMS quads of outputs at a time, SPLITS splits of them asked for together
    constexpr int ITEMS = R > 32 ? 4 : R > 16 ? 2 : 1, SPLITS = R > 32 ? 2 : R > 16 ? 4 : 8;
    for (int i0 = (int)threadIdx.x; i0 < rows * d4; i0 += THREADS * ITEMS) {
        int r[ITEMS], d[ITEMS];
        float mx[ITEMS], sum[ITEMS];
        f32x4 o[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = min(i0 + k * THREADS, rows * d4 - 1);
            r[k] = i / d4;
            d[k] = 4 * (i - r[k] * d4);
            mx[k] = -INFINITY;
            sum[k] = 0.0f;
            o[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int s0 = 0; s0 < splits; s0 += SPLITS) {
            f32x2 ml[SPLITS][ITEMS];
            f32x4 ov[SPLITS][ITEMS];
#pragma unroll
            for (int u = 0; u < SPLITS; ++u)
#pragma unroll
                for (int k = 0; k < ITEMS; ++k) {
                    const int rec = it.record + min(s0 + u, splits - 1);
                    ml[u][k] = parts.load_ml(rec, r[k]);
                    ov[u][k] = parts.load_out(rec, r[k], d[k]);
                }
#pragma unroll
            for (int u = 0; u < SPLITS; ++u)
#pragma unroll
                for (int k = 0; k < ITEMS; ++k) {
                    if (s0 + u >= splits || (ml[u][k][0] == -INFINITY && ml[u][k][1] == 0.0f)) continue;   // past the end, or saw no key
                    const float mn = fmaxf(mx[k], ml[u][k][0]);
                    const float f0 = __builtin_amdgcn_exp2f(mx[k] - mn), f1 = __builtin_amdgcn_exp2f(ml[u][k][0] - mn);
                    sum[k] = sum[k] * f0 + ml[u][k][1] * f1;
                    o[k] = o[k] * f0 + ov[u][k] * f1;
                    mx[k] = mn;
                }
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (i0 + k * THREADS < rows * d4)
                paged_store4<BF>(a, sp, h, it.tile * R + r[k], d[k], sum[k] == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o[k] * (1.0f / sum[k]));
    }
}

// ---- few new rows (the method is described in attention_paged.hip) -------------
constexpr int PAGED_KEYS = 32;     // keys per wave and step

// threadIdx.x, computed anew where it is called: what follows from it is not kept in
// registers from item to item.
__device__ __forceinline__ int own_thread() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

template <int R> struct PagedAcc;
template <> struct PagedAcc<16> { typedef f32x4 type; };
template <> struct PagedAcc<32> { typedef f32x16 type; };

// v_mfma_f32_16x16x32 (R = 16) or v_mfma_f32_32x32x16 (R = 32): lane l gives row or
// column l % R and 8 consecutive k from 8 (l / R) on
template <int R, bool BF>
__device__ __forceinline__ typename PagedAcc<R>::type mfma_paged(u32x4 a, u32x4 b, typename PagedAcc<R>::type c) {
    if constexpr (R == 16) {
        if constexpr (BF)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        if constexpr (BF)
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// LDS of a wave: 32 V rows while it runs, R rows of output and their statistics
// when it merges.  V's pitch is 32 mod 64 bytes, so that the 8 rows of 32 bytes
// that half a transposed read touches lie in different banks (R = 16; of R = 32's 4
// rows of 64 bytes, two share banks).
template <int R, int KS32>
struct PagedLayout {
    static constexpr int DP = 32 * KS32;                       // padded head_dim
    static constexpr int VP = DP + 16;                         // halfs
    static constexpr int OP = DP + 4;                          // floats
    static constexpr int P = PAGED_KEYS * VP * 2, STAGE = P + (R > 16 ? PAGED_KEYS * R * 4 : 0);   // V, then probabilities (by key)
    static constexpr int MERGE = R * OP * 4 + 2 * R * 4;
    static constexpr int REGION = ((STAGE > MERGE ? STAGE : MERGE) + 15) / 16 * 16;
};

// The block of R f-rows of a tile and one kv head.  KS: head_dim <= 32 KS; BF: bf16
// cache; PP: parts of P; NW: waves of the block; lds: NW REGIONs and a word.
// Makes the index-th item, if there is one.
template <int R, int KS, bool BF, int PP, int NW>
__device__ __forceinline__ void paged_few_item(const PagedAttnArgs& a, const PagedShare& share, int index, int h, uint8_t* lds) {
    using L = PagedLayout<R, KS>;
    using Acc = typename PagedAcc<R>::type;
    constexpr int NG = 64 / R;                                 // lane groups: l / R
    constexpr int U = 32 / R, S = KS * 4 / NG;                 // products of 32 keys, steps of 8 NG dims
    constexpr int NE = R / 2, STEPS = NE / 8;                  // a lane's keys of 32, steps of 8 of them
    constexpr int DT = L::DP / R, NR = R == 16 ? 4 : 16, VI = 2 * KS;
    const int tid = own_thread(), lane = tid & 63, wave = tid >> 6;
    const int rl = lane % R, g = lane / R;
    const int D = a.kv.D;
    PagedItem it;
    if (!paged_locate<R, false>(a, share, index, &it)) return;
    const PagedSpan sp = it.span;

    // this lane's row of the tile
    const int f = it.tile * R + rl, rows_f = sp.n * a.group;
    const int j = f / a.group, gh = f - j * a.group;
    const int last = f < rows_f ? sp.visible(j) : 0;           // keys below it are visible
    const int first_row = it.tile * R / a.group, last_row = min(it.tile * R + R - 1, rows_f - 1) / a.group;
    const int open_end = sp.visible(first_row);                // keys below it are visible to every row
    const int k_begin = it.split * it.unit, k_end = min(k_begin + it.unit, sp.visible(last_row));
    if (it.split > 0 && k_begin >= k_end) return;              // the merge counts on it (paged_merge)

    u32x4 qf[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int d = 8 * NG * s + 8 * g;
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
    // page of key kv0 + lane % 32 (asked for a tile before it is needed), and where that
    // key is, in 16-byte chunks of the cache (below 2^32, checked on the host)
    const int* table = a.batch.table + (int64_t)it.seq * a.batch.width;
    auto ask_page = [&](int kv0) {
        const int key = kv0 + (lane & 31);
        return key < k_end ? table[a.kv.page.quotient(key)] : -1;
    };
    auto exists = [&](int page) { return page >= 0 && page < a.kv.num_pages; };
    auto chunk_of = [&](int kv0, int page) -> uint32_t {       // a hidden key's: the first, so that it may be read
        const int key = kv0 + (lane & 31);
        return exists(page) ? (uint32_t)a.kv.slot(page, h, key - a.kv.page.quotient(key) * a.kv.page.div) * (uint32_t)cpr : 0u;
    };

    float mrun = -INFINITY, lrun = 0.0f;                       // the reference (PagedP), and this lane's keys' sum
    Acc oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < NR; ++r) oacc[t][r] = 0.0f;

    // K and V of a tile are asked for while the tile before is computed.  For R = 16 K
    // comes as fragments, 64 bytes of each key per load, whose registers are free once its
    // scores are.  For R = 32 those would be 32 bytes, and the L1's accesses per load what
    // bounds it (the texture addresser was busy 65% of the time), so K comes in whole rows,
    // like V, and goes through V's place in LDS before V does: 256 rows and 11 single tokens,
    // 32 heads of 64, 35.7 -> 28.7 us, 8 heads of 128 64 -> 53, 768 rows 14.0 -> 12.1.  Not
    // for head_dims of 72 .. 96, whose rows are no multiple of a line or leave loads half empty
    // (768 rows of 32 heads of 80 22.4 us, staged 23.4; 256 and 11 of 96 41.4 and 40.7), and not
    // for 128 inside the kernel for many rows, more of whose registers it would spill (306 -> 330 us;
    // here 3 spill, outside the key loop).
    constexpr bool STAGED = R == 32 && KS != 3 && (KS < 4 || NW == 4);
    u32x4 kf[U][S], kr[STAGED ? VI : 1], vf[VI];
    uint32_t at[VI];                                           // where this lane's chunks are
    // in the global address space: a generic load counts as one of LDS too, and every wait for LDS
    // would be one for it
    typedef const __attribute__((address_space(1))) u32x4 global_u32x4;
    auto chunk_at = [](const uint16_t* base, uint32_t c) { return (global_u32x4*)((uintptr_t)base + ((uint64_t)c << 4)); };
    auto locate = [&](uint32_t where) {
#pragma unroll
        for (int i = 0; i < VI; ++i) at[i] = __shfl(where, vkey[i] & 31, 64) + (uint32_t)(vdim[i] >> 3);
    };
    auto load_k = [&](uint32_t where) {
        if constexpr (STAGED) {
#pragma unroll
            for (int i = 0; i < VI; ++i) kr[i] = *chunk_at(a.kv.k, at[i]);
            return;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t c = __shfl(where, R * u + rl, 64);  // a hidden key's score is replaced below
            global_u32x4* row = chunk_at(a.kv.k, c + (uint32_t)g);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (NG * (s + 1) * 8 <= 32 * (KS - 1)) kf[u][s] = row[NG * s];
                else kf[u][s] = *chunk_at(a.kv.k, c + (NG * s + g < cpr ? NG * s + g : 0));   // may be past head_dim
            }
        }
    };
    auto load_v = [&] {
#pragma unroll
        for (int i = 0; i < VI; ++i) vf[i] = *chunk_at(a.kv.v, at[i]);
    };
    auto store = [&](const u32x4* from) {                      // a tile's chunks into LDS
#pragma unroll
        for (int i = 0; i < VI; ++i)
            if (64 * i + 64 <= 128 * (KS - 1) || vkey[i] < PAGED_KEYS) *reinterpret_cast<u32x4*>(vt + vkey[i] * L::VP + vdim[i]) = from[i];
    };
    int kv0 = k_begin + PAGED_KEYS * wave;
    constexpr int STEP = PAGED_KEYS * NW;
    int page_next = ask_page(kv0 + STEP);
    const int page = ask_page(kv0);
    uint32_t where = chunk_of(kv0, page), gone_next = (uint32_t)__builtin_amdgcn_ballot_w64(!exists(page));
    locate(where);
    load_k(where);
    load_v();
    for (; kv0 < k_end; kv0 += STEP) {
        const uint32_t gone = gone_next;
        // the page of the tile after next is asked for before the loads, so that its
        // wait, an iteration later, does not wait for them
        auto next = [&] {
            where = chunk_of(kv0 + STEP, page_next);
            gone_next = (uint32_t)__builtin_amdgcn_ballot_w64(!exists(page_next));
            page_next = ask_page(kv0 + 2 * STEP);
            locate(where);
        };
        // dims past head_dim: K's registers hold other dims there
        auto clear_dims = [&] {
            if (D < 32 * KS) {
                asm volatile("");
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < S; ++k)
                        if (NG * (k + 1) * 8 > 32 * (KS - 1) && NG * k + g >= cpr) kf[u][k] = u32x4{0u, 0u, 0u, 0u};
            }
        };
        float p[NE];
        auto scores = [&] {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                Acc s;
#pragma unroll
                for (int r = 0; r < NR; ++r) s[r] = 0.0f;
#pragma unroll
                for (int k = 0; k < S; ++k) s = mfma_paged<R, BF>(kf[u][k], qf[k], s);
#pragma unroll
                for (int r = 0; r < NR; ++r) p[NR * u + r] = s[r];
            }
        };
        if constexpr (STAGED) {
            store(kr);
            asm volatile("" ::: "memory");                     // this wave's LDS: its reads follow its stores
#pragma unroll
            for (int k = 0; k < S; ++k) kf[0][k] = *reinterpret_cast<const u32x4*>(vt + rl * L::VP + 8 * NG * k + 8 * g);
            asm volatile("" ::: "memory");
            next();
            if constexpr (KS < 4) load_k(where);
            clear_dims();
            scores();
            if constexpr (KS == 4) load_k(where);              // the registers do not hold both
        }
        // some rows see only part of this tile: if it holds values that are not finite,
        // 0 x infinity would reach the rows that do not see them (R = 16: the rows are one
        // token's, whose hidden keys are behind k_end)
        bool by_key = false;
        if (R > 16 && kv0 + PAGED_KEYS > open_end && open_end < k_end) {
            asm volatile("");
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < VI; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t e = BF ? 0x7F80u : 0x7C00u;
                    bad |= vkey[i] < PAGED_KEYS && !((gone >> (vkey[i] & 31)) & 1u) && ((vf[i][x] & e) == e || ((vf[i][x] >> 16) & e) == e);
                }
            by_key = __builtin_amdgcn_ballot_w64(bad) != 0;
        }
        if (gone) {
            asm volatile("");                                  // a branch: few tiles need this
#pragma unroll
            for (int i = 0; i < VI; ++i)
                if ((gone >> (vkey[i] & 31)) & 1u) vf[i] = u32x4{0u, 0u, 0u, 0u};
        }
        store(vf);
        if constexpr (!STAGED) next();
        load_v();
        asm volatile("" ::: "memory");                         // this wave's LDS: its reads follow its stores
        if constexpr (!STAGED) {
            clear_dims();
            scores();
            load_k(where);
        }
        if (gone || kv0 + PAGED_KEYS > open_end) {
            asm volatile("");                                  // a branch: few tiles need this
            const int seen = last - kv0 - 4 * g;
            const uint32_t hid = gone >> (4 * g);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int key = 4 * NG * (e >> 2) + (e & 3);   // and 4 g
                if (key >= seen || (hid & (1u << key))) p[e] = -INFINITY;
            }
        }
        float tmax = p[0];
#pragma unroll
        for (int e = 1; e < NE; ++e) tmax = fmaxf(tmax, p[e]);
        tmax *= a.scale_log2;
        if (__builtin_amdgcn_ballot_w64(tmax > mrun + (PagedP<BF>::BIAS + PagedP<BF>::SLACK))) {
            if constexpr (R == 16) tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
            tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
            const float mnew = fmaxf(mrun, tmax - PagedP<BF>::BIAS);
            const float factor = mnew == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mrun - mnew);
            lrun *= factor;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < NR; ++r) oacc[t][r] *= factor;
            mrun = mnew;
        }
        const float msafe = mrun == -INFINITY ? 0.0f : mrun;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[e], a.scale_log2, -msafe));
            lrun += p[e];
        }
        if (R > 16 && by_key) {                                // key by key, over the rows that see the key
            float* pw = (float*)(lds + wave * L::REGION + L::P);
#pragma unroll
            for (int e = 0; e < NE; ++e) pw[(4 * NG * (e >> 2) + 4 * g + (e & 3)) * R + rl] = p[e];
            asm_wait_lgkmcnt<0>();
            for (int key = 0; key < PAGED_KEYS; ++key) {
                const float pk = pw[key * R + rl];
                if (kv0 + key >= last) continue;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const uint16_t v = vt[key * L::VP + R * t + 4 * NG * (r >> 2) + 4 * g + (r & 3)];
                        oacc[t][r] = __builtin_fmaf(pk, BF ? bf16_bits_to_f32(v) : f16_bits_to_f32(v), oacc[t][r]);
                    }
            }
            asm_wait_lgkmcnt<0>();
            for (int i = lane; i < PAGED_KEYS * L::VP / 8; i += 64)   // what follows adds zeros
                *reinterpret_cast<u32x4*>(vt + 8 * i) = u32x4{0u, 0u, 0u, 0u};
            asm_wait_lgkmcnt<0>();
        }
        {
            const uint16_t* vg = vt + (4 * g + ((lane & 15) >> 2)) * L::VP + 16 * ((lane >> 4) & (R / 16 - 1)) + 4 * (lane & 3);
            auto values = [&](int k, int t) {
                lds_i16x4* p0 = (lds_i16x4*)(uintptr_t)lds_offset(vg + 8 * NG * k * L::VP + R * t);
                lds_i16x4* p1 = (lds_i16x4*)(uintptr_t)lds_offset(vg + (8 * NG * k + 4 * NG) * L::VP + R * t);
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p0));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p1));
                return u32x4{lo[0], lo[1], hi[0], hi[1]};
            };
            u32x4 pb[STEPS][PP];
            auto parts = [&](int k) {
#pragma unroll
                for (int w = 0; w < PP; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float &lo = p[8 * k + 2 * e], &hi = p[8 * k + 2 * e + 1];
                        if (w == 1) lo *= PagedP<BF>::REST, hi *= PagedP<BF>::REST;
                        pb[k][w][e] = round2<BF, true>(lo, hi);
                    }
            };
            if constexpr (PP > 1 && PagedP<BF>::REST != 1.0f) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) parts(k);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    Acc rest;
#pragma unroll
                    for (int r = 0; r < NR; ++r) rest[r] = 0.0f;
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) {
                        const u32x4 v = values(k, t);
                        rest = mfma_paged<R, BF>(v, pb[k][1], rest);
                        oacc[t] = mfma_paged<R, BF>(v, pb[k][0], oacc[t]);
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) oacc[t][r] = __builtin_fmaf(rest[r], 1.0f / PagedP<BF>::REST, oacc[t][r]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    parts(k);
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        const u32x4 v = values(k, t);
#pragma unroll
                        for (int w = 0; w < PP; ++w) oacc[t] = mfma_paged<R, BF>(v, pb[k][w], oacc[t]);
                    }
                }
            }
        }
        asm volatile("" ::: "memory");
    }
    if constexpr (R == 16) lrun += __shfl_xor(lrun, 16, 64);
    lrun += __shfl_xor(lrun, 32, 64);

    // merge the waves: each parks its rows, then the block combines them
    float* om = (float*)(lds + wave * L::REGION);              // [R][OP]
    float* ml = om + R * L::OP;                                // max[R], sum[R]
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < NR; r += 4)
            *reinterpret_cast<f32x4*>(om + rl * L::OP + R * t + NG * r + 4 * g) = f32x4{oacc[t][r], oacc[t][r + 1], oacc[t][r + 2], oacc[t][r + 3]};
    if (g == 0) {
        ml[rl] = mrun;
        ml[R + rl] = lrun;
    }
    __syncthreads();
    const PagedParts<R> parts(a, a.few, h);
    const int d4 = D / 4;
    for (int i = tid; i < R * d4; i += 64 * NW) {
        const int r = i / d4, d = 4 * (i - r * d4);
        if (it.tile * R + r >= rows_f) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) mx = fmaxf(mx, ((const float*)(lds + w * L::REGION))[R * L::OP + r]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float* rw = (const float*)(lds + w * L::REGION);
            const float e = __builtin_amdgcn_exp2f(rw[R * L::OP + r] - ref);
            sum += e * rw[R * L::OP + R + r];
            o += e * *reinterpret_cast<const f32x4*>(rw + r * L::OP + d);
        }
        if (it.record >= 0) {
            parts.store_out(it.record + it.split, r, d, o);
            if (d == 0) parts.store_ml(it.record + it.split, r, mx, sum);
            continue;
        }
        paged_store4<BF>(a, sp, h, it.tile * R + r, d, sum == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * (1.0f / sum));
    }
    if (it.record >= 0) paged_merge<BF, R, 64 * NW>(a, a.few, it, h, (uint32_t*)(lds + NW * L::REGION));
}

constexpr int CHUNK_KEYS = 64;     // keys per tile of the kernel for many new rows
constexpr int CHUNK_R = 256;       // its f-rows per tile
constexpr int CHUNK_UNIT = 1024;   // its least keys per split
// The launch that comes first where a batch may be worth tiles of 256 rows (a.many.tile).
hipError_t launch_attention_paged_chunk(hipStream_t s, const PagedAttnArgs& a, int num_cus);

}  // namespace mvlm
