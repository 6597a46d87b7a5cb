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
    constexpr int ITEMS = R > 16 ? 4 : 1, SPLITS = R > 16 ? 2 : 8;
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
constexpr int PAGED_R = 16;        // rows per tile
constexpr int PAGED_KEYS = 32;     // keys per wave and step

// threadIdx.x, computed anew where it is called: what follows from it is not kept in
// registers from item to item.
__device__ __forceinline__ int own_thread() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

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

// KS: head_dim <= 32 KS; BF: bf16 cache; PP: parts of P; NW: waves of the block.
// Makes the index-th item, if there is one.
template <int KS, bool BF, int PP, int NW>
__device__ __forceinline__ void paged_few_item(const PagedAttnArgs& a, int unit, int index, int h, uint8_t* lds) {
    using L = PagedLayout<KS>;
    constexpr int DT = 2 * KS, VI = 2 * KS;
    const int tid = own_thread(), lane = tid & 63, wave = tid >> 6;
    const int c16 = lane & 15, g4 = lane >> 4;
    const int D = a.kv.D;
    PagedItem it;
    if (!paged_locate<PAGED_R, false>(a, unit, index, &it)) return;
    const PagedSpan sp = it.span;

    // this lane's row of the tile
    const int f = it.tile * PAGED_R + c16, rows_f = sp.n * a.group;
    const int j = f / a.group, gh = f - j * a.group;
    const int last = f < rows_f ? sp.visible(j) : 0;           // keys below it are visible
    const int first_row = it.tile * PAGED_R / a.group, last_row = min(it.tile * PAGED_R + PAGED_R - 1, rows_f - 1) / a.group;
    const int open_end = sp.visible(first_row);                // keys below it are visible to every row
    const int k_begin = it.split * it.unit, k_end = min(k_begin + it.unit, sp.visible(last_row));
    if (it.split > 0 && k_begin >= k_end) return;              // the merge counts on it (paged_merge)

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
    // page of key kv0 + lane % 32 (asked for a tile before its slot is needed), and
    // that key's slot, -1 where there is none
    const int* table = a.batch.table + (int64_t)it.seq * a.batch.width;
    auto ask_page = [&](int kv0) {
        const int key = kv0 + (lane & 31);
        return key < k_end ? table[a.kv.page.quotient(key)] : -1;
    };
    auto slot_of = [&](int kv0, int page) {
        const int key = kv0 + (lane & 31);
        return page >= 0 && page < a.kv.num_pages ? a.kv.slot(page, h, key - a.kv.page.quotient(key) * a.kv.page.div) : -1;
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
    constexpr int STEP = PAGED_KEYS * NW;
    int page_next = ask_page(kv0 + STEP);
    int slot = slot_of(kv0, ask_page(kv0));
    load_k(slot);
    load_v(slot);
    for (; kv0 < k_end; kv0 += PAGED_KEYS * NW) {
        const uint32_t gone = (uint32_t)__builtin_amdgcn_ballot_w64(slot < 0);
#pragma unroll
        for (int i = 0; i < VI; ++i)
            if (vkey[i] < PAGED_KEYS) {
                if (gone && ((gone >> vkey[i]) & 1u)) vf[i] = u32x4{0u, 0u, 0u, 0u};
                *reinterpret_cast<u32x4*>(vt + vkey[i] * L::VP + vdim[i]) = vf[i];
            }
        // the page of the tile after next is asked for before the loads, so that its
        // wait, an iteration later, does not wait for them
        slot = slot_of(kv0 + STEP, page_next);
        page_next = ask_page(kv0 + 2 * STEP);
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
        if (gone || kv0 + PAGED_KEYS > open_end) {
            asm volatile("");                                  // a branch: few tiles need this
            const int seen = last - kv0 - 4 * g4;
            const uint32_t hid = gone >> (4 * g4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = 16 * (e >> 2) + (e & 3);       // and 4 g4
                if (key >= seen || (hid & (1u << key))) p[e] = -INFINITY;
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
    const PagedParts<PAGED_R> parts(a, a.few, h);
    const int d4 = D / 4;
    for (int i = tid; i < PAGED_R * d4; i += 64 * NW) {
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
            parts.store_out(it.record + it.split, r, d, o);
            if (d == 0) parts.store_ml(it.record + it.split, r, mx, sum);
            continue;
        }
        paged_store4<BF>(a, sp, h, it.tile * PAGED_R + r, d, sum == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * (1.0f / sum));
    }
    if (it.record >= 0) paged_merge<BF, PAGED_R, 64 * NW>(a, a.few, it, h, (uint32_t*)(lds + NW * L::REGION));
}

constexpr int CHUNK_KEYS = 64;     // keys per tile of the kernel for many new rows
constexpr int CHUNK_R = 256;       // its f-rows per tile
hipError_t launch_attention_paged_chunk(hipStream_t s, const PagedAttnArgs& a, int num_cus);

}  // namespace mvlm
