// Attention over a paged cache for sequences with many new rows (see
// attention_paged.hip for the operator and its division into items).
//
// A block of four waves owns 128 RW f-rows of one kv head, wave w rows
// 32 RW w .. of them, and walks the keys in tiles of 64 that all its waves share:
// the matrix cores bound it, and each K or V fragment a wave reads from LDS serves
// its RW products.
//  * K and V tiles go straight from memory to LDS, two buffers each, a tile ahead
//    (16-byte chunks, the waves' loads finding their rows through the table);
//    a hidden key's chunks come from zeros.
//  * LDS rows are CH chunks; chunk c of key k lies at c ^ key_swizzle(k), so that
//    16 lanes reading one chunk of 16 keys touch all 64 banks, and c ^
//    value_swizzle(k), so that the four keys x 64 bytes of half a transposed read do.
//  * S^T = K Q^T and O^T = V^T P^T as above on v_mfma_f32_32x32x16: lane l's
//    results are row l % 32 and keys 8 (r / 4) + 4 (l / 32) + r % 4.
#include "attention_paged.h"

namespace mvlm {

constexpr int CHUNK_KEYS = 64;

__device__ const u32x4 paged_zeros = {0u, 0u, 0u, 0u};

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int CH>
__device__ __forceinline__ int key_swizzle(int key) { return CH == 16 ? key & 15 : (key >> 1) & 7; }
template <int CH>
__device__ __forceinline__ int value_swizzle(int key) { return CH == 16 ? (key & 3) << 2 : ((key >> 1) & 1) << 2; }

// KS: head_dim <= 16 KS; DT: head_dim <= 32 DT; RW: 32-row tiles per wave
template <int KS, int DT, bool BF, int PP, int RW>
__global__ __launch_bounds__(256, RW == 1 ? 2 : 1) void paged_chunk_kernel(const PagedAttnArgs a) {
    constexpr int CH = DT > 2 ? 16 : 8, PB = 16 * CH, TILE = CHUNK_KEYS * PB, R = 128 * RW;
    constexpr int NL = CHUNK_KEYS * CH / 256;                  // chunks of K (and of V) per thread and tile
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TILE];   // K0 V0 K1 V1
    const int lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int l32 = lane & 31, h2 = lane >> 5;
    const int D = a.kv.D, index = (int)(blockIdx.x / (uint32_t)a.kv.kv_heads);
    const int h = (int)blockIdx.x - index * a.kv.kv_heads;
    PagedItem it;
    if (!paged_find<R, true, false>(a, index, &it)) return;
    const PagedSpan sp = it.span;
    const int rows_f = sp.n * a.group;
    const int tile_f = it.tile * R, wave_f = tile_f + 32 * RW * wave;
    const int k_begin = it.split * it.unit;
    const int k_end = min(k_begin + it.unit, sp.visible(min(tile_f + R - 1, rows_f - 1) / a.group));
    if (it.split > 0 && k_begin >= k_end) return;              // the combine knows (paged_combine_kernel)
    const int wave_open = wave_f < rows_f ? sp.visible(wave_f / a.group) : 0;   // keys below it are visible to all the wave's rows
    const int wave_end = wave_f < rows_f ? min(k_end, sp.visible(min(wave_f + 32 * RW - 1, rows_f - 1) / a.group)) : 0;

    u32x4 qf[RW][KS];
    int last[RW];                                              // keys below it are visible to the lane's row
#pragma unroll
    for (int t = 0; t < RW; ++t) {
        const int f = wave_f + 32 * t + l32, j = f / a.group, g = f - j * a.group;
        last[t] = f < rows_f ? sp.visible(j) : 0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * h2;
            qf[t][s] = u32x4{0u, 0u, 0u, 0u};
            if (f < rows_f && d < D)
                qf[t][s] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(sp.row0 + j) * a.heads + h * a.group + g) * D + d);
        }
    }

    // the chunks of a row past head_dim: K's are contracted with Q's zeros, and no load reaches them
    if (D < 8 * CH) {
        for (int i = (int)threadIdx.x; i < 4 * TILE / 16; i += 256) *reinterpret_cast<u32x4*>(lds + 16 * i) = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
    }

    const int* table = a.batch.table + (int64_t)it.seq * a.batch.width;
    // slot of key kv0 + lane, -1 where there is none
    auto find_slot = [&](int kv0) {
        const int key = kv0 + lane;
        if (key >= k_end) return -1;
        const int pi = a.kv.page.quotient(key), page = table[pi];
        return page >= 0 && page < a.kv.num_pages ? a.kv.slot(page, h, key - pi * a.kv.page.div) : -1;
    };
    const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_offset(lds));
    auto load_tile = [&](int buf, int slot) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int first = 64 * wave + 256 * i;             // this wave's chunks first .. +63
            const int key = (first + lane) / CH, c = (first + lane) % CH;
            const int sl = __shfl(slot, key, 64);
            const int ck = c ^ key_swizzle<CH>(key), cv = c ^ value_swizzle<CH>(key);
            const uint16_t* k = sl >= 0 ? a.kv.k + (int64_t)sl * D + 8 * ck : (const uint16_t*)&paged_zeros;
            const uint16_t* v = sl >= 0 ? a.kv.v + (int64_t)sl * D + 8 * cv : (const uint16_t*)&paged_zeros;
            const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + 2 * buf * TILE + 16 * first));
            if (8 * ck < D) asm_global_load_lds_b128(k, to);
            if (8 * cv < D) asm_global_load_lds_b128(v, to + TILE);
        }
    };

    float mrun[RW], lrun[RW];                                  // lrun: this lane's keys only
    f32x16 oacc[RW][DT];
#pragma unroll
    for (int t = 0; t < RW; ++t) {
        mrun[t] = -INFINITY;
        lrun[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[t][i][r] = 0.0f;
    }

    int slot = find_slot(k_begin);
    if (k_begin < k_end) load_tile(0, slot);
    int slot_next = find_slot(k_begin + CHUNK_KEYS);
    int buf = 0;
    for (int kv0 = k_begin; kv0 < k_end; kv0 += CHUNK_KEYS, buf ^= 1) {
        const uint64_t gone = __builtin_amdgcn_ballot_w64(slot < 0);
        asm_wait_vmcnt<0>();
        __syncthreads();                                       // this tile is in LDS, and the one before is done with
        slot = slot_next;
        if (kv0 + CHUNK_KEYS < k_end) load_tile(buf ^ 1, slot);
        slot_next = find_slot(kv0 + 2 * CHUNK_KEYS);
        if (kv0 >= wave_end) continue;
        const uint8_t* kt = lds + 2 * buf * TILE;
        const uint8_t* vt = kt + TILE;

        f32x16 s[RW][2];
#pragma unroll
        for (int t = 0; t < RW; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][u][r] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                const int key = 32 * u + l32;
                const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + key * PB + 16 * ((2 * st + h2) ^ key_swizzle<CH>(key)));
#pragma unroll
                for (int t = 0; t < RW; ++t) s[t][u] = mfma32<BF>(kf, qf[t][st], s[t][u]);
            }
        if (gone || kv0 + CHUNK_KEYS > wave_open) {
            asm volatile("");                                  // a branch: few tiles need this
#pragma unroll
            for (int t = 0; t < RW; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = 32 * u + 8 * (r >> 2) + 4 * h2 + (r & 3);
                        if (kv0 + i >= last[t] || ((gone >> i) & 1u)) s[t][u][r] = -INFINITY;
                    }
        }
#pragma unroll
        for (int t = 0; t < RW; ++t) {
            float tmax = s[t][0][0];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[t][u][r]);
            tmax *= a.scale_log2;
            if (__builtin_amdgcn_ballot_w64(tmax > mrun[t] + 8.0f)) {
                const float mnew = fmaxf(mrun[t], fmaxf(tmax, __shfl_xor(tmax, 32, 64)));
                const float factor = mnew == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mrun[t] - mnew);
                lrun[t] *= factor;
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) oacc[t][i][r] *= factor;
                mrun[t] = mnew;
            }
            const float msafe = mrun[t] == -INFINITY ? 0.0f : mrun[t];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[t][u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][r], a.scale_log2, -msafe));
                    lrun[t] += s[t][u][r];
                }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u32x4 pb[RW][PP];
#pragma unroll
                for (int t = 0; t < RW; ++t) {
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = s[t][u][8 * kk + e];
#pragma unroll
                    for (int w = 0; w < PP; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) pb[t][w][e] = round2<BF, true>(p[2 * e], p[2 * e + 1]);
                }
                // this lane's address: key 4 h2 + (lane & 15) / 4 of the step, dims 16 ((lane / 16) & 1) + 4 (lane & 3)
                const int key = 32 * u + 16 * kk + 4 * h2 + ((lane & 15) >> 2);
                const int dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                const uint8_t* vk = vt + key * PB + 2 * (dim & 7);
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    const int c = (4 * i + (dim >> 3)) ^ value_swizzle<CH>(key);   // the same for key + 8
                    lds_i16x4* p0 = (lds_i16x4*)(uintptr_t)lds_offset(vk + 16 * c);
                    lds_i16x4* p1 = (lds_i16x4*)(uintptr_t)lds_offset(vk + 16 * c + 8 * PB);
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p0));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p1));
#pragma unroll
                    for (int t = 0; t < RW; ++t)
#pragma unroll
                        for (int w = 0; w < PP; ++w) oacc[t][i] = mfma32<BF>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pb[t][w], oacc[t][i]);
                }
            }
    }

#pragma unroll
    for (int t = 0; t < RW; ++t) {
        const float sum = lrun[t] + __shfl_xor(lrun[t], 32, 64);
        const int f = wave_f + 32 * t + l32;
        if (f >= rows_f) continue;
        if (it.record >= 0) {
            float* wo = paged_ws_out<R>(a, it.record + it.split, h) + (int64_t)(f - tile_f) * D;
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int d = 32 * i + 8 * q + 4 * h2;
                    if (d < D)
                        *reinterpret_cast<f32x4*>(wo + d) = f32x4{oacc[t][i][4 * q], oacc[t][i][4 * q + 1], oacc[t][i][4 * q + 2], oacc[t][i][4 * q + 3]};
                }
            if (h2 == 0) paged_ws_ml<R, true>(a, it.record + it.split, h)[f - tile_f] = f32x2{mrun[t], sum};
            continue;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * i + 8 * q + 4 * h2;
                if (d < D)
                    paged_store4<BF>(a, sp, h, f, d, f32x4{oacc[t][i][4 * q] * inv, oacc[t][i][4 * q + 1] * inv,
                                                           oacc[t][i][4 * q + 2] * inv, oacc[t][i][4 * q + 3] * inv});
            }
    }
}

template <int KS, int DT, bool BF, int PP>
static void launch_many(PagedLaunch& go) {
    if (go.a.many.tile == 256) {
        go(paged_chunk_kernel<KS, DT, BF, PP, 2>, go.a.many.items);
        go(paged_combine_kernel<BF, 256, true>, go.a.many.tiles);
    } else {
        go(paged_chunk_kernel<KS, DT, BF, PP, 1>, go.a.many.items);
        go(paged_combine_kernel<BF, 128, true>, go.a.many.tiles);
    }
}

template <int KS, int DT>
static void launch_many_dims(PagedLaunch& go) {
    const bool wide = go.a.o_dtype == MVLM_F32;
    if (go.a.kv.dtype == MVLM_F16) {
        if (wide) launch_many<KS, DT, false, 2>(go);
        else launch_many<KS, DT, false, 1>(go);
    } else {
        if (wide) launch_many<KS, DT, true, 3>(go);
        else launch_many<KS, DT, true, 1>(go);
    }
}

void launch_attention_paged_chunk(PagedLaunch& go) {
    const int D = go.a.kv.D;
    if (D <= 32) launch_many_dims<2, 1>(go);
    else if (D <= 64) launch_many_dims<4, 2>(go);
    else if (D <= 80) launch_many_dims<5, 3>(go);
    else if (D <= 96) launch_many_dims<6, 3>(go);
    else launch_many_dims<8, 4>(go);
}

}  // namespace mvlm
