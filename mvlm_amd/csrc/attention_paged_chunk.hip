// Attention over a paged cache for batches in which some sequence may have many new
// rows (attention_paged.hip describes the operator and its division into items).
//
// A block of eight waves owns 256 f-rows of one kv head, wave w rows 32 w .. of
// them, and walks the keys in tiles of 64 that all its waves share.  The matrix
// cores and the vector ALUs bound it about equally: a tile costs a wave 32
// matrix instructions of 32 cycles (head_dim 128) and, for its 2048 scores, about as
// many cycles of exponentials, maxima, sums and conversions.  So the two waves of a
// SIMD (w and w + 4) are half a tile apart.  Iteration i, between two barriers, holds
// the products O^T += V^T P^T of tile i - 1 and S^T = K Q^T of tile i of all waves;
// waves 0..3 run them first and then the softmax of tile i, waves 4..7 run the softmax
// of tile i - 1 first and then the products, so that one wave of a SIMD has matrix
// instructions while the other has vector ones.  The products, and the softmax of waves 4..7, have
// the higher priority.  One barrier per tile is enough, as both groups read K of tile i and V of
// tile i - 1 there, while the tiles after them are on their way into the other buffers
// of a ring: the blocks of one kv head walk its keys in step, so each tile comes from
// memory once for all of them and its loads have to cover that latency.
// 2048 bf16 rows on 8192 positions, 32 heads of 128 over 8 kv heads (309 GFLOP): 302 ..
// 322 us as the clock allows, 960 .. 1023 TFLOP/s, of the 1229 .. 1275 that a large
// library product of that type reaches here; with both groups in step 384 us, with two
// barriers per tile 349.  For an fp32 O, whose probabilities have two (fp16) or three (bf16) parts, 470
// and 510.  At head_dim 128 all 256 registers are in use and 13 to 18 values spill, outside
// the key loop of the tiles of 256 rows.
//  * K and V tiles go straight from memory to LDS in 16-byte chunks; a hidden
//    key's chunks and those past head_dim come from zeros.  Their rows are found through
//    the page table for SLOT_KEYS keys at a time, kept in LDS, so that no load that a wave waits for
//    comes between them.
//  * LDS rows are CH chunks; chunk c of key k lies at c ^ key_swizzle(k), so that
//    16 lanes reading one chunk of 16 keys touch all 64 banks, and c ^
//    value_swizzle(k), so that the four keys x 64 bytes of half a transposed read do.
//  * v_mfma_f32_32x32x16: lane l's results are row l % 32 and keys
//    8 (r / 4) + 4 (l / 32) + r % 4, which are the B operand of the second product
//    as they stand when V^T is read in the same key order.
//  * a tile with keys that some of a wave's rows do not see is checked for values that are
//    not finite (0 x infinity would reach rows that do not see them); if it holds any,
//    its second product is made key by key over the rows that see the key.
// Whether tiles of 256 rows pay depends on the lengths, which only the device knows
// (chunk_worth): this kernel is launched before the one for few rows, and either makes
// the whole batch, the sequences with few new rows as items of paged_few_item behind
// those with many, or ends at once and leaves it to that one (made).  A block fills a
// CU (its LDS), so there is one per CU, and they take items from queues, one per XCD:
// item w belongs to queue w % 8, so with a multiple of 8 kv heads the tiles of a head
// run on one XCD and share its L2.  A sequence's tiles come in order of their keys, the
// most first, and the blocks take them in turn, from the last block to the first in
// every other round, so that who had the longest takes the shortest next.
#include "attention_paged.h"

#include <algorithm>

namespace mvlm {

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

// Barrier between iterations: this wave's LDS reads are complete, its direct loads
// stay in flight, and no instruction moves to the other side.
__device__ __forceinline__ void phase_barrier() {
    asm_wait_lgkmcnt<0>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

constexpr int CHUNK_THREADS = 512;

constexpr uint32_t NOWHERE = 0xFFFFFFFFu;
constexpr int SLOT_KEYS = 2048;                                // keys whose slots LDS holds, twice

template <int DT>
struct ChunkLayout {
    static constexpr int CH = DT > 2 ? 16 : 8;                 // chunks per LDS row
    static constexpr int PB = 16 * CH, TILE = CHUNK_KEYS * PB;
    static constexpr int NB = DT > 2 ? 3 : 4;                  // tiles of the K ring, and of the V ring behind it
    static constexpr int V = NB * TILE, SLOTS = 2 * NB * TILE, P = SLOTS + 2 * SLOT_KEYS * 4;
    static constexpr int P_WAVE = 32 * 32 * 4;                 // 32 keys x 32 rows of probabilities (slow path)
    static constexpr int ZEROS = P + 8 * P_WAVE, BYTES = ZEROS + TILE;   // a V tile of zeros
};

// KS: head_dim <= 16 KS; DT: head_dim <= 32 DT; PP: parts of P
template <int KS, int DT, bool BF, int PP>
__device__ __forceinline__ void paged_chunk_item(const PagedAttnArgs& a, const PagedShare& share, int index, int h, uint8_t* lds) {
    using L = ChunkLayout<DT>;
    constexpr int CH = L::CH, PB = L::PB, TILE = L::TILE, NB = L::NB, R = CHUNK_R;
    constexpr int NL = CHUNK_KEYS * CH / CHUNK_THREADS;        // chunks of K (and of V) per thread and tile
    const int tid = own_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, h2 = lane >> 5;
    const bool second = wave >= 4;
    const int D = a.kv.D;
    PagedItem it;
    if (!paged_locate<R, true>(a, share, index, &it)) return;
    const PagedSpan sp = it.span;
    const int rows_f = sp.n * a.group;
    const int tile_f = it.tile * R, wave_f = tile_f + 32 * wave;
    const int k_begin = it.split * it.unit;
    const int k_end = min(k_begin + it.unit, sp.visible(min(tile_f + R - 1, rows_f - 1) / a.group));
    if (it.split > 0 && k_begin >= k_end) return;              // the merge counts on it (paged_merge)
    const int wave_open = wave_f < rows_f ? sp.visible(wave_f / a.group) : 0;   // keys below it are visible to all the wave's rows
    const int wave_end = wave_f < rows_f ? min(k_end, sp.visible(min(wave_f + 31, rows_f - 1) / a.group)) : 0;

    const int f = wave_f + l32, fj = f / a.group, fg = f - fj * a.group;
    const int last = f < rows_f ? sp.visible(fj) : 0;          // keys below it are visible to the lane's row
    u32x4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = 16 * s + 8 * h2;
        qf[s] = u32x4{0u, 0u, 0u, 0u};
        if (f < rows_f && d < D)
            qf[s] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(sp.row0 + fj) * a.heads + h * a.group + fg) * D + d);
    }
    for (int i = tid; i < TILE / 16; i += CHUNK_THREADS) *reinterpret_cast<u32x4*>(lds + L::ZEROS + 16 * i) = u32x4{0u, 0u, 0u, 0u};
    const int n = (max(k_end - k_begin, 0) + CHUNK_KEYS - 1) / CHUNK_KEYS;
    // where the part-th SLOT_KEYS keys are, in 16-byte chunks of the cache (below 2^32, checked
    // on the host) or NOWHERE, into their half of the buffer
    const int* table = a.batch.table + (int64_t)it.seq * a.batch.width;
    uint32_t* slots = (uint32_t*)(lds + L::SLOTS);
    auto find_slots = [&](int part) {
#pragma unroll
        for (int u = 0; u < SLOT_KEYS / CHUNK_THREADS; ++u) {
            const int i = u * CHUNK_THREADS + tid, key = k_begin + part * SLOT_KEYS + i;
            uint32_t at = NOWHERE;
            if (key < k_end) {
                const int pi = a.kv.page.quotient(key), page = table[pi];
                if (page >= 0 && page < a.kv.num_pages)
                    at = (uint32_t)a.kv.slot(page, h, key - pi * a.kv.page.div) * (uint32_t)(D / 8);
            }
            slots[(part & 1) * SLOT_KEYS + i] = at;
        }
    };
    find_slots(0);
    __syncthreads();

    const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_offset(lds));
    // this wave's l-th 64 chunks of a tile: chunk 64 wave + 512 l + lane
    const int chunk = 64 * wave + lane, wave_lds = lds0 + 1024 * wave;
    auto slot_of = [&](int tile, int l) {
        return slots[(uint32_t)(tile * CHUNK_KEYS + (chunk + CHUNK_THREADS * l) / CH) % (2 * SLOT_KEYS)];
    };
    auto load_chunks = [&](const uint16_t* from, uint32_t slot, int l, uint32_t to, bool keys) {
        const int key = (chunk + CHUNK_THREADS * l) / CH, c = (chunk + CHUNK_THREADS * l) % CH;
        const uint32_t cs = c ^ (keys ? key_swizzle<CH>(key) : value_swizzle<CH>(key));
        const uint64_t p = (uint64_t)(uintptr_t)from + 16 * (uint64_t)(slot + cs), zeros = (uint64_t)(uintptr_t)&paged_zeros;
        asm_global_load_lds_b128((const void*)(uintptr_t)(slot != NOWHERE && 8 * (int)cs < D ? p : zeros),
                                 (uint32_t)wave_lds + to + 16 * CHUNK_THREADS * l);
    };
    // K of tile i + NB - 1 and V of tile i + NB - 2 go into the buffers that iteration i
    // does not read: of the ring, before tile i's and two before it.  A wave asks for
    // its 2 NL pieces of them between its products (a load takes the memory pipeline some
    // 100 cycles to accept), past the last tile too (of zeros or of keys
    // nobody reads), so that a count of them says which are done.
    auto before = [](int ring) { return ring ? ring - 1 : NB - 1; };
    auto piece = [&](int ring, int j, uint32_t slot) {
        const int k_ring = before(ring), v_ring = before(k_ring);
        if (j < NL) load_chunks(a.kv.k, slot, j, k_ring * TILE, true);
        else load_chunks(a.kv.v, slot, j - NL, L::V + v_ring * TILE, false);
    };
    auto next_slots = [&](int i) {
        // half a part ahead: the slots of the next one, in the half whose tiles are done
        constexpr int PART = SLOT_KEYS / CHUNK_KEYS;
        const int tv = i + NB - 2;
        if (tv % PART == PART / 2 && (tv / PART + 1) * PART <= n + NB) find_slots(tv / PART + 1);
    };
    // where this lane reads: K chunk 2 st + h2 of key l32, V at key 4 h2 + (lane & 15) / 4
    // and dims 32 t + 16 ((lane / 16) & 1) + 4 (lane & 3); st and t are one exclusive or
    // in the row (32 st, 64 t), and the swizzles do not change with the multiples of 32
    // and 8 keys that the reads add
    const int vkey = 4 * h2 + ((lane & 15) >> 2), vdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const uint32_t kat = lds0 + l32 * PB + 16 * (h2 ^ key_swizzle<CH>(l32));
    const uint32_t vat = lds0 + L::V + vkey * PB + 2 * (vdim & 7) + 16 * ((vdim >> 3) ^ value_swizzle<CH>(vkey));

    float mrun = -INFINITY, lrun = 0.0f;                       // the reference (PagedP), and this lane's keys' sum
    f32x16 oacc[DT], s[2];
    u32x4 pb[PP][4] = {};                                      // P of the tile before, 16 keys each
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[i][r] = 0.0f;
    bool partial = false;                                      // the tile holds keys that some of the wave's rows do not see

    // Where tile i's values are read for the second product; the slow path makes it itself.
    auto values_at = [&](int i, int ring) {
        uint32_t base = vat + ring * TILE;
        if (partial) {
            const uint8_t* vt = lds + L::V + ring * TILE;
            uint32_t bad = 0;
            for (int c = lane; c < TILE / 16; c += 64) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(vt + 16 * c);
                const uint32_t e = BF ? 0x7F80u : 0x7C00u;
                if (8 * ((c % CH) ^ value_swizzle<CH>(c / CH)) < D)
#pragma unroll
                    for (int x = 0; x < 4; ++x) bad |= (w[x] & e) == e || ((w[x] >> 16) & e) == e;
            }
            if (__builtin_amdgcn_ballot_w64(bad)) {
                float* pw = (float*)(lds + L::P + wave * L::P_WAVE);       // [32 keys][32 rows]
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float p = 0.0f;
#pragma unroll
                            for (int w = 0; w < PP; ++w)
                                p += (w == 1 ? 1.0f / PagedP<BF>::REST : 1.0f) *
                                     bits_to_f32<std::conditional_t<BF, __hip_bfloat16, __half>>((uint16_t)(pb[w][2 * u + k][e >> 1] >> (16 * (e & 1))));
                            pw[(16 * k + 8 * (e >> 2) + 4 * h2 + (e & 3)) * 32 + l32] = p;
                        }
                    asm_wait_lgkmcnt<0>();
                    for (int key = 0; key < 32; ++key) {
                        const float p = pw[key * 32 + l32];
                        if (k_begin + i * CHUNK_KEYS + 32 * u + key >= last) continue;
#pragma unroll
                        for (int t = 0; t < DT; ++t)
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int c = (4 * t + q) ^ value_swizzle<CH>(key);
                                const u32x2 w = *reinterpret_cast<const u32x2*>(vt + (32 * u + key) * PB + 16 * c + 8 * h2);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float v = bits_to_f32<std::conditional_t<BF, __hip_bfloat16, __half>>((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
                                    oacc[t][4 * q + e] = __builtin_fmaf(p, v, oacc[t][4 * q + e]);
                                }
                            }
                    }
                    asm_wait_lgkmcnt<0>();
                }
                base = vat - L::V + L::ZEROS;                  // what follows adds zeros
            }
        }
        return base;
    };
    // The products of an iteration: O^T += V^T P^T of tile i - 1 in four steps of 16 keys (or, where
    // the second parts are summed apart (PagedP), in steps of 32 dims), then S^T = K Q^T of tile i in steps
    // of 32 dims.  A step's fragments are read from LDS AHEAD steps before they are multiplied.
    // Both are always made, a branch around either would cost copies of the accumulators:
    // without a tile before, from values of zero (pv false), and behind the last tile into
    // scores that nobody reads.
    auto products = [&](int i, int ring, bool pv) {
        constexpr bool APART = PP > 1 && PagedP<BF>::REST != 1.0f;
        constexpr int PV = APART ? DT : 4, STEPS = PV + (KS + 1) / 2;
        static_assert(2 * NL <= STEPS, "a step asks for one piece at most");
        constexpr int AHEAD = DT > 2 ? 1 : 3, SETS = AHEAD + 1;
        const uint32_t v_at = pv ? values_at(i - 1, before(ring)) : vat - L::V + L::ZEROS, k_at = kat + ring * TILE;
        const f32x16 zero = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t slot[2 * NL];
        u32x4 frag[SETS][4];
        auto read = [&](auto step) {
            constexpr int st = decltype(step)::value;
            if constexpr (st < PV) {
#pragma unroll
                for (int x = 0; x < (APART ? 4 : DT); ++x) {   // the step's keys of one t, or its t of 16 keys
                    const int t = APART ? st : x, k16 = APART ? x : st;
                    const uint32_t at = (v_at ^ (64 * t)) + 16 * k16 * PB;
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)at));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)(at + 8 * PB)));
                    frag[st % SETS][x] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                }
            } else if constexpr (st < STEPS) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (2 * (st - PV) + e < KS)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            frag[st % SETS][2 * e + u] = *(const lds_u32x4*)(uintptr_t)((k_at ^ (32 * (2 * (st - PV) + e))) + 32 * u * PB);
            }
        };
        static_for<AHEAD>(read);
#pragma unroll
        for (int j = 0; j < 2 * NL; ++j) slot[j] = slot_of(i + NB - 1 - j / NL, j % NL);
        static_for<STEPS>([&](auto step) {
            constexpr int st = decltype(step)::value;
            read(std::integral_constant<int, st + AHEAD>{});
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (st < PV && APART) {
                f32x16 rest = zero;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    rest = mfma32<BF>(frag[st % SETS][x], pb[PP - 1][x], rest);
                    oacc[st] = mfma32<BF>(frag[st % SETS][x], pb[0][x], oacc[st]);
                    if constexpr (st < 2 * NL)
                        if (x == 0) piece(ring, st, slot[st]);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[st][r] = __builtin_fmaf(rest[r], 1.0f / PagedP<BF>::REST, oacc[st][r]);
            } else if constexpr (st < PV) {
#pragma unroll
                for (int t = 0; t < DT; ++t) oacc[t] = mfma32<BF>(frag[st % SETS][t], pb[0][st], oacc[t]);
                if constexpr (st < 2 * NL) piece(ring, st, slot[st]);
#pragma unroll
                for (int w = 1; w < PP; ++w)
#pragma unroll
                    for (int t = 0; t < DT; ++t) oacc[t] = mfma32<BF>(frag[st % SETS][t], pb[w][st], oacc[t]);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (2 * (st - PV) + e < KS)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int d = 2 * (st - PV) + e;
                            s[u] = mfma32<BF>(frag[st % SETS][2 * e + u], qf[d], d == 0 ? zero : s[u]);
                        }
                if constexpr (st < 2 * NL) piece(ring, st, slot[st]);
            }
        });
    };
    auto softmax = [&](int i) {
        const int kv0 = k_begin + i * CHUNK_KEYS;
        const uint64_t hidden = __builtin_amdgcn_ballot_w64(slots[(uint32_t)(i * CHUNK_KEYS + lane) % (2 * SLOT_KEYS)] == NOWHERE);
        // keys up to k_end are in LDS with their values: the last of a tile may be hidden from all the wave's rows
        // (group >= 32: one token's) and visible to later waves' only
        partial = kv0 + CHUNK_KEYS > wave_open && wave_open < k_end;
        if (hidden || kv0 + CHUNK_KEYS > wave_open) {
            asm volatile("");                                  // a branch: few tiles need this
            const int seen = last - kv0 - 4 * h2;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t hid = (uint32_t)(hidden >> (32 * u)) >> (4 * h2);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = 8 * (r >> 2) + (r & 3);    // and 32 u + 4 h2
                    if (32 * u + key >= seen || (hid & (1u << key))) s[u][r] = -INFINITY;
                }
            }
        }
        float tmax = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[u][r]);
        tmax *= a.scale_log2;
        if (__builtin_amdgcn_ballot_w64(tmax > mrun + (PagedP<BF>::BIAS + PagedP<BF>::SLACK))) {
            const float mnew = fmaxf(mrun, fmaxf(tmax, __shfl_xor(tmax, 32, 64)) - PagedP<BF>::BIAS);
            const float factor = mnew == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mrun - mnew);
            lrun *= factor;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[t][r] *= factor;
            mrun = mnew;
        }
        const float msafe = mrun == -INFINITY ? 0.0f : mrun;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k >> 1][8 * (k & 1) + e], a.scale_log2, -msafe));
                lrun += p[e];
            }
#pragma unroll
            for (int w = 0; w < PP; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (w == 1) p[2 * e] *= PagedP<BF>::REST, p[2 * e + 1] *= PagedP<BF>::REST;
                    pb[w][k][e] = round2<BF, true>(p[2 * e], p[2 * e + 1]);
                }
        }
    };

#pragma unroll
    for (int t = 0; t < NB - 1; ++t)
#pragma unroll
        for (int l = 0; l < NL; ++l) {
            load_chunks(a.kv.k, slot_of(t, l), l, t * TILE, true);
            if (t < NB - 2) load_chunks(a.kv.v, slot_of(t, l), l, L::V + t * TILE, false);
        }
    asm_wait_vmcnt<0>();
    phase_barrier();
    auto in_reach = [&](int i) { return i < n && k_begin + i * CHUNK_KEYS < wave_end; };
    for (int i = 0, ring = 0; i <= n; ++i, ring = ring == NB - 1 ? 0 : ring + 1) {
        next_slots(i);
        // a softmax of the second group goes before one of the first, or its products, which come after it,
        // find no vector instructions to run beside (2048 fp16 rows on 8192, 32 heads of 64: 234 -> 224 us, with fp32 O
        // 341 -> 316; head_dim 128 the same)
        __builtin_amdgcn_s_setprio(1);
        if (second && i > 0 && in_reach(i - 1)) softmax(i - 1);
        products(i, ring, i > 0 && in_reach(i - 1));
        __builtin_amdgcn_s_setprio(0);
        if (!second && in_reach(i)) softmax(i);
        // what this wave asked for NB - 2 iterations ago has arrived: K of tile i + 1 and V of tile i
        asm_wait_vmcnt<(NB - 2) * 2 * NL>();
        phase_barrier();
    }
    asm_wait_vmcnt<0>();                                       // loads past the last tile write LDS that is about to be reused

    const float sum = lrun + __shfl_xor(lrun, 32, 64);
    if (f < rows_f) {
        const PagedParts<R> parts(a, a.many, h);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * t + 8 * q + 4 * h2;
                const f32x4 o = {oacc[t][4 * q], oacc[t][4 * q + 1], oacc[t][4 * q + 2], oacc[t][4 * q + 3]};
                if (d >= D) continue;
                if (it.record >= 0) parts.store_out(it.record + it.split, f - tile_f, d, o);
                else paged_store4<BF>(a, sp, h, f, d, o * inv);
            }
        if (it.record >= 0 && h2 == 0) parts.store_ml(it.record + it.split, f - tile_f, mrun, sum);
    }
    if (it.record >= 0) paged_merge<BF, R, CHUNK_THREADS>(a, a.many, it, h, (uint32_t*)lds);
}

// Full tiles of 256 rows per kv head, each times the splits its keys could make: whether
// they would fill the chip (plan_attention_paged asks the same of what the tables can
// hold).  The same in all lanes; first: the lane-th sequence's span.
__device__ __forceinline__ int chunk_worth(const PagedAttnArgs& a, const PagedSpan& first) {
    int worth = 0;
    for (int base = 0; base < a.batch.seqs; base += 64) {
        const PagedSpan p = base ? paged_lane_span(a.batch, base + (int)(threadIdx.x & 63)) : first;
        const int64_t tiles = (int64_t)p.n * a.group / CHUNK_R;
        worth = min(worth + (int)min(tiles, (int64_t)4096) * min(max(p.len / CHUNK_UNIT, 1), 4096), 1 << 24);
    }
    return __builtin_amdgcn_readlane(wave_scan(worth), 63);
}

// The kernel's arguments, loaded anew for an item.  Kept from item to item, what both kinds of item
// use is more than the scalar registers hold, and 128 of them are kept in lanes of vector registers and read back inside
// the loops: 51 when they are loaded anew (2048 rows on 8192, 32 heads of 64: 221 -> 211 us, with fp32 O
// 309 -> 292).  With more than two accumulators that cost more than it gave (heads of 80 155 -> 157 us, of 128 307 -> 324).
template <int DT>
__device__ __forceinline__ const PagedAttnArgs& item_args(const PagedAttnArgs& a) {
    if constexpr (DT > 2) return a;
    uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();     // where a, the only argument, is
    asm volatile("" : "+s"(p));
    return *(const PagedAttnArgs*)(const __attribute__((address_space(4))) PagedAttnArgs*)p;
}

template <int KS, int DT, bool BF, int PP>
__global__ __launch_bounds__(CHUNK_THREADS, 2) void paged_chunk_kernel(const PagedAttnArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int kv_heads = a.kv.kv_heads, q = (int)blockIdx.x % PAGED_QUEUES, own = (int)blockIdx.x / PAGED_QUEUES;
    const int blocks = ((int)gridDim.x - q + PAGED_QUEUES - 1) / PAGED_QUEUES;              // of this queue
    const PagedSpan span = paged_lane_span(a.batch, (int)(threadIdx.x & 63));
    const bool worth = chunk_worth(a, span) >= a.many_least;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.made = worth;
    if (!worth) return;                                        // the kernel for few rows makes everything
    const PagedShare many = paged_share<CHUNK_R, true>(a, span, PAGED_FEW), few = paged_share<32, false>(a, span, PAGED_FEW);
    const int many_items = (many.items * kv_heads - q + PAGED_QUEUES - 1) / PAGED_QUEUES;
    const int all_items = many_items + (few.items * kv_heads - q + PAGED_QUEUES - 1) / PAGED_QUEUES;
    for (int round = 0; round * blocks < all_items; ++round) {
        const int i = round * blocks + (round & 1 ? blocks - 1 - own : own);
        if (i < many_items) {
            const int w = i * PAGED_QUEUES + q, index = w / kv_heads;
            paged_chunk_item<KS, DT, BF, PP>(item_args<DT>(a), many, index, w - index * kv_heads, lds);
        } else if (i < all_items) {
            const int w = (i - many_items) * PAGED_QUEUES + q, index = w / kv_heads;
            paged_few_item<32, DT, BF, PP, 8>(item_args<DT>(a), few, index, w - index * kv_heads, lds);
        }
        __syncthreads();                                       // LDS is free
    }
}

template <int KS, int DT, bool BF, int PP>
static hipError_t launch_chunk(hipStream_t s, const PagedAttnArgs& a, int num_cus) {
    constexpr int few = 8 * PagedLayout<32, DT>::REGION + 16, bytes = ChunkLayout<DT>::BYTES > few ? ChunkLayout<DT>::BYTES : few;
    if (const hipError_t e = allow_dynamic_lds<paged_chunk_kernel<KS, DT, BF, PP>>(bytes); e != hipSuccess) return e;
    const int64_t most = ((int64_t)a.many.items + a.few.items) * a.kv.kv_heads;
    launch_kernel_part(LaunchPart::First, paged_chunk_kernel<KS, DT, BF, PP>, dim3((unsigned)std::min<int64_t>(num_cus, most)), dim3(CHUNK_THREADS),
                  (uint32_t)bytes, s, a);
    return hipGetLastError();
}

template <int KS, int DT>
static hipError_t launch_chunk_dims(hipStream_t s, const PagedAttnArgs& a, int num_cus) {
    const bool wide = a.o_dtype == MVLM_F32;
    if (a.kv.dtype == MVLM_F16) return wide ? launch_chunk<KS, DT, false, 2>(s, a, num_cus) : launch_chunk<KS, DT, false, 1>(s, a, num_cus);
    return wide ? launch_chunk<KS, DT, true, 3>(s, a, num_cus) : launch_chunk<KS, DT, true, 1>(s, a, num_cus);
}

hipError_t launch_attention_paged_chunk(hipStream_t s, const PagedAttnArgs& a, int num_cus) {
    const int D = a.kv.D;
    if (D <= 32) return launch_chunk_dims<2, 1>(s, a, num_cus);
    if (D <= 64) return launch_chunk_dims<4, 2>(s, a, num_cus);
    if (D <= 80) return launch_chunk_dims<5, 3>(s, a, num_cus);
    if (D <= 96) return launch_chunk_dims<6, 3>(s, a, num_cus);
    return launch_chunk_dims<8, 4>(s, a, num_cus);
}

}  // namespace mvlm
