// Rows of keys and values out of a paged cache (paged.h), contiguous, in any of the 16- and 32-bit types: what
// kv_append.hip wrote for the same rows of a batch.  An element of an 8-bit cache is its code times its block's
// power of two, which is exact in fp32.
//
// Bytes bound it: each is read once and written once.  A thread makes 8 elements of one head, of one row or of
// four that follow one another.
// Measured: 65536 bf16 rows of 8 heads of 128 out of an 8-bit cache, 406 MB: 88 us, 4.6 TB/s (a large copy reaches
// 5.1), out of a bf16 cache, 535 MB: 98 us, 5.5 TB/s; 729 fp16 rows of 32 heads of 64, 9 MB: 4.3 us, little more than a
// launch, out of an fp16 cache 4.2.
#include "common.h"
#include "device_math.h"
#include "paged_ops.h"

namespace mvlm {

constexpr int READ_THREADS = 256;

typedef _Float16 f16x2_r __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_r __attribute__((ext_vector_type(2)));

// 8 elements of a slot as they lie in the cache, and their scales' word
struct ReadRaw {
    u32x4 w;
    uint32_t scale;
};
template <bool MX>
__device__ __forceinline__ ReadRaw read_raw(const PagedKv& kv, bool keys, int64_t slot, int d) {
    const uint16_t* base = keys ? kv.k : kv.v;
    ReadRaw r{};
    if constexpr (MX) {
        const u32x2 c = *reinterpret_cast<const u32x2*>((const uint8_t*)base + slot * kv.D + d);
        r.w[0] = c[0], r.w[1] = c[1];
        r.scale = kv.scales(base)[slot];
    } else
        r.w = *reinterpret_cast<const u32x4*>(base + slot * kv.D + d);
    return r;
}
template <bool MX>
__device__ __forceinline__ void read_values(const PagedKv& kv, const ReadRaw& r, int d, float (&v)[8]) {
    if constexpr (MX) {
        const float up = __uint_as_float(((r.scale >> (d / MX_BLOCK * 8)) & 0xFFu) << 23);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)r.w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)r.w[j], true);
            v[4 * j] = lo[0] * up, v[4 * j + 1] = lo[1] * up, v[4 * j + 2] = hi[0] * up, v[4 * j + 3] = hi[1] * up;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t h = (uint16_t)(r.w[e >> 1] >> (16 * (e & 1)));
            v[e] = kv.dtype == MVLM_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
        }
    }
}

template <int OD, bool VEC>
__device__ __forceinline__ void read_store8(void* out, int64_t at, const float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int e = 0; e < 8; ++e) store_out(out, at + e, v[e], OD);
    } else if constexpr (OD == MVLM_F32) {
        f32x4* to = reinterpret_cast<f32x4*>((float*)out + at);
        to[0] = f32x4{v[0], v[1], v[2], v[3]};
        to[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x2 pair = {v[2 * j], v[2 * j + 1]};
            w[j] = OD == MVLM_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, f16x2_r))
                                  : __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_r));
        }
        *reinterpret_cast<u32x4*>((uint16_t*)out + at) = w;
    }
}

// Where a row's keys are: slot of kv head 0; -1: it has no place, -2: it is no sequence's
__device__ __forceinline__ int read_slot(const KvReadArgs& a, int row) {
    PagedSpan sp;
    const int seq = paged_seq_of_row(a.batch, row, &sp);
    if (seq < 0) return -2;
    const int p = sp.position(row - sp.row0);
    if (p < 0 || p >= a.batch.positions) return -1;
    const int pi = a.kv.page.quotient(p);
    const int page = a.batch.table[(int64_t)seq * a.batch.width + pi];
    return page >= 0 && page < a.kv.num_pages ? a.kv.slot(page, 0, p - pi * a.kv.page.div) : -1;
}

// OD: type of the outputs; VEC: their rows are 16-byte aligned; MX: 8-bit cache; ROWS: rows of a block
template <int OD, bool VEC, bool MX, int ROWS>
__global__ __launch_bounds__(READ_THREADS) void kv_read_kernel(const KvReadArgs a) {
    // an XCD's blocks (every eighth) have rows that follow one another, whose scales share lines
    const int eighth = (int)gridDim.x / 8, b = ROWS == 1 ? (int)blockIdx.x : (int)(blockIdx.x % 8) * eighth + (int)blockIdx.x / 8;
    const int row0 = b * ROWS;
    if (ROWS > 1 && row0 >= a.batch.rows) return;
    const PagedKv& kv = a.kv;
    int slots[ROWS];
    if constexpr (ROWS == 1) slots[0] = read_slot(a, row0);
    else {
        static_assert(ROWS <= READ_THREADS / 64, "a wave finds a row's place");
        __shared__ int found[ROWS];
        const int wave = (int)threadIdx.x >> 6;
        if (wave < ROWS) {
            const int slot = row0 + wave < a.batch.rows ? read_slot(a, row0 + wave) : -2;
            if ((threadIdx.x & 63) == 0) found[wave] = slot;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROWS; ++r) slots[r] = found[r];
    }
    const int cpr = kv.D / 8, chunks = kv.kv_heads * cpr;
    for (int c = (int)threadIdx.x; c < 2 * chunks; c += READ_THREADS) {
        const bool keys = c < chunks;
        void* out = keys ? a.k_out : a.v_out;
        if (!out) continue;
        const int i = keys ? c : c - chunks, head = a.chunk.quotient(i), d = 8 * (i - head * cpr);
        ReadRaw raw[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) raw[r] = read_raw<MX>(kv, keys, max(slots[r], 0) + (int64_t)head * kv.page.div, d);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (slots[r] == -2) continue;
            float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (slots[r] >= 0) read_values<MX>(kv, raw[r], d, v);
            read_store8<OD, VEC>(out, (int64_t)(row0 + r) * a.ld + 8 * (int64_t)i, v);
        }
    }
}

hipError_t launch_kv_read(hipStream_t s, const KvReadArgs& a) {
    const size_t es = dtype_size(a.dtype);
    const bool vec = (((uintptr_t)a.k_out | (uintptr_t)a.v_out) & 15u) == 0 && (a.ld * (int64_t)es) % 16 == 0;
    auto go = [&](auto dt, auto mx) {
        constexpr int OD = decltype(dt)::value;
        constexpr bool MX = decltype(mx)::value;
        auto rows = [&](auto n) {
            constexpr int ROWS = decltype(n)::value;
            const int blocks = (a.batch.rows + ROWS - 1) / ROWS;
            const dim3 grid((unsigned)(ROWS == 1 ? blocks : (blocks + 7) / 8 * 8)), block(READ_THREADS);
            if (vec) launch_kernel(kv_read_kernel<OD, true, MX, ROWS>, grid, block, 0, s, a);
            else launch_kernel(kv_read_kernel<OD, false, MX, ROWS>, grid, block, 0, s, a);
        };
        // four rows to a block have four times the loads in flight behind one chain of lookups (65536 rows of 8 heads of
        // 128: 112 -> 88 us), which few rows pay for with CUs that have none.  Four and one, 8 bits: 1024 rows of 32 heads of 64
        // 5.8 and 4.7 us, 1536 6.6 and 6.6, 2048 7.3 and 8.2, 4096 11.6 and 13.4; of 8 heads of 128 4.1 and 4.2, 4.5 and
        // 4.1, 4.8 and 4.8, 7.1 and 7.8, of 16 bits 3.9 and 4.1, 4.4 and 4.2, 4.8 and 5.0, 8.2 and 8.3
        if (a.batch.rows >= 2048) rows(std::integral_constant<int, 4>{});
        else rows(std::integral_constant<int, 1>{});
    };
    auto type = [&](auto mx) {
        if (a.dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{}, mx);
        else if (a.dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{}, mx);
        else go(std::integral_constant<int, MVLM_BF16>{}, mx);
    };
    if (a.kv.dtype == MVLM_MXFP8) type(std::true_type{});
    else type(std::false_type{});
    return hipGetLastError();
}

}  // namespace mvlm
