// Rows of keys and values out of a paged cache (paged.h), contiguous, in any of the 16- and 32-bit types: what
// kv_append.hip wrote for the same rows of a batch.  An element of an 8-bit cache is its code times its block's
// power of two, which is exact in fp32.
//
// Bytes bound it: each is read once and written once.  A thread makes 8 elements of one head; one block per row.
#include "common.h"
#include "device_math.h"
#include "paged_ops.h"

namespace mvlm {

constexpr int READ_THREADS = 256;

typedef _Float16 f16x2_r __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_r __attribute__((ext_vector_type(2)));

// 8 elements of a slot from dim d on, fp32
__device__ __forceinline__ void read_load8(const PagedKv& kv, bool keys, int64_t slot, int d, float (&v)[8]) {
    const uint16_t* base = keys ? kv.k : kv.v;
    if (kv.dtype == MVLM_MXFP8) {
        const u32x2 c = *reinterpret_cast<const u32x2*>((const uint8_t*)base + slot * kv.D + d);
        const uint32_t word = (keys ? kv.k_scale : kv.v_scale)[slot];
        const float up = __uint_as_float(((word >> (d / MX_BLOCK * 8)) & 0xFFu) << 23);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], true);
            v[4 * j] = lo[0] * up, v[4 * j + 1] = lo[1] * up, v[4 * j + 2] = hi[0] * up, v[4 * j + 3] = hi[1] * up;
        }
        return;
    }
    const u32x4 w = *reinterpret_cast<const u32x4*>(base + slot * kv.D + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        v[e] = kv.dtype == MVLM_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
    }
}

// OD: type of the outputs; VEC: their rows are 16-byte aligned
template <int OD, bool VEC>
__global__ __launch_bounds__(READ_THREADS) void kv_read_kernel(const KvReadArgs a) {
    const int row = (int)blockIdx.x;
    const PagedKv& kv = a.kv;
    PagedSpan sp;
    const int seq = paged_seq_of_row(a.batch, row, &sp);
    if (seq < 0) return;                                   // behind the last sequence: left as it is
    const int p = sp.position(row - sp.row0);
    int slot0 = -1;                                        // slot of kv head 0, or no place
    if (p >= 0 && p < a.batch.positions) {
        const int pi = kv.page.quotient(p);
        const int page = a.batch.table[(int64_t)seq * a.batch.width + pi];
        if (page >= 0 && page < kv.num_pages) slot0 = kv.slot(page, 0, p - pi * kv.page.div);
    }
    const int cpr = kv.D / 8, chunks = kv.kv_heads * cpr;
    for (int c = (int)threadIdx.x; c < 2 * chunks; c += READ_THREADS) {
        const bool keys = c < chunks;
        void* out = keys ? a.k_out : a.v_out;
        if (!out) continue;
        const int i = keys ? c : c - chunks, head = a.chunk.quotient(i), d = 8 * (i - head * cpr);
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (slot0 >= 0) read_load8(kv, keys, slot0 + (int64_t)head * kv.page.div, d, v);
        const int64_t at = (int64_t)row * a.ld + 8 * (int64_t)i;
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
}

hipError_t launch_kv_read(hipStream_t s, const KvReadArgs& a) {
    const size_t es = dtype_size(a.dtype);
    const bool vec = (((uintptr_t)a.k_out | (uintptr_t)a.v_out) & 15u) == 0 && (a.ld * (int64_t)es) % 16 == 0;
    const dim3 grid((unsigned)a.batch.rows), block(READ_THREADS);
    auto go = [&](auto dt) {
        constexpr int OD = decltype(dt)::value;
        if (vec) launch_kernel(kv_read_kernel<OD, true>, grid, block, 0, s, a);
        else launch_kernel(kv_read_kernel<OD, false>, grid, block, 0, s, a);
    };
    if (a.dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
