// New rows of q | k | v for sequences with a paged cache: rotary positions on q
// and k, keys and values into their pages, q out, in one pass.
//
//   x = one row of qkv: heads q heads, then kv_heads k heads, then kv_heads v
//   heads of D elements; p = the row's position (paged.h); (c, s) = rope[p][i]
//   rotated pairs i < rot / 2 of a q or k head, (a, b) = (x[i], x[i + rot/2]) or,
//   interleaved, (x[2i], x[2i + 1]):   a' = a c - b s,   b' = b c + a s
// in fp32, rounded once (to nearest even) to the cache's type, since that is what
// the matrix products of the attention read.
//
// Bytes bound it: each element is read once and written once.  A thread makes 8
// elements of one head: a 16-byte store whatever the types are, and its partner
// elements (a chunk further on in the same head, or its own) come from the lines
// that its neighbours read.  One block per row, so sequence, position, page
// and table row are found once per wave; the elements are asked for before that chain of
// loads (95 -> 80 us below).
// Measured: 4 x 4096 bf16 rows, 32 + 2 x 8 heads of 128, 405 MB: 80 us, 5.1 TB/s, what a
// large copy reaches; 768 fp16 rows, 3 x 32 heads of 64, 19 MB: 6.1 us; one row 3.8 us, a
// launch.
#include "common.h"
#include "device_math.h"
#include "paged_ops.h"

namespace mvlm {

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_AHEAD = 3;

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));   // the rope table's rows may start anywhere

// 8 elements from x[i], fp32
template <int XD, bool VEC>
__device__ __forceinline__ void append_load8(const void* x, int64_t i, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = load_as_f32(x, i + e, XD);
    } else if constexpr (XD == MVLM_F32) {
        const f32x4* p = reinterpret_cast<const f32x4*>((const float*)x + i);
        const f32x4 lo = p[0], hi = p[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>((const uint16_t*)x + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            v[e] = XD == MVLM_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
        }
    }
}

// XD: type of qkv; VEC: its rows are 16-byte aligned
template <int XD, bool VEC>
__global__ __launch_bounds__(APPEND_THREADS) void kv_append_kernel(const KvAppendArgs a) {
    const int row = (int)blockIdx.x;
    const PagedKv& kv = a.kv;
    const int D = kv.D, cpr = D / 8, half = a.rot / 2;
    const int chunks = (a.heads + 2 * kv.kv_heads) * cpr;
    const int64_t xrow = (int64_t)row * a.ld;
    // a thread's first chunks are asked for before its sequence is looked up
    float first[APPEND_AHEAD][8];
#pragma unroll
    for (int u = 0; u < APPEND_AHEAD; ++u) {
        const int c = min((int)threadIdx.x + u * APPEND_THREADS, chunks - 1);
        append_load8<XD, VEC>(a.qkv, xrow + 8 * (int64_t)c, first[u]);
    }
    PagedSpan sp;
    const int seq = paged_seq_of_row(a.batch, row, &sp);
    if (seq < 0) return;                                   // behind the last sequence: left as it is
    const int p = sp.position(row - sp.row0);
    // a row without a place: no position, past the table or the rotary table, a page that does not exist
    int slot0 = -1;                                        // slot of kv head 0
    if (p >= 0 && p < a.batch.positions && (a.rot == 0 || p < a.rope_positions)) {
        const int pi = kv.page.quotient(p);
        const int page = a.batch.table[(int64_t)seq * a.batch.width + pi];
        if (page >= 0 && page < kv.num_pages) slot0 = kv.slot(page, 0, p - pi * kv.page.div);
    }
    const float* cs = a.rope + (int64_t)p * a.rot;         // [rot / 2][2], read only with a place
    auto make = [&](int c, const float (&v)[8]) {
        const int head = a.chunk.quotient(c), d = 8 * (c - head * cpr);
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e];
        if (d < a.rot && head < a.heads + kv.kv_heads && slot0 >= 0) {
            const int64_t h0 = xrow + (int64_t)head * D;
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    if (d + e < a.rot) {
                        const float co = cs[d + e], si = cs[d + e + 1];
                        o[e] = v[e] * co - v[e + 1] * si;
                        o[e + 1] = v[e + 1] * co + v[e] * si;
                    }
            } else if (half % 8 == 0) {                    // a chunk lies in one half, its partner chunk in the other
                const bool first = d < half;
                const int i = first ? d : d - half;
                float w[8];
                append_load8<XD, VEC>(a.qkv, h0 + (first ? d + half : i), w);
                const f32x4_any* t = reinterpret_cast<const f32x4_any*>(cs + 2 * i);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const f32x4_any q = t[e / 2];
                    o[e] = v[e] * q[0] + (first ? -w[e] : w[e]) * q[1];
                    o[e + 1] = v[e + 1] * q[2] + (first ? -w[e + 1] : w[e + 1]) * q[3];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (d + e < a.rot) {
                        const bool first = d + e < half;
                        const int i = first ? d + e : d + e - half;
                        const float w = load_as_f32(a.qkv, h0 + (first ? i + half : i), XD);
                        const float co = cs[2 * i], si = cs[2 * i + 1];
                        o[e] = v[e] * co + (first ? -w : w) * si;
                    }
            }
        }
        u32x4 out;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x2 pair = {o[2 * j], o[2 * j + 1]};
            out[j] = kv.dtype == MVLM_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, f16x2_t))
                                          : __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_t));
        }
        if (head < a.heads) {
            if (slot0 < 0) out = u32x4{0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4*>(a.q_out + ((int64_t)row * a.heads + head) * D + d) = out;
        } else if (slot0 >= 0) {
            const bool key = head < a.heads + kv.kv_heads;
            const int h = head - a.heads - (key ? 0 : kv.kv_heads);
            const int64_t at = (int64_t)(slot0 + h * kv.page.div) * D + d;
            *reinterpret_cast<u32x4*>((key ? kv.k : kv.v) + at) = out;
        }
    };
#pragma unroll
    for (int u = 0; u < APPEND_AHEAD; ++u)
        if ((int)threadIdx.x + u * APPEND_THREADS < chunks) make((int)threadIdx.x + u * APPEND_THREADS, first[u]);
    for (int c = (int)threadIdx.x + APPEND_AHEAD * APPEND_THREADS; c < chunks; c += APPEND_THREADS) {
        float v[8];
        append_load8<XD, VEC>(a.qkv, xrow + 8 * (int64_t)c, v);
        make(c, v);
    }
}

hipError_t launch_kv_append(hipStream_t s, const KvAppendArgs& a) {
    const size_t es = dtype_size(a.x_dtype);
    const bool vec = ((uintptr_t)a.qkv & 15u) == 0 && (a.ld * (int64_t)es) % 16 == 0;
    const dim3 grid((unsigned)a.batch.rows), block(APPEND_THREADS);
    auto go = [&](auto dt) {
        constexpr int XD = decltype(dt)::value;
        if (vec) launch_kernel(kv_append_kernel<XD, true>, grid, block, 0, s, a);
        else launch_kernel(kv_append_kernel<XD, false>, grid, block, 0, s, a);
    };
    if (a.x_dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.x_dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
