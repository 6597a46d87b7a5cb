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

// The same where a head's elements need each other: norms (a sum of squares over the head) and 8-bit caches (the
// largest magnitude of 32 dims).
//   x' = x w / sqrt(sum x^2 / D + eps), then the rotation; e = mx_exponent(max |x|), code = e4m3(x 2^-e)
// Bytes bound it as well.  L = 1 .. 16 lanes make a head, 8 dims each, and sum over one another; a lane has the
// same dims of every head that it makes, so the weights and the row's cos and sin are in its registers once.  Codes
// leave in 8-byte stores, a head's scales in one word.
// Measured: 16162 bf16 rows of 32 + 2 x 8 heads of 128 with both norms into an 8-bit cache, 303 MB: 84 us, 3.6 TB/s
// (a wave's chain of lookup, sums over lanes and conversions; the 16-bit append without norms 5.1); 768 fp16 rows
// of 3 x 32 heads of 64 with norms, 19 MB: 6.5 us; one row 4.0 us, a launch.  Sums over lanes by DPP, loads ahead and
// weights, cos and sin in registers brought the first from 176 us, halves and lanes known to the compiler from 93.
constexpr int HEADS_AHEAD = 3;

// 8 elements as they lie in memory
template <int XD, bool VEC>
struct AppendRaw {
    u32x4 w[VEC && XD != MVLM_F32 ? 1 : 2];
    __device__ __forceinline__ void load(const void* x, int64_t i) {
        if constexpr (!VEC) {
            float v[8];
            append_load8<XD, false>(x, i, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2][e & 3] = __float_as_uint(v[e]);
        } else if constexpr (XD == MVLM_F32) {
            const u32x4* p = reinterpret_cast<const u32x4*>((const float*)x + i);
            w[0] = p[0], w[1] = p[1];
        } else
            w[0] = *reinterpret_cast<const u32x4*>((const uint16_t*)x + i);
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (!VEC || XD == MVLM_F32) return __uint_as_float(w[e >> 2][e & 3]);
        else if constexpr (XD == MVLM_BF16) return __uint_as_float(e & 1 ? w[0][e >> 1] & 0xFFFF0000u : w[0][e >> 1] << 16);
        else return f16_bits_to_f32((uint16_t)(w[0][e >> 1] >> (16 * (e & 1))));
    }
};

// f(v, the value of the lane that is off away by exclusive or), over groups of `lanes` lanes; off = 1, 2, 4, 8
// in turn, after which a group's lanes agree where f is a sum or a maximum (the mirrors reach the lane 4 or 8 away because
// its neighbours agree by then)
template <class T, class F>
__device__ __forceinline__ T over_lanes(T v, int from, int lanes, F&& f) {
    auto move = [](T x, auto ctrl) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    if (from <= 1 && lanes > 1) v = f(v, move(v, std::integral_constant<int, 0xB1>{}));      // quad_perm [1, 0, 3, 2]
    if (from <= 2 && lanes > 2) v = f(v, move(v, std::integral_constant<int, 0x4E>{}));      // quad_perm [2, 3, 0, 1]
    if (from <= 4 && lanes > 4) v = f(v, move(v, std::integral_constant<int, 0x141>{}));     // row_half_mirror
    if (lanes > 8) v = f(v, move(v, std::integral_constant<int, 0x140>{}));                  // row_mirror
    return v;
}

// XD: type of qkv; VEC: its rows are 16-byte aligned; MX: 8-bit cache; NORM: of q or k heads; LANES: of a head, all with
// 8 dims, 0: any number; HALVES: rotated pairs are halves of multiples of 8
template <int XD, bool VEC, bool MX, bool NORM, int LANES, bool HALVES>
__global__ __launch_bounds__(APPEND_THREADS) void kv_append_heads_kernel(const KvAppendArgs a) {
    const int row = (int)blockIdx.x;
    const PagedKv& kv = a.kv;
    const int D = kv.D, half = a.rot / 2, qk = a.heads + kv.kv_heads, all = qk + kv.kv_heads;
    const int shift = LANES == 16 ? 4 : LANES == 8 ? 3 : D > 64 ? 4 : D > 32 ? 3 : D > 16 ? 2 : D > 8 ? 1 : 0, lanes = 1 << shift;
    const int sub = (int)threadIdx.x & (lanes - 1), d = 8 * sub, step = (int)blockDim.x >> shift;
    const int own = (int)threadIdx.x >> shift;
    const int dl = min(d, D - 8);                          // a lane past the head's end reads its last dims
    const int64_t xrow = (int64_t)row * a.ld;
    AppendRaw<XD, VEC> ahead[HEADS_AHEAD];
#pragma unroll
    for (int u = 0; u < HEADS_AHEAD; ++u) ahead[u].load(a.qkv, xrow + (int64_t)min(own + u * step, all - 1) * D + dl);
    // the weights of the kind of head that the lane is at, of which each follows the other
    float wt[8];
    const float* weight = nullptr;
    auto weigh = [&](const float* w) {
        weight = w;
        if (!w) return;
        const f32x4_any lo = *reinterpret_cast<const f32x4_any*>(w + dl), hi = *reinterpret_cast<const f32x4_any*>(w + dl + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) wt[e] = lo[e], wt[4 + e] = hi[e];
    };
    int kind_end = a.heads;                                // heads below it are of that kind
    if constexpr (NORM) weigh(a.q_weight);
    PagedSpan sp;
    const int seq = paged_seq_of_row(a.batch, row, &sp);
    if (seq < 0) return;                                   // behind the last sequence: left as it is
    const int p = sp.position(row - sp.row0);
    int slot0 = -1;                                        // slot of kv head 0; no place: as in kv_append_kernel
    if (p >= 0 && p < a.batch.positions && (a.rot == 0 || p < a.rope_positions)) {
        const int pi = kv.page.quotient(p);
        const int page = a.batch.table[(int64_t)seq * a.batch.width + pi];
        if (page >= 0 && page < kv.num_pages) slot0 = kv.slot(page, 0, p - pi * kv.page.div);
    }
    // cos and signed sin of this lane's dims: x' = x co + (its pair's other element) si
    float co[8], si[8];
    const bool turns = d < a.rot && slot0 >= 0;
    const bool whole = HALVES || (a.interleaved ? a.rot : half) % 8 == 0;   // a chunk turns as a whole
    const bool inter = !HALVES && a.interleaved;
    const float* cs = a.rope + (int64_t)p * a.rot;         // [rot / 2][2]
    if (turns) {
        if (whole && inter) {
            const f32x4_any lo = *reinterpret_cast<const f32x4_any*>(cs + d), hi = *reinterpret_cast<const f32x4_any*>(cs + d + 4);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const f32x4_any& q = e < 4 ? lo : hi;
                co[e] = co[e + 1] = q[e & 2];
                si[e] = -q[(e & 2) + 1];
                si[e + 1] = q[(e & 2) + 1];
            }
        } else if (whole) {
            const f32x4_any* t = reinterpret_cast<const f32x4_any*>(cs + 2 * (d < half ? d : d - half));
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const f32x4_any q = t[e / 2];
                co[e] = q[0], co[e + 1] = q[2];
                si[e] = d < half ? -q[1] : q[1], si[e + 1] = d < half ? -q[3] : q[3];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool first = inter ? (e & 1) == 0 : d + e < half;
                const int i = min(inter ? (d + e) / 2 : first ? d + e : d + e - half, half - 1);
                co[e] = cs[2 * i];
                si[e] = first ? -cs[2 * i + 1] : cs[2 * i + 1];
            }
        }
    }
    // where the lane's dims of q head 0 and of kv head 0 go; a kv head further on is a page's slots further on
    uint16_t* const q_to = a.q_out + (int64_t)row * a.heads * D + d;
    const int64_t kv_to = (int64_t)max(slot0, 0) * D + d;
    const int64_t kv_step = (int64_t)kv.page.div * D;      // past 2^31 in pages of 2^24 positions and more
    const int partner = ((int)threadIdx.x & 63) + (d < half ? half / 8 : -(half / 8));
    auto make = [&](int head, const AppendRaw<XD, VEC>& x) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = x.get(e);
        if (LANES == 0 && 8 * lanes > D) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = d < D ? v[e] : 0.0f;
        }
        const bool is_q = head < a.heads, is_k = !is_q && head < qk;
        float r = 1.0f;
        if constexpr (NORM) {
            if (head >= kind_end) {
                weigh(is_k ? a.k_weight : nullptr);
                kind_end = is_k ? qk : all;
            }
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
            ss = over_lanes(ss, 1, lanes, [](float u, float w) { return u + w; });
            if (weight) {
                const float mean = __builtin_fmaf(ss, a.per_dim, a.eps);
                r = mean >= 0x1p-120f ? __builtin_amdgcn_rsqf(mean) : 1.0f / sqrtf(mean);   // the first, off by a bit, takes no subnormals
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = v[e] * r * wt[e];
            }
        }
        if (HALVES || a.rot) {
            float w[8];                                    // the pairs' other elements
            if (inter) {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = v[e ^ 1];
            } else if (whole) {                            // a chunk lies in one half, its partner chunk in the other
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __shfl(v[e], partner & 63, 64);
            } else if (turns && (is_q || is_k)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = min(d + e, a.rot - 1), j = i < half ? i + half : i - half;
                    w[e] = load_as_f32(a.qkv, xrow + (int64_t)head * D + j, XD);
                    if (weight) w[e] = w[e] * r * weight[j];
                }
            }
            if (turns && (is_q || is_k)) {
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = v[e] * co[e] + w[e] * si[e];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = w[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = d + e < a.rot ? v[e] * co[e] + w[e] * si[e] : v[e];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = w[e];
                }
            }
        }
        if (is_q || !MX) {
            u32x4 out;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x2 pair = {v[2 * j], v[2 * j + 1]};
                out[j] = !MX && kv.dtype == MVLM_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, f16x2_t))
                                                     : __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_t));
            }
            if (LANES == 0 && d >= D) return;
            if (is_q) {
                if (slot0 < 0) out = u32x4{0u, 0u, 0u, 0u};
                *reinterpret_cast<u32x4*>(q_to + head * D) = out;
            } else if (slot0 >= 0)
                *reinterpret_cast<u32x4*>((is_k ? kv.k : kv.v) + (kv_to + (head - (is_k ? a.heads : qk)) * kv_step)) = out;
            return;
        }
        if constexpr (MX) {
            const auto larger = [](float u, float w) { return fmaxf(u, w); };
            float most = 0.0f;                             // of |v|; a NaN is not taken
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
            if (most == INFINITY) {                        // few have any: the largest of the others
                most = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fabsf(v[e]) < INFINITY ? fmaxf(most, fabsf(v[e])) : most;
            }
            most = over_lanes(most, 1, min(lanes, MX_BLOCK / 8), larger);
            const int ex = mx_exponent(__float_as_uint(most));
            const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = v[e] * down;
            if (ex == MX_MOST) {                           // 248 and above would round to 2^8, a value of 2^128
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (fabsf(v[e]) < INFINITY) y[e] = fminf(fmaxf(y[e], -240.0f), 240.0f);
            }
            u32x2 code;                                    // the conversion makes NaN of infinities as well
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j], y[4 * j + 1], 0, false);
                code[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2], y[4 * j + 3], c, true);
            }
            uint32_t word = (uint32_t)(ex + MX_BIAS) << (d / MX_BLOCK * 8);
            word = over_lanes(word, MX_BLOCK / 8, lanes, [](uint32_t u, uint32_t w) { return u | w; });
            if (slot0 < 0) return;
            const int h = head - (is_k ? a.heads : qk);
            if (LANES > 0 || d < D) *reinterpret_cast<u32x2*>((uint8_t*)(is_k ? kv.k : kv.v) + (kv_to + h * kv_step)) = code;
            if (sub == 0) kv.scales(is_k ? kv.k : kv.v)[slot0 + h * kv.page.div] = word;
        }
    };
    // The lanes of a head go round together, so that each finds the others.
    for (int head = own; head < all; head += step) {
        const AppendRaw<XD, VEC> x = ahead[0];
#pragma unroll
        for (int u = 0; u + 1 < HEADS_AHEAD; ++u) ahead[u] = ahead[u + 1];
        ahead[HEADS_AHEAD - 1].load(a.qkv, xrow + (int64_t)min(head + HEADS_AHEAD * step, all - 1) * D + dl);
        make(head, x);
    }
}

hipError_t launch_kv_append(hipStream_t s, const KvAppendArgs& a) {
    const size_t es = dtype_size(a.x_dtype);
    const bool vec = ((uintptr_t)a.qkv & 15u) == 0 && (a.ld * (int64_t)es) % 16 == 0;
    const dim3 grid((unsigned)a.batch.rows), block(APPEND_THREADS);
    // a row's prologue is paid by each of its waves: two of them where the rows fill the chip (16162 rows of 32 + 2 x 8
    // heads of 128: 93 us, with four 102, with one 93, all since 9 less), four where they do not.  fp16 rows of 3 x 32 heads
    // of 64 with two and with four waves: 512 rows 7.2 and 5.7 us, 1024 8.8 and 7.9, 1536 10.9 and 10.7, 2048 11.8 and 13.3, 4096
    // 19.1 and 21.1; bf16 of 32 + 2 x 8 heads of 128 the same within 6%
    const dim3 hblock(a.batch.rows >= 2048 ? APPEND_THREADS / 2 : APPEND_THREADS);
    const bool by_head = a.kv.dtype == MVLM_MXFP8 || a.q_weight || a.k_weight;
    auto go = [&](auto dt) {
        constexpr int XD = decltype(dt)::value;
        if (by_head) {
            auto heads = [&](auto mx, auto norm) {
                constexpr bool MX = decltype(mx)::value, NORM = decltype(norm)::value;
                auto lanes = [&](auto n) {
                    constexpr int LANES = decltype(n)::value;
                    if (a.rot > 0 && !a.interleaved && a.rot % 16 == 0) launch_kernel(kv_append_heads_kernel<XD, true, MX, NORM, LANES, true>, grid, hblock, 0, s, a);
                    else launch_kernel(kv_append_heads_kernel<XD, true, MX, NORM, LANES, false>, grid, hblock, 0, s, a);
                };
                if (!vec) launch_kernel(kv_append_heads_kernel<XD, false, MX, NORM, 0, false>, grid, hblock, 0, s, a);
                else if (a.kv.D == 128) lanes(std::integral_constant<int, 16>{});
                else if (a.kv.D == 64) lanes(std::integral_constant<int, 8>{});
                else lanes(std::integral_constant<int, 0>{});
            };
            const bool norm = a.q_weight || a.k_weight;
            if (a.kv.dtype != MVLM_MXFP8) heads(std::false_type{}, std::true_type{});
            else if (norm) heads(std::true_type{}, std::true_type{});
            else heads(std::true_type{}, std::false_type{});
            return;
        }
        if (vec) launch_kernel(kv_append_kernel<XD, true>, grid, block, 0, s, a);
        else launch_kernel(kv_append_kernel<XD, false>, grid, block, 0, s, a);
    };
    if (a.x_dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.x_dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
