// Penalties of repeated tokens, biases and grammar masks on a batch's logits, in
// one pass over them.  For token t of row r, with c and g the number of times it
// occurs in the row's history and in the generated part of it:
//   x = x > 0 ? x / rep : x rep            if c > 0
//   x = x - (g freq + (g > 0) pres)
//   x = x + bias                           of the last entry that names t
//   x = -inf                               where the mask does not allow t
// in fp32, rounded once to the logits' type.
//
// Reading and writing the logits once bounds it, and for one row the launch.  A
// block owns a slice of a row's tokens and counts the history's tokens that fall
// into it in LDS (one word per token: generated occurrences, and the top bit for
// one in the prompt), so no count ever reaches memory; every block of a row reads
// the row's history, from L2 after the first, which costs history / slice of the
// logits' own traffic.  Integer counts and the maximum of entry numbers do not
// depend on the order in which the threads arrive.
#include "common.h"
#include "device_math.h"
#include "logits.h"

#include <algorithm>

namespace mvlm {

constexpr int LOGITS_THREADS = 256;
constexpr uint32_t IN_PROMPT = 0x80000000u;

template <int DT>
__device__ __forceinline__ float logit_elem(const u32x4& w, int e) {
    if constexpr (DT == MVLM_F32) return __uint_as_float(w[e]);
    const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    return DT == MVLM_F16 ? f16_bits_to_f32(b) : bf16_bits_to_f32(b);
}

template <int DT, bool VEC>
__global__ __launch_bounds__(LOGITS_THREADS) void logits_kernel(const LogitsArgs a) {
    extern __shared__ uint32_t counts[];                       // [slice] counts, then [slice] last bias entries + 1
    constexpr int ES = DT == MVLM_F32 ? 4 : 2, EPC = VEC ? 16 / ES : 1;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices);
    const int v0 = ((int)blockIdx.x - row * a.slices) * a.slice, v1 = min(v0 + a.slice, a.n);
    const int tid = (int)threadIdx.x;
    uint32_t* entries = counts + a.slice;
    if (a.penalties)
        for (int i = tid; i < a.slice; i += LOGITS_THREADS) counts[i] = 0u;
    if (a.bias_ids)
        for (int i = tid; i < a.slice; i += LOGITS_THREADS) entries[i] = 0u;
    __syncthreads();
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.penalties) {
        rep = a.penalties[3 * (int64_t)row];
        freq = a.penalties[3 * (int64_t)row + 1];
        pres = a.penalties[3 * (int64_t)row + 2];
        const int len = min(max(a.history_len[row], 0), a.history_width);
        const int from = a.generated_from ? a.generated_from[row] : 0;
        const int* ids = a.history + (int64_t)row * a.history_width;
        for (int i = tid; i < len; i += LOGITS_THREADS) {
            const int id = ids[i];
            if (id >= v0 && id < v1) {
                if (i >= from) atomicAdd(&counts[id - v0], 1u);
                else atomicOr(&counts[id - v0], IN_PROMPT);
            }
        }
    }
    const float* bias = nullptr;
    if (a.bias_ids) {
        const int len = min(max(a.bias_len[row], 0), a.bias_width);
        const int* ids = a.bias_ids + (int64_t)row * a.bias_width;
        bias = a.bias_values + (int64_t)row * a.bias_width;
        for (int i = tid; i < len; i += LOGITS_THREADS) {
            const int id = ids[i];
            if (id >= v0 && id < v1) atomicMax(&entries[id - v0], (uint32_t)i + 1u);
        }
    }
    __syncthreads();
    const uint32_t* allowed = a.allowed ? a.allowed + (int64_t)row * ((a.n + 31) / 32) : nullptr;
    auto one = [&](float x, int t) {
        if (a.penalties) {
            const uint32_t w = counts[t - v0], g = w & ~IN_PROMPT;
            if (w) x = x > 0.0f ? x / rep : x * rep;
            if (g) x -= __builtin_fmaf((float)g, freq, pres);
        }
        if (bias) {
            const uint32_t e = entries[t - v0];
            if (e) x += bias[e - 1];
        }
        if (allowed && !((allowed[t >> 5] >> (t & 31)) & 1u)) x = -INFINITY;
        return x;
    };
    const int64_t base = (int64_t)row * a.ld;
    const uint8_t* x = (const uint8_t*)a.x + base * ES;
    uint8_t* out = (uint8_t*)a.out + base * ES;
    if constexpr (VEC) {
        const int whole = v0 + (v1 - v0) / EPC * EPC;
        for (int t = v0 + tid * EPC; t < whole; t += LOGITS_THREADS * EPC) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(x + (int64_t)t * ES);
            u32x4 o;
            if constexpr (DT == MVLM_F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __float_as_uint(one(logit_elem<DT>(w, e), t + e));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = one(logit_elem<DT>(w, 2 * e), t + 2 * e), hi = one(logit_elem<DT>(w, 2 * e + 1), t + 2 * e + 1);
                    o[e] = DT == MVLM_F16 ? (uint32_t)f32_to_f16_bits(lo) | (uint32_t)f32_to_f16_bits(hi) << 16
                                          : (uint32_t)f32_to_bf16_bits(lo) | (uint32_t)f32_to_bf16_bits(hi) << 16;
                }
            }
            *reinterpret_cast<u32x4*>(out + (int64_t)t * ES) = o;
        }
        for (int t = whole + tid; t < v1; t += LOGITS_THREADS) store_out(out, t, one(load_as_f32(x, t, DT), t), DT);
    } else {
        for (int t = v0 + tid; t < v1; t += LOGITS_THREADS) store_out(out, t, one(load_as_f32(x, t, DT), t), DT);
    }
}

hipError_t launch_logits(hipStream_t s, const LogitsArgs& in, int num_cus) {
    LogitsArgs a = in;
    // the largest slice that still gives every CU a block: large slices read the
    // history less often, small ones share a row among more CUs
    a.slice = 8192;
    while (a.slice > 1024 && (int64_t)a.rows * ((a.n + a.slice - 1) / a.slice) < num_cus) a.slice /= 2;
    a.slices = (a.n + a.slice - 1) / a.slice;
    const int es = a.dtype == MVLM_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)a.x | (uintptr_t)a.out) & 15u) == 0 && (a.ld * es) % 16 == 0;
    const uint32_t shmem = (uint32_t)a.slice * 4u * (a.bias_ids ? 2u : 1u);
    const dim3 grid((unsigned)(a.rows * a.slices)), block(LOGITS_THREADS);
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (vec) launch_kernel(logits_kernel<DT, true>, grid, block, shmem, s, a);
        else launch_kernel(logits_kernel<DT, false>, grid, block, shmem, s, a);
    };
    if (a.dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
