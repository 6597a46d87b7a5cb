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
// block owns a slice of a row's tokens, T of them per thread, and counts the
// history's tokens that fall into it in LDS (one word per token: generated
// occurrences, and the top bit for one in the prompt), so no count ever reaches
// memory.  A thread asks for its logits, its mask bits and its share of the
// history before it waits for any of them.  Every block of a row reads the row's
// history, from L2 after the first: history / slice of the logits' own traffic.
// Measured: 128 rows of 128000 fp32 logits with mask, 64 biases and 4096 tokens of
// history, 135 MB: 29 .. 31 us, 4.4 .. 4.6 TB/s (116 us where each load was waited for
// before the next, 32.7 with the mask words read by every thread itself); one row of
// 51200: 3.8 us, a launch.
// Integer counts and the maximum of entry numbers do not depend on the order in
// which the threads arrive.
#include "common.h"
#include "device_math.h"
#include "logits.h"

#include <algorithm>

namespace mvlm {

constexpr uint32_t IN_PROMPT = 0x80000000u;
constexpr int LOGITS_IDS = 8;          // history entries in flight per thread

// N consecutive logits from x[t], N of them past v1 read as 0
template <int DT, int N, bool VEC>
__device__ __forceinline__ void load_logits(const void* x, int64_t t, int left, float (&v)[N]) {
    if (VEC && left >= N) {
        if constexpr (DT == MVLM_F32) {
            static_assert(N == 4, "16 bytes");
            const f32x4 w = *reinterpret_cast<const f32x4*>((const float*)x + t);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = w[e];
        } else {
            uint32_t w[N / 2];
            if constexpr (N == 8) {
                const u32x4 q = *reinterpret_cast<const u32x4*>((const uint16_t*)x + t);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = q[e];
            } else {
                const u32x2 q = *reinterpret_cast<const u32x2*>((const uint16_t*)x + t);
                w[0] = q[0], w[1] = q[1];
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const uint16_t h = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
                v[e] = DT == MVLM_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < left ? load_as_f32(x, t + e, DT) : 0.0f;
}

template <int DT, int N, bool VEC>
__device__ __forceinline__ void store_logits(void* y, int64_t t, int left, const float (&v)[N]) {
    if (VEC && left >= N) {
        if constexpr (DT == MVLM_F32) {
            *reinterpret_cast<f32x4*>((float*)y + t) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
            uint32_t w[N / 2];
#pragma unroll
            for (int e = 0; e < N / 2; ++e)
                w[e] = DT == MVLM_F16 ? (uint32_t)f32_to_f16_bits(v[2 * e]) | (uint32_t)f32_to_f16_bits(v[2 * e + 1]) << 16
                                      : (uint32_t)f32_to_bf16_bits(v[2 * e]) | (uint32_t)f32_to_bf16_bits(v[2 * e + 1]) << 16;
            if constexpr (N == 8) *reinterpret_cast<u32x4*>((uint16_t*)y + t) = u32x4{w[0], w[1], w[2], w[3]};
            else *reinterpret_cast<u32x2*>((uint16_t*)y + t) = u32x2{w[0], w[1]};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < left) store_out(y, t + e, v[e], DT);
}

// A thread's share of a list, entries tid, tid + THREADS, ...: asked for LOGITS_IDS
// at a time, the first of them before the list's length is known (its room is).
template <int THREADS, int BATCH>
struct ListShare {
    int id[BATCH];
    const int* list;
    int room, tid;
    __device__ __forceinline__ void ask(int base) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u) id[u] = list[min(base + u * THREADS, room - 1)];
    }
    __device__ __forceinline__ ListShare(const int* l, int width, int t) : list(l), room(width), tid(t) {
        if (list) ask(tid);
    }
    // f(i, list[i]) for the thread's entries below len
    template <class F>
    __device__ __forceinline__ void each(int len, F&& f) {
        for (int base = tid; base < len; base += THREADS * BATCH) {
            if (base != tid) ask(base);
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (base + u * THREADS < len) f(base + u * THREADS, id[u]);
        }
    }
};

// T tokens per thread; VEC: rows of x and out start 16-byte aligned
template <int DT, bool VEC, int THREADS, int T>
__global__ __launch_bounds__(THREADS) void logits_kernel(const LogitsArgs a) {
    constexpr int N = DT == MVLM_F32 || T == 4 ? 4 : 8, NV = T / N, SLICE = THREADS * T;
    extern __shared__ __attribute__((aligned(16))) uint32_t words[];   // [SLICE] counts, then [SLICE] last bias entries + 1
    uint32_t* counts = words;
    uint32_t* entries = words + (a.penalties ? SLICE : 0);
    const int row = (int)(blockIdx.x / (uint32_t)a.slices);
    const int v0 = ((int)blockIdx.x - row * a.slices) * SLICE, size = min(SLICE, a.n - v0);
    const int tid = (int)threadIdx.x;
    const int64_t base = (int64_t)row * a.ld + v0;
    __shared__ uint32_t allow[SLICE / 32];
    float v[NV][N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int t = (i * THREADS + tid) * N;
        load_logits<DT, N, VEC>(a.x, base + t, size - t, v[i]);
    }
    if (a.allowed && 32 * tid < size) allow[tid] = a.allowed[(int64_t)row * ((a.n + 31) / 32) + v0 / 32 + tid];
    ListShare<THREADS, LOGITS_IDS> history(a.penalties ? a.history + (int64_t)row * a.history_width : nullptr,
                                           a.history_width, tid);
    ListShare<THREADS, 1> biases(a.bias_ids ? a.bias_ids + (int64_t)row * a.bias_width : nullptr, a.bias_width, tid);
    const int used = (a.penalties ? SLICE : 0) + (a.bias_ids ? SLICE : 0);
    for (int i = 4 * tid; i < used; i += 4 * THREADS) *reinterpret_cast<u32x4*>(words + i) = u32x4{0u, 0u, 0u, 0u};
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    int len = 0, from = 0, bias_len = 0;
    if (a.penalties) {
        rep = a.penalties[3 * (int64_t)row];
        freq = a.penalties[3 * (int64_t)row + 1];
        pres = a.penalties[3 * (int64_t)row + 2];
        len = min(max(a.history_len[row], 0), a.history_width);
        from = a.generated_from ? a.generated_from[row] : 0;
    }
    if (a.bias_ids) bias_len = min(max(a.bias_len[row], 0), a.bias_width);
    __syncthreads();
    if (a.penalties) {
        history.each(len, [&](int i, int id) {
            if ((uint32_t)(id - v0) < (uint32_t)size) {
                if (i >= from) atomicAdd(&counts[id - v0], 1u);
                else atomicOr(&counts[id - v0], IN_PROMPT);
            }
        });
    }
    const float* bias = a.bias_values + (int64_t)row * a.bias_width;
    if (a.bias_ids) {
        biases.each(bias_len, [&](int i, int id) {
            if ((uint32_t)(id - v0) < (uint32_t)size) atomicMax(&entries[id - v0], (uint32_t)i + 1u);
        });
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int t = (i * THREADS + tid) * N;
        if (a.penalties) {
#pragma unroll
            for (int q = 0; q < N; q += 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(counts + t + q);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& x = v[i][q + e];
                    const uint32_t g = w[e] & ~IN_PROMPT;
                    if (w[e]) x = x > 0.0f ? x / rep : x * rep;
                    if (g) x -= __builtin_fmaf((float)g, freq, pres);
                }
            }
        }
        if (a.bias_ids) {
#pragma unroll
            for (int q = 0; q < N; q += 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(entries + t + q);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (w[e]) v[i][q + e] += bias[w[e] - 1];
            }
        }
        if (a.allowed && t < size) {
            const uint32_t mask = allow[t >> 5] >> (t & 31);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (!((mask >> e) & 1u)) v[i][e] = -INFINITY;
        }
        store_logits<DT, N, VEC>(a.out, base + t, size - t, v[i]);
    }
}

template <int DT, bool VEC, int THREADS, int T>
static void launch_slices(hipStream_t s, LogitsArgs a) {
    constexpr int SLICE = THREADS * T;
    a.slices = (a.n + SLICE - 1) / SLICE;
    const uint32_t shmem = SLICE * 4u * ((a.penalties ? 1u : 0u) + (a.bias_ids ? 1u : 0u));
    launch_kernel(logits_kernel<DT, VEC, THREADS, T>, dim3((unsigned)(a.rows * a.slices)), dim3(THREADS), shmem, s, a);
}

hipError_t launch_logits(hipStream_t s, const LogitsArgs& a, int num_cus) {
    const int es = a.dtype == MVLM_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)a.x | (uintptr_t)a.out) & 15u) == 0 && (a.ld * es) % 16 == 0;
    // slices of 4096 tokens read the history a quarter as often as slices of 1024, which
    // share few rows among more CUs (16 rows of 128000 5.7 us against 6.5, 128 rows 25
    // against 32; one row of 51200 4.3 us against 3.5, from 8 rows of 128000 on no difference)
    const bool large = (int64_t)a.rows * ((a.n + 4095) / 4096) >= 2 * (int64_t)num_cus;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (vec) {
            if (large) launch_slices<DT, true, 512, 8>(s, a);
            else launch_slices<DT, true, 256, 4>(s, a);
        } else {
            if (large) launch_slices<DT, false, 512, 8>(s, a);
            else launch_slices<DT, false, 256, 4>(s, a);
        }
    };
    if (a.dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
