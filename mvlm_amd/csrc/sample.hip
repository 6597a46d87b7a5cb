// A token of each row of logits by temperature, min-p, top-k, top-p and a given uniform number (mvlm_sample).
//
// With m the row's largest value and t_i = (v_i - m) log2(e) / T <= 0 in 64 bits, a token's weight is
//   W_i = round(2^(bits + t_i)), an integer: 2^bits for the largest, 0 below 2^-(bits + 1) of it.
// Integers below 2^62 / n add up exactly in any order and in any parts, so that a row's token is the same whichever
// blocks make it.  In the order of falling value (the lower index first among
// equals) everything asked for is a start of the row or a place in it:
//   live     t_i >= max(log2(min_p), -(bits + 1))
//   top-k    the place of the k-th live token
//   top-p    the first place at which the running sum of W reaches ceil(top_p x the sum so far kept)
//   picked   the first at which it reaches floor(u x the sum kept) + 1
// so one search serves all three.  Values are compared as integers that order like them (sample_key).
//
//  * Few tokens can be kept: the candidates, the tokens above a bound, go into LDS.  With the k-th largest of the
//    threads' largest values as bound, k tokens at least lie above it (some THREADS ln(THREADS / (THREADS - k)) of
//    them where values do not depend on their places).  So top_k of up to RANKS has all that it may keep among the
//    candidates, and min_p has with the bound that it sets itself.
//  * Up to LIST candidates are sorted (128 by one wave, two to a lane), and running sums give the answers.  More of them
//    are counted in steps of t first, and top_k's cut away; what is still more (or all live tokens of the row) is
//    searched by steps of 1 / STEPS, counted with their weights.  A search finds its step in the running sums,
//    sorts the step's tokens, and finds its place among them; a step of more tokens than the list holds is counted
//    again in ranges of keys, down to equal values, of which the index decides.
// A row whose candidates are enough and that a block can hold is made by one block.  A longer one is looked through by
// as many as can hold it, and the block that ends last puts their candidates together.  Of the others, whose weights all
// count, each of `slices` blocks looks for the row's largest value, so that it need not wait to be told the weights' unit, and
// counts a slice; the block that ends last adds the slices up and searches.  No block waits for another.  A row's blocks
// are on one XCD where there are 8 rows, whose L2 has the row after the first of them (64 open rows of 128000 82 us, spread 98).
// Running sums are over THREADS bins or entries, one of each thread's, which then knows whether a place is its own.
//
// Its floor is one look at the row, but few rows leave most of the chip without work, and what bounds it are chains of
// barriers, LDS atomics and searches.  Measured: one fp32 row of 51200, top_k 50, top_p 0.95: 9.2 us (a launch 3.7,
// tokens 2, bound and candidates 2, sort and draw 1.5; found one by one 28, in bins 11); 16 bf16 rows, half masked,
// top_p 0.9: 32 us (largest value 3.4, slices 9, arrival and their sum 2, two searches 16; by one block each 83, steps of
// 1/8 octave 38); 128 fp32 rows of 128000, 65.5 MB, top_p 0.9: 138 us, 0.5 TB/s (two blocks a row, which count for 62 of them,
// and search for 28); the same rows with top_k to 1250, min_p 0.02: 39 us, 1.7 TB/s (tokens 19, as many as greedy rows take; a row
// to a block 41, candidates counted in bins 86); one row of 128000, top_k 1000: 32 us (its tail read without a bound 216).
#include "common.h"
#include "device_math.h"
#include "sample.h"

#include <algorithm>

namespace mvlm {

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_BATCH = 4;        // 16-byte chunks in flight per thread behind the held ones
constexpr int HOLD = 52;               // words of tokens that a thread keeps: 53248 fp32 tokens of a row, twice as many of 16 bits
constexpr int CANDIDATES = 8192;       // room for them in LDS
constexpr int LIST = SAMPLE_THREADS;   // entries that are sorted at once
constexpr int RANKED = 256;            // of which so many by counting
constexpr int RANKS = 1000;            // of the threads' largest values
constexpr int RANK_BINS = 256, RANK_STEPS = 8;   // in which they are counted, per factor of two of the weight
constexpr int BINS = SAMPLE_THREADS;
constexpr int STEPS = 48;              // bins per factor of two of the weight; the last has all that lies 2^21 and more below the first

typedef unsigned long long u64;

// An integer that orders like the value with these bits: NaN as the infinity of its sign, -0 as 0.
__device__ __forceinline__ uint32_t sample_key(float f) {
    uint32_t b = __float_as_uint(f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) b = (b & 0x80000000u) | 0x7F800000u;
    if (b == 0x80000000u) b = 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float as_number(float v) { return v == v ? v : __uint_as_float((__float_as_uint(v) & 0x80000000u) | 0x7F800000u); }
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
constexpr uint32_t KEY_NEG_INF = 0x007FFFFFu, KEY_INF = 0xFF800000u;

// 2^x for -1 <= x <= 51: 2^n times the exponential series of f ln 2, n the integer next to x, f = x - n; its 14th
// term is below 2^-57 of the sum.  Adding 1.5 2^52 leaves n in the low bits: additions go at four times the
// rate of conversions and roundings in 64 bits.
__device__ __forceinline__ double exp2_series(double x) {
    constexpr double L1 = 0.69314718055994530942, L2 = L1 * L1, L4 = L2 * L2, L8 = L4 * L4;
    constexpr double HALVES = 6755399441055744.0;
    const double r = x + HALVES, f = x - (r - HALVES);
    double p = L8 * L4 * L1 / 6227020800.0;
    p = __builtin_fma(p, f, L8 * L4 / 479001600.0);
    p = __builtin_fma(p, f, L8 * L2 * L1 / 39916800.0);
    p = __builtin_fma(p, f, L8 * L2 / 3628800.0);
    p = __builtin_fma(p, f, L8 * L1 / 362880.0);
    p = __builtin_fma(p, f, L8 / 40320.0);
    p = __builtin_fma(p, f, L4 * L2 * L1 / 5040.0);
    p = __builtin_fma(p, f, L4 * L2 / 720.0);
    p = __builtin_fma(p, f, L4 * L1 / 120.0);
    p = __builtin_fma(p, f, L4 / 24.0);
    p = __builtin_fma(p, f, L2 * L1 / 6.0);
    p = __builtin_fma(p, f, L2 / 2.0);
    p = __builtin_fma(p, f, L1);
    p = __builtin_fma(p, f, 1.0);
    const u64 b = (u64)__double_as_longlong(p);
    return __longlong_as_double((long long)(b + ((u64)(uint32_t)__double_as_longlong(r) << 52)));
}

// 2^x rounded to an integer, -1 <= x <= 51
__device__ __forceinline__ u64 integer_power(double x) {
    return (u64)__double_as_longlong(exp2_series(x) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // + 2^52: its unit is 1
}

// What a row's block knows of it.
struct SampleRow {
    uint32_t top;                      // key of the largest value
    double m, c;                       // that value, log2(e) / T; where it is infinite, 0 and 0: its like have t = 0
    double bits;
    // Each operation rounds by itself: t's product and the sum below made one fma in one place and not in another would make
    // two weights of a token, and a sum would not be that of its tokens'.
    __device__ __forceinline__ double t(float v) const {
#pragma clang fp contract(off)
        return ((double)fminf(v, 3.402823466e38f) - m) * c;
    }
    __device__ __forceinline__ u64 weight(double t) const {
#pragma clang fp contract(off)
        const double x = t + bits;
        return integer_power(x);
    }
    // The bin of a value: how many steps of v log2(e) / T lie between its own and the largest's.
    double steps = STEPS, step0;
    __device__ __forceinline__ double step(float v, double c) const { return __builtin_floor((double)fminf(v, 3.402823466e38f) * c * steps); }
    __device__ __forceinline__ int bin(float v) const { return (int)fmin(step0 - step(v, c), BINS - 1.0); }
};

// ceil(p z) (p in (0, 1), UP) or floor(p z) of a float p in [0, 1) and an integer z, exactly
template <bool UP>
__device__ __forceinline__ u64 part_of(float p, u64 z) {
    const uint32_t b = __float_as_uint(p);
    const int ex = (int)(b >> 23);
    const uint32_t mant = ex ? (b & 0x7FFFFFu) | 0x800000u : b & 0x7FFFFFu;
    const int k = 150 - (ex ? ex : 1);                             // p = mant 2^-k, k >= 24
    const u64 lo = z * mant, hi = __umul64hi(z, mant);             // below 2^88
    u64 q, rest;
    if (k < 64) {
        q = lo >> k | hi << (64 - k);
        rest = lo & ((1ull << k) - 1);
    } else if (k < 128) {
        q = k == 64 ? hi : hi >> (k - 64);
        rest = lo | (k == 64 ? 0 : hi & ((1ull << (k - 64)) - 1));
    } else {
        q = 0;
        rest = lo | hi;
    }
    return q + (UP && rest ? 1 : 0);
}

// A row's tokens as a thread sees them: chunks of 16 bytes (EPC tokens), THREADS apart, -inf behind the row's end.
template <int DT, bool VEC>
struct RowTokens {
    static constexpr int EPC = DT == MVLM_F32 ? 4 : 8, CHUNKS = HOLD / 4;
    const void* x;
    int64_t row;
    int n, chunks;                     // tokens, chunks (the last may be short)
    u32x4 held[CHUNKS];

    __device__ __forceinline__ u32x4 whole_chunk(int c) const {
        return *reinterpret_cast<const u32x4*>((const char*)x + (row + (int64_t)c * EPC) * (DT == MVLM_F32 ? 4 : 2));
    }
    __device__ __forceinline__ u32x4 load(int c) const {
        if (VEC && (c + 1) * EPC <= n) return whole_chunk(c);
        constexpr uint32_t NONE = DT == MVLM_F32 ? 0xFF800000u : DT == MVLM_F16 ? 0xFC00u : 0xFF80u;
        uint32_t t[EPC];
#pragma unroll
        for (int e = 0; e < EPC; ++e) {
            const int64_t i = row + (int64_t)c * EPC + e;
            t[e] = c * EPC + e >= n ? NONE : DT == MVLM_F32 ? ((const uint32_t*)x)[i] : ((const uint16_t*)x)[i];
        }
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = EPC == 4 ? t[e] : t[(2 * e) % EPC] | t[(2 * e + 1) % EPC] << 16;
        return w;
    }
    __device__ __forceinline__ static float value(uint32_t w, int e) {
        if constexpr (DT == MVLM_F32) return __uint_as_float(w);
        else if constexpr (DT == MVLM_BF16) return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
        else return f16_bits_to_f32((uint16_t)(e & 1 ? w >> 16 : w));
    }
    __device__ __forceinline__ float at(int i) const { return load_as_f32(x, row + i, DT); }
    // f(value) for the held tokens
    template <class F>
    __device__ __forceinline__ void each_held(F&& f) const {
#pragma unroll
        for (int u = 0; u < CHUNKS; ++u) {
            if (u * SAMPLE_THREADS >= chunks) break;
#pragma unroll
            for (int e = 0; e < EPC; ++e) f(value(held[u][e * 4 / EPC], e));
        }
    }
    // index of the nth of them
    __device__ __forceinline__ int held_index(int nth) const {
        return ((int)threadIdx.x + nth / EPC * SAMPLE_THREADS) * EPC + nth % EPC;
    }
    // f(value, nth of the batch) for the tokens of chunks [first, last), end(first index of the batch, THREADS apart by
    // chunks) after each batch, then rest(value, index) for those of a chunk that the row cuts short
    template <class F, class E, class R>
    __device__ __forceinline__ void each_batch(int first, int last, F&& f, E&& end, R&& rest) const {
        const int whole = VEC ? min(last, n / EPC) : last;     // chunks read in one load, but where rows are not aligned
        u32x4 next[SAMPLE_BATCH];
        auto ask = [&](int base) {
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u) {
                const int c = min(base + (int)threadIdx.x + u * SAMPLE_THREADS, whole - 1);
                if constexpr (VEC) next[u] = whole_chunk(c);
                else next[u] = load(c);
            }
        };
        if (first < whole) ask(first);
        for (int base = first; base < whole; base += SAMPLE_THREADS * SAMPLE_BATCH) {
            u32x4 w[SAMPLE_BATCH];
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u) w[u] = next[u];
            if (base + SAMPLE_THREADS * SAMPLE_BATCH < whole) ask(base + SAMPLE_THREADS * SAMPLE_BATCH);
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u)
                if (base + (int)threadIdx.x + u * SAMPLE_THREADS < whole)
#pragma unroll
                    for (int e = 0; e < EPC; ++e) f(value(w[u][e * 4 / EPC], e), u * EPC + e);
            end((base + (int)threadIdx.x) * EPC);
        }
        if constexpr (VEC)
            for (int i = max(whole, first) * EPC + (int)threadIdx.x; i < min(last * EPC, n); i += SAMPLE_THREADS) rest(at(i), i);
    }
    __device__ __forceinline__ static int batch_index(int from, int nth) { return from + nth / EPC * SAMPLE_THREADS * EPC + nth % EPC; }
    // f(value, index) for the tokens of chunks [first, last)
    template <class F>
    __device__ __forceinline__ void each_between(int first, int last, F&& f) const {
        const int whole = VEC ? min(last, n / EPC) : last;
        for (int base = (int)threadIdx.x + first; base < whole; base += SAMPLE_THREADS * SAMPLE_BATCH) {
            u32x4 w[SAMPLE_BATCH];
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u) {
                const int c = min(base + u * SAMPLE_THREADS, whole - 1);
                if constexpr (VEC) w[u] = whole_chunk(c);
                else w[u] = load(c);
            }
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u)
                if (base + u * SAMPLE_THREADS < whole)
#pragma unroll
                    for (int e = 0; e < EPC; ++e) f(value(w[u][e * 4 / EPC], e), (base + u * SAMPLE_THREADS) * EPC + e);
        }
        if constexpr (VEC)
            for (int i = max(whole, first) * EPC + (int)threadIdx.x; i < min(last * EPC, n); i += SAMPLE_THREADS) f(at(i), i);
    }
    // The largest of this thread's tokens of the row, a NaN as as_number takes it.  Nothing else is kept of them, so more
    // are in flight.
    __device__ __forceinline__ float most() const {
        constexpr int FLIGHT = 2 * SAMPLE_BATCH;
        const int whole = VEC ? n / EPC : chunks;
        float own = -INFINITY;
        bool odd = false;
        for (int base = (int)threadIdx.x; base < whole; base += SAMPLE_THREADS * FLIGHT) {
            u32x4 w[FLIGHT];
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) {                 // those past the end: the last chunk again
                const int c = min(base + u * SAMPLE_THREADS, whole - 1);
                if constexpr (VEC) w[u] = whole_chunk(c);
                else w[u] = load(c);
            }
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u)
#pragma unroll
                for (int e = 0; e < EPC; e += 2) {
                    const float a = value(w[u][e * 4 / EPC], e), b = value(w[u][(e + 1) * 4 / EPC], e + 1);
                    own = fmaxf(own, fmaxf(a, b));             // a NaN is not taken
                    odd |= __builtin_isunordered(a, b);
                }
        }
        if (odd) each([&](float v, int) { own = fmaxf(own, as_number(v)); });
        else if constexpr (VEC)
            for (int i = whole * EPC + (int)threadIdx.x; i < n; i += SAMPLE_THREADS) own = fmaxf(own, as_number(at(i)));
        return own;
    }
    template <class F>
    __device__ __forceinline__ void each_other(F&& f) const { each_between(CHUNKS * SAMPLE_THREADS, chunks, f); }
    template <class F>
    __device__ __forceinline__ void each(F&& f) const { each_between(0, chunks, f); }
    __device__ __forceinline__ void hold() {
        const uint32_t none = DT == MVLM_F32 ? 0xFF800000u : DT == MVLM_F16 ? 0xFC00FC00u : 0xFF80FF80u;
#pragma unroll
        for (int u = 0; u < CHUNKS; ++u) {
            const int c = (int)threadIdx.x + u * SAMPLE_THREADS;
            held[u] = c < chunks ? load(c) : u32x4{none, none, none, none};
        }
    }
};

// The least key of [lo, hi] for which f holds; f holds for hi and from some key on.  By a wave.
template <class F>
__device__ __forceinline__ uint32_t least_where(uint32_t lo, uint32_t hi, F&& f) {
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1, lane = threadIdx.x & 63;
        const uint32_t key = hi - lo >= lane * step ? lo + lane * step : hi;
        const uint64_t holds = __builtin_amdgcn_ballot_w64(f(key));
        // lane l's key is lo + l step or hi; the first that holds bounds the least from above, the one before from below
        const uint32_t l = holds ? (uint32_t)__builtin_ctzll(holds) : 64u;
        const uint32_t above = l < 64 && hi - lo >= l * step ? lo + l * step : hi;
        if (l) lo += (l - 1) * step + 1;
        hi = above;
    }
    return hi;
}

// A bin or a list entry of each thread: what lies before it, and its own.
struct Share {
    u64 before, own;
    uint32_t above, count;
};
struct SamplePlace {
    u64 before, own;
    uint32_t above, count;
    int index;
};

struct SampleLds {
    u64 candidates[CANDIDATES];        // ~key, index
    u64 list[LIST];                    // the same
    u64 sums[BINS], part_sums[BINS];   // weights of the bins, and of those of a range of keys
    uint32_t counts[BINS], part_counts[BINS];
    u64 wave_sums[SAMPLE_THREADS / 64];
    uint32_t wave_counts[SAMPLE_THREADS / 64];
    float wave_values[SAMPLE_THREADS / 64];
    SamplePlace place[2];
    uint32_t listed, word;
};

// v plus the values of the lanes before
__device__ __forceinline__ u64 scan_wave(u64 v) {
    auto step = [&](auto ctrl, auto rows, auto bound) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, decltype(ctrl)::value, decltype(rows)::value, 0xF, decltype(bound)::value);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xF, decltype(bound)::value);
        v += (u64)hi << 32 | lo;
    };
    using all = std::integral_constant<int, 0xF>;
    step(std::integral_constant<int, 0x111>{}, all{}, std::true_type{});   // row_shr:1
    step(std::integral_constant<int, 0x112>{}, all{}, std::true_type{});   // row_shr:2
    step(std::integral_constant<int, 0x114>{}, all{}, std::true_type{});   // row_shr:4
    step(std::integral_constant<int, 0x118>{}, all{}, std::true_type{});   // row_shr:8
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{}, std::false_type{});   // row_bcast:15 into rows 1 and 3
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{}, std::false_type{});   // row_bcast:31 into rows 2 and 3
    return v;
}

// The shares of threads that own w and c, and the sums of all; by all threads, which have synchronised since they
// read what an earlier call left.
__device__ __forceinline__ Share share_out(u64 w, uint32_t c, SampleLds& s, u64* sum, uint32_t* count) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const u64 iw = scan_wave(w);
    const uint32_t ic = (uint32_t)scan_wave((u64)c);
    if (lane == 63) s.wave_sums[wave] = iw, s.wave_counts[wave] = ic;
    __syncthreads();
    Share m{iw - w, w, ic - c, c};
    u64 sw = 0;
    uint32_t sc = 0;
#pragma unroll
    for (int i = 0; i < SAMPLE_THREADS / 64; ++i) {
        const u64 a = s.wave_sums[i];
        const uint32_t b = s.wave_counts[i];
        m.before += i < wave ? a : 0;
        m.above += i < wave ? b : 0;
        sw += a;
        sc += b;
    }
    *sum = sw;
    *count = sc;
    return m;
}

// v over the lanes of a wave with f, in all lanes
template <class F>
__device__ __forceinline__ float over_wave(float v, F&& f) {
    auto move = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, false));
    };
    v = f(v, move(v, std::integral_constant<int, 0xB1>{}));        // quad_perm [1, 0, 3, 2]
    v = f(v, move(v, std::integral_constant<int, 0x4E>{}));        // quad_perm [2, 3, 0, 1]
    v = f(v, move(v, std::integral_constant<int, 0x141>{}));       // row_half_mirror
    v = f(v, move(v, std::integral_constant<int, 0x140>{}));       // row_mirror: 16 lanes agree
    v = f(v, __shfl_xor(v, 16, 64));
    return f(v, __shfl_xor(v, 32, 64));
}

// list[0 .. size) in ascending order (entries differ), by all threads; size <= RANKED.  Each entry's place is the
// number of entries below it; THREADS / RANKED threads count for one.
__device__ __forceinline__ void rank_list(u64* list, int size) {
    constexpr int PARTS = SAMPLE_THREADS / RANKED;
    const int i = (int)threadIdx.x / PARTS, part = (int)threadIdx.x % PARTS;
    const u64 own = list[max(min(i, size - 1), 0)];
    int below = 0;
    for (int j = part; j < size; j += PARTS) below += list[j] < own;
    below += __shfl_xor(below, 1, 64);
    below += __shfl_xor(below, 2, 64);
    static_assert(PARTS == 4, "two exchanges");
    __syncthreads();
    if (part == 0 && i < size) list[below] = own;
    __syncthreads();
}

// the same for size <= LIST, by exchanges: each thread has an entry, and its partner's comes from the wave's lanes or
// through LDS
__device__ __forceinline__ void sort_list(u64* list, int size) {
    if (size <= RANKED) return rank_list(list, size);
    const int tid = (int)threadIdx.x;
    u64 own = tid < size ? list[tid] : ~0ull;
    for (int k = 2; k < 2 * size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            u64 other;
            if (j >= 64) {
                __syncthreads();
                list[tid] = own;
                __syncthreads();
                other = list[tid ^ j];
            } else
                other = __shfl_xor(own, j, 64);
            own = ((tid & j) == 0) == ((tid & k) == 0) ? min(own, other) : max(own, other);
        }
    __syncthreads();
    list[tid] = own;
    __syncthreads();
}

// Up to 128 entries in their order, two to a lane of a wave, with running sums of their weights.
struct WaveList {
    u64 entry0, entry1, upto0, upto1;  // of places 2 lane and 2 lane + 1
    int live;                          // entries that live
    __device__ __forceinline__ static u64 of_lane(u64 v, int l) {
        return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
    }
    __device__ __forceinline__ u64 sum_at(int place) const {
        const u64 even = of_lane(upto0, place >> 1), odd = of_lane(upto1, place >> 1);
        return place & 1 ? odd : even;
    }
    __device__ __forceinline__ int token_at(int place) const {
        const u64 even = of_lane(entry0, place >> 1), odd = of_lane(entry1, place >> 1);
        return (int)(uint32_t)(place & 1 ? odd : even);
    }
    // the first place whose running sum is need, which the sum of all is at least
    __device__ __forceinline__ int reaches(u64 need) const {
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(upto1 >= need);
        const int l = lanes ? __builtin_ctzll(lanes) : 63;
        return 2 * l + (of_lane(upto0, l) >= need ? 0 : 1);
    }
};
// from[0 .. size) through to[0 .. size), which may be the same
__device__ __forceinline__ WaveList wave_list(const u64* from, u64* to, int size, const SampleRow& r, double t_least) {
    const int lane = (int)threadIdx.x & 63;
    const u64 e0 = lane < size ? from[lane] : ~0ull, e1 = lane + 64 < size ? from[lane + 64] : ~0ull;
    int place0 = 0, place1 = 0;
    for (int j = 0; j < size; ++j) {
        const u64 other = from[j];
        place0 += other < e0;
        place1 += other < e1;
    }
    asm_wait_lgkmcnt<0>();
    if (lane < size) *(volatile u64*)&to[place0] = e0;
    if (lane + 64 < size) *(volatile u64*)&to[place1] = e1;
    asm_wait_lgkmcnt<0>();
    WaveList l;
    const auto weigh = [&](int place, u64* entry) {
        *entry = place < size ? *(volatile u64*)&to[place] : 0ull;
        const double t = place < size ? r.t(key_value(~(uint32_t)(*entry >> 32))) : -INFINITY;
        return t >= t_least ? t : -INFINITY;
    };
    const double t0 = weigh(2 * lane, &l.entry0), t1 = weigh(2 * lane + 1, &l.entry1);
    const u64 w0 = t0 > -INFINITY ? r.weight(t0) : 0, w1 = t1 > -INFINITY ? r.weight(t1) : 0;
    l.live = __popcll(__builtin_amdgcn_ballot_w64(t0 > -INFINITY)) + __popcll(__builtin_amdgcn_ballot_w64(t1 > -INFINITY));
    l.upto1 = scan_wave(w0 + w1);
    l.upto0 = l.upto1 - w1;
    return l;
}

// SPLIT: a row may be made by several blocks
template <int DT, bool VEC, bool SPLIT>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_kernel(const SampleArgs a) {
    __shared__ SampleLds s;
    int row = (int)blockIdx.x, slice = 0;
    if constexpr (SPLIT) {                                     // a row's blocks on one XCD (every eighth block's), while rows are left for all
        const int eight = 8 * a.slices, group = a.rows < 8 ? 0 : row / eight;
        row -= group * eight;
        if (8 * group + 8 <= a.rows) slice = row / 8, row %= 8;
        else {
            const int of_these = row / a.slices;
            slice = row - of_these * a.slices, row = of_these;
        }
        row += 8 * group;
    }
    const int tid = (int)threadIdx.x, n = a.n;
    RowTokens<DT, VEC> tokens;
    tokens.x = a.x;
    auto whole_row = [&] {
        tokens.row = (int64_t)row * a.ld;
        tokens.n = n;
        tokens.chunks = (n + tokens.EPC - 1) / tokens.EPC;
    };
    whole_row();
    if constexpr (!SPLIT) tokens.hold();
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    float min_p = a.min_p ? a.min_p[row] : 0.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, u = a.uniform[row];
    const int top_k = a.top_k ? a.top_k[row] : 0;
    if (!(u > 0.0f)) u = 0.0f;
    if (tid == 0) s.word = (uint32_t)n, s.listed = 0, s.place[0] = s.place[1] = SamplePlace{};

    // the largest value over all threads
    auto largest = [&](float v) {
        v = over_wave(v, [](float x, float y) { return fmaxf(x, y); });
        __syncthreads();
        if ((tid & 63) == 0) s.wave_values[tid >> 6] = v;
        __syncthreads();
        v = s.wave_values[0];
#pragma unroll
        for (int w = 1; w < SAMPLE_THREADS / 64; ++w) v = fmaxf(v, s.wave_values[w]);
        return v;
    };
    // The candidates are enough where `closed`: no other token can be kept.
    const bool by_rank = top_k > 0 && top_k <= RANKS, closed = by_rank || min_p > 0.0f;
    const double c = 1.4426950408889634074 / (double)T;
    const bool split = SPLIT && T > 0.0f && !closed;
    // Blocks that look for candidates: as many as it takes to hold the row.  1: this one looks at all of it.
    int parts = 1;
    if (SPLIT && T > 0.0f && closed) parts = min(a.slices, (tokens.chunks + tokens.CHUNKS * SAMPLE_THREADS - 1) / (tokens.CHUNKS * SAMPLE_THREADS));
    if (slice >= (split ? a.slices : parts)) return;
    // Parts cross workgroups: device-scope stores and loads, complete before a block counts itself in.  Whether this is
    // the last of `blocks`.
    auto arrive = [&](int blocks) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const uint32_t before = __hip_atomic_fetch_add(a.arrived + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (before == (uint32_t)blocks - 1) __hip_atomic_store(a.arrived + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s.word = before;
        }
        __syncthreads();
        return s.word == (uint32_t)blocks - 1;
    };
    const int64_t first_part = (int64_t)row * (SPLIT ? a.slices : 1), own_part = first_part + slice;
    float own = -INFINITY, top;                                // the largest of those that this thread holds, of all
    u64 slice_sum = 0;                                         // of this thread's bin, where the slices are added up
    uint32_t slice_count = 0;
    bool summed = false;
    SampleRow r;
    r.bits = (double)a.bits;
    auto with_top = [&] {
        r.top = sample_key(top);
        r.m = top < INFINITY ? (double)top : 0.0;
        r.c = top < INFINITY ? c : 0.0;
        r.step0 = r.step(top, r.c);
    };
    double t_least = -(r.bits + 1.0) + 0x1p-30;                // what lives has a weight of 1 at least
    if (min_p > 0.0f) t_least = fmax(t_least, log2((double)fminf(min_p, 1.0f)));
    if (split) {
        // each block finds the row's largest value, so that all count in the same unit and the sums are the row's
        top = largest(tokens.most());
        with_top();
        summed = top > -INFINITY && top < INFINITY;
        if (!summed && slice) return;                          // nothing to count, or infinities only: one block's work
    }
    if (summed) {
        const int per = (tokens.chunks + a.slices - 1) / a.slices, from = min(slice * per, tokens.chunks), to = min(from + per, tokens.chunks);
        s.counts[tid] = 0, s.sums[tid] = 0;
        __syncthreads();
        tokens.each_between(from, to, [&](float v, int) {
            if (!(v > -INFINITY)) return;                      // a NaN lies below all others here
            const double t = r.t(v);
            if (!(t >= t_least)) return;
            const int b = r.bin(v);
            atomicAdd(&s.counts[b], 1u);
            atomicAdd(&s.sums[b], r.weight(t));
        });
        __syncthreads();
        __hip_atomic_store(a.slice_sums + own_part * BINS + tid, s.sums[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.slice_counts + own_part * BINS + tid, s.counts[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!arrive(a.slices)) return;
        constexpr int AHEAD = 8;
        for (int i = 0; i < a.slices; i += AHEAD) {
            u64 w[AHEAD];
            uint32_t k[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int64_t at = (first_part + min(i + q, a.slices - 1)) * BINS + tid;
                w[q] = __hip_atomic_load(a.slice_sums + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                k[q] = __hip_atomic_load(a.slice_counts + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (i + q < a.slices) slice_sum += w[q], slice_count += k[q];
        }
    }
    const int per_part = (tokens.chunks + parts - 1) / parts;
    int base = 0;                                              // index of the tokens' first in the row
    if (parts > 1) {
        base = slice * per_part * tokens.EPC;
        tokens.row += base;
        tokens.n = min(n - base, per_part * tokens.EPC);
        tokens.chunks = (tokens.n + tokens.EPC - 1) / tokens.EPC;
    }
    // a finite value that is below those of all tokens with t >= t_to, by a little
    auto value_below = [&](double t_to) {
        if (!(c > 0.0)) return -3.402823466e38f;               // an infinite temperature: every finite value has t = 0
        const uint32_t k = sample_key((float)(r.m + t_to / c));
        return key_value(max(k, KEY_NEG_INF + 9) - 8);
    };
    auto to_list = [&](uint32_t key, int i) {
        const uint32_t to = atomicAdd(&s.listed, 1u);
        if (to < LIST) s.list[to] = (u64)~key << 32 | (uint32_t)i;
    };
    // the indices of marked tokens to the candidates, from place `to` on
    auto put = [&](u64 marks, uint32_t to, auto&& index) {
        for (; marks; marks &= marks - 1, ++to)
            if (to < CANDIDATES) s.candidates[to] = (u64)(uint32_t)index(__builtin_ctzll(marks));
    };
    // room for `own` of them from each lane of a wave
    auto places = [&](uint32_t own) {
        const uint32_t upto = (uint32_t)scan_wave((u64)own);
        uint32_t to = 0;
        if ((tid & 63) == 63) to = atomicAdd(&s.listed, upto);
        return (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + upto - own;
    };
    float least = -3.402823466e38f;                            // the candidates: from this value on
    int candidates = 0;
    bool compact = false;                                      // all of them are in LDS
    // Steps as fine as the bins allow for the candidates, and of many those that top_k may keep.
    auto refine = [&] {
        if (!compact) return;
        const double span = 2.0 - fmax(t_least, r.t(least));
        r.steps = STEPS;
        while (r.steps * 2.0 * span < BINS && r.steps < 65536.0) r.steps *= 2.0;
        with_top();
        if (!by_rank || candidates <= 128 || candidates <= top_k) return;
        s.counts[tid] = 0;
        if (tid == 0) s.word = BINS - 1, s.listed = 0;
        __syncthreads();
        for (int i = tid; i < candidates; i += SAMPLE_THREADS) atomicAdd(&s.counts[r.bin(key_value(~(uint32_t)(s.candidates[i] >> 32)))], 1u);
        __syncthreads();
        const uint32_t count = s.counts[tid], upto = (uint32_t)scan_wave((u64)count);
        if ((tid & 63) == 63) s.wave_counts[tid >> 6] = upto;
        __syncthreads();
        uint32_t above = upto - count;
        for (int w = 0; w < tid >> 6; ++w) above += s.wave_counts[w];
        if (above < (uint32_t)top_k && above + count >= (uint32_t)top_k) s.word = (uint32_t)tid;
        __syncthreads();
        const int bin = (int)s.word;
        for (int i = tid; i < candidates; i += SAMPLE_THREADS)
            if (const u64 entry = s.candidates[i]; r.bin(key_value(~(uint32_t)(entry >> 32))) <= bin) {
                const uint32_t to = atomicAdd(&s.listed, 1u);
                if (to < LIST) s.list[to] = entry;
            }
        __syncthreads();
        if (s.listed > LIST) return;
        candidates = (int)s.listed;
        if (tid < candidates) s.candidates[tid] = s.list[tid];
        if (bin < BINS - 1) least = fmaxf(least, value_below((r.step0 - bin) / r.steps - r.m * r.c));
        __syncthreads();
    };
    if (!split) {
        if constexpr (SPLIT) tokens.hold();
        bool odd = false;
        own = -INFINITY;
        tokens.each_held([&](float v) {
            own = fmaxf(own, v);                               // a NaN is not taken
            odd |= v != v;
        });
        if (odd) tokens.each_held([&](float v) { own = fmaxf(own, as_number(v)); });
        top = largest(own);
        with_top();
    }
    const bool more = !split && tokens.chunks > tokens.CHUNKS * SAMPLE_THREADS;

    if (!(T > 0.0f)) {                                         // the first token of the largest value
        const float held = own;
        int at = n;
        if (more) {
            tokens.each_other([&](float x, int i) {
                if (as_number(x) > own) own = as_number(x), at = i;
            });
            top = largest(own);
            if (own < top) at = n;
        }
        if (held == top) {
            int nth = 0;
            at = n;
            tokens.each_held([&](float v) {
                if (as_number(v) == top) at = min(at, tokens.held_index(nth));
                ++nth;
            });
        }
        for (int off = 32; off; off >>= 1) at = min(at, __shfl_xor(at, off, 64));
        if ((tid & 63) == 0) atomicMin(&s.word, (uint32_t)at);
        __syncthreads();
        if (tid == 0) a.out[row] = top == -INFINITY ? 0 : (int)s.word;
        return;
    }

    // A bound of many tokens is worth another look at those that are not held: with theirs among the threads' largest
    // it leaves fewer candidates, where they might be too many else, which costs far more (160 rows of 128000, with the look and
    // without: top_k 60 28 and 23 us, 250 35 and 30, 500 39 and 35, 1000 48 and 240; 200 of 60000 17 and 16, 23 and 21, 27 and 26,
    // 35 and 34).
    if (more && by_rank && top_k > RANKS / 4) {
        tokens.each_other([&](float x, int) { own = fmaxf(own, as_number(x)); });
        top = largest(own);
        with_top();
    }
    if (closed && top > -INFINITY && top < INFINITY) {
        if (by_rank) {                                         // the step of the k-th of the threads' largest
            if (tid < RANK_BINS) s.counts[tid] = 0;
            __syncthreads();
            if (own > -INFINITY) atomicAdd(&s.counts[(int)fmin(r.t(own) * -RANK_STEPS, RANK_BINS - 1.0)], 1u);
            __syncthreads();
            const uint32_t kth = (uint32_t)top_k;
            uint32_t n4[RANK_BINS / 64], run = 0;
#pragma unroll
            for (int i = 0; i < RANK_BINS / 64; ++i) run += n4[i] = s.counts[(tid & 63) * (RANK_BINS / 64) + i];
            const uint32_t upto = (uint32_t)scan_wave((u64)run);
            const uint64_t reached = __builtin_amdgcn_ballot_w64(upto >= kth);
            if (reached) {
                const int l = __builtin_ctzll(reached);
                uint32_t sum = (uint32_t)__builtin_amdgcn_readlane((int)(upto - run), l);
                int bin = l * (RANK_BINS / 64) - 1;
#pragma unroll
                for (int i = 0; i < RANK_BINS / 64; ++i) {
                    const uint32_t v = (uint32_t)__builtin_amdgcn_readlane((int)n4[i], l);
                    if (sum < kth) sum += v, ++bin;
                }
                if (bin < RANK_BINS - 1) least = value_below(-(bin + 1.0) / RANK_STEPS);
            }
        }
        if (min_p > 0.0f) least = fmaxf(least, value_below(t_least));
    }
    if (more) {
        float v = own;
        u64 marks = 0;
        tokens.each_batch(tokens.CHUNKS * SAMPLE_THREADS, tokens.chunks, [&](float x, int nth) {
            v = fmaxf(v, as_number(x));
            if (closed && x >= least) marks |= 1ull << nth;
        }, [&](int from) {
            if (!__builtin_amdgcn_ballot_w64(marks != 0)) return;
            put(marks, places((uint32_t)__popcll(marks)), [&](int nth) { return tokens.batch_index(from, nth); });
            marks = 0;
        }, [&](float x, int i) {
            v = fmaxf(v, as_number(x));
            if (closed && x >= least) put(1, atomicAdd(&s.listed, 1u), [&](int) { return i; });
        });
        top = largest(v);
        with_top();
        if (min_p > 0.0f && top < INFINITY) least = fmaxf(least, value_below(t_least));
    }
    if (closed && top > -INFINITY) {
        u64 marks[2] = {0, 0};
        int nth = 0;
        tokens.each_held([&](float v) {
            if (v >= least) marks[nth / 52] |= 1ull << nth % 52;
            ++nth;
        });
        const uint32_t first = (uint32_t)__popcll(marks[0]), to = places(first + (uint32_t)__popcll(marks[1]));
        put(marks[0], to, [&](int nth) { return tokens.held_index(nth); });
        put(marks[1], to + first, [&](int nth) { return tokens.held_index(52 + nth); });
        __syncthreads();
        candidates = (int)min(s.listed, CANDIDATES + 1u);
        compact = candidates <= CANDIDATES && top < INFINITY;
        if (compact) {
            // their values, again from memory
            constexpr int EACH = CANDIDATES / SAMPLE_THREADS;
            float v[EACH];
            int at[EACH];
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                at[q] = tid + q * SAMPLE_THREADS < candidates ? (int)(uint32_t)s.candidates[tid + q * SAMPLE_THREADS] : 0;
                v[q] = q * SAMPLE_THREADS < candidates ? tokens.at(at[q]) : 0.0f;
            }
#pragma unroll
            for (int q = 0; q < EACH; ++q)
                if (tid + q * SAMPLE_THREADS < candidates) s.candidates[tid + q * SAMPLE_THREADS] = (u64)~sample_key(v[q]) << 32 | (uint32_t)at[q];
        }
        __syncthreads();
    }
    if (parts > 1) {
    // the part's candidates, to the block that ends last
    refine();
    const bool fits = top == -INFINITY || compact;
    if (fits)
        for (int i = tid; i < candidates; i += SAMPLE_THREADS)
            __hip_atomic_store(a.part_entries + own_part * CANDIDATES + i, s.candidates[i] + (u64)base, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (tid == 0) {
        __hip_atomic_store(a.slice_counts + own_part * BINS, fits ? (uint32_t)candidates : CANDIDATES + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.slice_counts + own_part * BINS + 1, __float_as_uint(least), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.slice_tops + own_part, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!arrive(parts)) return;
    whole_row();
    r.steps = STEPS;                                           // those of the part's candidates are too fine for a row
    bool all_fit = true;
    top = -INFINITY;
    for (int i = 0; i < parts; ++i) {
        const uint32_t count = __hip_atomic_load(a.slice_counts + (first_part + i) * BINS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        all_fit = all_fit && count <= CANDIDATES;
        // what bounds a part's candidates from below bounds the row's: there are as many above it, or more
        least = fmaxf(least, __uint_as_float(__hip_atomic_load(a.slice_counts + (first_part + i) * BINS + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)));
        top = fmaxf(top, __hip_atomic_load(a.slice_tops + first_part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
    with_top();
    if (min_p > 0.0f && top > -INFINITY && top < INFINITY) least = fmaxf(least, value_below(t_least));
    if (tid == 0) s.listed = 0;
    __syncthreads();
    if (all_fit)
        for (int i = 0; i < parts; ++i) {
            const int count = (int)__hip_atomic_load(a.slice_counts + (first_part + i) * BINS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll 1
            for (int from = 0; from < count; from += SAMPLE_THREADS) {
                const int j = from + tid;
                const u64 entry = j < count ? __hip_atomic_load(a.part_entries + (first_part + i) * CANDIDATES + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : ~0ull;
                const bool takes = key_value(~(uint32_t)(entry >> 32)) >= least;   // of none: a NaN
                const uint32_t to = places(takes ? 1u : 0u);
                if (takes && to < CANDIDATES) s.candidates[to] = entry;
            }
        }
    __syncthreads();
    candidates = (int)min(s.listed, CANDIDATES + 1u);
    compact = all_fit && candidates <= CANDIDATES;
    __syncthreads();                                           // all have read the count, which refine() starts anew
    }
    if (top == -INFINITY) {
        if (tid == 0) a.out[row] = 0;
        return;
    }
    refine();

    const auto top_p_need = [&](u64 kept) { return top_p > 0.0f ? max(part_of<true>(top_p, kept), (u64)1) : (u64)1; };
    const auto token_need = [&](u64 kept) { return u < 1.0f ? part_of<false>(u, kept) + 1 : kept; };
    if (compact && candidates <= 128) {                        // a wave's work: two entries to a lane, and no barriers
        if (tid >= 64) return;
        const WaveList list = wave_list(s.candidates, s.list, candidates, r, t_least);
        u64 kept = list.sum_at(max(top_k > 0 ? min(top_k, list.live) : list.live, 1) - 1);
        if (top_p < 1.0f) kept = list.sum_at(list.reaches(top_p_need(kept)));
        const int token = list.token_at(list.reaches(token_need(kept)));
        if (tid == 0) a.out[row] = token;
        return;
    }

    int turn = 0;
    // what the thread with `mine` knows, to all threads
    auto announce = [&](bool mine, const Share& m) {
        if (mine) s.place[turn] = SamplePlace{m.before, m.own, m.above, m.count, tid};
        __syncthreads();
        const SamplePlace p = s.place[turn];
        turn ^= 1;                                             // the next one is written while this is still read
        return p;
    };
    // Where the running count or sum reaches need, which is 1 at least and the whole at most: a weight is the same integer
    // wherever it is counted.
    auto reaches = [&](const Share& m, bool by_count, u64 need) {
        const u64 before = by_count ? (u64)m.above : m.before;
        return announce(before < need && before + (by_count ? (u64)m.count : m.own) >= need, m);
    };
    // the list sorted, an entry to each thread
    auto share_list = [&](int size, u64* sum) __attribute__((always_inline)) {
        sort_list(s.list, size);
        uint32_t count;
        const double t = tid < size ? r.t(key_value(~(uint32_t)(s.list[tid] >> 32))) : -INFINITY;
        return share_out(t >= t_least ? r.weight(t) : 0, tid < size ? 1u : 0u, s, sum, &count);
    };
    if (compact && candidates <= LIST) {
        const int size = candidates;
        if (tid < size) s.list[tid] = s.candidates[tid];
        __syncthreads();
        u64 sum;
        const Share m = share_list(size, &sum);
        const int live = __syncthreads_count(tid < size && r.t(key_value(~(uint32_t)(s.list[tid] >> 32))) >= t_least);
        SamplePlace p = announce(tid == (top_k > 0 ? min(top_k, live) : live) - 1, m);
        if (top_p < 1.0f) p = reaches(m, false, top_p_need(p.before + p.own));
        p = reaches(m, false, token_need(p.before + p.own));
        if (tid == 0) a.out[row] = (int)(uint32_t)s.list[p.index];
        return;
    }

    const uint32_t live = r.top == KEY_INF ? KEY_INF : least_where(KEY_NEG_INF + 1, r.top, [&](uint32_t key) { return r.t(key_value(key)) >= t_least; });
    const float live_value = key_value(live);
    // f(t, key, index) for the live tokens of the row (a NaN passes the first test)
    auto each_live = [&](auto&& f) __attribute__((always_inline)) {
        tokens.each([&](float v, int i) {
            if (v < live_value) return;
            const uint32_t key = sample_key(v);
            if (key >= live) f(r.t(v), key, i);
        });
    };
    // the same for the candidates, or the row
    auto each = [&](bool of_row, auto&& f) __attribute__((always_inline)) {
        if (of_row) return each_live(f);
        for (int i = tid; i < candidates; i += SAMPLE_THREADS) {
            const uint32_t key = ~(uint32_t)(s.candidates[i] >> 32);
            if (key >= live) f(r.t(key_value(key)), key, (int)(uint32_t)s.candidates[i]);
        }
    };

    const bool of_row = !compact;
    u64 bin_sum = 0;
    uint32_t bin_count = 0;
    if (!summed) {
        s.counts[tid] = 0, s.sums[tid] = 0;
        __syncthreads();
        each(of_row, [&](double t, uint32_t key, int) {
            const int b = r.bin(key_value(key));
            atomicAdd(&s.counts[b], 1u);
            atomicAdd(&s.sums[b], r.weight(t));
        });
        __syncthreads();
        bin_sum = s.sums[tid], bin_count = s.counts[tid];
    } else {
        bin_sum = slice_sum, bin_count = slice_count;
    }
    {
        u64 sum_here;
        uint32_t all;
        const Share bins = share_out(bin_sum, bin_count, s, &sum_here, &all);
        const uint32_t k = top_k > 0 && (uint32_t)top_k < all ? (uint32_t)top_k : all;   // tokens kept by count
        u64 kept = sum_here;
        int token = 0;
        for (int step = 0; step < 3; ++step) {                 // top-k, top-p, the token
            if ((step == 0 && k == all) || (step == 1 && !(top_p < 1.0f))) continue;
            const bool by_count = step == 0;
            const u64 need = by_count ? k : step == 1 ? top_p_need(kept) : token_need(kept);
            u64 sum;
            SamplePlace p = reaches(bins, by_count, need);
            const int bin = p.index;
            u64 before = p.before;                             // of the tokens above the range
            uint32_t above = p.above, inside = p.count;
            // the range's keys: from the least with a bin <= this one to the one before the least with a bin below it
            uint32_t lo = least_where(live, r.top, [&](uint32_t key) { return r.bin(key_value(key)) <= bin; });
            uint32_t hi = bin == 0 ? r.top : least_where(lo, r.top, [&](uint32_t key) { return r.bin(key_value(key)) < bin; }) - 1;
            while (inside > LIST && lo < hi) {
                const uint32_t span = hi - lo;                 // keys less one
                int shift = 0;
                while ((span >> shift) >= (uint32_t)BINS) ++shift;
                s.part_counts[tid] = 0, s.part_sums[tid] = 0;
                __syncthreads();
                each(of_row, [&](double t, uint32_t key, int) {
                    if (key < lo || key > hi) return;
                    const uint32_t b = (hi - key) >> shift;
                    atomicAdd(&s.part_counts[b], 1u);
                    atomicAdd(&s.part_sums[b], r.weight(t));
                });
                __syncthreads();
                uint32_t count;
                const Share parts = share_out(s.part_sums[tid], s.part_counts[tid], s, &sum, &count);
                p = reaches(parts, by_count, need - (by_count ? (u64)above : before));
                inside = p.count;
                before += p.before;
                above += p.above;
                hi -= (uint32_t)p.index << shift;
                lo = max(lo, hi - ((1u << shift) - 1u));
            }
            if (inside <= LIST) {
                if (tid == 0) s.listed = 0;
                __syncthreads();
                if (of_row && top < INFINITY) {                // there is no NaN but below
                    const float low = key_value(lo), high = key_value(hi);
                    tokens.each([&](float v, int i) {
                        if (v >= low && v <= high) to_list(sample_key(v), i);
                    });
                } else
                    each(of_row, [&](double, uint32_t key, int i) {
                        if (key >= lo && key <= hi) to_list(key, i);
                    });
                __syncthreads();
                const int size = min((int)s.listed, LIST);
                if (size <= 128) {                             // a wave's work
                    if (tid < 64) {
                        const WaveList list = wave_list(s.list, s.list, size, r, t_least);
                        const u64 rest = need - (by_count ? (u64)above : before);
                        const int at = by_count ? (int)rest - 1 : list.reaches(rest);
                        const u64 upto = list.sum_at(at);
                        const int index = list.token_at(at);
                        if (tid == 0) s.place[turn] = SamplePlace{upto, 0, 0, 0, index};
                    }
                    __syncthreads();
                    kept = before + s.place[turn].before;
                    token = s.place[turn].index;
                    turn ^= 1;
                    continue;
                }
                const Share m = share_list(size, &sum);
                p = reaches(m, by_count, need - (by_count ? (u64)above : before));
                token = (int)(uint32_t)s.list[p.index];
                kept = before + p.before + p.own;
                __syncthreads();
                continue;
            }
            // equal values: the rank among them, and its index (or the last one's) where the token is asked for
            const u64 w = r.weight(r.t(key_value(lo)));
            const u64 rank = min(by_count ? need - above : (need - before + w - 1) / max(w, (u64)1), (u64)inside);
            kept = before + rank * w;
            if (step < 2) continue;
            // THREADS tokens at a time, in their order
            uint32_t seen = 0, latest = 0;
            if (tid == 0) s.word = 0;
            for (int from = 0; from < n; from += SAMPLE_THREADS) {
                const int i = from + tid;
                const bool same = i < n && sample_key(tokens.at(i)) == lo;
                const uint64_t mask = __builtin_amdgcn_ballot_w64(same);
                if ((tid & 63) == 0) s.wave_counts[tid >> 6] = (uint32_t)__popcll(mask);
                __syncthreads();
                uint32_t mine = seen + (uint32_t)__popcll(mask & ((1ull << (tid & 63)) - 1)), total = 0;
                for (int w2 = 0; w2 < SAMPLE_THREADS / 64; ++w2) {
                    if (w2 < (tid >> 6)) mine += s.wave_counts[w2];
                    total += s.wave_counts[w2];
                }
                if (same && mine < rank) latest = (uint32_t)i;
                __syncthreads();
                if (seen + total >= rank) break;
                seen += total;
            }
            if (latest) atomicMax(&s.word, latest);
            __syncthreads();
            token = (int)s.word;
        }
        if (tid == 0) a.out[row] = token;
    }
}

// Blocks per row: so many that they fill the chip once (a block's LDS leaves room for no other on its CU), each with
// SAMPLE_THREADS chunks of 16 bytes at least (16 bf16 rows of 51200 32.3 us; with half of that 34.4, twice 36.4; one fp32 row of
// 128000 51.5, 68.6, 48.0).
int sample_slices(int dtype, int rows, int n, int num_cus) {
    const int chunks = (n + (dtype == MVLM_F32 ? 3 : 7)) / (dtype == MVLM_F32 ? 4 : 8);
    return std::max(1, std::min(num_cus / rows, chunks / SAMPLE_THREADS));
}

// Bytes of the slices' parts; placing them.
size_t sample_workspace_bytes(const SampleArgs& a) {
    return a.slices == 1 ? 0 : (size_t)a.rows * a.slices * ((BINS + CANDIDATES) * sizeof(u64) + BINS * sizeof(uint32_t) + sizeof(float));
}
void sample_place(SampleArgs* a, void* workspace) {
    const size_t parts = (size_t)a->rows * a->slices;
    a->slice_sums = (unsigned long long*)workspace;
    a->part_entries = a->slice_sums + parts * BINS;
    a->slice_counts = (uint32_t*)(a->part_entries + parts * CANDIDATES);
    a->slice_tops = (float*)(a->slice_counts + parts * BINS);
}

hipError_t launch_sample(hipStream_t s, const SampleArgs& a) {
    const int es = a.dtype == MVLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)a.x & 15u) == 0 && (a.ld * es) % 16 == 0;
    const dim3 grid((unsigned)(a.rows * a.slices));
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto split = [&](auto sp) {
            constexpr bool SPLIT = decltype(sp)::value;
            if (vec) launch_kernel(sample_kernel<DT, true, SPLIT>, grid, dim3(SAMPLE_THREADS), 0, s, a);
            else launch_kernel(sample_kernel<DT, false, SPLIT>, grid, dim3(SAMPLE_THREADS), 0, s, a);
        };
        if (a.slices > 1) split(std::true_type{});
        else split(std::false_type{});
    };
    if (a.dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
