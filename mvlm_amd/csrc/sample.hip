// A token of each row of logits by temperature, min-p, top-k, top-p and a given uniform number (mvlm_sample).
//
// With m the row's largest value and t_i = (v_i - m) log2(e) / T <= 0 in 64 bits, a token's weight is
//   W_i = round(2^(bits + t_i)), an integer: 2^bits for the largest, 0 below 2^-(bits + 1) of it.
// Integers below 2^62 / n add up exactly in any order.  In the order of falling value (the lower index first among
// equals) everything asked for is a start of the row or a place in it:
//   live     t_i >= max(log2(min_p), -(bits + 1))
//   top-k    the place of the k-th live token
//   top-p    the first place at which the running sum of W reaches ceil(top_p x the sum so far kept)
//   picked   the first at which it reaches floor(u x the sum kept) + 1
// so one search serves all three.  Values are compared as integers that order like them (sample_key).
//
// One block per row.  It reads the row for m, then counts the live tokens by t in steps of 1/32 (at most 1664 of
// them), with their weights where more than LIST tokens may be kept.  If those that matter fit a list in LDS, a
// pass collects them, they are sorted, and running sums give all answers.  Otherwise each search goes on inside its
// step: by list if that fits, else by counting in ranges of keys, and among equal values by index.
#include "common.h"
#include "device_math.h"
#include "sample.h"

namespace mvlm {

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_BATCH = 4;        // 16-byte chunks in flight per thread
constexpr int BINS = 2048;
constexpr int LIST = 4096;             // entries of the list in LDS
constexpr int STEPS = 32;              // bins per factor of two of the weight; (51 + 1) 32 < BINS

typedef unsigned long long u64;

// An integer that orders like the value with these bits: NaN as the infinity of its sign, -0 as 0.
__device__ __forceinline__ uint32_t sample_key(float f) {
    uint32_t b = __float_as_uint(f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) b = (b & 0x80000000u) | 0x7F800000u;
    if (b == 0x80000000u) b = 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
constexpr uint32_t KEY_NEG_INF = 0x007FFFFFu, KEY_INF = 0xFF800000u;

// 2^x for x <= 0: 2^round(x) times the exponential series of (x - round(x)) ln 2, |..| <= 0.347, whose 14th term is
// below 2^-57 of the sum
__device__ __forceinline__ double exp2_series(double x) {
    const double n = __builtin_rint(x), f = (x - n) * 0.69314718055994530942;
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, f, 1.0 / 479001600.0);
    p = __builtin_fma(p, f, 1.0 / 39916800.0);
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// What a row's block knows of it.
struct SampleRow {
    uint32_t top;                      // key of the largest value
    double m, c;                       // that value, log2(e) / T
    int bits;
    // t of a key that is not above top
    __device__ __forceinline__ double t(uint32_t key) const { return key == top ? 0.0 : ((double)key_value(key) - m) * c; }
    __device__ __forceinline__ u64 weight(uint32_t key) const {
        const double w = exp2_series(t(key) + bits);               // at most 2^51
        return (u64)__double_as_longlong(w + 4503599627370496.0) - 0x4330000000000000ull;   // + 2^52: rounded to an integer
    }
    __device__ __forceinline__ int bin(uint32_t key) const { return min((int)(t(key) * -STEPS), BINS - 1); }
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

// f(key, index) for every token of a row
template <int DT, bool VEC, class F>
__device__ __forceinline__ void each_token(const void* x, int64_t row, int n, F&& f) {
    constexpr int EPC = DT == MVLM_F32 ? 4 : 8;
    const int tid = (int)threadIdx.x;
    int from = 0;
    if constexpr (VEC) {
        const int chunks = n / EPC;
        const u32x4* p = reinterpret_cast<const u32x4*>((const char*)x + row * (DT == MVLM_F32 ? 4 : 2));
        for (int base = tid; base < chunks; base += SAMPLE_THREADS * SAMPLE_BATCH) {
            u32x4 w[SAMPLE_BATCH];
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u) w[u] = p[min(base + u * SAMPLE_THREADS, chunks - 1)];
#pragma unroll
            for (int u = 0; u < SAMPLE_BATCH; ++u) {
                const int c = base + u * SAMPLE_THREADS;
                if (c >= chunks) break;
#pragma unroll
                for (int e = 0; e < EPC; ++e) {
                    float v;
                    if constexpr (DT == MVLM_F32) v = __uint_as_float(w[u][e]);
                    else {
                        const uint16_t h = (uint16_t)(w[u][e >> 1] >> (16 * (e & 1)));
                        v = DT == MVLM_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
                    }
                    f(sample_key(v), c * EPC + e);
                }
            }
        }
        from = chunks * EPC;
    }
    for (int i = from + tid; i < n; i += SAMPLE_THREADS) f(sample_key(load_as_f32(x, row + i, DT)), i);
}

struct SampleLds {
    u64 sums[BINS];                    // weights of the bins, then running sums
    uint32_t counts[BINS];             // tokens of the bins, then running counts
    union {
        struct {
            u64 list[LIST];            // ~key, index
            u64 weights[LIST];         // running sums of their weights
        };
        struct {
            u64 part_sums[BINS];       // of a range of keys
            uint32_t part_counts[BINS];
        };
    };
    u64 wave_sums[SAMPLE_THREADS / 64];
    uint32_t wave_counts[SAMPLE_THREADS / 64];
    uint32_t listed, word;
    u64 found[4];
};

// Running sums of sums[] and counts[], size of them a multiple of SAMPLE_THREADS or below it, by all threads.
template <bool COUNTS>
__device__ __forceinline__ void running(u64* sums, uint32_t* counts, int size, SampleLds& s) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = (size + SAMPLE_THREADS - 1) / SAMPLE_THREADS, from = min(tid * each, size), to = min(from + each, size);
    u64 w = 0;
    uint32_t c = 0;
    for (int i = from; i < to; ++i) {
        w += sums[i];
        if (COUNTS) c += counts[i];
    }
    u64 iw = w;
    uint32_t ic = c;
    for (int off = 1; off < 64; off <<= 1) {
        const u64 a = __shfl_up(iw, off, 64);
        const uint32_t b = __shfl_up(ic, off, 64);
        if (lane >= off) iw += a, ic += b;
    }
    if (lane == 63) s.wave_sums[wave] = iw, s.wave_counts[wave] = ic;
    __syncthreads();
    for (int i = 0; i < wave; ++i) iw += s.wave_sums[i], ic += s.wave_counts[i];
    iw -= w;
    ic -= c;
    for (int i = from; i < to; ++i) {
        iw += sums[i];
        sums[i] = iw;
        if (COUNTS) ic += counts[i], counts[i] = ic;
    }
    __syncthreads();
}

// list[0 .. size) in ascending order, by all threads; size <= LIST
__device__ __forceinline__ void sort_list(u64* list, int size) {
    int padded = 2;
    while (padded < size) padded *= 2;
    for (int i = size + (int)threadIdx.x; i < padded; i += SAMPLE_THREADS) list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= padded; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = (int)threadIdx.x; i < padded / 2; i += SAMPLE_THREADS) {
                const int lo = (i & ~(j - 1)) * 2 + (i & (j - 1)), hi = lo + j;
                const u64 a = list[lo], b = list[hi];
                if ((a > b) == ((lo & k) == 0)) list[lo] = b, list[hi] = a;
            }
            __syncthreads();
        }
}

// Where a search ends: the place's token and the sum of weights up to and with it.
struct SamplePlace {
    uint32_t key;
    int token;                         // -1: not looked for
    u64 sum;
};

template <int DT, bool VEC>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_kernel(const SampleArgs a) {
    __shared__ SampleLds s;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, n = a.n;
    const int64_t base = (int64_t)row * a.ld;

    // the largest value, and its first token
    uint32_t best = 0;
    int at = n;
    each_token<DT, VEC>(a.x, base, n, [&](uint32_t key, int i) {
        if (key > best) best = key, at = i;
    });
    for (int off = 32; off; off >>= 1) {
        const uint32_t k = (uint32_t)__shfl_xor((int)best, off, 64);
        const int i = __shfl_xor(at, off, 64);
        if (k > best || (k == best && i < at)) best = k, at = i;
    }
    if ((tid & 63) == 0) s.wave_sums[tid >> 6] = (u64)best << 32 | (uint32_t)~at;
    __syncthreads();
    u64 first = 0;
    for (int w = 0; w < SAMPLE_THREADS / 64; ++w) first = max(first, s.wave_sums[w]);
    __syncthreads();
    if (tid == 0) s.word = 0;
    SampleRow r;
    r.top = (uint32_t)(first >> 32);
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    if (r.top == KEY_NEG_INF || !(T > 0.0f)) {
        if (tid == 0) a.out[row] = r.top == KEY_NEG_INF ? 0 : ~(int)(uint32_t)first;
        return;
    }
    r.m = (double)key_value(r.top);
    r.c = 1.4426950408889634074 / (double)T;
    r.bits = a.bits;
    float min_p = a.min_p ? a.min_p[row] : 0.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, u = a.uniform[row];
    const int top_k = a.top_k ? a.top_k[row] : 0;
    if (!(u > 0.0f)) u = 0.0f;

    // the least key with t >= t_least; t does not fall as keys rise
    auto least_key = [&](double t_least) {
        uint32_t lo = KEY_NEG_INF + 1, hi = r.top;             // hi has it
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (r.t(mid) >= t_least) hi = mid;
            else lo = mid + 1;
        }
        return hi;
    };
    double t_least = -(double)(a.bits + 1);
    if (min_p > 0.0f) t_least = fmax(t_least, log2((double)fminf(min_p, 1.0f)));
    const uint32_t live = r.top == KEY_INF ? KEY_INF : least_key(t_least);

    // tokens by t; their weights too unless few may be kept
    const bool few = top_k > 0 || min_p > 0.0f;
    auto count_bins = [&](bool weights) __attribute__((always_inline)) {
        for (int i = tid; i < BINS; i += SAMPLE_THREADS) s.counts[i] = 0, s.sums[i] = 0;
        __syncthreads();
        each_token<DT, VEC>(a.x, base, n, [&](uint32_t key, int) {
            if (key < live) return;
            const int b = r.bin(key);
            atomicAdd(&s.counts[b], 1u);
            if (weights) atomicAdd(&s.sums[b], r.weight(key));
        });
        __syncthreads();
        running<true>(s.sums, s.counts, BINS, s);
    };
    count_bins(!few);
    const uint32_t all = s.counts[BINS - 1];
    const uint32_t k = top_k > 0 && (uint32_t)top_k < all ? (uint32_t)top_k : all;   // tokens kept by count

    // tokens with keys in [lo, hi] into the list, sorted, with running sums of their weights
    auto make_list = [&](uint32_t lo, uint32_t hi) __attribute__((always_inline)) {
        if (tid == 0) s.listed = 0;
        __syncthreads();
        each_token<DT, VEC>(a.x, base, n, [&](uint32_t key, int i) {
            if (key < lo || key > hi) return;
            const uint32_t to = atomicAdd(&s.listed, 1u);
            if (to < LIST) s.list[to] = (u64)~key << 32 | (uint32_t)i;
        });
        __syncthreads();
        const int size = min((int)s.listed, LIST);
        sort_list(s.list, size);
        for (int i = tid; i < size; i += SAMPLE_THREADS) s.weights[i] = r.weight(~(uint32_t)(s.list[i] >> 32));
        __syncthreads();
        running<false>(s.weights, nullptr, size, s);
        return size;
    };
    // the first entry of the list with entry + 1 >= need (by count) or running sum >= need
    auto in_list = [&](int size, bool by_count, u64 need) {
        if (by_count) return (int)need - 1;
        for (int i = tid; i < size; i += SAMPLE_THREADS)
            if (s.weights[i] >= need && (i == 0 || s.weights[i - 1] < need)) s.word = (uint32_t)i;
        __syncthreads();
        const int i = max(min((int)s.word, size - 1), 0);
        __syncthreads();
        return i;
    };
    // the bin (of running sums and counts) in which the place lies
    auto in_bins = [&](const u64* sums, const uint32_t* counts, bool by_count, u64 need) {
        for (int i = tid; i < BINS; i += SAMPLE_THREADS) {
            const u64 end = by_count ? counts[i] : sums[i], begin = i == 0 ? 0 : by_count ? counts[i - 1] : sums[i - 1];
            if (end >= need && begin < need) s.word = (uint32_t)i;
        }
        __syncthreads();
        const int i = min((int)s.word, BINS - 1);
        __syncthreads();
        return i;
    };
    // the keys of a bin of t
    auto keys_of = [&](int bin, uint32_t* lo, uint32_t* hi) {
        uint32_t l = live, h = r.top;                          // the least key with a bin <= this one
        while (l < h) {
            const uint32_t mid = l + (h - l) / 2;
            if (r.bin(mid) <= bin) h = mid;
            else l = mid + 1;
        }
        *lo = h;
        l = h, h = r.top;                                      // the largest with a bin >= this one
        while (l < h) {
            const uint32_t mid = l + (h - l + 1) / 2;
            if (r.bin(mid) >= bin) l = mid;
            else h = mid - 1;
        }
        *hi = l;
    };

    if (few) {
        // all that the count lets through, if the list has room for it
        const int last = in_bins(s.sums, s.counts, true, k);
        if (s.counts[last] <= LIST) {
            uint32_t lo, hi;
            keys_of(last, &lo, &hi);
            const int size = make_list(lo, r.top);
            u64 kept = s.weights[k - 1];
            if (top_p < 1.0f) kept = s.weights[in_list(size, false, top_p > 0.0f ? max(part_of<true>(top_p, kept), (u64)1) : 1)];
            const u64 need = u < 1.0f ? part_of<false>(u, kept) + 1 : kept;
            const int i = in_list(size, false, need);
            if (tid == 0) a.out[row] = (int)(uint32_t)s.list[i];
            return;
        }
        count_bins(true);
    }

    // the place that a search ends in; `token`: whether its index is asked for
    auto search = [&](bool by_count, u64 need, bool token) __attribute__((always_inline)) {
        SamplePlace place{0, -1, 0};
        int bin = in_bins(s.sums, s.counts, by_count, need);
        u64 before = bin ? s.sums[bin - 1] : 0;                // of the tokens above the range
        uint32_t above = bin ? s.counts[bin - 1] : 0, inside = s.counts[bin] - above;
        uint32_t lo, hi;
        keys_of(bin, &lo, &hi);
        while (inside > LIST && lo < hi) {
            const uint32_t span = hi - lo;                     // keys less one
            int shift = 0;
            while ((span >> shift) >= (uint32_t)BINS) ++shift;
            for (int i = tid; i < BINS; i += SAMPLE_THREADS) s.part_counts[i] = 0, s.part_sums[i] = 0;
            __syncthreads();
            each_token<DT, VEC>(a.x, base, n, [&](uint32_t key, int) {
                if (key < lo || key > hi) return;
                const uint32_t b = (hi - key) >> shift;
                atomicAdd(&s.part_counts[b], 1u);
                atomicAdd(&s.part_sums[b], r.weight(key));
            });
            __syncthreads();
            running<true>(s.part_sums, s.part_counts, BINS, s);
            bin = in_bins(s.part_sums, s.part_counts, by_count, need - (by_count ? (u64)above : before));
            const u64 less = bin ? s.part_sums[bin - 1] : 0;
            const uint32_t fewer = bin ? s.part_counts[bin - 1] : 0;
            inside = s.part_counts[bin] - fewer;
            before += less;
            above += fewer;
            hi -= (uint32_t)bin << shift;
            lo = max(lo, hi - ((1u << shift) - 1u));
            __syncthreads();
        }
        if (inside <= LIST) {
            const int size = make_list(lo, hi);
            const int i = in_list(size, by_count, need - (by_count ? (u64)above : before));
            place.key = ~(uint32_t)(s.list[i] >> 32);
            place.token = (int)(uint32_t)s.list[i];
            place.sum = before + s.weights[i];
            __syncthreads();
            return place;
        }
        // equal values: the rank among them, and its index where asked for
        const u64 w = r.weight(lo);
        const u64 rank = by_count ? need - above : (need - before + w - 1) / w;
        place.key = lo;
        place.sum = before + rank * w;
        if (!token) return place;
        // THREADS tokens at a time, in their order
        uint32_t seen = 0;
        for (int from = 0; from < n; from += SAMPLE_THREADS) {
            const int i = from + tid;
            const bool same = i < n && sample_key(load_as_f32(a.x, base + i, DT)) == lo;
            const uint64_t mask = __builtin_amdgcn_ballot_w64(same);
            if ((tid & 63) == 0) s.wave_counts[tid >> 6] = (uint32_t)__popcll(mask);
            __syncthreads();
            uint32_t mine = seen + (uint32_t)__popcll(mask & ((1ull << (tid & 63)) - 1)), total = 0;
            for (int w2 = 0; w2 < SAMPLE_THREADS / 64; ++w2) {
                if (w2 < (tid >> 6)) mine += s.wave_counts[w2];
                total += s.wave_counts[w2];
            }
            if (same && mine + 1 == rank) s.word = (uint32_t)i;
            __syncthreads();
            if (seen + total >= rank) break;
            seen += total;
        }
        place.token = (int)s.word;
        return place;
    };
    u64 kept = s.sums[BINS - 1];
    SamplePlace place{0, 0, 0};
    for (int step = 0; step < 3; ++step) {                     // top-k, top-p, the token
        if ((step == 0 && k == all) || (step == 1 && !(top_p < 1.0f))) continue;
        u64 need = k;
        if (step == 1) need = top_p > 0.0f ? max(part_of<true>(top_p, kept), (u64)1) : 1;
        if (step == 2) need = u < 1.0f ? part_of<false>(u, kept) + 1 : kept;
        place = search(step == 0, need, step == 2);
        kept = place.sum;
    }
    if (tid == 0) a.out[row] = place.token;
}

hipError_t launch_sample(hipStream_t s, const SampleArgs& a, int) {
    const int es = a.dtype == MVLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)a.x & 15u) == 0 && (a.ld * es) % 16 == 0;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (vec) launch_kernel(sample_kernel<DT, true>, dim3((unsigned)a.rows), dim3(SAMPLE_THREADS), 0, s, a);
        else launch_kernel(sample_kernel<DT, false>, dim3((unsigned)a.rows), dim3(SAMPLE_THREADS), 0, s, a);
    };
    if (a.dtype == MVLM_F32) go(std::integral_constant<int, MVLM_F32>{});
    else if (a.dtype == MVLM_F16) go(std::integral_constant<int, MVLM_F16>{});
    else go(std::integral_constant<int, MVLM_BF16>{});
    return hipGetLastError();
}

}  // namespace mvlm
