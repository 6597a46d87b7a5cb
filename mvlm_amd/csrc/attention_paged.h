// What the kernels of the attention over a paged cache share (attention_paged.hip for
// few new rows, attention_paged_chunk.hip for many).
#pragma once

#include "common.h"
#include "device_math.h"
#include "paged_ops.h"

namespace mvlm {

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

// (lo, hi) rounded to nearest even, packed; with REST, lo and hi become what was lost
template <bool BF, bool REST>
__device__ __forceinline__ uint32_t round2(float& lo, float& hi) {
    if constexpr (BF) {
        const bf16x2v h = __builtin_convertvector(f32x2{lo, hi}, bf16x2v);
        if constexpr (REST) lo -= (float)h[0], hi -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    } else {
        const f16x2v h = __builtin_convertvector(f32x2{lo, hi}, f16x2v);
        if constexpr (REST) lo -= (float)h[0], hi -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    }
}

// Workspace: per record (tile of one split and kv head) its R rows of D floats of
// unnormalized output, then, behind all records, R (max, sum) pairs each.
template <int R>
__device__ __forceinline__ float* paged_ws_out(const PagedAttnArgs& a, int record, int h) {
    return a.ws + ((int64_t)record * a.kv.kv_heads + h) * R * a.kv.D;
}
template <int R, bool MANY>
__device__ __forceinline__ f32x2* paged_ws_ml(const PagedAttnArgs& a, int record, int h) {
    const int64_t records = (int64_t)(MANY ? a.many.records : a.few.records) * a.kv.kv_heads;
    return reinterpret_cast<f32x2*>(a.ws + records * R * a.kv.D) + ((int64_t)record * a.kv.kv_heads + h) * R;
}

// four outputs of row f of a tile's sequence, from dim d on
template <bool BF>
__device__ __forceinline__ void paged_store4(const PagedAttnArgs& a, const PagedSpan& sp, int h, int f, int d, f32x4 v) {
    const int j = f / a.group, g = f - j * a.group;
    const int64_t at = ((int64_t)(sp.row0 + j) * a.heads + h * a.group + g) * a.kv.D + d;
    if (a.o_dtype == MVLM_F32)
        *reinterpret_cast<f32x4*>((float*)a.o + at) = v;
    else {
        float e[4] = {v[0], v[1], v[2], v[3]};
        *reinterpret_cast<u32x2*>((uint16_t*)a.o + at) = u32x2{round2<BF, false>(e[0], e[1]), round2<BF, false>(e[2], e[3])};
    }
}

// Merges the splits of a tile of R rows, in their order.
template <bool BF, int R, bool MANY>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedAttnArgs a) {
    const int D = a.kv.D, index = (int)(blockIdx.x / (uint32_t)a.kv.kv_heads);
    const int h = (int)blockIdx.x - index * a.kv.kv_heads;
    PagedItem it;
    if (!paged_find<R, MANY, true>(a, index, &it) || it.record < 0) return;
    const PagedSpan sp = it.span;
    const int rows_f = sp.n * a.group, rows = min(R, rows_f - it.tile * R);
    const int splits = max(1, (sp.visible((it.tile * R + rows - 1) / a.group) + it.unit - 1) / it.unit);   // those that saw keys
    const int d4 = D / 4;
    for (int i = (int)threadIdx.x; i < rows * d4; i += 256) {
        const int r = i / d4, d = 4 * (i - r * d4);
        float mx = -INFINITY, sum = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int BATCH = 8;
        for (int s0 = 0; s0 < splits; s0 += BATCH) {
            f32x2 ml[BATCH];
            f32x4 ov[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int rec = it.record + min(s0 + u, splits - 1);
                ml[u] = paged_ws_ml<R, MANY>(a, rec, h)[r];
                ov[u] = *reinterpret_cast<const f32x4*>(paged_ws_out<R>(a, rec, h) + (int64_t)r * D + d);
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                if (s0 + u >= splits || (ml[u][0] == -INFINITY && ml[u][1] == 0.0f)) continue;   // past the end, or saw no key
                const float mn = fmaxf(mx, ml[u][0]);
                const float f0 = __builtin_amdgcn_exp2f(mx - mn), f1 = __builtin_amdgcn_exp2f(ml[u][0] - mn);
                sum = sum * f0 + ml[u][1] * f1;
                o = o * f0 + ov[u] * f1;
                mx = mn;
            }
        }
        paged_store4<BF>(a, sp, h, it.tile * R + r, d, sum == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * (1.0f / sum));
    }
}

// The kernels of one call, each share's attention and the combine of its splits.
struct PagedLaunch {
    hipStream_t s;
    const PagedAttnArgs& a;
    int left;
    bool first = true;
    template <class K>
    void operator()(K kernel, int per_head) {
        const LaunchPart part = first ? LaunchPart::First : left == 1 ? LaunchPart::Last : LaunchPart::Middle;
        --left;
        first = false;
        launch_kernel_part(part, kernel, dim3((unsigned)(a.kv.kv_heads * per_head)), dim3(256), 0, s, a);
    }
};
void launch_attention_paged_chunk(PagedLaunch& go);

}  // namespace mvlm
