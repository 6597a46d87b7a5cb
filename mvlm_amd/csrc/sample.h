// Arguments of the token draw (sample.hip).
#pragma once

#include "common.h"

namespace mvlm {

constexpr int SAMPLE_MAX_TOKENS = 1 << 24;     // of a row

struct SampleArgs {
    const void* x;
    int dtype, rows, n;
    int64_t ld;
    const float* uniform;          // [rows] each; all but the first may be null
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* out;
    int bits;                      // weights are multiples of 2^-bits
    int slices;                    // blocks per row
    // where slices > 1: what the slices found, and the row's finished slices, zero between launches
    unsigned long long* slice_sums;
    unsigned long long* part_entries;
    uint32_t* slice_counts;
    float* slice_tops;
    uint32_t* arrived;
};
int sample_slices(int dtype, int rows, int n, int num_cus);
size_t sample_workspace_bytes(const SampleArgs& a);
void sample_place(SampleArgs* a, void* workspace);
hipError_t launch_sample(hipStream_t s, const SampleArgs& a);

}  // namespace mvlm
