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
};
hipError_t launch_sample(hipStream_t s, const SampleArgs& a, int num_cus);

}  // namespace mvlm
