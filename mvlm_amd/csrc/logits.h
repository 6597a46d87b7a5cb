// Arguments of the logits operator (logits.hip).
#pragma once

#include "common.h"

namespace mvlm {

struct LogitsArgs {
    const void* x;
    void* out;
    int dtype, rows, n;
    int64_t ld;
    const int* history;            // [rows][history_width]
    const int* history_len;
    const int* generated_from;     // null: 0
    int history_width;
    const float* penalties;        // [rows][3] repetition, frequency, presence; null: none
    const int* bias_ids;           // [rows][bias_width]; null: none
    const float* bias_values;
    const int* bias_len;
    int bias_width;
    const uint32_t* allowed;       // [rows][(n + 31) / 32]; null: everything
    int slices;                    // blocks per row (set by the launcher)
};
hipError_t launch_logits(hipStream_t s, const LogitsArgs& a, int num_cus);

}  // namespace mvlm
