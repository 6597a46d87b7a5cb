// Limits of the operators over a paged cache beyond which their kernels' arithmetic would not hold, checked
// without a GPU (run by tests/test_paged_limits.py).  Handles are made by hand: a refused call reads only sizes and
// addresses and reaches no device.
#include "common.h"

#include <cfloat>
#include <climits>
#include <cstdio>
#include <cstdlib>

using namespace mvlm;

static int failures = 0;
static mvlm_device dev;

static mvlm_buffer buffer(size_t bytes, uintptr_t address) {
    mvlm_buffer b;
    b.dev = &dev;
    b.ptr = (void*)address;
    b.bytes = bytes;
    return b;
}
static void refused(const char* what, int status) {
    if (status == MVLM_ERR_INVALID_ARG) return;
    ++failures;
    std::printf("%s: status %d (%s)\n", what, status, mvlm_last_error());
}

// A list's entries are walked in steps of up to 4096, which the index of the last step has to have room for.
static void logits_lists(const char* kind) {
    mvlm_buffer x = buffer(4000, 0x1000), out = buffer(4000, 0x2000), hist = buffer((size_t)1 << 34, (uintptr_t)1 << 40),
                len = buffer(16, 0x3000), pen = buffer(48, 0x4000), ids = buffer((size_t)1 << 34, (uintptr_t)2 << 40),
                values = buffer((size_t)1 << 34, (uintptr_t)3 << 40), count = buffer(16, 0x5000);
    for (int width : {(1 << 30) + 1, INT_MAX - 4096, INT_MAX}) {
        mvlm_logit_controls h{}, b{};
        h.history = &hist, h.history_len = &len, h.penalties = &pen, h.history_width = width;
        b.bias_ids = &ids, b.bias_values = &values, b.bias_len = &count, b.bias_width = width;
        for (const mvlm_logit_controls& c : {h, b})
            refused(kind, mvlm_logits_process(&dev, &x, MVLM_F32, 1, 1000, 1000, &c, &out, nullptr));
    }
}

// Scores are scaled by scale log2(e) in fp32; were that infinite, a score of 0 would become NaN.
static void attention_scales() {
    mvlm_buffer k = buffer(1 << 20, 0x10000000), v = buffer(1 << 20, 0x20000000), len = buffer(16, 0x30000000),
                table = buffer(64, 0x40000000), q = buffer(1 << 20, 0x50000000), o = buffer(1 << 20, 0x60000000);
    const mvlm_paged_kv kv{&k, &v, MVLM_F16, 16, 16, 4, 64};
    const mvlm_paged_batch batch{4, 4, nullptr, &len, &table, 4};
    for (float scale : {FLT_MAX, FLT_MAX / 1.4426f})
        refused("a scale that log2(e) makes infinite", mvlm_attention_paged(&dev, &q, &batch, &kv, &o, MVLM_F32, 4, scale, nullptr));
}

int main() {
    setenv("MVLM_QUIET", "1", 1);
    logits_lists("a list of more than 2^30 entries");
    attention_scales();
    std::printf("%d failures\n", failures);
    return failures != 0;
}
