// Host checks of the operators over a paged cache, without a GPU (run by
// tests/test_paged_host.py): the index arithmetic of paged.h over hostile
// values, and every refusal of the entry points.  Handles are made by hand: a
// refused call reads only sizes and addresses and reaches no device.
#include "common.h"
#include "paged.h"

#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>

using namespace mvlm;

static int failures = 0;
#define CHECK(cond, ...)                                   \
    do {                                                   \
        if (!(cond)) {                                     \
            ++failures;                                    \
            std::printf("FAILED %s:%d: ", __FILE__, __LINE__); \
            std::printf(__VA_ARGS__);                      \
            std::printf("\n");                             \
        }                                                  \
    } while (0)

static void test_division() {
    std::mt19937_64 rng(1);
    for (int i = 0; i < 200000; ++i) {
        const int d = i < 3000 ? i + 1 : 1 + (int)(rng() % ((uint64_t)1 << (1 + rng() % 30)));
        const FastDiv f = fast_div(d);
        const int64_t near = (int64_t)(rng() % ((uint64_t)INT_MAX / d + 1)) * d;   // multiples and their neighbours
        for (int64_t n : {(int64_t)0, (int64_t)INT_MAX, near - 1, near, near + 1, near + d - 1, (int64_t)(rng() >> 33)})
            if (n >= 0 && n <= INT_MAX) CHECK(f.quotient((int)n) == (int)n / d, "%lld / %d", (long long)n, d);
    }
}

static void test_spans() {
    const int bad[] = {INT_MIN, INT_MIN + 1, -1, 0, 1, 2, 7, 8, 9, 1 << 30, INT_MAX - 1, INT_MAX};
    for (int rows : {1, 8, 1 << 22})
        for (int positions : {1, 8, 1 << 30})
            for (int start : bad)
                for (int stop : bad)
                    for (int held : bad) {
                        const PagedSpan p = paged_span(start, stop, held, rows, positions);
                        CHECK(p.row0 >= 0 && p.n >= 0 && p.row0 + p.n <= rows, "rows of %d %d", start, stop);
                        CHECK(p.len >= 0 && p.len <= positions && p.len <= p.held, "len of %d", held);
                        for (int j : {0, p.n / 2, p.n - 1})
                            if (j >= 0 && j < p.n) {
                                CHECK(p.visible(j) >= 0 && p.visible(j) <= p.len, "visible");
                                CHECK(p.position(j) < p.held, "position");
                            }
                    }
    const PagedSpan p = paged_span(2, 5, 10, 100, 9);
    CHECK(p.row0 == 2 && p.n == 3 && p.position(0) == 7 && p.visible(0) == 8 && p.visible(1) == 9 && p.visible(2) == 9, "plain");
}

static mvlm_device dev, other;
static mvlm_buffer buffer(size_t bytes, uintptr_t address, mvlm_device* d = &dev) {
    mvlm_buffer b;
    b.dev = d;
    b.ptr = (void*)address;
    b.bytes = bytes;
    return b;
}

// the arguments of a call that would be taken; each refusal changes one thing
struct Append {
    mvlm_buffer k = buffer(1 << 20, 0x10000000), v = buffer(1 << 20, 0x20000000), len = buffer(16, 0x30000000),
                table = buffer(64, 0x40000000), start = buffer(20, 0x50000000), x = buffer(1 << 20, 0x60000000),
                q = buffer(1 << 20, 0x70000000), cs = buffer(1 << 20, 0x80000000), o = buffer(1 << 20, 0x90000000);
    mvlm_paged_kv kv{&k, &v, MVLM_F16, 16, 16, 4, 64};
    mvlm_paged_batch batch{4, 8, &start, &len, &table, 4};
    mvlm_rope rope{&cs, 64, 64, 0};
    int x_dtype = MVLM_F32, heads = 8, o_dtype = MVLM_F16;
    int64_t ld = 16 * 64;
    float scale = 0.0f;
    int append() { return mvlm_kv_append_paged(&dev, &x, x_dtype, ld, &batch, &kv, heads, &q, &rope, nullptr); }
    int attend() { return mvlm_attention_paged(&dev, &q, &batch, &kv, &o, o_dtype, heads, scale, nullptr); }
};
template <class F>
static void refuses(int code, const char* what, F change, bool append = true, bool attend = true) {
    if (append) {
        Append a;
        change(a);
        const int got = a.append();
        CHECK(got == code, "append, %s: %d (%s)", what, got, mvlm_last_error());
    }
    if (attend) {
        Append a;
        change(a);
        const int got = a.attend();
        CHECK(got == code, "attention, %s: %d (%s)", what, got, mvlm_last_error());
    }
}

static void test_paged_refusals() {
    const int BAD = MVLM_ERR_INVALID_ARG, SMALL = MVLM_ERR_BUFFER_TOO_SMALL, NOT = MVLM_ERR_UNSUPPORTED;
    refuses(BAD, "null k", [](Append& a) { a.kv.k = nullptr; });
    refuses(BAD, "null v", [](Append& a) { a.kv.v = nullptr; });
    refuses(BAD, "null kv_len", [](Append& a) { a.batch.kv_len = nullptr; });
    refuses(BAD, "null table", [](Append& a) { a.batch.page_table = nullptr; });
    refuses(BAD, "fp32 cache", [](Append& a) { a.kv.dtype = MVLM_F32; });
    refuses(BAD, "no pages", [](Append& a) { a.kv.num_pages = 0; });
    refuses(BAD, "page size 0", [](Append& a) { a.kv.page_size = 0; });
    refuses(BAD, "negative heads", [](Append& a) { a.kv.kv_heads = -1; });
    refuses(BAD, "no dims", [](Append& a) { a.kv.head_dim = 0; });
    refuses(NOT, "head_dim 60", [](Append& a) { a.kv.head_dim = 60; });
    refuses(NOT, "head_dim 136", [](Append& a) { a.kv.head_dim = 136; });
    refuses(NOT, "2^31 slots", [](Append& a) { a.kv.num_pages = 1 << 25; });
    refuses(NOT, "64 GiB of keys", [](Append& a) { a.kv.num_pages = 1 << 22, a.kv.head_dim = 128, a.k.bytes = a.v.bytes = SIZE_MAX; });
    refuses(NOT, "1025 kv heads", [](Append& a) { a.kv.kv_heads = 1025; });
    refuses(SMALL, "cache too small", [](Append& a) { a.k.bytes = 16 * 16 * 4 * 64 * 2 - 1; });
    refuses(SMALL, "v too small", [](Append& a) { a.v.bytes = 16 * 16 * 4 * 64 * 2 - 1; });
    refuses(BAD, "misaligned cache", [](Append& a) { a.k = buffer(1 << 20, 0x10000008); });
    refuses(BAD, "k is v", [](Append& a) { a.v = a.k; });
    refuses(BAD, "another device's cache", [](Append& a) { a.v.dev = &other; });
    refuses(BAD, "another device's table", [](Append& a) { a.table.dev = &other; });
    refuses(BAD, "no sequences", [](Append& a) { a.batch.num_seqs = 0; });
    refuses(BAD, "no rows", [](Append& a) { a.batch.rows = 0; });
    refuses(BAD, "no table", [](Append& a) { a.batch.table_width = 0; });
    refuses(BAD, "rows without row_start", [](Append& a) { a.batch.row_start = nullptr; });
    refuses(BAD, "too many sequences", [](Append& a) { a.batch.num_seqs = 65537; });
    refuses(BAD, "too many rows", [](Append& a) { a.batch.rows = (1 << 22) + 1; });
    refuses(BAD, "too many positions", [](Append& a) { a.batch.table_width = (1 << 26) + 1; });
    refuses(SMALL, "short kv_len", [](Append& a) { a.len.bytes = 15; });
    refuses(SMALL, "short table", [](Append& a) { a.table.bytes = 63; });
    refuses(SMALL, "short row_start", [](Append& a) { a.start.bytes = 19; });
    refuses(BAD, "misaligned kv_len", [](Append& a) { a.len = buffer(16, 0x30000002); });
    refuses(BAD, "heads off the group", [](Append& a) { a.heads = 6; });
    refuses(BAD, "no heads", [](Append& a) { a.heads = 0; });
    refuses(SMALL, "short q", [](Append& a) { a.q.bytes = 8 * 8 * 64 * 2 - 1; });
    refuses(BAD, "misaligned q", [](Append& a) { a.q = buffer(1 << 20, 0x70000002); });
    refuses(BAD, "another device's q", [](Append& a) { a.q.dev = &other; });

    refuses(BAD, "qkv of int8", [](Append& a) { a.x_dtype = MVLM_Q8_0; }, true, false);
    refuses(BAD, "short ld", [](Append& a) { a.ld = 16 * 64 - 1; }, true, false);
    refuses(BAD, "huge ld", [](Append& a) { a.ld = INT64_MAX; }, true, false);
    refuses(SMALL, "short qkv", [](Append& a) { a.x.bytes = 8 * 1024 * 4 - 1; }, true, false);
    refuses(BAD, "misaligned qkv", [](Append& a) { a.x = buffer(1 << 20, 0x60000002); }, true, false);
    refuses(BAD, "odd rot_dim", [](Append& a) { a.rope.rot_dim = 7; }, true, false);
    refuses(BAD, "rot_dim over head_dim", [](Append& a) { a.rope.rot_dim = 66; }, true, false);
    refuses(BAD, "rot_dim 0", [](Append& a) { a.rope.rot_dim = 0; }, true, false);
    refuses(BAD, "no rope positions", [](Append& a) { a.rope.positions = 0; }, true, false);
    refuses(BAD, "null rope table", [](Append& a) { a.rope.table = nullptr; }, true, false);
    refuses(SMALL, "short rope table", [](Append& a) { a.cs.bytes = 64 * 64 * 4 - 1; }, true, false);
    refuses(BAD, "q_out in qkv", [](Append& a) { a.q = a.x; }, true, false);
    refuses(BAD, "q_out in the cache", [](Append& a) { a.q = a.k; }, true, false);
    refuses(BAD, "cache over the table", [](Append& a) { a.table = buffer(64, 0x10000100); }, true, false);
    refuses(BAD, "cache over the rope table", [](Append& a) { a.cs = buffer(1 << 20, 0x20000000); }, true, false);

    refuses(BAD, "bf16 output of an fp16 cache", [](Append& a) { a.o_dtype = MVLM_BF16; }, false);
    refuses(BAD, "negative scale", [](Append& a) { a.scale = -1.0f; }, false);
    refuses(BAD, "infinite scale", [](Append& a) { a.scale = INFINITY; }, false);
    refuses(BAD, "NaN scale", [](Append& a) { a.scale = NAN; }, false);
    refuses(SMALL, "short O", [](Append& a) { a.o.bytes = 8 * 8 * 64 * 2 - 1; }, false);
    refuses(BAD, "misaligned O", [](Append& a) { a.o = buffer(1 << 20, 0x90000008); }, false);
    refuses(BAD, "O is Q", [](Append& a) { a.o = a.q; }, false);
    refuses(BAD, "O in the cache", [](Append& a) { a.o = a.v; }, false);
    refuses(BAD, "more blocks than a launch takes", [](Append& a) {
        a.batch = mvlm_paged_batch{65536, 65536, nullptr, &a.len, &a.table, 1};
        a.kv.kv_heads = a.heads = 128;
        for (mvlm_buffer* b : {&a.k, &a.v, &a.len, &a.table, &a.q, &a.o}) b->ptr = (void*)((uintptr_t)b->ptr << 8), b->bytes = (size_t)1 << 33;
    }, false);
    refuses(BAD, "O over kv_len", [](Append& a) { a.len = buffer(16, 0x90000000); }, false);
    Append a;
    CHECK(mvlm_kv_append_paged(nullptr, &a.x, 0, a.ld, &a.batch, &a.kv, 8, &a.q, nullptr, nullptr) == BAD, "null device");
    CHECK(mvlm_kv_append_paged(&dev, nullptr, 0, a.ld, &a.batch, &a.kv, 8, &a.q, nullptr, nullptr) == BAD, "null qkv");
    CHECK(mvlm_kv_append_paged(&dev, &a.x, 0, a.ld, nullptr, &a.kv, 8, &a.q, nullptr, nullptr) == BAD, "null batch");
    CHECK(mvlm_kv_append_paged(&dev, &a.x, 0, a.ld, &a.batch, nullptr, 8, &a.q, nullptr, nullptr) == BAD, "null cache");
    CHECK(mvlm_attention_paged(&dev, nullptr, &a.batch, &a.kv, &a.o, 0, 8, 0.0f, nullptr) == BAD, "null Q");
    CHECK(mvlm_attention_paged(&dev, &a.q, &a.batch, &a.kv, nullptr, 0, 8, 0.0f, nullptr) == BAD, "null O");
    CHECK(mvlm_plan_add_kv_append_paged(nullptr, &a.x, 0, a.ld, &a.batch, &a.kv, 8, &a.q, nullptr) == BAD, "null plan");
    CHECK(mvlm_plan_add_attention_paged(nullptr, &a.q, &a.batch, &a.kv, &a.o, 0, 8, 0.0f) == BAD, "null plan");
}

struct Logits {
    mvlm_buffer x = buffer(4 * 1000 * 4, 0x10000000), out = buffer(4 * 1000 * 4, 0x20000000),
                hist = buffer(4 * 50 * 4, 0x30000000), len = buffer(16, 0x40000000), from = buffer(16, 0x50000000),
                pen = buffer(48, 0x60000000), ids = buffer(4 * 5 * 4, 0x70000000), val = buffer(4 * 5 * 4, 0x80000000),
                cnt = buffer(16, 0x90000000), mask = buffer(4 * 32 * 4, 0xA0000000);
    mvlm_logit_controls c{&hist, &len, &from, 50, &pen, &ids, &val, &cnt, 5, &mask};
    int dtype = MVLM_F32, rows = 4, n = 1000;
    int64_t ld = 1000;
    int call() { return mvlm_logits_process(&dev, &x, dtype, rows, n, ld, &c, &out, nullptr); }
};
template <class F>
static void refuses_logits(int code, const char* what, F change) {
    Logits a;
    change(a);
    const int got = a.call();
    CHECK(got == code, "logits, %s: %d (%s)", what, got, mvlm_last_error());
}

static void test_logits_refusals() {
    const int BAD = MVLM_ERR_INVALID_ARG, SMALL = MVLM_ERR_BUFFER_TOO_SMALL;
    refuses_logits(BAD, "dtype", [](Logits& a) { a.dtype = MVLM_Q4_0; });
    refuses_logits(BAD, "no rows", [](Logits& a) { a.rows = 0; });
    refuses_logits(BAD, "no tokens", [](Logits& a) { a.n = 0; });
    refuses_logits(BAD, "short ld", [](Logits& a) { a.ld = 999; });
    refuses_logits(BAD, "too many rows", [](Logits& a) { a.rows = (1 << 20) + 1; });
    refuses_logits(BAD, "more blocks than a launch takes", [](Logits& a) { a.rows = 1 << 20, a.n = 7 * 4096 + 1, a.ld = a.n; });
    refuses_logits(BAD, "huge ld", [](Logits& a) { a.ld = INT64_MAX; });
    refuses_logits(SMALL, "short x", [](Logits& a) { a.x.bytes -= 1; });
    refuses_logits(SMALL, "short out", [](Logits& a) { a.out.bytes -= 1; });
    refuses_logits(BAD, "misaligned x", [](Logits& a) { a.x = buffer(1 << 20, 0x10000002); });
    refuses_logits(BAD, "out across x", [](Logits& a) { a.out = buffer(1 << 20, 0x10000010); });
    refuses_logits(BAD, "another device's out", [](Logits& a) { a.out.dev = &other; });
    refuses_logits(BAD, "history without penalties", [](Logits& a) { a.c.penalties = nullptr; });
    refuses_logits(BAD, "penalties without history", [](Logits& a) { a.c.history = nullptr; });
    refuses_logits(BAD, "no history_len", [](Logits& a) { a.c.history_len = nullptr; });
    refuses_logits(BAD, "generated_from alone", [](Logits& a) { a.c.history = a.c.history_len = a.c.penalties = nullptr; });
    refuses_logits(BAD, "history width 0", [](Logits& a) { a.c.history_width = 0; });
    refuses_logits(SMALL, "short history", [](Logits& a) { a.hist.bytes -= 1; });
    refuses_logits(SMALL, "short history_len", [](Logits& a) { a.len.bytes -= 1; });
    refuses_logits(SMALL, "short generated_from", [](Logits& a) { a.from.bytes -= 1; });
    refuses_logits(SMALL, "short penalties", [](Logits& a) { a.pen.bytes -= 1; });
    refuses_logits(BAD, "bias without values", [](Logits& a) { a.c.bias_values = nullptr; });
    refuses_logits(BAD, "bias without counts", [](Logits& a) { a.c.bias_len = nullptr; });
    refuses_logits(BAD, "bias width -1", [](Logits& a) { a.c.bias_width = -1; });
    refuses_logits(SMALL, "short bias ids", [](Logits& a) { a.ids.bytes -= 1; });
    refuses_logits(SMALL, "short bias values", [](Logits& a) { a.val.bytes -= 1; });
    refuses_logits(SMALL, "short mask", [](Logits& a) { a.mask.bytes -= 1; });
    refuses_logits(BAD, "misaligned mask", [](Logits& a) { a.mask = buffer(1 << 20, 0xA0000001); });
    refuses_logits(BAD, "out over the history", [](Logits& a) { a.hist = buffer(1 << 20, 0x20000000); });
    Logits a;
    CHECK(mvlm_logits_process(&dev, &a.x, 0, 4, 1000, 1000, nullptr, &a.out, nullptr) == BAD, "null controls");
    CHECK(mvlm_logits_process(&dev, &a.x, 0, 4, 1000, 1000, &a.c, nullptr, nullptr) == BAD, "null out");
    CHECK(mvlm_plan_add_logits_process(nullptr, &a.x, 0, 4, 1000, 1000, &a.c, &a.out) == BAD, "null plan");
}

int main() {
    setenv("MVLM_QUIET", "1", 1);
    test_division();
    test_spans();
    test_paged_refusals();
    test_logits_refusals();
    std::printf("%d failures\n", failures);
    return failures != 0;
}
