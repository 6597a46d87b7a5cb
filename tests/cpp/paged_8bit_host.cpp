// Host checks of the 8-bit paged cache, the norms of its append and the token draw, without a GPU (run by
// tests/test_paged_8bit_host.py): the rule of a block's power of two, the sizes of buffers, and the refusals of the
// entry points.  Handles are made by hand: a refused call reads only sizes and addresses and reaches no device.
#include "common.h"
#include "paged.h"

#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
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

static void test_exponent() {
    std::mt19937 rng(1);
    for (int i = 0; i < 300000; ++i) {
        uint32_t b = i < 2000 ? (uint32_t)i : rng() & 0x7FFFFFFFu;
        if (i % 5 == 0) b = (b & 0x7F800000u) | 0x600000u | (i / 5 % 3 == 1 ? 1u : 0u);    // 1.75 and just above
        if (b >= 0x7F800000u) continue;
        float a;
        std::memcpy(&a, &b, 4);
        const int e = mx_exponent(b);
        CHECK(e >= MX_LEAST && e <= MX_MOST, "%g: %d", (double)a, e);
        CHECK((double)a <= std::ldexp(448.0, e), "%g is above 448 2^%d", (double)a, e);
        CHECK(e == MX_LEAST || (double)a > std::ldexp(448.0, e - 1), "%g would fit 448 2^%d", (double)a, e - 1);
    }
}

static mvlm_device dev, other;
static mvlm_buffer buffer(size_t bytes, uintptr_t address, mvlm_device* d = &dev) {
    mvlm_buffer b;
    b.dev = d;
    b.ptr = (void*)address;
    b.bytes = bytes;
    return b;
}
static const int BAD = MVLM_ERR_INVALID_ARG, SMALL = MVLM_ERR_BUFFER_TOO_SMALL, NOT = MVLM_ERR_UNSUPPORTED;

static void test_sizes() {
    size_t n = 0;
    mvlm_paged_kv kv{nullptr, nullptr, MVLM_MXFP8, 3, 5, 7, 24};
    CHECK(mvlm_paged_kv_bytes(&kv, &n) == MVLM_OK && n == 2528 + 420, "105 slots of 24: %zu", n);
    kv.head_dim = 64;
    CHECK(mvlm_paged_kv_bytes(&kv, &n) == MVLM_OK && n == 6720 + 420, "105 slots of 64: %zu", n);
    kv.dtype = MVLM_BF16;
    CHECK(mvlm_paged_kv_bytes(&kv, &n) == MVLM_OK && n == 13440, "16 bits: %zu", n);
    CHECK(mvlm_paged_kv_bytes(&kv, nullptr) == BAD && mvlm_paged_kv_bytes(nullptr, &n) == BAD, "null");
    kv.dtype = MVLM_Q8_0;
    CHECK(mvlm_paged_kv_bytes(&kv, &n) == BAD, "dtype");
    kv = {nullptr, nullptr, MVLM_MXFP8, 1 << 20, 1 << 10, 2, 64};
    CHECK(mvlm_paged_kv_bytes(&kv, &n) == NOT, "2^31 slots");
    kv = {nullptr, nullptr, MVLM_MXFP8, 4, 16, 2, 60};
    CHECK(mvlm_paged_kv_bytes(&kv, &n) == NOT, "head_dim");
    // a load of 16 codes from the last chunk of any row stays inside (rows lie at multiples of 8 bytes)
    for (int D = 8; D <= 128; D += 8)
        for (int slots = 1; slots <= 6; ++slots) {
            kv = {nullptr, nullptr, MVLM_MXFP8, slots, 1, 1, D};
            CHECK(mvlm_paged_kv_bytes(&kv, &n) == MVLM_OK && (size_t)(slots - 1) * D + (size_t)(D + 15) / 16 * 16 <= n, "%d slots of %d", slots, D);
        }
}

// the arguments of calls that would be taken; each refusal changes one thing
struct Call {
    mvlm_buffer k = buffer(1024 * 68, 0x10000000), v = buffer(1024 * 68, 0x20000000), len = buffer(16, 0x30000000),
                table = buffer(64, 0x40000000), start = buffer(20, 0x50000000), x = buffer(1 << 20, 0x60000000),
                q = buffer(1 << 20, 0x70000000), cs = buffer(1 << 20, 0x80000000), o = buffer(1 << 20, 0x90000000),
                qw = buffer(256, 0xA0000000), kw = buffer(256, 0xB0000000), ko = buffer(1 << 20, 0xC0000000), vo = buffer(1 << 20, 0xD0000000);
    mvlm_paged_kv kv{&k, &v, MVLM_MXFP8, 16, 16, 4, 64};
    mvlm_paged_batch batch{4, 8, &start, &len, &table, 4};
    mvlm_rope rope{&cs, 64, 64, 0};
    mvlm_head_norm norm{&qw, &kw, 1e-6f};
    int x_dtype = MVLM_F32, heads = 8, o_dtype = MVLM_BF16, out_dtype = MVLM_F16;
    int64_t ld = 16 * 64, out_ld = 256;
    mvlm_buffer *k_out = &ko, *v_out = &vo;
    int append() { return mvlm_kv_append_paged_ex(&dev, &x, x_dtype, ld, &batch, &kv, heads, &q, &rope, &norm, nullptr); }
    int attend() { return mvlm_attention_paged(&dev, &q, &batch, &kv, &o, o_dtype, heads, 0.0f, nullptr); }
    int read() { return mvlm_kv_read_paged(&dev, &batch, &kv, k_out, v_out, out_dtype, out_ld, nullptr); }
};
enum { APPEND = 1, ATTEND = 2, READ = 4, ALL = 7 };
template <class F>
static void refuses(int code, int calls, const char* what, F change) {
    for (int c : {APPEND, ATTEND, READ}) {
        if (!(calls & c)) continue;
        Call a;
        change(a);
        const int got = c == APPEND ? a.append() : c == ATTEND ? a.attend() : a.read();
        CHECK(got == code, "call %d, %s: %d (%s)", c, what, got, mvlm_last_error());
    }
}

static void test_cache_refusals() {
    refuses(BAD, ALL, "null k", [](Call& a) { a.kv.k = nullptr; });
    refuses(BAD, ALL, "cache of int8 blocks", [](Call& a) { a.kv.dtype = MVLM_Q8_0; });
    refuses(SMALL, ALL, "room for codes alone", [](Call& a) { a.k.bytes = 1024 * 64; });
    refuses(SMALL, ALL, "a byte short", [](Call& a) { a.v.bytes -= 1; });
    refuses(BAD, ALL, "misaligned", [](Call& a) { a.k = buffer(1 << 20, 0x10000008); });
    refuses(BAD, ALL, "v in k's scales", [](Call& a) { a.v = buffer(1 << 20, 0x10000000 + 65536); });
    refuses(NOT, ALL, "head_dim 60", [](Call& a) { a.kv.head_dim = 60; });
    refuses(NOT, ALL, "32 GiB of codes", [](Call& a) { a.kv.num_pages = 1 << 22, a.kv.head_dim = 128, a.k.bytes = a.v.bytes = SIZE_MAX; });
    refuses(BAD, ALL, "another device's cache", [](Call& a) { a.v.dev = &other; });
    refuses(BAD, ALL, "another device's table", [](Call& a) { a.table.dev = &other; });
    refuses(BAD, ALL, "no rows", [](Call& a) { a.batch.rows = 0; });
    refuses(SMALL, ALL, "short table", [](Call& a) { a.table.bytes = 63; });
    refuses(BAD, ATTEND, "fp16 output", [](Call& a) { a.o_dtype = MVLM_F16; });
    refuses(BAD, ATTEND, "8-bit output", [](Call& a) { a.o_dtype = MVLM_MXFP8; });
    refuses(BAD, ATTEND, "O in v's scales", [](Call& a) { a.o = buffer(1 << 20, 0x20000000 + 65536); });
    refuses(BAD, APPEND, "8-bit qkv", [](Call& a) { a.x_dtype = MVLM_MXFP8; });
    refuses(BAD, APPEND, "q_out in k's scales", [](Call& a) { a.q = buffer(1 << 20, 0x10000000 + 65536); });
    refuses(BAD, APPEND, "k's scales over kv_len", [](Call& a) { a.len = buffer(16, 0x10000000 + 65536 + 1024); });
}

static void test_norm_refusals() {
    refuses(BAD, APPEND, "no weights", [](Call& a) { a.norm.q_weight = a.norm.k_weight = nullptr; });
    refuses(BAD, APPEND, "negative eps", [](Call& a) { a.norm.eps = -1e-6f; });
    refuses(BAD, APPEND, "infinite eps", [](Call& a) { a.norm.eps = INFINITY; });
    refuses(BAD, APPEND, "NaN eps", [](Call& a) { a.norm.eps = NAN; });
    refuses(SMALL, APPEND, "short q weight", [](Call& a) { a.qw.bytes = 255; });
    refuses(SMALL, APPEND, "short k weight", [](Call& a) { a.kw.bytes = 255; });
    refuses(BAD, APPEND, "misaligned k weight", [](Call& a) { a.kw = buffer(512, 0xB0000002); });
    refuses(BAD, APPEND, "another device's weight", [](Call& a) { a.qw.dev = &other; });
    refuses(BAD, APPEND, "q_out over a weight", [](Call& a) { a.qw = buffer(256, 0x70000000); });
    refuses(BAD, APPEND, "the cache over a weight", [](Call& a) { a.kw = buffer(256, 0x20000100); });
}

static void test_read_refusals() {
    refuses(BAD, READ, "no outputs", [](Call& a) { a.k_out = a.v_out = nullptr; });
    refuses(BAD, READ, "8-bit output", [](Call& a) { a.out_dtype = MVLM_MXFP8; });
    refuses(BAD, READ, "short ld", [](Call& a) { a.out_ld = 255; });
    refuses(BAD, READ, "huge ld", [](Call& a) { a.out_ld = INT64_MAX; });
    refuses(SMALL, READ, "short K", [](Call& a) { a.ko.bytes = 8 * 256 * 2 - 1; });
    refuses(SMALL, READ, "short V", [](Call& a) { a.vo.bytes = 8 * 256 * 2 - 1, a.k_out = nullptr; });
    refuses(BAD, READ, "misaligned K", [](Call& a) { a.ko = buffer(1 << 20, 0xC0000001); });
    refuses(BAD, READ, "another device's V", [](Call& a) { a.vo.dev = &other; });
    refuses(BAD, READ, "K is V", [](Call& a) { a.v_out = &a.ko; });
    refuses(BAD, READ, "V inside K", [](Call& a) { a.vo = buffer(1 << 20, 0xC0000000 + 4094); });
    refuses(BAD, READ, "rows between rows, too near", [](Call& a) { a.out_ld = 500, a.vo = buffer(1 << 20, 0xC0000000 + 512); });
    refuses(BAD, READ, "K in the cache", [](Call& a) { a.ko = buffer(1 << 20, 0x10000000 + 65536); });
    refuses(BAD, READ, "V over the table", [](Call& a) { a.table = buffer(64, 0xD0000000); });
    Call a;
    CHECK(mvlm_kv_read_paged(nullptr, &a.batch, &a.kv, &a.ko, &a.vo, MVLM_F16, 256, nullptr) == BAD, "null device");
    CHECK(mvlm_kv_read_paged(&dev, nullptr, &a.kv, &a.ko, &a.vo, MVLM_F16, 256, nullptr) == BAD, "null batch");
    CHECK(mvlm_kv_read_paged(&dev, &a.batch, nullptr, &a.ko, &a.vo, MVLM_F16, 256, nullptr) == BAD, "null cache");
    CHECK(mvlm_plan_add_kv_read_paged(nullptr, &a.batch, &a.kv, &a.ko, &a.vo, MVLM_F16, 256) == BAD, "null plan");
    CHECK(mvlm_plan_add_kv_append_paged_ex(nullptr, &a.x, 0, a.ld, &a.batch, &a.kv, 8, &a.q, nullptr, nullptr) == BAD, "null plan");
}

struct Draw {
    mvlm_buffer x = buffer(4 * 1000 * 4, 0x10000000), out = buffer(16, 0x20000000), u = buffer(16, 0x30000000),
                t = buffer(16, 0x40000000), k = buffer(16, 0x50000000), p = buffer(16, 0x60000000), least = buffer(16, 0x70000000);
    mvlm_sampling s{&u, &t, &k, &p, &least};
    int dtype = MVLM_F32, rows = 4, n = 1000;
    int64_t ld = 1000;
    int call() { return mvlm_sample(&dev, &x, dtype, rows, n, ld, &s, &out, nullptr); }
};
template <class F>
static void refuses_draw(int code, const char* what, F change) {
    Draw a;
    change(a);
    const int got = a.call();
    CHECK(got == code, "draw, %s: %d (%s)", what, got, mvlm_last_error());
}

static void test_draw_refusals() {
    refuses_draw(BAD, "dtype", [](Draw& a) { a.dtype = MVLM_MXFP8; });
    refuses_draw(BAD, "no rows", [](Draw& a) { a.rows = 0; });
    refuses_draw(BAD, "no tokens", [](Draw& a) { a.n = 0; });
    refuses_draw(BAD, "short ld", [](Draw& a) { a.ld = 999; });
    refuses_draw(BAD, "huge ld", [](Draw& a) { a.ld = INT64_MAX; });
    refuses_draw(BAD, "too many rows", [](Draw& a) { a.rows = (1 << 20) + 1; });
    refuses_draw(BAD, "too many tokens", [](Draw& a) { a.n = (1 << 24) + 1, a.ld = a.n; });
    refuses_draw(SMALL, "short x", [](Draw& a) { a.x.bytes -= 1; });
    refuses_draw(SMALL, "short out", [](Draw& a) { a.out.bytes -= 1; });
    refuses_draw(SMALL, "short uniform", [](Draw& a) { a.u.bytes -= 1; });
    refuses_draw(SMALL, "short temperature", [](Draw& a) { a.t.bytes -= 1; });
    refuses_draw(SMALL, "short top_k", [](Draw& a) { a.k.bytes -= 1; });
    refuses_draw(SMALL, "short top_p", [](Draw& a) { a.p.bytes -= 1; });
    refuses_draw(SMALL, "short min_p", [](Draw& a) { a.least.bytes -= 1; });
    refuses_draw(BAD, "misaligned x", [](Draw& a) { a.x = buffer(1 << 20, 0x10000002); });
    refuses_draw(BAD, "misaligned out", [](Draw& a) { a.out = buffer(64, 0x20000002); });
    refuses_draw(BAD, "misaligned top_p", [](Draw& a) { a.p = buffer(64, 0x60000001); });
    refuses_draw(BAD, "another device's x", [](Draw& a) { a.x.dev = &other; });
    refuses_draw(BAD, "another device's out", [](Draw& a) { a.out.dev = &other; });
    refuses_draw(BAD, "another device's min_p", [](Draw& a) { a.least.dev = &other; });
    refuses_draw(BAD, "no random numbers", [](Draw& a) { a.s.uniform = nullptr; });
    refuses_draw(BAD, "out in x", [](Draw& a) { a.out = buffer(16, 0x10000100); });
    refuses_draw(BAD, "out over the random numbers", [](Draw& a) { a.out = buffer(16, 0x30000008); });
    Draw a;
    CHECK(mvlm_sample(&dev, &a.x, 0, 4, 1000, 1000, nullptr, &a.out, nullptr) == BAD, "null settings");
    CHECK(mvlm_sample(&dev, &a.x, 0, 4, 1000, 1000, &a.s, nullptr, nullptr) == BAD, "null out");
    CHECK(mvlm_sample(nullptr, &a.x, 0, 4, 1000, 1000, &a.s, &a.out, nullptr) == BAD, "null device");
    CHECK(mvlm_plan_add_sample(nullptr, &a.x, 0, 4, 1000, 1000, &a.s, &a.out) == BAD, "null plan");
}

int main() {
    setenv("MVLM_QUIET", "1", 1);
    test_exponent();
    test_sizes();
    test_cache_refusals();
    test_norm_refusals();
    test_read_refusals();
    test_draw_refusals();
    std::printf("%d failures\n", failures);
    return failures != 0;
}
