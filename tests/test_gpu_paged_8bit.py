"""The 8-bit paged cache on the GPU against its definition in 64 bits, through the C ABI: appended with and without
norms, read back, attended over.  What no sequence has written is garbage (NaN codes, scales of 0xFF), outputs start as NaN
patterns, and rows of no sequence must come back as they were."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
import mx_ref
from paged_ref import HALF_STEP, SMALLEST, Batch, attention, cache_on, close, from_bits, nan_cache, values
from test_gpu_paged import NAN, NP, rope_table, same_or_close

pytestmark = pytest.mark.gpu

F32, F16, BF16, MX = m.F32, m.F16, m.BF16, m.MXFP8


def say(*a):
    print("[8 bit]", *a, flush=True)


# ---- append, with norms ---------------------------------------------------------------

def made_rows(x, heads, kv_heads, D, p, table, rot, inter, qw, kw, eps):
    """q | k | v heads of one row in 64 bits, and how far fp32 may be off before it is rounded to the cache's type"""
    y = x.reshape(-1, D).copy()
    t = np.zeros(y.shape)
    for lo, hi, w in ((0, heads, qw), (heads, heads + kv_heads, kw)):
        if w is not None:
            # the sum of squares: D fma, 4 sums over lanes, a division, eps, a square root, its inverse, two products
            y[lo:hi] *= w.astype(np.float64) / np.sqrt((y[lo:hi] ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
            t[lo:hi] = ((D + 8) / 2 + 4) * 2.0 ** -24 * np.abs(y[lo:hi])
    if rot:
        n = heads + kv_heads
        a, b = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if inter else (np.arange(rot // 2), np.arange(rot // 2, rot))
        c, s = table[p, :, 0].astype(np.float64), table[p, :, 1].astype(np.float64)
        ya, yb, ta, tb = y[:n, a].copy(), y[:n, b].copy(), t[:n, a].copy(), t[:n, b].copy()
        y[:n, a], y[:n, b] = ya * c - yb * s, yb * c + ya * s
        t[:n, a] = ta * np.abs(c) + tb * np.abs(s) + 3 * 2.0 ** -24 * (np.abs(ya * c) + np.abs(yb * s))
        t[:n, b] = tb * np.abs(c) + ta * np.abs(s) + 3 * 2.0 ** -24 * (np.abs(yb * c) + np.abs(ya * s))
    return y, t


def in_8_bits(got, y, t):
    """values of codes within half a step of y, off by t before: 2^-4 of the value, or 2^-10 of the block's power of
    two where that is more (the block's largest value may be off by t as well, so its power one higher)"""
    e = np.repeat(mx_ref.exponents(np.abs(y) + t), 32, -1)[..., :y.shape[-1]]
    half = np.maximum(2.0 ** -4 * (np.abs(y) + t), 2.0 ** (e - 10.0))
    assert np.all(np.abs(got - y) <= half + t)


APPENDS = [
    # news, lens, heads, kv_heads, D, rot, interleaved, page, x, cache, q norm, k norm, options
    ([1], [1], 1, 1, 8, 0, False, 16, F32, MX, False, False, {}),
    ([1], [1], 1, 1, 8, 8, False, 16, F32, F16, True, True, {}),
    ([1], [512], 32, 32, 64, 32, False, 16, F32, MX, False, False, {}),
    ([1], [512], 32, 8, 128, 128, False, 16, F32, MX, True, True, {"ragged": False}),
    ([1] * 16, [1, 2, 15, 16, 17, 31, 32, 33, 100, 0, 511, 512, 7, 9, 0, 1000], 32, 32, 64, 32, False, 16, F32, MX, True, True, {"ragged": False}),
    ([5, 0, 1, 33, 1], [5, 0, 70, 50, 1], 8, 2, 128, 128, True, 48, BF16, MX, True, False, {"lead": 2, "spare": 3}),
    ([5, 0, 1, 33, 1], [5, 0, 70, 50, 1], 8, 2, 128, 128, True, 48, BF16, BF16, False, True, {"lead": 2, "spare": 3}),
    ([7, 3], [20, 3], 12, 4, 72, 36, False, 5, F16, MX, True, True, {}),
    ([7, 3], [20, 3], 12, 4, 72, 36, True, 5, F32, F16, True, True, {}),
    ([4, 2], [9, 2], 6, 3, 80, 40, False, 1, F32, MX, True, True, {"pad": 3}),
    ([4, 2], [9, 2], 6, 3, 80, 10, False, 64, F16, MX, False, True, {"pad": 1, "offset": 1}),
    ([4, 2], [9, 2], 6, 3, 16, 16, False, 64, F16, MX, True, False, {}),
    ([4, 2], [9, 2], 6, 3, 24, 24, False, 3, BF16, MX, True, True, {}),
    ([4, 2], [9, 2], 6, 3, 40, 20, True, 3, F32, BF16, True, True, {"pad": 8}),
    ([4, 2], [9, 2], 6, 3, 96, 96, True, 64, BF16, MX, False, False, {"pad": 8}),
    ([3], [40], 4, 4, 64, 64, False, 16, F16, MX, False, False, {"table": 39}),       # the last position is past the rotary table
    ([4], [2], 4, 2, 64, 64, False, 16, F16, MX, True, True, {}),                     # two rows before position 0
    ([20], [20], 4, 2, 64, 64, False, 8, F16, MX, True, True, {"width": 2}),          # four past the page table
    ([20, 4], [20, 4], 4, 2, 120, 64, True, 8, F32, MX, True, True, {"drop": {(0, 1): -1, (1, 0): 1 << 30}}),
    ([300], [300], 200, 100, 104, 32, False, 7, F16, MX, True, True, {}),             # more heads than a block makes at once
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(dev, case):
    news, lens, heads, kv_heads, D, rot, inter, page, xd, cd, qn, kn, opt = APPENDS[case]
    say("append", case, APPENDS[case])
    rng = np.random.default_rng(700 + case)
    opt = dict(opt)
    pad, offset, positions = opt.pop("pad", 0), opt.pop("offset", 0), opt.pop("table", max(lens) + 1)
    batch = Batch(rng, news, lens, page, **opt)
    width = (heads + 2 * kv_heads) * D
    ld = width + pad
    flat = values(rng, offset + batch.rows * ld, xd, 3.0)
    x = from_bits(flat, xd)[offset:].reshape(batch.rows, ld)[:, :width]
    table = rope_table(positions, rot) if rot else None
    qw, kw = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float32) if w else None for w in (qn, kn))
    eps = 1e-6
    mx = cd == MX
    qd = BF16 if mx else cd
    shape = (batch.pages, kv_heads, page, D)
    if mx:
        start = [mx_ref.garbage(rng, batch, kv_heads, D) for _ in range(2)]
        cache = mx_ref.cache_on(dev, batch, *start)
    else:
        start = nan_cache(batch, kv_heads, D, cd)
        cache = cache_on(dev, batch, *start, cd)
    es = flat.itemsize
    q = dev.upload(np.full(batch.rows * heads * D, NAN[qd]))
    rope = m.Rope(dev.upload(table), positions, rot, inter) if rot else None
    norm = m.HeadNorm(dev.upload(qw) if qn else None, dev.upload(kw) if kn else None, eps) if qn or kn else None
    dev.kv_append_paged_ex(dev.upload(flat).view(offset * es, (batch.rows * ld - pad) * es), xd, ld, batch.device(dev), cache,
                           heads, q, rope, norm)
    got = from_bits(q.download(np.uint16), qd).reshape(batch.rows, heads, D)
    held = mx_ref.cache_from(cache, shape) if mx else [b.download(np.uint16).reshape(shape) for b in cache.buffers]
    ref, tol = np.full(got.shape, np.nan), np.zeros(got.shape)
    for r, s, p in batch.each_row():
        at = batch.place(s, p)
        if at is None or (rot and p >= positions):
            ref[r] = 0.0
            continue
        y, t = made_rows(x[r], heads, kv_heads, D, p, table, rot, inter, qw, kw, eps)
        ref[r], tol[r] = y[:heads], t[:heads]
        for what, lo, exact in ((0, heads, not rot and not kn), (1, heads + kv_heads, True)):
            y_, t_ = y[lo:lo + kv_heads], t[lo:lo + kv_heads]
            if not mx:
                bits = held[what][at[0], :, at[1]]
                assert close(from_bits(bits, cd), y_, t_, cd) <= 1.0
                start[what][at[0], :, at[1]] = bits
                continue
            codes, word = (z[at[0], :, at[1]] for z in held[what])
            used = np.uint32(0xFFFFFFFF >> (32 - 8 * len(mx_ref.blocks(D))))
            if exact:                                          # nothing rounds before the codes do
                assert np.array_equal(codes, mx_ref.encode(y_)[0]) and np.array_equal(word & used, mx_ref.encode(y_)[1])
            else:
                in_8_bits(mx_ref.decode(codes, word & used), y_, t_)
            start[what][0][at[0], :, at[1]], start[what][1][at[0], :, at[1]] = codes, word
    assert same_or_close(got, ref, tol, qd) <= 1.0
    for a, b in zip(held, start):                              # nothing else was written
        assert all(np.array_equal(u, v) for u, v in zip(a, b)) if mx else np.array_equal(a, b)


def test_append_of_extreme_values(dev):
    """infinities, NaN, the largest and smallest fp32 values: each block on its own"""
    D, heads = 128, 2
    x = np.ones((6, 3 * heads, D), np.float32)
    x[0] = 0.0
    x[1, :, 3], x[1, :, 40], x[1, :, 100] = np.inf, -np.inf, np.nan
    x[2] = np.finfo(np.float32).max
    x[3] = 2.0 ** -149
    x[4, :, ::2], x[4, :, 1::2] = 1e30, -1e-30
    x[5] = (2.0 ** np.linspace(-120, 127, D)).astype(np.float32)
    rng = np.random.default_rng(3)
    batch = Batch(rng, [6], [6], 4)
    cache = mx_ref.cache_on(dev, batch, *(mx_ref.garbage(rng, batch, heads, D) for _ in range(2)))
    q = dev.alloc(6 * heads * D * 2)
    dev.kv_append_paged(dev.upload(x), F32, 3 * heads * D, batch.device(dev), cache, heads, q)
    held = mx_ref.cache_from(cache, (batch.pages, heads, batch.page, D))
    for r in range(6):
        page, slot = batch.place(0, r)
        for what, (codes, word) in enumerate(held):
            want = mx_ref.encode(x[r, heads * (1 + what):heads * (2 + what)])
            bad = want[0] & 0x7F == 0x7F
            got = codes[page, :, slot]
            assert np.array_equal(got[~bad], want[0][~bad]) and np.all(got[bad] & 0x7F == 0x7F)
            assert np.array_equal(word[page, :, slot], want[1])


# ---- read back ------------------------------------------------------------------------

READS = [
    # news, lens, kv_heads, D, page, cache, out, options
    ([1], [1], 1, 8, 16, MX, F32, {}),
    ([1] * 3, [40, 0, 7], 4, 64, 16, MX, F16, {"ragged": False}),
    ([729], [729], 32, 64, 16, MX, F16, {}),
    ([5, 0, 1, 33, 1], [9, 0, 70, 50, 1], 2, 128, 48, MX, BF16, {"lead": 2, "spare": 3}),
    ([5, 0, 1, 33, 1], [9, 0, 70, 50, 1], 2, 128, 48, F16, BF16, {"lead": 2, "spare": 3}),
    ([20, 20], [20, 20], 3, 72, 5, MX, F32, {"drop": {(0, 1): -1, (1, 0): 1 << 30}}),
    ([20, 20], [18, 20], 3, 80, 8, BF16, F32, {"width": 2, "pad": 8}),        # rows before position 0, and past the table
    ([20], [20], 5, 24, 1, MX, F16, {"pad": 3, "offset": 1}),
    ([9], [30], 5, 40, 64, F16, F16, {"pad": 120}),
    ([300], [300], 100, 104, 7, MX, BF16, {}),
]


@pytest.mark.parametrize("case", range(len(READS)))
@pytest.mark.parametrize("which", ["both", "k", "v"])
def test_read(dev, case, which):
    news, lens, kv_heads, D, page, cd, od, opt = READS[case]
    say("read", case, which, READS[case])
    rng = np.random.default_rng(800 + case)
    opt = dict(opt)
    pad, offset = opt.pop("pad", 0), opt.pop("offset", 0)
    batch = Batch(rng, news, lens, page, **opt)
    if cd == MX:
        held = mx_ref.filled(rng, batch, kv_heads, D)
        cache, vals = mx_ref.cache_on(dev, batch, *held), [mx_ref.decode(*x) for x in held]
    else:
        held = [values(rng, (batch.pages, kv_heads, page, D), cd) for _ in range(2)]
        cache, vals = cache_on(dev, batch, *held, cd), [from_bits(x, cd) for x in held]
    ld = kv_heads * D + pad
    flat = np.full(offset + batch.rows * ld, NAN[od])
    bufs = [dev.upload(flat) for _ in range(2)]
    size = (batch.rows * ld - pad) * flat.itemsize
    views = [b.view(offset * flat.itemsize, size) for b in bufs]
    dev.kv_read_paged(batch.device(dev), cache, views[0] if which != "v" else None, views[1] if which != "k" else None, od, ld)
    for what, (buf, x) in enumerate(zip(bufs, vals)):
        got = buf.download(NP[od])
        if which not in ("both", "kv"[what]):
            assert np.array_equal(got.view(np.uint8), flat.view(np.uint8))
            continue
        rows = from_bits(got, od)[offset:].reshape(batch.rows, ld)
        assert np.all(np.isnan(rows[:, kv_heads * D:])) and np.all(np.isnan(from_bits(got, od)[:offset]))
        ref = np.full((batch.rows, kv_heads, D), np.nan)
        for r, s, p in batch.each_row():
            at = batch.place(s, p)
            ref[r] = 0.0 if at is None else x[at[0], :, at[1]]
        assert same_or_close(rows[:, :kv_heads * D].reshape(ref.shape), ref, np.zeros(ref.shape), od) <= 1.0


def test_read_of_interleaved_rows(dev):
    """K and V rows between one another, as in one tensor of k | v rows"""
    rng = np.random.default_rng(5)
    batch = Batch(rng, [30], [30], 8)
    held = mx_ref.filled(rng, batch, 2, 64)
    out = dev.upload(np.full((30, 2, 128), np.float32(np.nan)))
    dev.kv_read_paged(batch.device(dev), mx_ref.cache_on(dev, batch, *held), out.view(0, (29 * 256 + 128) * 4),
                      out.view(512, (29 * 256 + 128) * 4), F32, 256)
    got = out.download(np.float32).reshape(30, 2, 2, 64)
    for r in range(30):
        page, slot = batch.place(0, r)
        for what in range(2):
            assert np.array_equal(got[r, what], mx_ref.decode(held[what][0], held[what][1])[page, :, slot])


def test_what_was_appended_is_read(dev):
    """append and read in one graph, replayed as the sequences grow: the values of the codes, and the rows' own keys"""
    rng = np.random.default_rng(7)
    heads, kv_heads, D, S = 4, 2, 96, 3
    width = (heads + 2 * kv_heads) * D
    lens = np.array([0, 15, 63], np.int32)
    batch = Batch(rng, [1] * S, lens + 4, 16, ragged=False)
    cache = mx_ref.cache_on(dev, batch, *(mx_ref.garbage(rng, batch, kv_heads, D) for _ in range(2)))
    b = batch.device(dev)
    x, q = dev.alloc(S * width * 4), dev.alloc(S * heads * D * 2)
    k, v = (dev.alloc(S * kv_heads * D * 4) for _ in range(2))
    plan = m.Plan(dev)
    plan.add_kv_append_paged(x, F32, width, b, cache, heads, q)
    plan.add_kv_read_paged(b, cache, k, v, F32, kv_heads * D)
    plan.use_graph(True)
    for _ in range(4):
        lens = lens + 1
        b.buffers[0].upload(lens)
        xs = rng.standard_normal((S, heads + 2 * kv_heads, D)).astype(np.float32)
        x.upload(xs)
        plan.run()
        for buf, lo in ((k, heads), (v, heads + kv_heads)):
            want = mx_ref.decode(*mx_ref.encode(xs[:, lo:lo + kv_heads]))
            assert np.array_equal(buf.download(np.float32).reshape(want.shape), want)


# ---- attention over the codes -------------------------------------------------------------

def run_attention(dev, batch, q, K, V, od, heads, scale=0.0):
    D = K[0].shape[3]
    cache = mx_ref.cache_on(dev, batch, K, V)
    o = dev.upload(np.full(batch.rows * heads * D, NAN[od]))
    dev.attention_paged(dev.upload(q), batch.device(dev), cache, o, od, heads, scale)
    return from_bits(o.download(NP[od]), od).reshape(batch.rows, heads, D)


def check_attention(dev, batch, heads, kv_heads, D, od, seed, std=1.0, scale=0.0):
    rng = np.random.default_rng(seed)
    K, V = mx_ref.filled(rng, batch, kv_heads, D, std)
    q = values(rng, (batch.rows, heads, D), BF16, std)
    got = run_attention(dev, batch, q, K, V, od, heads, scale)
    # garbage where nothing is held is not read by the reference
    ref, tol = attention(batch, q, mx_ref.bf16_of(*K), mx_ref.bf16_of(*V), BF16, scale or D ** -0.5, 1 if od != F32 else 2)
    worst = same_or_close(got, ref, tol, od)
    say("worst", worst)
    assert worst <= 1.0


ATTENTIONS = [
    # news, lens, heads, kv_heads, D, page, out, options
    ([1], [1], 1, 1, 8, 16, F32, {}),
    ([1], [512], 4, 4, 64, 16, F32, {"ragged": False}),
    ([1] * 9, [1, 2, 31, 32, 33, 0, 127, 129, 700], 4, 4, 64, 16, BF16, {"ragged": False}),
    ([1] * 9, [1, 2, 31, 32, 33, 0, 127, 129, 700], 16, 2, 128, 48, BF16, {"ragged": False}),
    ([1] * 3, [5, 0, 260], 40, 2, 64, 7, F32, {"ragged": False}),            # a group of 20: two tiles a token
    ([1] * 70, list(range(70)), 2, 1, 64, 1, F32, {"ragged": False}),        # more sequences than lanes
    ([1] * 3, [1, 40, 33], 2, 2, 72, 3, F32, {"ragged": False}),
    ([1] * 3, [1, 40, 33], 2, 2, 24, 1, BF16, {"ragged": False}),
    ([1] * 3, [1, 40, 333], 2, 1, 104, 16, BF16, {"ragged": False}),
    ([1] * 3, [1, 40, 333], 8, 2, 40, 16, F32, {"ragged": False}),
    ([1] * 3, [9, 40, 333], 8, 2, 96, 16, F32, {"ragged": False}),
    ([1] * 3, [9, 40, 333], 8, 2, 16, 16, BF16, {"ragged": False}),
    ([1], [1], 1, 1, 120, 1, F32, {"ragged": False}),
    ([17], [17], 4, 4, 64, 16, BF16, {}),
    ([33, 1, 0, 64, 2], [33, 40, 0, 200, 2], 4, 2, 72, 16, BF16, {"lead": 1, "spare": 2}),
    ([100], [357], 4, 1, 80, 64, BF16, {}),
    ([130, 1, 1], [130, 300, 7], 8, 8, 96, 32, F32, {}),
    ([65], [65], 2, 2, 128, 256, F32, {"spare": 5}),
    ([9], [4], 2, 2, 64, 16, BF16, {}),                                      # five rows before position 0: zeros
    ([40], [40], 4, 2, 64, 8, BF16, {"width": 3}),                           # sixteen positions past the page table
    ([40, 30], [40, 300], 4, 2, 64, 8, F32, {"drop": {(0, 0): -1, (1, 5): 1 << 30, (1, 36): -7}}),
    ([1, 1], [20, 20], 4, 2, 64, 16, F32, {"drop": {(0, 0): -1, (0, 1): -1}, "ragged": False}),   # sees nothing
    ([300], [1000], 2, 1, 64, 16, BF16, {}),
    ([257], [257], 3, 3, 24, 16, BF16, {}),
    ([60], [61], 3, 3, 8, 16, F32, {}),
    ([50], [70], 6, 2, 56, 16, F32, {}),
]


@pytest.mark.parametrize("case", range(len(ATTENTIONS)))
def test_attention(dev, case):
    news, lens, heads, kv_heads, D, page, od, opt = ATTENTIONS[case]
    say("attention", case, ATTENTIONS[case])
    batch = Batch(np.random.default_rng(900 + case), news, lens, page, **opt)
    check_attention(dev, batch, heads, kv_heads, D, od, 950 + case)


@pytest.mark.parametrize("lens,heads,kv_heads,D", [([5000, 3, 900], 2, 1, 64), ([9000], 8, 1, 128), ([2100] * 3, 4, 4, 72)])
def test_attention_splits_long_caches(dev, lens, heads, kv_heads, D):
    say("long", lens, heads, kv_heads, D)
    batch = Batch(np.random.default_rng(7), [1] * len(lens), lens, 64, ragged=False)
    check_attention(dev, batch, heads, kv_heads, D, F32, 8)


# Batches that fill the chip with tiles of 256 rows (rows x group / 256 per kv head, times the thousands of keys, at
# least 256 / kv_heads)
LARGE = [
    ([300], [300], 256, 256, 64, 16, BF16, {}),
    ([293, 1, 3], [500, 700, 3], 256, 128, 128, 48, BF16, {"lead": 1, "spare": 4}),
    ([256, 0, 70], [256, 0, 70], 256, 64, 72, 16, F32, {}),
    ([270, 5], [333, 400], 256, 64, 80, 7, F32, {"drop": {(0, 1): -1, (0, 40): 1 << 30, (1, 0): -5}}),
    ([290], [290], 256, 128, 96, 64, BF16, {"width": 4}),                    # rows past the page table
    ([260, 16], [200, 16], 256, 256, 8, 16, BF16, {}),                       # rows before position 0
    ([257] * 2 + [1] * 66, [257, 300] + list(range(66)), 256, 256, 32, 32, BF16, {}),   # more sequences than lanes
    ([512, 1], [4200, 9000], 32, 32, 64, 16, F32, {}),                       # splits
    ([260], [5000], 64, 64, 128, 1, BF16, {}),                               # splits of more keys than LDS holds slots for
    ([257], [4097], 64, 64, 48, 100, F32, {}),
    ([257], [600], 256, 128, 128, 16, F32, {}),
    ([257], [600], 256, 128, 104, 16, F32, {}),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_attention_of_many_rows(dev, case):
    news, lens, heads, kv_heads, D, page, od, opt = LARGE[case]
    say("many rows", case, news[:4], lens[:4], *LARGE[case][2:])
    batch = Batch(np.random.default_rng(1000 + case), news, lens, page, **opt)
    check_attention(dev, batch, heads, kv_heads, D, od, 1100 + case)


@pytest.mark.parametrize("std,scale", [(6.0, 0.0), (1.0, 3.0), (0.0, 0.0)])
def test_attention_sharp_and_flat_scores(dev, std, scale):
    """scores of some hundred (one key takes all, the running maximum moves often) and of 0"""
    batch = Batch(np.random.default_rng(11), [20, 1], [150, 400], 16)
    check_attention(dev, batch, 4, 2, 64, F32, 12, std, scale)


def test_attention_repeats_itself_and_leaves_the_cache(dev):
    rng = np.random.default_rng(13)
    batch = Batch(rng, [40, 1, 1], [700, 2000, 3], 16)
    K, V = mx_ref.filled(rng, batch, 2, 64)
    q = dev.upload(values(rng, (batch.rows, 4, 64), BF16))
    cache, b, o = mx_ref.cache_on(dev, batch, K, V), batch.device(dev), dev.alloc(batch.rows * 4 * 64 * 4)
    outs = []
    for _ in range(3):
        dev.attention_paged(q, b, cache, o, F32, 4)
        outs.append(o.download(np.uint32))
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])
    for buf, x in zip(cache.buffers, (K, V)):
        assert np.array_equal(buf.download(np.uint8), mx_ref.packed(*x))


@pytest.mark.parametrize("news,lens,heads,kv_heads,D,od,key", [
    ([40], [100], 4, 2, 64, BF16, 83), ([40], [40], 2, 2, 128, F32, 17), ([33], [33], 3, 3, 72, F32, 32),
    ([300], [300], 256, 256, 64, BF16, 200), ([256], [600], 256, 128, 128, BF16, 500), ([256], [600], 256, 128, 72, F32, 500)])
def test_attention_hidden_values_may_be_anything(dev, news, lens, heads, kv_heads, D, od, key):
    """NaN values of a new position reach the rows that see it and no row before"""
    say("not finite at", key, news, lens, heads, kv_heads, D)
    rng = np.random.default_rng(19)
    batch = Batch(rng, news, lens, 16)
    K, V = mx_ref.filled(rng, batch, kv_heads, D)
    q = values(rng, (batch.rows, heads, D), BF16)
    page, slot = batch.place(0, key)
    clean = V[0].copy()
    V[0][page, :, slot, 1], V[0][page, :, slot, D - 1], V[0][page, 0, slot, 5] = 0x7F, 0xFF, 0x7F
    clean[page, :, slot, 1] = clean[page, :, slot, D - 1] = clean[page, 0, slot, 5] = 0
    got = run_attention(dev, batch, q, K, V, od, heads)
    ref, tol = attention(batch, q, mx_ref.bf16_of(*K), mx_ref.bf16_of(clean, V[1]), BF16, D ** -0.5, 1 if od != F32 else 2)
    sees = np.arange(news[0]) >= key - (lens[0] - news[0])
    bad = np.zeros(got.shape, bool)
    bad[np.ix_(sees, np.arange(heads), [1, D - 1])] = True
    bad[np.ix_(sees, np.arange(heads // kv_heads), [5])] = True
    assert np.all(np.isnan(got[bad]))
    got[bad] = ref[bad] = 0.0
    assert same_or_close(got, ref, tol, od) <= 1.0


def test_attention_not_finite_where_seen(dev):
    """a NaN key makes the rows that see it NaN, and no other"""
    rng = np.random.default_rng(15)
    batch = Batch(rng, [8], [40], 16)
    K, V = mx_ref.filled(rng, batch, 2, 64)
    page, slot = batch.place(0, 36)
    K[0][page, 1, slot, 3] = 0x7F
    got = run_attention(dev, batch, values(rng, (8, 4, 64), BF16), K, V, BF16, 4)
    seen = np.zeros(got.shape, bool)
    seen[4:, 2:] = True                                     # rows 4 .. are positions 36 ..; heads 2, 3 read kv head 1
    assert np.array_equal(np.isnan(got), seen)


def test_over_int32_offsets(dev):
    """pages past 2^31 codes of a cache: append, attention and read"""
    D, page, kv_heads = 128, 64, 4
    pages = (1 << 32) // (page * kv_heads * D) + 3            # codes of K pass 2^32
    rng = np.random.default_rng(5)
    size = m.paged_kv_bytes(MX, pages, page, kv_heads, D)
    cache = m.PagedKV(dev.alloc(size), dev.alloc(size), MX, pages, page, kv_heads, D)
    batch = m.PagedBatch(1, 70, dev.upload(np.array([70], np.int32)), dev.upload(np.array([[pages - 1, 0]], np.int32)), 2,
                         row_start=dev.upload(np.array([0, 70], np.int32)))
    x = values(rng, (70, 3, kv_heads, D), BF16)
    q, o = dev.alloc(70 * kv_heads * D * 2), dev.alloc(70 * kv_heads * D * 4)
    k, v = (dev.alloc(70 * kv_heads * D * 4) for _ in range(2))
    say("page", pages - 1)
    dev.kv_append_paged(dev.upload(x), BF16, 3 * kv_heads * D, batch, cache, kv_heads, q)
    dev.attention_paged(q, batch, cache, o, F32, kv_heads)
    dev.kv_read_paged(batch, cache, k, v, F32, kv_heads * D)
    held = [mx_ref.encode(from_bits(x[:, i], BF16)) for i in (1, 2)]
    for buf, z in zip((k, v), held):
        assert np.array_equal(buf.download(np.float32).reshape(70, kv_heads, D), mx_ref.decode(*z))
    b = Batch(rng, [70], [70], page)
    b.pages, b.table = 2, np.array([[1, 0, -1]], np.int32)
    Kh, Vh = (np.zeros((2, kv_heads, page, D), np.uint16) for _ in range(2))
    for r in range(70):
        for to, z in ((Kh, held[0]), (Vh, held[1])):
            to[1 - r // 64, :, r % 64] = mx_ref.bf16_of(z[0][r], z[1][r])
    ref, tol = attention(b, x[:, 0], Kh, Vh, BF16, D ** -0.5, 2)
    assert close(o.download(np.float32).reshape(ref.shape).astype(np.float64), ref, tol, F32) <= 1.0


@pytest.mark.parametrize("cd", [MX, BF16])
def test_pages_past_int32(dev, cd):
    """one page of 2^25 positions: the second head's elements start 2^32 further on"""
    D, page, kv_heads = 128, 1 << 25, 2
    rng = np.random.default_rng(6)
    size = m.paged_kv_bytes(cd, 1, page, kv_heads, D)
    cache = m.PagedKV(dev.alloc(size), dev.alloc(size), cd, 1, page, kv_heads, D)
    batch = m.PagedBatch(1, 3, dev.upload(np.array([page], np.int32)), dev.upload(np.zeros(1, np.int32)), 1,
                         row_start=dev.upload(np.array([0, 3], np.int32)))
    x = values(rng, (3, 3, kv_heads, D), BF16)
    norm = m.HeadNorm(dev.upload(np.ones(D, np.float32)), None, 1e-6)
    q = dev.alloc(3 * kv_heads * D * 2)
    k, v = (dev.alloc(3 * kv_heads * D * 4) for _ in range(2))
    say("a page of", page)
    dev.kv_append_paged_ex(dev.upload(x), BF16, 3 * kv_heads * D, batch, cache, kv_heads, q, None, norm)
    dev.kv_read_paged(batch, cache, k, v, F32, kv_heads * D)
    for i, buf in ((1, k), (2, v)):
        want = from_bits(x[:, i], BF16)
        assert np.array_equal(buf.download(np.float32).reshape(3, kv_heads, D), mx_ref.decode(*mx_ref.encode(want)) if cd == MX else want)


def test_graphs_of_one_device_share_workspaces(dev):
    """two captured graphs with split attention, over 8 and over 16 bits, replayed in turn with eager calls between"""
    rng = np.random.default_rng(31)
    jobs = []
    for news, lens, heads, kv_heads, mx in (([1] * 3, [3000, 20, 1500], 8, 2, True), ([512, 1], [4200, 600], 32, 32, True),
                                            ([1] * 3, [2000, 7, 900], 4, 4, False)):
        batch = Batch(rng, news, lens, 16, ragged=len(news) != 3)
        if mx:
            cache = mx_ref.cache_on(dev, batch, *mx_ref.filled(rng, batch, kv_heads, 64))
        else:
            cache = cache_on(dev, batch, *(values(rng, (batch.pages, kv_heads, 16, 64), BF16) for _ in range(2)), BF16)
        q = dev.upload(values(rng, (batch.rows, heads, 64), BF16))
        b = batch.device(dev)
        o, eager = (dev.alloc(batch.rows * heads * 64 * 4).zero() for _ in range(2))
        dev.attention_paged(q, b, cache, eager, F32, heads)
        plan = m.Plan(dev)
        plan.add_attention_paged(q, b, cache, o, F32, heads)
        plan.use_graph(True)
        jobs.append((plan, o, eager.download(np.uint32), (q, b, cache, eager, heads)))
    for _ in range(3):
        for plan, o, _, _ in jobs:
            o.zero()
            plan.run(2)
        for plan, o, first, (q, b, cache, eager, heads) in jobs:
            dev.attention_paged(q, b, cache, eager, F32, heads)
            assert np.array_equal(o.download(np.uint32), first)
            assert np.array_equal(eager.download(np.uint32), first)
