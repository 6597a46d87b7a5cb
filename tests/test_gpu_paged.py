"""mvlm_kv_append_paged and mvlm_attention_paged on the GPU against their
definitions in 64 bits (paged_ref), through the C ABI.  Caches hold NaN wherever
no sequence has written, outputs start as NaN patterns, and rows of no sequence
must come back as they were."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import (HALF_STEP, SMALLEST, Batch, attention, cache_on, close, filled_cache, from_bits, nan_cache,
                       to_bits, values)

pytestmark = pytest.mark.gpu

F32, F16, BF16 = m.F32, m.F16, m.BF16
NP = {F32: np.float32, F16: np.uint16, BF16: np.uint16}
NAN = {F32: np.float32(np.nan), F16: np.uint16(0x7E00), BF16: np.uint16(0x7FC0)}


def say(*a):
    print("[paged]", *a, flush=True)


# ---- append ------------------------------------------------------------------------

def rope_table(positions, rot):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)


def append_reference(batch, x, heads, kv_heads, D, dtype, table, rot, interleaved, K, V):
    """(q, its tolerance, K, V, their tolerances) in 64 bits; NaN in rows of no sequence"""
    q, qt = np.full((batch.rows, heads, D), np.nan), np.zeros((batch.rows, heads, D))
    K, V = from_bits(K, dtype), from_bits(V, dtype)
    Kt = np.zeros(K.shape)
    for r, s, p in batch.each_row():
        at = batch.place(s, p)
        if at is None or (rot and p >= len(table)):
            q[r] = 0.0
            continue
        y, yt = x[r].reshape(-1, D).copy(), np.zeros((heads + 2 * kv_heads, D))
        if rot:
            a, b = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2),
                                                                                     np.arange(rot // 2, rot))
            c, sn = table[p, :, 0].astype(np.float64), table[p, :, 1].astype(np.float64)
            n = heads + kv_heads
            ya, yb = y[:n, a].copy(), y[:n, b].copy()
            y[:n, a], y[:n, b] = ya * c - yb * sn, yb * c + ya * sn
            # two products and a sum in fp32
            yt[:n, a] = 3 * 2.0 ** -24 * (np.abs(ya * c) + np.abs(yb * sn))
            yt[:n, b] = 3 * 2.0 ** -24 * (np.abs(yb * c) + np.abs(ya * sn))
        q[r], qt[r] = y[:heads], yt[:heads]
        K[at[0], :, at[1]], Kt[at[0], :, at[1]] = y[heads:heads + kv_heads], yt[heads:heads + kv_heads]
        V[at[0], :, at[1]] = y[heads + kv_heads:]
    return q, qt, K, V, Kt


def same_or_close(got, ref, tol, dtype):
    """NaN where the reference is NaN, else within tol and half a step"""
    gone = np.isnan(ref)
    assert np.array_equal(np.isnan(got), gone)
    return close(got[~gone], ref[~gone], tol[~gone], dtype)


APPENDS = [
    # news, lens, heads, kv_heads, D, rot, interleaved, page, x, cache, options
    ([1], [1], 1, 1, 8, 0, False, 16, F32, F16, {}),
    ([1], [512], 32, 32, 64, 32, False, 16, F32, F16, {}),
    ([1] * 16, [1, 2, 15, 16, 17, 31, 32, 33, 100, 0, 511, 512, 7, 9, 0, 1000], 32, 32, 64, 32, False, 16, F32, F16, {"ragged": False}),
    ([5, 0, 1, 33, 1], [5, 0, 70, 50, 1], 8, 2, 128, 128, True, 48, BF16, BF16, {"lead": 2, "spare": 3}),
    ([7, 3], [20, 3], 12, 4, 72, 36, False, 5, F16, F16, {}),
    ([7, 3], [20, 3], 12, 4, 72, 36, True, 5, F32, BF16, {}),
    ([4, 2], [9, 2], 6, 3, 80, 40, False, 1, F32, F16, {"pad": 3}),
    ([4, 2], [9, 2], 6, 3, 80, 10, False, 64, F16, F16, {"pad": 1, "offset": 1}),
    ([4, 2], [9, 2], 6, 3, 96, 96, True, 64, BF16, BF16, {"pad": 8}),
    ([3], [40], 4, 4, 64, 64, False, 16, F16, BF16, {"table": 39}),      # the last position is past the rotary table
    ([4], [2], 4, 2, 64, 64, False, 16, F16, F16, {}),                    # two rows before position 0
    ([20], [20], 4, 2, 64, 64, False, 8, F16, F16, {"width": 2}),         # four past the page table
    ([20, 4], [20, 4], 4, 2, 64, 64, True, 8, F32, F16, {"drop": {(0, 1): -1, (1, 0): 1 << 30}}),
    ([300], [300], 2, 1, 64, 32, False, 7, F16, F16, {}),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(dev, case):
    news, lens, heads, kv_heads, D, rot, inter, page, xd, cd, opt = APPENDS[case]
    say("append", case, APPENDS[case])
    rng = np.random.default_rng(100 + case)
    opt = dict(opt)
    pad, offset, positions = opt.pop("pad", 0), opt.pop("offset", 0), opt.pop("table", max(lens) + 1)
    batch = Batch(rng, news, lens, page, **opt)
    width = (heads + 2 * kv_heads) * D
    ld = width + pad
    flat = values(rng, offset + batch.rows * ld, xd)
    x = from_bits(flat, xd)[offset:].reshape(batch.rows, ld)[:, :width]
    table = rope_table(positions, rot) if rot else None
    K, V = nan_cache(batch, kv_heads, D, cd)
    cache = cache_on(dev, batch, K, V, cd)
    es = flat.itemsize
    whole = dev.upload(flat)
    q = dev.upload(np.full(batch.rows * heads * D, NAN[cd]))
    rope = m.Rope(dev.upload(table), positions, rot, inter) if rot else None
    dev.kv_append_paged(whole.view(offset * es, (batch.rows * ld - pad) * es), xd, ld, batch.device(dev), cache, heads, q, rope)
    got = from_bits(q.download(np.uint16), cd).reshape(batch.rows, heads, D)
    gK, gV = (from_bits(b.download(np.uint16), cd).reshape(K.shape) for b in cache.buffers)
    ref, qt, rK, rV, Kt = append_reference(batch, x, heads, kv_heads, D, cd, table, rot, inter, K, V)
    worst = [same_or_close(got, ref, qt, cd), same_or_close(gK, rK, Kt, cd), same_or_close(gV, rV, np.zeros(V.shape), cd)]
    say("worst", worst)
    assert max(worst) <= 1.0


def test_append_over_int32_offsets(dev):
    """pages past 2^31 elements of a cache: only the page's own slots change"""
    D, page, kv_heads = 128, 64, 4
    pages = (1 << 32) // (page * kv_heads * D) + 3            # elements of K pass 2^32
    rng = np.random.default_rng(5)
    K, V = dev.alloc(pages * page * kv_heads * D * 2), dev.alloc(pages * page * kv_heads * D * 2)
    cache = m.PagedKV(K, V, F16, pages, page, kv_heads, D)
    table = np.array([[pages - 1, 0]], np.int32)
    batch = m.PagedBatch(1, 70, dev.upload(np.array([70], np.int32)), dev.upload(table), 2,
                         row_start=dev.upload(np.array([0, 70], np.int32)))
    x = values(rng, (70, 3 * kv_heads * D), F16)
    q, o = dev.alloc(70 * kv_heads * D * 2), dev.alloc(70 * kv_heads * D * 4)
    say("append and attention at page", pages - 1)
    dev.kv_append_paged(dev.upload(x), F16, 3 * kv_heads * D, batch, cache, kv_heads, q)
    dev.attention_paged(q, batch, cache, o, F32, kv_heads)
    block = page * kv_heads * D * 2
    x = x.reshape(70, 3, kv_heads, D)
    for buf, what in ((K, 1), (V, 2)):
        last = buf.download(np.uint16, block // 2, (pages - 1) * block).reshape(kv_heads, page, D)
        assert np.array_equal(last, x[:64, what].transpose(1, 0, 2))
        first = buf.download(np.uint16, block // 2, 0).reshape(kv_heads, page, D)
        assert np.array_equal(first[:, :6], x[64:, what].transpose(1, 0, 2))
    b = Batch(rng, [70], [70], page)
    b.pages, b.table = 2, np.array([[1, 0, -1]], np.int32)
    Kh, Vh = (np.zeros((2, kv_heads, page, D), np.uint16) for _ in range(2))
    for r in range(70):
        Kh[1 - r // 64, :, r % 64], Vh[1 - r // 64, :, r % 64] = x[r, 1], x[r, 2]
    ref, tol = attention(b, x[:, 0], Kh, Vh, F16, D ** -0.5, 2)
    assert close(o.download(np.float32).reshape(ref.shape).astype(np.float64), ref, tol, F32) <= 1.0


# ---- attention -----------------------------------------------------------------------

def run_attention(dev, batch, q, K, V, cd, od, heads, scale=0.0):
    D = K.shape[3]
    cache = cache_on(dev, batch, K, V, cd)
    o = dev.upload(np.full(batch.rows * heads * D, NAN[od]))
    dev.attention_paged(dev.upload(q), batch.device(dev), cache, o, od, heads, scale)
    return from_bits(o.download(NP[od]), od).reshape(batch.rows, heads, D)


def check_attention(dev, batch, heads, kv_heads, D, cd, od, seed, std=1.0, scale=0.0):
    rng = np.random.default_rng(seed)
    K, V = filled_cache(rng, batch, kv_heads, D, cd, std)
    q = values(rng, (batch.rows, heads, D), cd, std)
    got = run_attention(dev, batch, q, K, V, cd, od, heads, scale)
    ref, tol = attention(batch, q, K, V, cd, scale or D ** -0.5, 1 if od != F32 else 2)
    worst = same_or_close(got, ref, tol, od)
    say("worst", worst)
    assert worst <= 1.0


ATTENTIONS = [
    # news, lens, heads, kv_heads, D, page, cache, out, options
    ([1], [1], 1, 1, 8, 16, F16, F32, {}),
    ([1], [512], 4, 4, 64, 16, F16, F32, {"ragged": False}),
    ([1] * 9, [1, 2, 31, 32, 33, 0, 127, 129, 700], 4, 4, 64, 16, F16, F16, {"ragged": False}),
    ([1] * 9, [1, 2, 31, 32, 33, 0, 127, 129, 700], 16, 2, 128, 48, BF16, BF16, {"ragged": False}),
    ([1] * 3, [5, 0, 260], 40, 2, 64, 7, BF16, F32, {"ragged": False}),   # a group of 20: two tiles a token
    ([1] * 70, list(range(70)), 2, 1, 64, 1, F16, F32, {"ragged": False}),  # more sequences than lanes
    ([17], [17], 4, 4, 64, 16, F16, F16, {}),
    ([33, 1, 0, 64, 2], [33, 40, 0, 200, 2], 4, 2, 72, 16, F16, F16, {"lead": 1, "spare": 2}),
    ([100], [357], 4, 1, 80, 64, BF16, BF16, {}),
    ([130, 1, 1], [130, 300, 7], 8, 8, 96, 32, F16, F32, {}),
    ([65], [65], 2, 2, 128, 256, BF16, F32, {"spare": 5}),
    ([9], [4], 2, 2, 64, 16, F16, F16, {}),                                # five rows before position 0: zeros
    ([40], [40], 4, 2, 64, 8, F16, F16, {"width": 3}),                     # sixteen positions past the page table
    ([40, 30], [40, 300], 4, 2, 64, 8, F16, F32, {"drop": {(0, 0): -1, (1, 5): 1 << 30, (1, 36): -7}}),
    ([1, 1], [20, 20], 4, 2, 64, 16, F16, F32, {"drop": {(0, 0): -1, (0, 1): -1}, "ragged": False}),   # sees nothing
    ([300], [1000], 2, 1, 64, 16, F16, F16, {}),
    ([257], [257], 3, 3, 24, 16, F16, F16, {}),
]


@pytest.mark.parametrize("case", range(len(ATTENTIONS)))
def test_attention(dev, case):
    news, lens, heads, kv_heads, D, page, cd, od, opt = ATTENTIONS[case]
    say("attention", case, ATTENTIONS[case])
    batch = Batch(np.random.default_rng(200 + case), news, lens, page, **opt)
    check_attention(dev, batch, heads, kv_heads, D, cd, od, 300 + case)


@pytest.mark.parametrize("lens,heads,kv_heads,D,cd", [([5000, 3, 900], 2, 1, 64, F16), ([9000], 8, 1, 128, BF16),
                                                      ([2100] * 3, 4, 4, 64, F16)])
def test_attention_splits_long_caches(dev, lens, heads, kv_heads, D, cd):
    say("long", lens, heads, kv_heads, D, cd)
    batch = Batch(np.random.default_rng(7), [1] * len(lens), lens, 64, ragged=False)
    check_attention(dev, batch, heads, kv_heads, D, cd, F32, 8)


def test_attention_chunk_with_splits(dev):
    batch = Batch(np.random.default_rng(9), [37, 1], [1800, 1000], 16)
    check_attention(dev, batch, 2, 2, 64, F16, F16, 10)


@pytest.mark.parametrize("std,scale", [(6.0, 0.0), (1.0, 3.0), (0.0, 0.0)])
def test_attention_sharp_and_flat_scores(dev, std, scale):
    """scores of some hundred (one key takes all, the running maximum moves often) and of 0"""
    batch = Batch(np.random.default_rng(11), [20, 1], [150, 400], 16)
    check_attention(dev, batch, 4, 2, 64, F16, F32, 12, std, scale)


def test_attention_repeats_itself_and_leaves_the_cache(dev):
    rng = np.random.default_rng(13)
    batch = Batch(rng, [40, 1, 1], [700, 2000, 3], 16)
    K, V = filled_cache(rng, batch, 2, 64, F16)
    q = dev.upload(values(rng, (batch.rows, 4, 64), F16))
    cache, b, o = cache_on(dev, batch, K, V, F16), batch.device(dev), dev.alloc(batch.rows * 4 * 64 * 4)
    outs = []
    for _ in range(3):
        dev.attention_paged(q, b, cache, o, F32, 4)
        outs.append(o.download(np.uint32))
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])
    assert np.array_equal(cache.buffers[0].download(np.uint16).reshape(K.shape), K)
    assert np.array_equal(cache.buffers[1].download(np.uint16).reshape(V.shape), V)


def test_attention_not_finite_where_seen(dev):
    """a NaN key or an infinite score makes the rows that see it NaN, and no other"""
    rng = np.random.default_rng(15)
    batch = Batch(rng, [8], [40], 16)
    K, V = filled_cache(rng, batch, 2, 64, F16)
    page, slot = batch.place(0, 36)
    K[page, 1, slot, 3] = 0x7E00
    q = values(rng, (8, 4, 64), F16)
    got = run_attention(dev, batch, q, K, V, F16, F16, 4)
    seen = np.zeros(got.shape, bool)
    seen[4:, 2:] = True                                     # rows 4 .. are positions 36 ..; heads 2, 3 read kv head 1
    assert np.array_equal(np.isnan(got), seen)


# Batches that fill the chip with tiles of 256 rows (rows x group / 256 per kv head, times
# the thousands of keys, at least 256 / kv_heads), so the second kernel makes them.
LARGE = [
    ([300], [300], 256, 256, 64, 16, F16, F16, {}),
    ([293, 1, 3], [500, 700, 3], 256, 128, 128, 48, BF16, BF16, {"lead": 1, "spare": 4}),
    ([256, 0, 70], [256, 0, 70], 256, 64, 72, 16, F16, F32, {}),
    ([270, 5], [333, 400], 256, 64, 80, 7, BF16, F32, {"drop": {(0, 1): -1, (0, 40): 1 << 30, (1, 0): -5}}),
    ([290], [290], 256, 128, 96, 64, F16, F16, {"width": 4}),                # rows past the page table
    ([260, 16], [200, 16], 256, 256, 8, 16, F16, F16, {}),                   # rows before position 0
    ([257] * 2 + [1] * 66, [257, 300] + list(range(66)), 256, 256, 32, 32, F16, F16, {}),   # more sequences than lanes
    ([512, 1], [4200, 9000], 32, 32, 64, 16, F16, F16, {}),                  # splits
    ([260], [5000], 64, 64, 128, 1, BF16, BF16, {}),                         # splits of more keys than LDS holds slots for
    ([257], [4097], 64, 64, 48, 100, F16, F32, {}),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_attention_of_many_rows(dev, case):
    news, lens, heads, kv_heads, D, page, cd, od, opt = LARGE[case]
    say("many rows", case, news[:4], lens[:4], *LARGE[case][2:])
    batch = Batch(np.random.default_rng(400 + case), news, lens, page, **opt)
    check_attention(dev, batch, heads, kv_heads, D, cd, od, 500 + case)


def test_attention_single_rows_of_many_heads(dev):
    """one row of 256 heads per sequence: a tile of 256 rows each, in tables that could hold a lot"""
    batch = Batch(np.random.default_rng(23), [1] * 3, [700, 0, 2100], 64, ragged=False, width=2048)
    check_attention(dev, batch, 512, 2, 64, F16, F16, 24)


@pytest.mark.parametrize("ragged", [False, True])
def test_attention_of_more_sequences_than_lanes(dev, ragged):
    lens = [(37 * i) % 90 for i in range(150)]
    lens[149] = 2500
    batch = Batch(np.random.default_rng(25), [1] * 150, lens, 16, ragged=ragged)
    check_attention(dev, batch, 8, 2, 64, F16, F32, 26)


def test_attention_short_rows_in_long_tables(dev):
    """tables that could hold a million positions, of which few are held"""
    batch = Batch(np.random.default_rng(17), [300, 1, 40], [300, 77, 40], 64, width=16384)
    check_attention(dev, batch, 4, 2, 64, F16, F16, 18)


@pytest.mark.parametrize("news,lens,heads,kv_heads,D,cd,od,key", [
    ([40], [100], 4, 2, 64, F16, F16, 83), ([40], [40], 2, 2, 128, BF16, F32, 17), ([33], [33], 3, 3, 72, F16, F32, 32),
    ([300], [300], 256, 256, 64, F16, F16, 200), ([256], [600], 256, 128, 128, BF16, BF16, 500)])
def test_attention_hidden_values_may_be_anything(dev, news, lens, heads, kv_heads, D, cd, od, key):
    """infinite and NaN values of a new position reach the rows that see it and no row before"""
    say("not finite at", key, news, lens, heads, kv_heads, D)
    rng = np.random.default_rng(19)
    batch = Batch(rng, news, lens, 16)
    K, V = filled_cache(rng, batch, kv_heads, D, cd)
    q = values(rng, (batch.rows, heads, D), cd)
    inf, nan = (0x7C00, 0x7E00) if cd == F16 else (0x7F80, 0x7FC0)
    page, slot = batch.place(0, key)
    V[page, :, slot, 1], V[page, :, slot, D - 1], V[page, 0, slot, 5] = inf, nan, inf | 0x8000
    got = run_attention(dev, batch, q, K, V, cd, od, heads)
    clean = V.copy()
    clean[page, :, slot, 1] = clean[page, :, slot, D - 1] = clean[page, 0, slot, 5] = 0
    ref, tol = attention(batch, q, K, clean, cd, D ** -0.5, 1 if od != F32 else 2)
    sees = np.arange(news[0]) >= key - (lens[0] - news[0])
    group = heads // kv_heads
    bad = np.zeros(got.shape, bool)
    bad[np.ix_(sees, np.arange(heads), [1, D - 1])] = True
    bad[np.ix_(sees, np.arange(group), [5])] = True
    assert np.all(np.isnan(got[sees][:, :, D - 1]))
    if od != F32:
        assert np.all(got[sees][:, :, 1] == np.inf) and np.all(got[sees][:, :group, 5] == -np.inf)
    else:
        # p = hi + lo (+ lower) with lo = p - round(p), which is 0 or negative as often as positive: p inf is
        # hi inf + lo inf, so inf + 0 inf = NaN or inf - inf = NaN, or inf
        assert not np.any(np.isfinite(got[sees][:, :, 1])) and not np.any(np.isfinite(got[sees][:, :group, 5]))
        assert not np.any(got[sees][:, :, 1] == -np.inf) and not np.any(got[sees][:, :group, 5] == np.inf)
    got[bad] = ref[bad] = 0.0
    assert same_or_close(got, ref, tol, od) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,rows,seqs", [(4, 2, 64, 200), (64, 64, 300, 80)])
def test_starts_that_decrease_leave_no_trace(dev, heads, kv_heads, rows, seqs):
    """a row_start that goes back and forth asks for more work than any batch of these rows; whatever it
    leaves undone, the calls after it, whose split keys are counted in the same words, are right"""
    say("decreasing starts", heads, kv_heads, rows, seqs)
    rng = np.random.default_rng(37)
    good = Batch(rng, [rows], [3000], 16)
    K, V = filled_cache(rng, good, kv_heads, 64, F16)
    bits = values(rng, (rows, heads, 64), F16)
    q, cache, b = dev.upload(bits), cache_on(dev, good, K, V, F16), good.device(dev)
    start = np.array([0, rows] * (seqs // 2 + 1), np.int32)[:seqs + 1]
    wild = m.PagedBatch(seqs, rows, dev.upload(np.full(seqs, 3000, np.int32)), dev.upload(np.repeat(good.table, seqs, 0)),
                        good.width, row_start=dev.upload(start))
    qkv = dev.upload(np.zeros((rows, (heads + 2 * kv_heads) * 64), np.float32))
    outs = [dev.alloc(rows * heads * 64 * 2) for _ in range(3)]
    for o in outs:
        dev.attention_paged(q, b, cache, o, F16, heads)
        dev.attention_paged(q, wild, cache, dev.alloc(o.nbytes), F16, heads)
        dev.kv_append_paged(qkv, F32, (heads + 2 * kv_heads) * 64, wild, cache_on(dev, good, K, V, F16), heads, dev.alloc(o.nbytes), None)
    ref, tol = attention(good, bits, K, V, F16, 64 ** -0.5, 1)
    first = outs[0].download(np.uint16)
    assert same_or_close(from_bits(first.reshape(ref.shape), F16), ref, tol, F16) <= 1.0
    assert all(np.array_equal(o.download(np.uint16), first) for o in outs)


# ---- plans ------------------------------------------------------------------------------

def test_plan_replays_as_lengths_grow(dev):
    """one captured graph appends and attends step after step: lengths and inputs change in device memory,
    with eager work between the replays; every step against the definitions"""
    rng = np.random.default_rng(21)
    heads, kv_heads, D, page, S, steps = 4, 2, 64, 8, 3, 5
    lens = np.array([0, 14, 700], np.int32)
    batch = Batch(rng, [1] * S, lens + steps, page, ragged=False)
    for s in range(S):
        batch.lens[s] = int(lens[s])
    K, V = filled_cache(rng, batch, kv_heads, D, F16)
    cache = cache_on(dev, batch, K, V, F16)
    width = (heads + 2 * kv_heads) * D
    table = rope_table(1000, 32)
    x, q, o = dev.alloc(S * width * 4), dev.alloc(S * heads * D * 2), dev.alloc(S * heads * D * 4)
    b = batch.device(dev)
    plan = m.Plan(dev)
    plan.add_kv_append_paged(x, F32, width, b, cache, heads, q, m.Rope(dev.upload(table), 1000, 32))
    plan.add_attention_paged(q, b, cache, o, F32, heads)
    assert len(plan) == 2
    plan.use_graph(True)
    for step in range(steps):
        lens = lens + 1
        batch.lens = [int(v) for v in lens]
        xs = rng.standard_normal((S, width)).astype(np.float32)
        x.upload(xs)
        b.buffers[0].upload(lens)
        plan.run()
        got = o.download(np.float32).reshape(S, heads, D).astype(np.float64)
        gq = q.download(np.uint16).reshape(S, heads, D)
        gK, gV = (c.download(np.uint16).reshape(K.shape) for c in cache.buffers)
        ref, qt, rK, rV, Kt = append_reference(batch, xs.astype(np.float64), heads, kv_heads, D, F16, table, 32, False, K, V)
        assert same_or_close(from_bits(gq, F16), ref, qt, F16) <= 1.0
        assert same_or_close(from_bits(gK, F16), rK, Kt, F16) <= 1.0
        assert same_or_close(from_bits(gV, F16), rV, np.zeros(V.shape), F16) <= 1.0
        ref, tol = attention(batch, gq, gK, gV, F16, D ** -0.5, 2)
        assert same_or_close(got, ref, tol, F32) <= 1.0
        eager = dev.alloc(o.nbytes)
        dev.attention_paged(q, b, cache, eager, F32, heads)
        assert np.array_equal(eager.download(np.uint32), o.download(np.uint32))
        K, V = gK, gV
    ms = plan.profile()
    assert len(ms) == 2 and np.all(ms > 0)


def test_graphs_of_one_device_share_workspaces(dev):
    """two captured graphs, both with split attention, replayed in turn with eager calls between"""
    rng = np.random.default_rng(31)
    jobs = []
    for news, lens, heads, kv_heads, ragged in (([1] * 3, [3000, 20, 1500], 8, 2, False), ([512, 1], [4200, 600], 32, 32, True)):
        batch = Batch(rng, news, lens, 16, ragged=ragged)
        K, V = filled_cache(rng, batch, kv_heads, 64, F16)
        q = dev.upload(values(rng, (batch.rows, heads, 64), F16))
        cache, b = cache_on(dev, batch, K, V, F16), batch.device(dev)
        o, eager = (dev.alloc(batch.rows * heads * 64 * 4).zero() for _ in range(2))
        dev.attention_paged(q, b, cache, eager, F32, heads)
        plan = m.Plan(dev)
        plan.add_attention_paged(q, b, cache, o, F32, heads)
        plan.use_graph(True)
        jobs.append((plan, o, eager.download(np.uint32), (q, b, cache, eager, heads)))
    for turn in range(3):
        for plan, o, _, _ in jobs:
            o.zero()
            plan.run(2)
        for plan, o, first, (q, b, cache, eager, heads) in jobs:
            dev.attention_paged(q, b, cache, eager, F32, heads)
            assert np.array_equal(o.download(np.uint32), first)
            assert np.array_equal(eager.download(np.uint32), first)


def test_two_handles_at_once(dev):
    """two device handles have streams, workspaces and counters of their own"""
    other = m.Device(0)
    rng = np.random.default_rng(33)
    work = []
    for d in (dev, other):
        batch = Batch(rng, [1] * 4, [2500, 900, 3100, 40], 16, ragged=False)
        K, V = filled_cache(rng, batch, 4, 64, F16)
        q = d.upload(values(rng, (4, 8, 64), F16))
        work.append((d, q, batch.device(d), cache_on(d, batch, K, V, F16), [d.alloc(4 * 8 * 64 * 4) for _ in range(20)]))
    for i in range(20):
        for d, q, b, cache, outs in work:
            d.attention_paged(q, b, cache, outs[i], F32, 8)
    for d, q, b, cache, outs in work:
        first = outs[0].download(np.uint32)
        assert all(np.array_equal(o.download(np.uint32), first) for o in outs)
    del work, d, q, b, cache, outs
    other.close()


def test_a_step_of_a_batch(dev, orc):
    """the operators together, as one graph: quantized QKV products, append, attention, dense product with
    residual, LM head, logits, pick; the tokens' histories and lengths move on between the replays"""
    rng = np.random.default_rng(35)
    S, heads, D, vocab, page, steps = 5, 4, 64, 1000, 16, 4
    hidden = heads * D
    W = {n: dev.random_weight(m.Q8_0, rows, hidden, 71 + i, 0.05) for i, (n, rows) in
         enumerate((("qkv", 3 * hidden), ("dense", hidden), ("head", vocab)))}
    deq = {n: w.dequant().astype(np.float64) for n, w in W.items()}
    lens = np.array([0, 3, 15, 40, 100], np.int32)
    batch = Batch(rng, [1] * S, lens + steps, page, ragged=False)
    batch.lens = [int(v) for v in lens]
    K, V = filled_cache(rng, batch, heads, D, F16)
    cache = cache_on(dev, batch, K, V, F16)
    b = batch.device(dev)
    x, qkv, o, y, logits, out = (dev.alloc(S * n * 4) for n in (hidden, 3 * hidden, hidden, hidden, vocab, vocab))
    q, token = dev.alloc(S * hidden * 2), dev.alloc(S * 4)
    history, hlen = dev.alloc(S * steps * 4).zero(), dev.alloc(S * 4).zero()
    pen = np.tile(np.array([[1.3, 0.4, 0.2]], np.float32), (S, 1))
    controls = m.LogitControls(history=history, history_len=hlen, history_width=steps, penalties=dev.upload(pen))
    table = rope_table(200, D)
    plan = m.Plan(dev)
    plan.add_gemm_quant_grouped(S, [(x, F32, W["qkv"], qkv, F32)])
    plan.add_kv_append_paged(qkv, F32, 3 * hidden, b, cache, heads, q, m.Rope(dev.upload(table), 200, D))
    plan.add_attention_paged(q, b, cache, o, F32, heads)
    plan.add_gemm_quant_grouped(S, [(o, F32, W["dense"], y, F32)], epilogues=[{"residual": x}])
    plan.add_gemv(y, F32, W["head"], logits, F32, S)
    plan.add_logits_process(logits, F32, S, vocab, vocab, controls, out)
    plan.add_argmax(out, F32, S, vocab, vocab, token)
    plan.use_graph(True)
    seen = np.zeros((S, steps), np.int32)
    for step in range(steps):
        lens = lens + 1
        batch.lens = [int(v) for v in lens]
        b.buffers[0].upload(lens)
        xs = rng.standard_normal((S, hidden)).astype(np.float32)
        x.upload(xs)
        history.upload(seen)
        hlen.upload(np.full(S, step, np.int32))
        plan.run()
        # each stage against its definition on the values that the stage before it stored
        got = {n: buf.download(np.float32).reshape(S, -1).astype(np.float64) for n, buf in
               (("qkv", qkv), ("o", o), ("y", y), ("logits", logits), ("out", out))}
        ref, S_ = xs.astype(np.float64) @ deq["qkv"].T, np.abs(xs.astype(np.float64)) @ np.abs(deq["qkv"]).T
        assert np.all(np.abs(got["qkv"] - ref) <= 1e-5 * S_)
        gq = q.download(np.uint16).reshape(S, heads, D)
        gK, gV = (c.download(np.uint16).reshape(K.shape) for c in cache.buffers)
        ref, qt, rK, rV, Kt = append_reference(batch, got["qkv"], heads, heads, D, F16, table, D, False, K, V)
        assert same_or_close(from_bits(gq, F16), ref, qt, F16) <= 1.0
        assert same_or_close(from_bits(gK, F16), rK, Kt, F16) <= 1.0
        assert same_or_close(from_bits(gV, F16), rV, np.zeros(V.shape), F16) <= 1.0
        K, V = gK, gV
        ref, tol = attention(batch, gq, gK, gV, F16, D ** -0.5, 2)
        assert same_or_close(got["o"].reshape(S, heads, D), ref, tol, F32) <= 1.0
        ref, S_ = got["o"] @ deq["dense"].T + xs, np.abs(got["o"]) @ np.abs(deq["dense"]).T + np.abs(xs)
        assert np.all(np.abs(got["y"] - ref) <= 1e-5 * S_)
        ref, S_ = got["y"] @ deq["head"].T, np.abs(got["y"]) @ np.abs(deq["head"]).T
        assert np.all(np.abs(got["logits"] - ref) <= 1e-5 * S_)
        ref = got["logits"].copy()
        for r in range(S):
            ids, times = np.unique(seen[r, :step], return_counts=True)
            z = ref[r, ids]
            ref[r, ids] = np.where(z > 0, z / np.float64(pen[0, 0]), z * np.float64(pen[0, 0])) - (times * np.float64(pen[0, 1]) + np.float64(pen[0, 2]))
        assert np.all(np.abs(got["out"] - ref) <= 4 * 2.0 ** -24 * (np.abs(ref) + 3.0))
        picked = token.download(np.int32)
        assert np.array_equal(picked, np.argmax(got["out"], 1))
        seen[:, step] = picked
