"""What values of the cache may be, and how small a probability may get, in mvlm_attention_paged on the GPU, against
the definitions in 64 bits (paged_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import HALF_STEP, Batch, attention, cache_on, close, filled_cache, to_bits, values
from test_gpu_paged import run_attention, same_or_close, say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = m.F32, m.F16, m.BF16


@pytest.mark.parametrize("news,lens,heads,kv_heads,D,cd,od,keys", [
    # with 32 heads and more over a kv head, all the rows of a wave may belong to one token
    ([256], [8192], 32, 1, 64, F16, F16, (7936 + 5, 7936 + 133)),
    ([256], [7300], 40, 1, 64, F16, F32, (7044 + 3, 7044 + 250)),
    ([300, 1], [4200, 900], 64, 2, 128, BF16, BF16, (3900 + 1, 3900 + 150)),
    ([300], [4200], 64, 2, 128, BF16, F32, (3900 + 2,)),
    # the same in tiles of 32 rows
    ([40], [200], 32, 1, 64, F16, F16, (163, 170)),
    ([20, 1], [100, 9], 40, 1, 128, BF16, F32, (83, 99))])
def test_not_finite_values_of_later_tokens_reach_no_row_before(dev, news, lens, heads, kv_heads, D, cd, od, keys):
    say("not finite at", keys, news, lens, heads, kv_heads, D)
    rng = np.random.default_rng(41)
    batch = Batch(rng, news, lens, 16)
    K, V = filled_cache(rng, batch, kv_heads, D, cd)
    q = values(rng, (batch.rows, heads, D), cd)
    inf, nan = (0x7C00, 0x7E00) if cd == F16 else (0x7F80, 0x7FC0)
    clean = V.copy()
    bad = np.zeros((batch.rows, heads, D), bool)
    position = lens[0] - news[0] + np.arange(news[0])
    for key in keys:
        page, slot = batch.place(0, key)
        V[page, :, slot, 1], V[page, :, slot, D - 1] = inf, nan
        clean[page, :, slot, 1] = clean[page, :, slot, D - 1] = 0
        bad[np.ix_(np.nonzero(position >= key)[0], np.arange(heads), [1, D - 1])] = True
    got = run_attention(dev, batch, q, K, V, cd, od, heads)
    assert np.array_equal(np.isfinite(got), ~bad)
    ref, tol = attention(batch, q, K, clean, cd, D ** -0.5, 1 if od != F32 else 2)
    got[bad] = ref[bad] = 0.0
    assert same_or_close(got, ref, tol, od) <= 1.0


@pytest.mark.parametrize("gap", [14, 18, 21])
@pytest.mark.parametrize("news,lens,heads,kv_heads,D,cd,od,opt", [
    ([1], [1000], 4, 2, 64, F16, F32, {"ragged": False}),
    ([1, 1], [5000, 700], 4, 2, 128, F16, F32, {"ragged": False}),                  # splits
    ([1], [1000], 32, 32, 64, F16, F16, {"ragged": False}),
    ([1] * 3, [600, 1, 900], 8, 2, 96, BF16, F32, {"ragged": False}),
    ([1] * 3, [600, 1, 900], 8, 2, 32, BF16, BF16, {"ragged": False}),
    ([40], [900], 4, 2, 64, F16, F32, {}),
    ([40, 1], [700, 950], 4, 4, 128, F16, F32, {}),
    ([33], [900], 6, 2, 80, F16, F16, {}),
    ([256], [600], 256, 256, 64, F16, F32, {}),
    ([256, 3], [500, 400], 256, 256, 64, F16, F16, {}),
    ([300], [500], 256, 128, 128, F16, F32, {}),
    ([300], [1100], 128, 64, 96, F16, F32, {}),
    ([256], [400], 256, 256, 32, F16, F32, {})])
def test_keys_far_below_the_largest(dev, news, lens, heads, kv_heads, D, cd, od, opt, gap):
    """Every 32nd key scores `gap` nats above the others and has values of zero, so that all of O comes from
    probabilities of exp(-gap).  Scores are exact (one product each), so with A as in paged_ref.attention what is
    rounded moves O by at most
      u_P A                   P in the cache's type, where O has it; in parts 2^-22
      F                       fp16: a part is a multiple of 2^-24 of a scale on which the row's largest is at least
                              2^12: 2^-37 a key, with the second part rounded 2^11 times as large 2^-48
      8 (1 + gap) 2^-23 A     the exponent's argument and the exponential, in numerator and denominator
      2 (N + 64) 2^-24 A      sums over N keys and the merge of their parts
    and the store by half a step."""
    say("far below", gap, news, lens, heads, kv_heads, D, cd, od)
    rng = np.random.default_rng(43)
    batch = Batch(rng, news, lens, 16, **opt)
    K, V = (np.zeros((batch.pages, kv_heads, 16, D), np.uint16) for _ in range(2))
    q = np.zeros((batch.rows, heads, D), np.float32)
    q[..., 0] = 8.0
    ref, tol = np.zeros(q.shape), np.zeros(q.shape)
    u_p = 2.0 ** -22 if od == F32 else HALF_STEP[cd]
    f = 0.0 if cd == BF16 else 2.0 ** -48 if od == F32 else 2.0 ** -37
    for s, (n, L) in enumerate(zip(news, lens)):
        at = np.array([batch.place(s, t) for t in range(L)])
        sink = np.arange(L) % 32 == 0
        v = rng.integers(1, 4, (L, kv_heads, D)) * 8192.0 * ~sink[:, None, None]
        K[at[:, 0], :, at[:, 1], 0] = to_bits(sink * float(gap), cd)[:, None]
        V[at[:, 0], :, at[:, 1]] = to_bits(v, cd)
        seen = np.arange(L - n, L)
        total = (np.cumsum(sink) + np.exp(-float(gap)) * np.cumsum(~sink))[seen]
        values_sum = np.repeat(np.cumsum(v, 0)[seen], heads // kv_heads, 1)
        A = np.exp(-float(gap)) * values_sum / total[:, None, None]
        r = slice(int(batch.start[s]), int(batch.start[s]) + n)
        ref[r] = A
        tol[r] = (u_p + 8 * (1 + gap) * 2.0 ** -23 + 2 * (L + 64) * 2.0 ** -24) * A + f * values_sum / total[:, None, None]
    got = run_attention(dev, batch, to_bits(q, cd), K, V, cd, od, heads, 0.125)
    worst = close(got, ref, tol, od)
    say("worst", worst)
    assert worst <= 1.0


@pytest.mark.parametrize("news,lens,heads,kv_heads,D", [([768], [768], 32, 32, 64), ([256] + [1] * 11, [900] + [700] * 11, 32, 32, 64),
                                                        ([768], [768], 32, 8, 128)])
def test_tables_with_room_choose_by_what_is_held(dev, news, lens, heads, kv_heads, D):
    """A table for 32768 positions of which few are held gives the values and, but for a launch that has
    nothing to do, the time of a table for just those: 20 calls in a graph, the two taken in turn, the best of 10.
    (Eight-wave blocks for what such tables hold took 1.4 to 1.9 times as long.)"""
    plans = []
    for width in (-(-max(lens) // 64), 512):
        rng = np.random.default_rng(45)
        batch = Batch(rng, news, lens, 64, width=width)
        K, V = filled_cache(rng, batch, kv_heads, D, F16)
        q, o = dev.upload(values(rng, (batch.rows, heads, D), F16)), dev.alloc(batch.rows * heads * D * 2)
        b, cache = batch.device(dev), cache_on(dev, batch, K, V, F16)
        plan = m.Plan(dev)
        for _ in range(20):
            plan.add_attention_paged(q, b, cache, o, F16, heads)
        plan.use_graph(True)
        plans.append((plan, o))
    best = [np.inf, np.inf]
    for _ in range(10):
        for i, (plan, _) in enumerate(plans):
            ev = plan.run(event=True)
            ev.wait()
            best[i] = min(best[i], ev.elapsed_ms() * 1000 / 20)
            ev.release()
    say("just wide enough, 32768 positions:", best, "us")
    outs = [o.download(np.uint16) for _, o in plans]
    assert np.array_equal(outs[0], outs[1])
    assert best[1] <= 1.25 * best[0] + 2.0


@pytest.mark.parametrize("lens,heads,kv_heads,D", [([2, 3, 5, 9, 40, 0, 1], 8, 8, 64), ([4, 6, 30, 700], 32, 4, 128),
                                                   ([1500, 7], 6, 2, 72)])
def test_bf16_single_tokens_round_once(dev, lens, heads, kv_heads, D):
    """A bf16 O of single tokens is its value in 64 bits rounded once, but for what fp32 arithmetic (the bound of
    paged_ref.attention) and probabilities of 16 bits (2^-17 each; values are positive, so 2^-17 O) move it by."""
    say("round once", lens, heads, kv_heads, D)
    rng = np.random.default_rng(47)
    batch = Batch(rng, [1] * len(lens), lens, 16, ragged=False)
    K, V = filled_cache(rng, batch, kv_heads, D, BF16)
    V &= np.uint16(0x7FFF)
    q = values(rng, (batch.rows, heads, D), BF16)
    got = run_attention(dev, batch, q, K, V, BF16, BF16, heads)
    ref, tol = attention(batch, q, K, V, BF16, D ** -0.5, 2)
    half_step = 2.0 ** (np.floor(np.log2(np.maximum(ref + tol, 1e-30))) - 8)
    assert np.all(np.abs(got - ref) <= half_step + tol + 2.0 ** -17 * ref)
