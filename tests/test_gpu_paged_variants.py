"""Kernel variants of the operators over a paged cache that no other test launches: fp32 outputs of tiles of 256 rows
at the head_dims of each accumulator count, and large slices of logits off the 16-byte grid."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import Batch, attention, cache_on, filled_cache, from_bits, values
from test_gpu_logits import NP, Controls, check
from test_gpu_paged import check_attention, same_or_close, say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = m.F32, m.F16, m.BF16


@pytest.mark.parametrize("news,lens,heads,kv_heads,D,page,cd", [
    # enough full tiles of 256 rows, times their keys in units of 1024, for 256 CUs
    ([260], [260], 256, 256, 128, 16, F16),
    ([260, 3], [2500, 70], 128, 128, 128, 64, BF16),         # with splits
    ([257], [4200], 64, 64, 128, 48, F16),
    ([258], [258], 256, 256, 96, 16, BF16),
    ([290], [2300], 128, 128, 104, 7, F16),
    ([256, 1], [400, 33], 256, 256, 32, 16, BF16),
    ([256], [500], 256, 256, 24, 16, F16),
    ([256], [300], 256, 256, 64, 16, BF16)])
def test_attention_of_many_rows_fp32_out(dev, news, lens, heads, kv_heads, D, page, cd):
    say("many rows, fp32 O", news, lens, heads, kv_heads, D, page, cd)
    batch = Batch(np.random.default_rng(51), news, lens, page)
    check_attention(dev, batch, heads, kv_heads, D, cd, F32, 52)


@pytest.mark.parametrize("rows,n,dt,history,bias,mask,extra,offset", [
    (300, 8201, F32, 100, 4, True, 0, 0),                    # an odd vocabulary: two slices of 4096 and a rest per row
    (300, 8201, F16, 100, 4, True, 0, 0),
    (260, 8195, BF16, 50, 3, True, 2, 1),
    (64, 50257, F16, 700, 9, False, 0, 0),
    (48, 50257, F32, 0, 9, True, 3, 3)])
def test_logits_of_many_rows_off_the_grid(dev, rows, n, dt, history, bias, mask, extra, offset):
    say("logits", rows, n, dt, extra, offset)
    rng = np.random.default_rng(53)
    c = Controls(rng, rows, n, history, bias, mask)
    ld = n + extra
    flat = values(rng, offset + rows * ld, dt, 4.0)
    es = flat.itemsize
    x, out = dev.upload(flat), dev.upload(np.full_like(flat, 7))
    views = [b.view(offset * es, (rows * ld - extra) * es) for b in (x, out)]
    dev.logits_process(views[0], dt, rows, n, ld, c.device(dev), views[1])
    got = out.download(NP[dt])
    ref, tol = c.reference(from_bits(flat, dt)[offset:].reshape(rows, ld)[:, :n])
    check(from_bits(got[offset:].reshape(rows, ld)[:, :n], dt), ref, tol, dt)
    assert np.all(got[offset:].reshape(rows, ld)[:, n:] == 7) and np.all(got[:offset] == 7)
    assert np.array_equal(x.download(NP[dt]), flat)


def test_one_graph_crosses_from_few_keys_to_many_and_back(dev):
    """a graph captured for a table with room: as the lengths change, tiles of 32 rows, of 256, and of 256 with split
    keys make the batch; every replay against the definition and an eager call, with two graphs in turn"""
    rng = np.random.default_rng(55)
    heads, D, steps = 64, 64, ([300, 20], [5000, 33], [256, 1], [4200, 900], [6000, 7])
    jobs = []
    for od in (F16, F32):
        batch = Batch(rng, [256, 1], [6000, 900], 16, width=500)
        K, V = filled_cache(rng, batch, heads, D, F16)
        bits = values(rng, (batch.rows, heads, D), F16)
        q, cache, b = dev.upload(bits), cache_on(dev, batch, K, V, F16), batch.device(dev)
        o, eager = (dev.alloc(batch.rows * heads * D * 4) for _ in range(2))
        plan = m.Plan(dev)
        plan.add_attention_paged(q, b, cache, o, od, heads)
        plan.use_graph(True)
        jobs.append((plan, batch, bits, K, V, q, cache, b, o, eager, od))
    for lens in steps:
        for plan, batch, *_, b, o, _, _ in jobs:
            batch.lens = lens
            b.buffers[0].upload(np.asarray(lens, np.int32))
            o.zero()
        for plan, *_ in jobs:
            plan.run(2)
        for plan, batch, bits, K, V, q, cache, b, o, eager, od in jobs:
            dev.attention_paged(q, b, cache, eager, od, heads)
            got = o.download(NP[od])[:bits.size]
            assert np.array_equal(got.view(np.uint8), eager.download(NP[od])[:bits.size].view(np.uint8))
            ref, tol = attention(batch, bits, K, V, F16, D ** -0.5, 1 if od != F32 else 2)
            worst = same_or_close(from_bits(got, od).reshape(ref.shape), ref, tol, od)
            say("lengths", lens, "worst", worst)
            assert worst <= 1.0
    ms = jobs[0][0].profile()
    assert len(ms) == 1 and ms[0] > 0
