"""What values of the cache may be, and how small a probability may get, in mvlm_attention_paged on the GPU, against
the definitions in 64 bits (paged_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import Batch, attention, filled_cache, values
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
