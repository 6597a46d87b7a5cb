"""mvlm_sample on the GPU against the places that its definition allows (sample_ref), one or two of a row."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import from_bits, values
from sample_ref import Places
from test_gpu_sample import draw

pytestmark = pytest.mark.gpu

F32, F16, BF16 = m.F32, m.F16, m.BF16


def check(dev, bits, dtype, u, rows=None, **kw):
    """the tokens drawn; rows: those that are looked at"""
    got = draw(dev, bits, dtype, u=u, **kw)
    for r in range(len(bits)) if rows is None else rows:
        f = {k: float(np.asarray(v, np.float32)[r]) for k, v in kw.items()}
        p = Places(from_bits(bits[r], dtype), **f | ({"top_k": int(kw["top_k"][r])} if "top_k" in kw else {}), u=float(np.float32(u[r])))
        assert p.allows(got[r]), (r, f, u[r], got[r], p.rank(got[r]), p.lo, p.hi)
        assert p.hi - p.lo <= 1 or p.order.size < 4
    return got


@pytest.mark.parametrize("rows,n,dt", [(1, 128000, F32), (3, 128000, F16), (5, 70000, F32), (100, 120000, F32)])
def test_candidates_of_several_blocks(dev, rows, n, dt):
    """rows that several blocks look through, whose candidates together are more than one wave draws from"""
    rng = np.random.default_rng(70)
    for std in (3.0, 0.5):
        x = values(rng, (rows, n), dt, std)
        for top_k in (130, 600, 1000):
            for more in ({}, {"top_p": np.full(rows, 0.95), "min_p": np.full(rows, 1e-3)}):
                check(dev, x, dt, rng.random(rows), range(min(rows, 8)), top_k=np.full(rows, top_k), **more)


@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("T", [1e-10, 1e-13, 1e-14, 1e-16])
def test_exponents_without_a_fraction(dev, rows, T):
    """v / T of 1e11 .. 1e17: their bins lie past 2^53, where not every integer is a double"""
    rng = np.random.default_rng(71)
    x = (3 * rng.standard_normal((rows, 30000))).astype(np.float32)
    x[:, 5::7] = x[:, :1].max() + 9                            # the largest, many times
    check(dev, x, F32, rng.random(rows), range(min(rows, 4)), T=np.full(rows, T))
    check(dev, x, F32, rng.random(rows), range(min(rows, 4)), T=np.full(rows, T), top_p=np.full(rows, 0.5))


@pytest.mark.parametrize("rows,n", [(4, 500), (3, 70000), (150, 70000)])
def test_infinite_temperatures_with_the_largest_min_p(dev, rows, n):
    """every finite value weighs 1, as much as min_p asks for"""
    rng = np.random.default_rng(72)
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    x[:, ::3] = -np.inf
    u, T, ones = rng.random(rows), np.full(rows, np.inf), np.ones(rows)
    for kw in ({}, {"top_k": np.full(rows, 40)}, {"top_p": np.full(rows, 0.25)}):
        check(dev, x, F32, u, range(min(rows, 3)), T=T, min_p=ones, **kw)


@pytest.mark.parametrize("rows,n,dt", [(2, 51200, F32), (16, 51200, F32), (3, 70001, F16), (150, 51200, F32)])
def test_one_as_random_number_picks_the_last_kept(dev, rows, n, dt):
    """many kept tokens whose weights are a unit or two, where a sum of roundings is not the rounding of a sum"""
    rng = np.random.default_rng(73)
    x = values(rng, (rows, n), dt, 3.0)
    looked = range(min(rows, 6))
    for T in (0.2, 0.3, 0.4):
        for kw in ({}, {"top_k": rng.integers(1001, 8000, rows)}, {"top_p": np.full(rows, 1 - 2.0 ** -24)},
                   {"top_k": rng.integers(3000, 8000, rows), "top_p": np.full(rows, 0.999)}):
            for u in (np.ones(rows), np.full(rows, 1 - 2.0 ** -24), np.zeros(rows)):
                check(dev, x, dt, u, looked, T=np.full(rows, T), **kw)


@pytest.mark.parametrize("n,dt", [(51200, F32), (70001, F16), (128000, BF16)])
def test_a_row_alone_and_in_a_batch(dev, n, dt):
    """a row's token depends on the row and its settings, not on the rows beside it, whose number says how many blocks make it"""
    rng = np.random.default_rng(74)
    x = values(rng, (3, n), dt, 3.0)
    for kw in ({}, {"T": 0.25}, {"T": 0.4}, {"T": 0.3, "top_k": 5000}, {"top_p": 0.9}, {"T": 0.2, "top_p": 1 - 2.0 ** -24}, {"T": 0.4, "top_k": 20000, "top_p": 0.999},
               {"top_k": 300}, {"min_p": 1e-3}):
        for u in (rng.random(3), np.ones(3), np.full(3, 1 - 2.0 ** -24)):
            got = [draw(dev, np.tile(x, (b, 1))[:max(3 * b, 1)], dt, u=np.tile(u, b), **{k: np.full(3 * b, v) for k, v in kw.items()})
                   for b in (1, 8, 50)]
            alone = [draw(dev, x[r:r + 1], dt, u=u[r:r + 1], **{k: np.full(1, v) for k, v in kw.items()})[0] for r in range(3)]
            assert all(np.array_equal(np.tile(alone, len(g) // 3), g) for g in got), (kw, u, alone, [g[:3] for g in got])


@pytest.mark.parametrize("rows,n,dt,std", [(3, 128000, F32, 3.0), (3, 128000, F16, 3.0), (130, 60000, F32, 2.0), (140, 9001, BF16, 2.0), (2, 300000, F32, 1.0)])
def test_more_live_tokens_than_candidates(dev, rows, n, dt, std):
    """a min_p that leaves more tokens than LDS has room for, and rows without any limit"""
    rng = np.random.default_rng(75)
    x = values(rng, (rows, n), dt, std)
    for T in (0.9, 1.6):
        for kw in ({}, {"min_p": np.full(rows, 1e-7)}, {"min_p": np.full(rows, 1e-7), "top_p": np.full(rows, 0.95)},
                   {"min_p": np.full(rows, 1e-5), "top_k": np.full(rows, 30000)}, {"min_p": np.full(rows, 1e-5), "top_k": np.full(rows, 900)}):
            for u in (rng.random(rows), np.ones(rows)):
                check(dev, x, dt, u, range(min(rows, 6)), T=np.full(rows, T), **kw)


@pytest.mark.parametrize("rows,n,top_k", [(1, 1 << 24, 50), (2, 1 << 22, 900)])
def test_candidates_of_too_many_blocks(dev, rows, n, top_k):
    """each block has few candidates, all of them together are more than one holds"""
    rng = np.random.default_rng(76)
    x = (3 * rng.standard_normal((rows, n), dtype=np.float32))
    check(dev, x, F32, rng.random(rows), top_k=np.full(rows, top_k), top_p=np.full(rows, 0.95))
