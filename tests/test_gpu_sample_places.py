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
