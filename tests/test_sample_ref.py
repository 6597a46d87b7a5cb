"""The places that the draw's reference allows, against a count token by token in exact fractions."""
import math
from fractions import Fraction

import numpy as np
import pytest

from sample_ref import Places, bits_of


def token(x, T, top_k, top_p, min_p, u):
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    w = [math.exp((x[i] - x[order[0]]) / T) for i in order]
    w = [round(z * 2 ** bits_of(len(x))) for z in w if z >= min_p]
    w = [z for z in w if z > 0]
    if top_k > 0:
        w = w[:top_k]
    for part, over in ((top_p, False), (u, True)):
        if part >= 1:
            if over:
                return order[len(w) - 1]
            continue
        need, run = Fraction(part) * sum(w), 0
        for i, z in enumerate(w):
            run += z
            if run > need or (not over and run >= need):
                break
        if over:
            return order[i]
        w = w[:i + 1]


@pytest.mark.parametrize("seed", range(60))
def test_places(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.choice([1, 2, 7, 60, 700]))
    x = (rng.choice([0.1, 3.0, 20.0]) * rng.standard_normal(n)).astype(np.float32).astype(np.float64)
    if seed % 3 == 0:
        x = np.round(x)
    T, top_k = float(rng.choice([0.3, 1.0, 1.7])), int(rng.choice([0, 1, 5, 50, 5000]))
    top_p, min_p = float(np.float32(rng.choice([1.0, 0.5, 0.95, 1e-6]))), float(np.float32(rng.choice([0.0, 0.01, 0.3])))
    u = float(rng.choice([0.0, 1.0, np.float32(rng.random()), np.float32(rng.random()), 1 - 2.0 ** -24]))
    p = Places(x, T, top_k, top_p, min_p, u)
    assert p.allows(token(x, T, top_k, top_p, min_p, u))
    assert p.lo <= p.hi <= p.last


def test_places_are_few():
    """ordinary rows leave one place, or two"""
    rng = np.random.default_rng(1)
    found = [Places((3 * rng.standard_normal(20000)).astype(np.float32), 0.9, k, p, q, float(np.float32(rng.random())))
             for k in (0, 50, 5000) for p in (1.0, 0.9) for q in (0.0, 1e-7, 0.05) for _ in range(3)]
    assert all(f.hi - f.lo <= 1 for f in found) and sum(f.hi > f.lo for f in found) <= 1


def test_places_of_rows_that_are_not_finite():
    inf = np.inf
    assert Places([-inf] * 3, u=0.9).allows(0) and not Places([-inf] * 3, u=0.9).allows(1)
    assert Places([1, inf, 2, np.nan, inf], u=0.99).allows(4)
    assert Places([3, 5, 5], T=0.0, u=0.9).allows(1) and not Places([3, 5, 5], T=0.0, u=0.9).allows(2)
    # what rounds to nothing does not live: of 8 tokens 51 bits
    x = [0.0] + [-52.1 * math.log(2)] * 7
    assert Places(x, u=1.0).last == 0 and Places(np.array(x) * 51.4 / 52.1, u=1.0).last == 7
