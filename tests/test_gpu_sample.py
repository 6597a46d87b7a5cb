"""mvlm_sample on the GPU against its definition in 64 bits, through the C ABI."""
from __future__ import annotations

import math

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import from_bits, to_bits, values

pytestmark = pytest.mark.gpu

F32, F16, BF16 = m.F32, m.F16, m.BF16


def pick(x, T, top_k, top_p, min_p, u):
    """The token, and how near (in parts of the sum) a random number or a top_p came to another outcome."""
    v = np.where(np.isnan(x), np.where(np.signbit(x), -np.inf, np.inf), x)
    order = np.argsort(-v, kind="stable")
    if v[order[0]] == -np.inf:
        return 0, 1.0
    if not T > 0:
        return int(order[0]), 1.0
    top = v[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(v[order] == top, 1.0, np.exp((v[order] - top) / T))
    w = np.where(v[order] == -np.inf, 0.0, w)
    # rounded as the interface says
    bits = min(51, 62 - max(0, math.ceil(math.log2(len(x)))))
    near = 1.0
    if min_p > 0:
        near = min(near, float(np.min(np.abs(w - min(min_p, 1.0))[w < 1.0], initial=1.0)))
        w = w[w >= min(min_p, 1.0)]
    if top_k > 0:
        w = w[:top_k]
    w = np.round(w * 2.0 ** bits)
    sums = np.cumsum([int(z) for z in w], dtype=object)
    if top_p < 1:
        need = max(float(top_p), 0.0) * float(sums[-1])
        near = min(near, min(abs(float(z) - need) for z in sums) / float(sums[-1]) if top_p > 0 else 1.0)
        end = next((i for i, z in enumerate(sums) if float(z) >= need), len(sums) - 1)
        sums = sums[:end + 1]
    u = 0.0 if not u > 0 else u
    if u >= 1:
        return int(order[next(i for i, z in enumerate(sums) if z == sums[-1])]), near
    need = u * float(sums[-1])
    if u > 0:
        near = min(near, min(abs(float(z) - need) for z in sums) / float(sums[-1]))
    return int(order[next(i for i, z in enumerate(sums) if float(z) > need)]), near


def slack(n):
    """How near an outcome may be for another to be right as well, in parts of the sum.  A token's weight is rounded by
    half of 2^-bits at most here and there, those of a slice's bin together once more, and what rounds to 0 may have
    been counted: 2 n 2^-bits in all.  Exponents v log2(e) / T of up to 1024 in 64 bits are off by 2^-43 twice, the
    series, the unit and the products by less: 2^-41 of a weight and of a sum."""
    return 2.0 * n * 2.0 ** -min(51, 62 - max(0, math.ceil(math.log2(n)))) + 2.0 ** -40


def draw(dev, x, dtype, T=None, top_k=None, top_p=None, min_p=None, u=None, ld=None, offset=0):
    rows, n = x.shape
    ld = ld or n
    flat = np.full(offset + rows * ld, to_bits(np.float32(1e4), dtype)[()] if dtype != F32 else np.float32(1e30))
    flat[offset:].reshape(rows, ld)[:, :n] = x
    es = flat.itemsize
    buf = dev.upload(flat)
    up = lambda a, t: None if a is None else dev.upload(np.asarray(a, t))  # noqa: E731
    s = m.Sampling(up(u, np.float32), temperature=up(T, np.float32), top_k=up(top_k, np.int32), top_p=up(top_p, np.float32),
                   min_p=up(min_p, np.float32))
    out = dev.upload(np.full(rows, -7, np.int32))
    view = buf.view(offset * es, (rows * ld - (ld - n)) * es)
    dev.sample(view, dtype, rows, n, ld, s, out)
    got = out.download(np.int32)
    dev.sample(view, dtype, rows, n, ld, s, out)                 # the same again
    assert np.array_equal(out.download(np.int32), got)
    assert np.array_equal(buf.download(flat.dtype).view(np.uint8), flat.view(np.uint8))
    return got


def check(dev, bits, dtype, T, top_k, top_p, min_p, u, **kw):
    rows, n = bits.shape
    got = draw(dev, bits, dtype, T, top_k, top_p, min_p, u, **kw)
    x = from_bits(bits, dtype)
    f = lambda a, r, none: none if a is None else float(np.float32(a[r]))  # noqa: E731
    for r in range(rows):
        want, near = pick(x[r], f(T, r, 1.0), int(f(top_k, r, 0)), f(top_p, r, 1.0), f(min_p, r, 0.0), f(u, r, 0.0))
        assert got[r] == want or near < slack(n), (r, got[r], want, near)


CASES = [
    # rows, n, dtype, std, top_k, top_p, min_p, extra columns, element offset
    (1, 1, F32, 1.0, 0, 1.0, 0.0, 0, 0),
    (4, 2, F16, 1.0, 0, 1.0, 0.0, 0, 0),
    (3, 33, BF16, 2.0, 5, 0.9, 0.0, 1, 3),
    (8, 1000, F32, 3.0, 0, 1.0, 0.0, 0, 0),
    (8, 1000, F32, 3.0, 40, 1.0, 0.0, 24, 0),
    (8, 1000, F16, 3.0, 0, 0.9, 0.0, 0, 0),
    (8, 1027, BF16, 3.0, 0, 1.0, 0.05, 5, 1),
    (5, 4096, F32, 3.0, 50, 0.8, 0.02, 0, 0),
    (5, 4097, F16, 0.5, 5000, 0.95, 0.001, 0, 0),
    (3, 51200, F32, 3.0, 50, 0.95, 0.0, 0, 0),
    (3, 51200, BF16, 3.0, 0, 0.9, 0.0, 0, 0),
    (3, 51203, F32, 3.0, 0, 1.0, 0.0, 1, 0),
    (3, 50000, F32, 1.0, 20000, 0.9, 0.0, 0, 0),            # more than the list holds, by count
    (3, 50000, F16, 0.1, 20000, 0.9, 0.0, 0, 0),            # many equal values
    (3, 50000, BF16, 0.01, 30000, 0.999, 0.5, 0, 0),
    (2, 128000, F32, 3.0, 1000, 0.95, 0.02, 0, 0),
    (300, 200, F32, 2.0, 7, 0.9, 0.01, 0, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_sample(dev, case):
    rows, n, dt, std, top_k, top_p, min_p, extra, offset = CASES[case]
    print("[sample]", case, CASES[case], flush=True)
    rng = np.random.default_rng(60 + case)
    for masked in (0.0, 0.6):
        x = values(rng, (rows, n), dt, std)
        if masked:
            x[rng.random((rows, n)) < masked] = to_bits(np.float32(-np.inf), dt)
        T = rng.uniform(0.4, 1.8, rows)
        if rows > 2:
            T[1] = 0.0
        check(dev, x, dt, T, rng.integers(top_k // 2, 2 * top_k + 1, rows) if top_k else None,
              np.full(rows, top_p) if top_p < 1 else None, np.full(rows, min_p) if min_p else None, rng.random(rows),
              ld=n + extra, offset=offset)


@pytest.mark.parametrize("case", range(6))
def test_sample_of_long_rows(dev, case):
    """rows of more tokens than a block holds, made by one block or by several, by all kinds of settings"""
    rows, n, dt, std = [(3, 128000, F32, 3.0), (3, 128000, F16, 3.0), (130, 60000, F32, 2.0), (140, 9001, BF16, 2.0),
                        (3, 120001, BF16, 0.3), (2, 300000, F32, 1.0)][case]
    print("[sample] long", rows, n, dt, flush=True)
    rng = np.random.default_rng(160 + case)
    x = values(rng, (rows, n), dt, std)
    few = min(rows, 12)                                      # rows that the reference looks at
    for kw in ({}, {"top_p": 0.9}, {"top_k": 50}, {"top_k": 1000}, {"top_k": 3000, "top_p": 0.8}, {"min_p": 0.05}, {"min_p": 1e-7, "top_p": 0.95},
               {"T": 0.0}, {"top_k": n - 5, "top_p": 0.99}):
        u = rng.random(rows)
        T = np.full(rows, kw.get("T", 0.9))
        args = [np.full(rows, kw[k]) if k in kw else None for k in ("top_k", "top_p", "min_p")]
        got = draw(dev, x, dt, T, *args, u)
        for r in range(few):
            f = [None if a is None else float(np.float32(a[r])) for a in args]
            want, near = pick(from_bits(x[r], dt), float(np.float32(T[r])), int(f[0] or 0), 1.0 if f[1] is None else f[1], f[2] or 0.0,
                              float(np.float32(u[r])))
            assert got[r] == want or near < slack(n), (kw, r, got[r], want, near)


@pytest.mark.parametrize("rows", [2, 150])
def test_sample_of_long_rows_that_are_not_ordinary(dev, rows):
    """infinities, NaN, values whose products with 1 / T leave no fraction, temperatures at their ends; one block and several"""
    n = 20000
    rng = np.random.default_rng(12)
    base = (2 * rng.standard_normal(n)).astype(np.float32)
    u = np.full(rows, 0.6, np.float32)
    def same(x, T=None, top_p=None):  # noqa: E306
        got = draw(dev, np.repeat(x[None], rows, 0), F32, None if T is None else np.full(rows, T), None,
                   None if top_p is None else np.full(rows, top_p), None, u)
        want, near = pick(x.astype(np.float64), 1.0 if T is None else float(np.float32(T)), 0, 1.0 if top_p is None else float(np.float32(top_p)), 0.0,
                          float(u[0]))
        assert near < slack(n) or np.all(got == want), (got[:3], want)
    x = base.copy()
    x[[5, 700, 19999]] = np.inf
    same(x)
    x = base.copy()
    x[[11, 12000]] = np.nan
    same(x, top_p=0.7)
    x = base.copy()
    x[3:9000] = np.copysign(np.float32(np.nan), np.float32(-1))
    same(x, top_p=0.7)
    x = np.full(n, -np.inf, np.float32)
    same(x)
    x[15000] = -7.0
    same(x)
    same(base * np.float32(1e30))
    same(base * np.float32(1e30), T=1e30)
    same(base + np.float32(3000.0))                          # 4300 octaves: 2^-43 of weights apart
    same(base, T=1e-30)
    same(base, T=1e-3, top_p=0.5)
    same(base, T=np.inf, top_p=0.5)
    same(np.abs(base) * np.float32(2.0 ** -140))             # subnormals


@pytest.mark.parametrize("rows,n", [(3, 128000), (100, 120000), (150, 70001)])
def test_sample_of_parts_that_differ(dev, rows, n):
    """few tokens kept of a row that more blocks than one look through: nothing in a part, all of them in one, ties across
    parts, more in a part than it may have, infinities"""
    rng = np.random.default_rng(30)
    base = (3 * rng.standard_normal(n)).astype(np.float32)
    rise = np.linspace(-20, 20, n).astype(np.float32)
    half = base.copy()
    half[:n // 2] = -np.inf
    one = np.full(n, -np.inf, np.float32)
    one[n - 3] = 1.0
    ties = np.round(base)
    inf = base.copy()
    inf[[17, n - 5]] = np.inf
    nan = base.copy()
    nan[[3, n - 2]] = np.nan
    flat = (1e-3 * base).astype(np.float32)                    # min_p keeps all of them
    for what, x in (("base", base), ("rise", rise), ("half", half), ("one", one), ("ties", ties), ("inf", inf), ("nan", nan), ("flat", flat),
                    ("none", np.full(n, -np.inf, np.float32))):
        for kw in ({"top_k": 1}, {"top_k": 50}, {"top_k": 1000}, {"top_k": 700, "min_p": 0.02, "top_p": 0.9}, {"min_p": 0.3}):
            args = [np.full(rows, kw[k]) if k in kw else None for k in ("top_k", "top_p", "min_p")]
            u = rng.random(rows)
            got = draw(dev, np.repeat(x[None], rows, 0), F32, np.full(rows, 0.8), *args, u)
            for r in range(2):
                f = [None if a is None else float(np.float32(a[r])) for a in args]
                want, near = pick(x.astype(np.float64), float(np.float32(0.8)), int(f[0] or 0), 1.0 if f[1] is None else f[1], f[2] or 0.0,
                                  float(np.float32(u[r])))
                assert got[r] == want or near < slack(n), (what, kw, r, got[r], want, near)


@pytest.mark.parametrize("rows", [3, 150])
@pytest.mark.parametrize("hidden", [-1e4, -3.4e38, -40.0, -30.0, -28.5])
def test_sample_of_rows_masked_by_finite_values(dev, rows, hidden):
    """most of a row at a value whose weight is nothing, or nearly: counted by top_k, picked by no number where it rounds to 0"""
    n, live = 40000, 300
    rng = np.random.default_rng(21)
    x = np.full((rows, n), hidden, np.float32)
    for r in range(rows):
        x[r, rng.choice(n, live, False)] = rng.standard_normal(live)
    few = 3
    for kw in ({}, {"top_k": 3000}, {"top_k": 200}, {"top_p": 1 - 2.0 ** -24}, {"top_k": 3000, "top_p": 0.9}, {"top_k": 39999, "top_p": 1 - 2.0 ** -24}):
        args = [np.full(rows, kw[k]) if k in kw else None for k in ("top_k", "top_p")]
        for u in (rng.random(rows), np.ones(rows), np.full(rows, 1 - 2.0 ** -24), np.zeros(rows)):
            got = draw(dev, x, F32, None, *args, None, u)
            for r in range(few):
                f = [None if a is None else float(np.float32(a[r])) for a in args]
                want, near = pick(x[r].astype(np.float64), 1.0, int(f[0] or 0), 1.0 if f[1] is None else f[1], 0.0, float(np.float32(u[r])))
                if (hidden - float(x[r].max())) * math.log2(math.e) < -47.001:   # 46 bits
                    assert x[r, got[r]] != np.float32(hidden)
                assert got[r] == want or near < slack(n), (kw, r, u[r], got[r], want, near)


def test_sample_of_weights_that_round_to_nothing(dev):
    """4194304 tokens: 40 bits.  One is at 0, the others' weights of 2^-41.5 each would make 2^-19.5 together"""
    n = 1 << 22
    x = np.full((2, n), -41.5 * math.log(2), np.float32)
    x[0, 777], x[1, n - 1] = 0.0, 0.0
    for kw in ({}, {"top_k": [5000] * 2}, {"top_p": [1 - 2.0 ** -24] * 2}):
        for u in (0.0, 0.5, 1 - 2.0 ** -24, 1.0):
            assert list(draw(dev, x, F32, u=[u] * 2, **kw)) == [777, n - 1], (kw, u)


@pytest.mark.parametrize("rows,n,dt", [(20, 70001, F32), (20, 120000, F16), (160, 3000, BF16), (160, 70000, F16)])
def test_sample_of_requests_of_all_kinds(dev, rows, n, dt):
    """one call whose rows ask for unlike things, with infinite, tiny and no temperatures, masks and NaN among them"""
    rng = np.random.default_rng(50)
    x = values(rng, (rows, n), dt, 3.0)
    x[rng.random((rows, n)) < 0.3] = to_bits(np.float32(-np.inf), dt)
    x[3, 11:12] = to_bits(np.float32(np.nan), dt)
    x[7, ::3] = to_bits(np.copysign(np.float32(np.nan), np.float32(-1)), dt)
    x[11, 1:] = to_bits(np.float32(-np.inf), dt)
    T = rng.choice([0.7, 1.0, 1.3, 0.0, np.inf, 1e-30, 1e-3], rows).astype(np.float32)
    top_k = rng.choice([0, 0, 1, 5, 50, 300, 1000, 5000], rows).astype(np.int32)
    top_p = rng.choice([1.0, 0.95, 0.5, 0.0], rows).astype(np.float32)
    min_p = rng.choice([0.0, 0.0, 0.01, 0.3, 1.0], rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    u[::9] = 1.0
    got = draw(dev, x, dt, T, top_k, top_p, min_p, u)
    for r in range(min(rows, 40)):
        want, near = pick(from_bits(x[r], dt), float(T[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]), float(u[r]))
        assert got[r] == want or near < slack(n), (r, T[r], top_k[r], top_p[r], min_p[r], u[r], got[r], want, near)


def test_sample_of_long_rows_in_a_graph(dev):
    """rows made by several blocks, whose parts are counted in the same words, replayed with eager calls between"""
    rng = np.random.default_rng(18)
    jobs = []
    for rows, n in ((3, 50000), (9, 30000)):
        x, out, eager = dev.alloc(rows * n * 4), dev.alloc(rows * 4), dev.alloc(rows * 4)
        u = dev.alloc(rows * 4)
        s = m.Sampling(u, top_p=dev.upload(np.full(rows, 0.9, np.float32)))
        plan = m.Plan(dev)
        plan.add_sample(x, F32, rows, n, n, s, out)
        plan.use_graph(True)
        jobs.append((rows, n, x, u, s, out, eager, plan))
    for _ in range(4):
        host = []
        for rows, n, x, u, s, out, eager, plan in jobs:
            host.append(((3 * rng.standard_normal((rows, n))).astype(np.float32), rng.random(rows).astype(np.float32)))
            x.upload(host[-1][0])
            u.upload(host[-1][1])
        for rows, n, x, u, s, out, eager, plan in jobs:
            plan.run(2)
        for (xs, us), (rows, n, x, u, s, out, eager, plan) in zip(host, jobs):
            dev.sample(x, F32, rows, n, n, s, eager)
            got = out.download(np.int32)
            assert np.array_equal(eager.download(np.int32), got)
            for r in range(rows):
                want, near = pick(xs[r].astype(np.float64), 1.0, 0, float(np.float32(0.9)), 0.0, float(us[r]))
                assert got[r] == want or near < slack(n)


@pytest.mark.parametrize("n", [1, 7, 5000, 40000])
def test_sample_of_equal_values(dev, n):
    """ties go to the lower index, also where there are more than any list holds"""
    x = np.zeros((6, n), np.float32)
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.999, 1.0])
    assert list(draw(dev, x, F32, u=u)) == [min(int(z * n), n - 1) for z in np.float32(u).astype(np.float64)]
    half = (n + 1) // 2
    got = draw(dev, x, F32, u=u, top_k=[half] * 6)
    assert list(got) == [min(int(z * half), half - 1) for z in np.float32(u).astype(np.float64)]
    got = draw(dev, x, F32, u=u, top_p=[0.5] * 6)
    assert list(got) == [min(int(z * half), half - 1) for z in np.float32(u).astype(np.float64)]
    x[:, n // 2] = -np.inf
    if n > 1:
        got = draw(dev, x, F32, u=u)
        order = np.delete(np.arange(n), n // 2)
        assert list(got) == [order[min(int(z * (n - 1)), n - 2)] for z in np.float32(u).astype(np.float64)]


def test_sample_of_values_that_are_not_finite(dev):
    inf, nan = np.inf, np.nan
    x = np.array([[-inf] * 5, [-inf, -inf, 3, -inf, -inf], [1, inf, 2, nan, inf], [nan, 1, 2, 3, 4], [-nan, 1, 1, -inf, 1],
                  [0.0, -0.0, 0.0, -1, -0.0], [1e38, -1e38, 3e38, 3e38, -3e38], [2.0 ** -149, 0, -2.0 ** -149, 0, 0]], np.float32)
    x[4, 0] = np.copysign(np.float32(nan), np.float32(-1))
    u = np.full(8, 0.99, np.float32)
    # [0, -0, 0, -1, -0]: 0.99 (4 + 1 / e) = 4.32 lies in the last of them, -1
    assert list(draw(dev, x, F32, u=u)) == [0, 2, 4, 0, 4, 3, 3, 2]
    assert list(draw(dev, x, F32, u=0 * u)) == [0, 2, 1, 0, 1, 0, 2, 0]
    assert list(draw(dev, x, F32, T=0 * u, u=u)) == [0, 2, 1, 0, 1, 0, 2, 0]


def test_sample_settings_at_their_ends(dev):
    rng = np.random.default_rng(9)
    x = (2 * rng.standard_normal((1, 300))).astype(np.float32)
    best = int(np.argmax(x))
    rows = lambda k: np.repeat(x, k, 0)  # noqa: E731
    # settings that leave one token, or that have no effect
    assert list(draw(dev, rows(4), F32, T=[0.0, -1.0, np.nan, 1e-30], u=[0.9] * 4)) == [best] * 4
    assert list(draw(dev, rows(3), F32, top_p=[0.0, -1.0, 1e-30], u=[0.9] * 3)) == [best] * 3
    assert list(draw(dev, rows(2), F32, min_p=[1.0, 7.0], u=[0.9] * 2)) == [best] * 2
    assert list(draw(dev, rows(1), F32, top_k=[1], u=[0.9])) == [best]
    u = [0.1, 0.5, 0.9]
    free = list(draw(dev, rows(3), F32, u=u))
    for kw in ({"T": [1.0] * 3}, {"top_k": [0, -5, 300]}, {"top_k": [2 ** 31 - 1] * 3}, {"top_p": [1.0, 2.0, np.nan]},
               {"min_p": [0.0, -1.0, np.nan]}, {"min_p": [1e-30] * 3}):
        assert list(draw(dev, rows(3), F32, u=u, **kw)) == free, kw
    # random numbers outside [0, 1)
    order = np.argsort(-x[0], kind="stable")
    assert list(draw(dev, rows(5), F32, u=[-1.0, np.nan, 1.0, 5.0, np.inf])) == [best, best] + [order[-1]] * 3
    # an infinite temperature: every token alike, the order by value stays
    assert list(draw(dev, rows(3), F32, T=[np.inf] * 3, u=[0.0, 0.5, 0.9999])) == [best, order[150], order[299]]


def test_sample_frequencies(dev):
    """numbers spread evenly over [0, 1) pick each token as often as its weight says, to one in N"""
    rng = np.random.default_rng(4)
    n, N = 50, 4000
    x = np.repeat((2 * rng.standard_normal((1, n))).astype(np.float32), N, 0)
    u = ((np.arange(N) + 0.5) / N).astype(np.float32)
    got = np.bincount(draw(dev, x, F32, u=u, T=[0.7] * N), minlength=n)
    w = np.exp((x[0].astype(np.float64) - x[0].max()) / np.float64(np.float32(0.7)))
    assert np.all(np.abs(got - N * w / w.sum()) <= 1.0 + 1e-3)


def test_logits_and_sample_in_a_graph(dev):
    """the end of a step: penalties, then the draw; numbers and logits change in device memory between replays"""
    rng = np.random.default_rng(8)
    rows, n, width = 5, 6000, 16
    x, out, token = dev.alloc(rows * n * 4), dev.alloc(rows * n * 4), dev.alloc(rows * 4)
    history = rng.integers(0, n, (rows, width)).astype(np.int32)
    controls = m.LogitControls(history=dev.upload(history), history_len=dev.upload(np.full(rows, width, np.int32)),
                               history_width=width, penalties=dev.upload(np.tile(np.float32([1.2, 0.1, 0.1]), (rows, 1))))
    u, k = dev.alloc(rows * 4), dev.alloc(rows * 4)
    T, p = rng.uniform(0.5, 1.2, rows).astype(np.float32), np.full(rows, 0.9, np.float32)
    s = m.Sampling(u, temperature=dev.upload(T), top_k=k, top_p=dev.upload(p))
    plan = m.Plan(dev)
    plan.add_logits_process(x, F32, rows, n, n, controls, out)
    plan.add_sample(out, F32, rows, n, n, s, token)
    plan.use_graph(True)
    for step in range(4):
        x.upload((3 * rng.standard_normal((rows, n))).astype(np.float32))
        us, ks = rng.random(rows).astype(np.float32), np.array([0, 5, 5000, 100, 1], np.int32)
        u.upload(us)
        k.upload(ks)
        plan.run()
        got = token.download(np.int32)
        logits = out.download(np.float32).reshape(rows, n).astype(np.float64)
        for r in range(rows):
            want, near = pick(logits[r], float(T[r]), int(ks[r]), float(p[r]), 0.0, float(us[r]))
            assert got[r] == want or near < slack(n)
        eager = dev.alloc(rows * 4)
        dev.sample(out, F32, rows, n, n, s, eager)
        assert np.array_equal(eager.download(np.int32), got)
    assert np.all(plan.profile() > 0)
