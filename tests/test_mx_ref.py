"""The host's 8-bit cache format against its rule (no GPU): every code is what rounding to the nearest makes of it."""
import numpy as np

import mx_ref


def test_codes_are_the_nearest():
    rng = np.random.default_rng(1)
    finite = np.sort(mx_ref.E4M3[np.isfinite(mx_ref.E4M3)])
    for scale in (1.0, 2.0 ** -40, 2.0 ** 90, 2.0 ** -104):
        x = (rng.standard_normal((200, 72)) * scale * 2.0 ** rng.integers(-12, 3, (200, 72))).astype(np.float32)
        codes, word = mx_ref.encode(x)
        e = mx_ref.exponents(x.astype(np.float64))
        for lo, hi in mx_ref.blocks(72):
            b = lo // 32
            y = x[:, lo:hi].astype(np.float64) * 2.0 ** -e[:, b, None].astype(np.float64)
            assert np.all(np.abs(y) <= 448) and np.all((np.abs(y).max(1) > 224) | (e[:, b] == mx_ref.LEAST))
            near = np.abs(finite[None, None] - y[..., None]).min(-1)
            assert np.array_equal(np.abs(mx_ref.E4M3[codes[:, lo:hi]] - y), near)
        assert np.array_equal(mx_ref.decode(codes, word) == 0, mx_ref.E4M3[codes] == 0)


def test_what_is_not_finite_and_ends_of_the_range():
    x = np.zeros((1, 40), np.float32)
    x[0, :4] = np.inf, -np.inf, np.nan, 1.0
    x[0, 32:36] = np.finfo(np.float32).max, -31 * 2.0 ** 123, np.nextafter(np.float32(31 * 2.0 ** 123), np.float32(0)), 2.0 ** -149
    v = mx_ref.decode(*mx_ref.encode(x))
    assert np.all(np.isnan(v[0, :3])) and v[0, 3] == 1.0
    assert list(v[0, 32:36]) == [15 * 2.0 ** 124, -15 * 2.0 ** 124, 15 * 2.0 ** 124, 0.0]


def test_buffers():
    rng = np.random.default_rng(2)
    codes, word = mx_ref.encode(rng.standard_normal((3, 1, 1, 24)))
    raw = mx_ref.packed(codes, word)
    assert raw.size == 80 + 12
    c, w = mx_ref.unpacked(raw, codes.shape)
    assert np.array_equal(c, codes) and np.array_equal(w, word)
