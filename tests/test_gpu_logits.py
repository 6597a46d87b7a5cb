"""mvlm_logits_process on the GPU against its definition in 64 bits, through the C ABI."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
from paged_ref import HALF_STEP, SMALLEST, from_bits, values

pytestmark = pytest.mark.gpu

F32, F16, BF16 = m.F32, m.F16, m.BF16
NP = {F32: np.float32, F16: np.uint16, BF16: np.uint16}


class Controls:
    """Histories that repeat tokens (and name some outside the vocabulary), biases with repeated tokens, a mask."""

    def __init__(self, rng, rows, n, history=0, bias=0, mask=False, generated=True):
        self.rows, self.n = rows, n
        few = rng.integers(0, n, max(1, n // 8))
        self.history = self.bias = self.mask = self.generated = None
        if history:
            self.history = np.where(rng.random((rows, history)) < 0.7, rng.choice(few, (rows, history)),
                                    rng.integers(-2, n + 3, (rows, history))).astype(np.int32)
            self.len = rng.integers(-3, history + 4, rows).astype(np.int32)
            self.len[0] = history
            if generated:
                self.generated = rng.integers(0, history + 1, rows).astype(np.int32)
            self.penalties = np.stack([rng.uniform(0.8, 1.6, rows), rng.uniform(-0.5, 1, rows),
                                       rng.uniform(-0.5, 1, rows)], 1).astype(np.float32)
        if bias:
            self.bias = np.where(rng.random((rows, bias)) < 0.5, rng.choice(few, (rows, bias)),
                                 rng.integers(-2, n + 3, (rows, bias))).astype(np.int32)
            self.bias_values = (5 * rng.standard_normal((rows, bias))).astype(np.float32)
            self.bias_len = rng.integers(-1, bias + 3, rows).astype(np.int32)
            self.bias_len[0] = bias
        if mask:
            self.mask = rng.integers(0, 1 << 32, (rows, (n + 31) // 32), dtype=np.uint64).astype(np.uint32)
            self.mask[-1] = 0                                # a row that may say nothing

    def device(self, dev):
        up = lambda a: None if a is None else dev.upload(a)  # noqa: E731
        h = self.history is not None
        b = self.bias is not None
        return m.LogitControls(history=up(self.history), history_len=up(self.len) if h else None,
                               generated_from=up(self.generated), history_width=self.history.shape[1] if h else 0,
                               penalties=up(self.penalties) if h else None, bias_ids=up(self.bias),
                               bias_values=up(self.bias_values) if b else None, bias_len=up(self.bias_len) if b else None,
                               bias_width=self.bias.shape[1] if b else 0, allowed=up(self.mask))

    def reference(self, x):
        """values in 64 bits and how far fp32 arithmetic may be off before the store"""
        x, tol = x.copy(), np.zeros(x.shape)
        n = self.n
        for r in range(self.rows):
            if self.history is not None:
                ids = self.history[r, :max(0, min(self.len[r], self.history.shape[1]))]
                inside = (ids >= 0) & (ids < n)
                made = np.arange(len(ids)) >= (0 if self.generated is None else self.generated[r])
                c = np.bincount(ids[inside], minlength=n)
                g = np.bincount(ids[inside & made], minlength=n)
                rep, freq, pres = (float(v) for v in self.penalties[r])
                hit = c > 0
                x[r, hit] = np.where(x[r, hit] > 0, x[r, hit] / rep, x[r, hit] * rep)
                tol[r, hit] += 2.0 ** -24 * np.abs(x[r, hit])
                less = np.where(g > 0, g * freq + pres, 0.0)
                x[r] -= less
                tol[r] += 2.0 ** -23 * (g * abs(freq) + abs(pres)) * (g > 0) + 2.0 ** -24 * np.abs(x[r]) * (g > 0)
            if self.bias is not None:
                last = {}
                for i in range(max(0, min(self.bias_len[r], self.bias.shape[1]))):
                    last[int(self.bias[r, i])] = float(self.bias_values[r, i])
                for t, v in last.items():
                    if 0 <= t < n:
                        x[r, t] += v
                        tol[r, t] += 2.0 ** -24 * abs(x[r, t])
            if self.mask is not None:
                t = np.arange(n)
                x[r, (self.mask[r, t // 32] >> (t % 32)) & 1 == 0] = -np.inf
        return x, tol


def check(got, ref, tol, dtype):
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf])
    step = tol[~inf] + HALF_STEP[dtype] * (np.abs(ref[~inf]) + tol[~inf]) + SMALLEST[dtype] / 2
    assert np.all(np.abs(got[~inf] - ref[~inf]) <= step)


CASES = [
    # rows, n, dtype, history, bias, mask, extra columns, element offset
    (1, 1, F32, 1, 1, True, 0, 0),
    (1, 51200, F32, 700, 9, True, 0, 0),
    (3, 1000, F32, 64, 0, False, 0, 0),
    (2, 33, F16, 5, 3, True, 0, 0),
    (5, 1027, F16, 300, 20, True, 5, 3),
    (4, 2048, BF16, 1, 0, True, 8, 0),
    (7, 5003, F32, 0, 40, False, 1, 1),
    (3, 4096, BF16, 0, 0, True, 0, 0),
    (2, 100, F32, 0, 0, False, 3, 0),
    (300, 8200, F32, 100, 4, True, 0, 0),          # slices of 8192: more blocks than compute units
    (40, 128000, F16, 2000, 64, True, 0, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_logits(dev, case):
    rows, n, dt, history, bias, mask, extra, offset = CASES[case]
    print("[logits]", case, CASES[case], flush=True)
    rng = np.random.default_rng(40 + case)
    c = Controls(rng, rows, n, history, bias, mask, generated=case % 2 == 0)
    ld = n + extra
    flat = values(rng, offset + rows * ld, dt, 4.0)
    es = flat.itemsize
    x, out = dev.upload(flat), dev.upload(np.full_like(flat, 7))
    views = [b.view(offset * es, (rows * ld - extra) * es) for b in (x, out)]
    controls = c.device(dev)
    dev.logits_process(views[0], dt, rows, n, ld, controls, views[1])
    got = out.download(NP[dt])
    ref, tol = c.reference(from_bits(flat, dt)[offset:].reshape(rows, ld)[:, :n])
    check(from_bits(got[offset:].reshape(rows, ld)[:, :n], dt), ref, tol, dt)
    assert np.all(got[offset:].reshape(rows, ld)[:, n:] == 7) and np.all(got[:offset] == 7)
    assert np.array_equal(x.download(NP[dt]), flat)
    dev.logits_process(views[0], dt, rows, n, ld, controls, views[0])          # in place: the same bits
    assert np.array_equal(x.download(NP[dt])[offset:].reshape(rows, ld)[:, :n], got[offset:].reshape(rows, ld)[:, :n])


def test_logits_keeps_what_is_not_finite(dev):
    """infinities and NaN stay what they are, except where the mask hides them"""
    x = np.array([[np.inf, -np.inf, np.nan, 1.0, np.inf, -np.inf, np.nan, 0.0, -0.0, 2.0]], np.float32)
    c = Controls(np.random.default_rng(1), 1, 10, history=10, bias=1, mask=True)
    c.history, c.len, c.generated = np.arange(10, dtype=np.int32)[None], np.array([10], np.int32), np.array([5], np.int32)
    c.penalties = np.array([[2.0, 0.5, 0.25]], np.float32)
    c.bias, c.bias_values, c.bias_len = np.array([[9]], np.int32), np.array([[-np.inf]], np.float32), np.array([1], np.int32)
    c.mask = np.array([[0b1110001111]], np.uint32)
    out = dev.alloc(40)
    dev.logits_process(dev.upload(x), F32, 1, 10, 10, c.device(dev), out)
    ref = np.array([np.inf, -np.inf, np.nan, 0.5, -np.inf, -np.inf, -np.inf, -0.75, -0.75, -np.inf], np.float32)
    assert np.array_equal(out.download(np.float32), ref, equal_nan=True)


def test_logits_then_argmax_in_a_graph(dev):
    """the pick of a step: penalties and mask change in device memory between replays"""
    rng = np.random.default_rng(3)
    rows, n, width = 5, 6000, 32
    x, out, token = dev.alloc(rows * n * 4), dev.alloc(rows * n * 4), dev.alloc(rows * 4)
    c = Controls(rng, rows, n, width, 4, True)
    d = c.device(dev)
    plan = m.Plan(dev)
    plan.add_logits_process(x, F32, rows, n, n, d, out)
    plan.add_argmax(out, F32, rows, n, n, token)
    plan.use_graph(True)
    for step in range(4):
        xs = (4 * rng.standard_normal((rows, n))).astype(np.float32)
        fresh = Controls(rng, rows, n, width, 4, True)
        for name in ("history", "len", "generated", "penalties", "bias", "bias_values", "bias_len", "mask"):
            setattr(c, name, getattr(fresh, name))
        for buf, arr in zip(d.buffers, (c.history, c.len, c.generated, c.penalties, c.bias, c.bias_values, c.bias_len, c.mask)):
            buf.upload(arr)
        x.upload(xs)
        plan.run()
        got = out.download(np.float32).reshape(rows, n)
        ref, tol = c.reference(xs.astype(np.float64))
        check(got.astype(np.float64), ref, tol, F32)
        assert np.array_equal(token.download(np.int32), np.argmax(got, 1))   # a row of -inf gives 0
