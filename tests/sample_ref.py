"""mvlm_sample's definition on the host: which places in the order of falling value may be the drawn one.

Weights are the interface's integers of 2^-bits, sums of them are exact.  What the library may do otherwise is round a
weight another way: its exponent (v - m) log2(e) / T takes a subtraction, a constant, a division and a product of 64
bits, 4 2^-53 of an exponent of 52 at most, 2^-45.3, and here a subtraction and a division, 2 2^-53 of 36 nats, 2^-46.8:
2^-45.8 and 2^-46.8 of the weight (ln 2 of the first), 2^-45 together."""
import math

import numpy as np

OFF = 2.0 ** -45


def bits_of(n):
    return min(51, 62 - (n - 1).bit_length())


class Places:
    """order: the row's tokens by falling value, the lower index first; the drawn one is at place lo .. hi of it"""

    def __init__(self, x, T=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
        x = np.asarray(x, np.float64)
        v = np.where(np.isnan(x), np.where(np.signbit(x), -np.inf, np.inf), x)
        self.order = np.argsort(-v, kind="stable")
        v = v[self.order]
        self.lo = self.hi = self.last = 0                    # last: of those that may be kept
        if v[0] == -np.inf or not T > 0:
            if v[0] == -np.inf:
                self.order = np.sort(self.order)
            return
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / T))
        w = np.where(v == -np.inf, 0.0, w)
        unit = 2.0 ** -bits_of(len(x))
        # the least and the most of them that live: what rounds to a unit or more, and reaches min_p
        live = [int(np.count_nonzero(w * s >= unit / 2)) for s in (1 - OFF, 1 + OFF)]
        if min_p > 0:
            least = min(min_p, 1.0)
            live = [min(a, int(np.count_nonzero((w >= least * s) | (w == 1.0)))) for a, s in zip(live, (1 + OFF, 1 - OFF))]
        kept = [min(a, top_k) if top_k > 0 else a for a in live]
        sums = [np.cumsum(np.round(w * s / unit).astype(np.uint64)) for s in (1 - OFF, 1 + OFF)]   # they lie between

        def place(part, over, limit):
            """the least and the most place, below limit's, at which the sum reaches part of (over: exceeds) the kept's"""
            if part >= 1:
                return [k - 1 for k in limit]
            found = []
            for i, k in enumerate(limit):
                total = int(sums[i][k - 1])
                mant, two = math.frexp(part)                 # exactly: part = mant 2^53 / 2^(53 - two)
                need = int(mant * 2 ** 53) * total
                down = 53 - two
                need = (need >> down) + 1 if over else -(-need >> down)
                found.append(min(int(np.searchsorted(sums[1 - i], np.uint64(max(need, 1)), "left")), k - 1))
            return found

        if top_p < 1:                                        # a NaN is none
            kept = [p + 1 for p in (place(float(top_p), False, kept) if top_p > 0 else [0, 0])]
        self.last = kept[1] - 1
        self.lo, self.hi = place(u if u > 0 else 0.0, True, kept) if u > 0 else [0, 0]

    def allows(self, token):
        return int(token) in self.order[self.lo:self.hi + 1]

    def rank(self, token):
        return int(np.nonzero(self.order == token)[0][0])
