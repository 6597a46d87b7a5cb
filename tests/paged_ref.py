"""Batches over a paged cache and their definitions in 64 bits, for the tests of
mvlm_kv_append_paged, mvlm_attention_paged and mvlm_logits_process."""
import numpy as np

import mvlm_amd as m

HALF_STEP = {m.F32: 2.0 ** -24, m.F16: 2.0 ** -11, m.BF16: 2.0 ** -8}
SMALLEST = {m.F32: 2.0 ** -149, m.F16: 2.0 ** -24, m.BF16: 2.0 ** -133}   # least positive value


def to_bits(x, dtype):
    """x rounded to nearest even, as the type's bit patterns (fp32: as it is)"""
    x = np.asarray(x, np.float32)
    if dtype == m.F32:
        return x
    if dtype == m.F16:
        return x.astype(np.float16).view(np.uint16)
    u = np.ascontiguousarray(x).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def from_bits(b, dtype):
    if dtype == m.F32:
        return np.asarray(b, np.float32).astype(np.float64)
    if dtype == m.F16:
        return np.asarray(b, np.uint16).view(np.float16).astype(np.float64)
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def values(rng, shape, dtype, std=1.0):
    return to_bits(rng.standard_normal(shape).astype(np.float32) * std, dtype)


class Batch:
    """news[s] new rows and lens[s] positions of each sequence; pages in a random
    order with spare ones between; `lead` rows before the first sequence and
    `spare` behind the last.  drop: {(s, page index): id} table entries replaced."""

    def __init__(self, rng, news, lens, page, ragged=True, lead=0, spare=0, width=None, drop=None):
        self.news, self.lens, self.page, self.ragged = list(news), list(lens), page, ragged
        self.seqs = len(self.news)
        self.start = lead + np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.rows = int(self.start[-1]) + spare
        need = [max(0, -(-L // page)) for L in self.lens]
        self.width = width or max(1, max(need) + 1)
        self.pages = sum(need) + 3
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.seqs, self.width), -1, np.int32)
        at = 0
        for s, k in enumerate(need):
            k = min(k, self.width)
            self.table[s, :k] = order[at:at + k]
            at += k
        for (s, i), page_id in (drop or {}).items():
            self.table[s, i] = page_id
        assert ragged or all(n == 1 for n in self.news) and lead == spare == 0

    def place(self, s, t):
        """(page, slot) of position t of sequence s, or None"""
        if t < 0 or t >= self.width * self.page:
            return None
        p = int(self.table[s, t // self.page])
        return (p, t % self.page) if 0 <= p < self.pages else None

    def device(self, dev):
        return m.PagedBatch(self.seqs, self.rows, dev.upload(np.asarray(self.lens, np.int32)), dev.upload(self.table),
                            self.width, row_start=dev.upload(self.start) if self.ragged else None)

    def each_row(self):
        """(row, sequence, position) of every row of a sequence"""
        for s, n in enumerate(self.news):
            for j in range(n):
                yield int(self.start[s]) + j, s, self.lens[s] - n + j


def nan_cache(batch, kv_heads, D, dtype):
    """A cache that holds NaN wherever nothing was written."""
    shape = (batch.pages, kv_heads, batch.page, D)
    return [np.full(shape, np.uint16(0x7E00 if dtype == m.F16 else 0x7FC0)) for _ in range(2)]


def filled_cache(rng, batch, kv_heads, D, dtype, std=1.0):
    """Values at every position the sequences hold, NaN elsewhere."""
    K, V = nan_cache(batch, kv_heads, D, dtype)
    for s, L in enumerate(batch.lens):
        at = np.array([a for a in (batch.place(s, t) for t in range(min(L, batch.width * batch.page))) if a])
        if len(at):
            K[at[:, 0], :, at[:, 1]] = values(rng, (len(at), kv_heads, D), dtype, std)
            V[at[:, 0], :, at[:, 1]] = values(rng, (len(at), kv_heads, D), dtype)
    return K, V


def cache_on(dev, batch, K, V, dtype):
    kv_heads, D = K.shape[1], K.shape[3]
    return m.PagedKV(dev.upload(K), dev.upload(V), dtype, batch.pages, batch.page, kv_heads, D)


def attention(batch, q, K, V, dtype, scale, parts):
    """O and its tolerance, [rows][heads][D] (NaN in rows of no sequence).

    With p_k = exp(score_k - max) and A = sum p |v| / sum p, what the kernel rounds
    moves O by at most
      u_P A               P in the cache's type (parts 1), its half step; kept in
                          two fp16 or three bf16 parts, 2^-22
      4 D 2^-24 R A       scores, D-term fp32 sums, R = max_k scale sum |q k|: each moves
                          p by that much of itself, in numerator and denominator
      8 (1 + R) 2^-23 A   the exponent's argument (two roundings of up to R log2(e) in
                          exp2) and the exponential (1 ulp), in both
      2 (N + 64) 2^-24 A  sums over N keys and the merge of their parts
      F                   parts below the type's normal range (fp16: p < 2^-14, or
                          p < 2^-3 for its second part): 2^-25 each
    and the store by half a step."""
    rows, heads, D = q.shape
    group = heads // K.shape[1]
    O, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    qd, Kd, Vd = from_bits(q, dtype), from_bits(K, dtype), from_bits(V, dtype)
    uP = HALF_STEP[dtype] if parts == 1 else 2.0 ** -22
    for s, (n, L) in enumerate(zip(batch.news, batch.lens)):
        if n == 0:
            continue
        r0 = int(batch.start[s])
        held = [t for t in range(min(L, batch.width * batch.page)) if batch.place(s, t)]
        pos = L - n + np.arange(n)
        O[r0:r0 + n] = 0.0
        if not held or pos[-1] < held[0]:
            continue
        at = np.array([batch.place(s, t) for t in held])
        seen = np.array(held)[None, :] <= pos[:, None]              # [n][keys]
        N = seen.sum(1)[:, None]
        some = N[:, 0] > 0
        for h in range(heads):
            k, v = Kd[at[:, 0], h // group, at[:, 1]], Vd[at[:, 0], h // group, at[:, 1]]
            qh = qd[r0:r0 + n, h]
            x = np.where(seen, scale * (qh @ k.T), -np.inf)
            R = np.where(seen, scale * (np.abs(qh) @ np.abs(k).T), 0.0).max(1)[:, None]
            w = np.exp(x - np.where(some, x.max(1), 0.0)[:, None])
            total = np.where(some, w.sum(1), 1.0)[:, None]
            O[r0:r0 + n, h] = w @ v / total
            A = w @ np.abs(v) / total
            small = seen & (w < (2.0 ** -13 if parts == 1 else 2.0 ** -2))
            F = 2.0 ** -25 * (small @ np.abs(v) if dtype == m.F16 else 0.0) / total
            tol[r0:r0 + n, h] = (uP + 4 * D * 2.0 ** -24 * R + 8 * (1 + R) * 2.0 ** -23 + 2 * (N + 64) * 2.0 ** -24) * A + F
    return O, tol


def close(got, ref, tol, out_dtype):
    """got (type's values) against ref within tol and a store's half step; worst ratio"""
    step = HALF_STEP[out_dtype] * (np.abs(ref) + tol) + SMALLEST[out_dtype] / 2
    err = np.abs(got - ref)
    assert np.all(np.isfinite(got) == np.isfinite(ref))
    return float(np.max(err / (tol + step + 1e-300))) if err.size else 0.0
