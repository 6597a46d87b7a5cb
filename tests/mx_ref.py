"""An 8-bit paged cache (MXFP8) on the host: its codes, its values, its buffers."""
import numpy as np

import mvlm_amd as m
from paged_ref import to_bits

LEAST, MOST = -100, 120                  # exponents of a block's power of two
_BYTE = np.arange(256)
_EXP, _MANT = _BYTE % 128 // 8, _BYTE % 8
E4M3 = np.where(_BYTE >= 128, -1.0, 1.0) * np.where(_EXP > 0, (8.0 + _MANT) * 2.0 ** (_EXP - 10.0), _MANT * 2.0 ** -9)
E4M3[[0x7F, 0xFF]] = np.nan


def blocks(D):
    return [(d, min(d + 32, D)) for d in range(0, D, 32)]


def exponents(x):
    """[..., blocks] of x [..., D]: the least e >= LEAST with max |x| <= 448 2^e, over what is finite"""
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = np.stack([a[..., lo:hi].max(-1) for lo, hi in blocks(x.shape[-1])], -1)
    with np.errstate(divide="ignore"):
        e = np.where(top > 0, np.ceil(np.log2(top / 448.0)), LEAST)
    e = np.where(top > 448.0 * 2.0 ** e, e + 1, e)
    e = np.where((top <= 448.0 * 2.0 ** (e - 1)) & (top > 0), e - 1, e)
    return np.maximum(e, LEAST).astype(np.int64)


def encode(x):
    """codes [..., D] and words [...] of fp32 values x, as the cache holds them"""
    x = np.asarray(x, np.float64)
    e = exponents(x)
    codes = np.zeros(x.shape, np.uint8)
    word = np.zeros(x.shape[:-1], np.uint32)
    for b, (lo, hi) in enumerate(blocks(x.shape[-1])):
        word |= (e[..., b] + 127).astype(np.uint32) << np.uint32(8 * b)
        y = x[..., lo:hi] * 2.0 ** -e[..., b, None].astype(np.float64)
        limit = np.where(e[..., b, None] == MOST, 240.0, 448.0)
        y = np.where(np.isfinite(y), np.clip(y, -limit, limit), y)
        a = np.abs(np.where(np.isfinite(y), y, 0.0))
        k = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6)
        r = np.round(a / 2.0 ** (k - 3)) * 2.0 ** (k - 3)                 # half to even
        k = np.maximum(np.floor(np.log2(np.maximum(r, 2.0 ** -20))), -6)
        code = np.where(r >= 2.0 ** -6, (k + 7) * 8 + r / 2.0 ** (k - 3) - 8, r * 2.0 ** 9).astype(np.uint8)
        code = np.where(np.isfinite(y), code, 0x7F).astype(np.uint8)
        codes[..., lo:hi] = code | (np.signbit(x[..., lo:hi]).astype(np.uint8) << 7)
    return codes, word


def decode(codes, word):
    """values of codes [..., D] under words [...]"""
    D = codes.shape[-1]
    e = np.stack([(word >> np.uint32(8 * b)) & 0xFF for b in range(len(blocks(D)))], -1).astype(np.float64) - 127.0
    return E4M3[codes] * 2.0 ** np.repeat(e, 32, -1)[..., :D]


def packed(codes, word):
    """a K or V buffer: the codes, from the next multiple of 16 bytes on the words"""
    flat = codes.reshape(-1)
    return np.concatenate([flat, np.zeros(-flat.size % 16, np.uint8), word.reshape(-1).view(np.uint8)])


def unpacked(raw, shape):
    size, slots = int(np.prod(shape)), int(np.prod(shape[:-1]))
    return raw[:size].reshape(shape), raw[raw.size - 4 * slots:].view(np.uint32).reshape(shape[:-1])


def bf16_of(codes, word):
    """the values as bf16 patterns, which is what they are"""
    return to_bits(decode(codes, word), m.BF16)


def garbage(rng, batch, kv_heads, D):
    """codes and words of a cache in which nothing was written: any bytes, many of them NaN codes and words of 0xFF"""
    shape = (batch.pages, kv_heads, batch.page, D)
    codes = np.where(rng.random(shape) < 0.5, 0x7F, rng.integers(0, 256, shape)).astype(np.uint8)
    return codes, np.where(rng.random(shape[:-1]) < 0.5, 0xFFFFFFFF, rng.integers(0, 1 << 32, shape[:-1])).astype(np.uint32)


def filled(rng, batch, kv_heads, D, std=1.0):
    """((codes, words) of K, of V): encoded values at every position the sequences hold, garbage elsewhere"""
    K, V = garbage(rng, batch, kv_heads, D), garbage(rng, batch, kv_heads, D)
    for s, L in enumerate(batch.lens):
        at = np.array([a for a in (batch.place(s, t) for t in range(min(L, batch.width * batch.page))) if a])
        if len(at):
            for (codes, word), scale in ((K, std), (V, 1.0)):
                # blocks of unlike size
                x = rng.standard_normal((len(at), kv_heads, D)) * scale * 2.0 ** np.repeat(
                    rng.integers(-2, 3, (len(at), kv_heads, len(blocks(D)))), 32, -1)[..., :D]
                codes[at[:, 0], :, at[:, 1]], word[at[:, 0], :, at[:, 1]] = encode(x.astype(np.float32))
    return K, V


def cache_on(dev, batch, K, V):
    kv_heads, D = K[0].shape[1], K[0].shape[3]
    bufs = [dev.upload(packed(*x)) for x in (K, V)]
    assert bufs[0].nbytes == m.paged_kv_bytes(m.MXFP8, batch.pages, batch.page, kv_heads, D)
    return m.PagedKV(*bufs, m.MXFP8, batch.pages, batch.page, kv_heads, D)


def cache_from(cache, shape):
    """((codes, words) of K, of V) as the device has them"""
    return [unpacked(b.download(np.uint8), shape) for b in cache.buffers]
