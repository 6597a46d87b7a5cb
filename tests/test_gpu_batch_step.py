"""A step of a batch over an 8-bit paged cache as one captured graph: products, append with norms, attention, LM head,
penalties, draw; and a chunk of a prompt that is appended, attended over and read back."""
from __future__ import annotations

import numpy as np
import pytest

import mvlm_amd as m
import mx_ref
from paged_ref import Batch, attention, close, from_bits, values
from test_gpu_paged import rope_table, same_or_close
from test_gpu_paged_8bit import in_8_bits, made_rows
from test_gpu_sample import pick, slack

pytestmark = pytest.mark.gpu

F32, BF16, MX = m.F32, m.BF16, m.MXFP8


@pytest.mark.parametrize("D,kv_heads", [(64, 4), (128, 2)])
def test_a_step_of_a_batch(dev, D, kv_heads):
    """lengths, histories and random numbers move on between the replays; each stage against its definition on the
    values that the stage before it stored"""
    rng = np.random.default_rng(41)
    S, heads, vocab, page, steps, eps = 5, 4, 5000, 16, 4, 1e-5
    hidden, width = heads * D, (heads + 2 * kv_heads) * D
    W = {n: dev.random_weight(m.Q8_0, rows, cols, 81 + i, 0.05) for i, (n, rows, cols) in
         enumerate((("qkv", width, hidden), ("dense", hidden, hidden), ("head", vocab, hidden)))}
    deq = {n: w.dequant().astype(np.float64) for n, w in W.items()}
    lens = np.array([0, 3, 15, 40, 700], np.int32)
    batch = Batch(rng, [1] * S, lens + steps, page, ragged=False)
    batch.lens = [int(v) for v in lens]
    held = mx_ref.filled(rng, batch, kv_heads, D)
    cache = mx_ref.cache_on(dev, batch, *held)
    shape = (batch.pages, kv_heads, page, D)
    b = batch.device(dev)
    x, qkv, o, y, logits, out = (dev.alloc(S * n * 4) for n in (hidden, width, hidden, hidden, vocab, vocab))
    q, token, u = dev.alloc(S * hidden * 2), dev.alloc(S * 4), dev.alloc(S * 4)
    history, hlen = dev.alloc(S * steps * 4).zero(), dev.alloc(S * 4).zero()
    pen = np.tile(np.array([[1.3, 0.4, 0.2]], np.float32), (S, 1))
    controls = m.LogitControls(history=history, history_len=hlen, history_width=steps, penalties=dev.upload(pen))
    qw, kw = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    table = rope_table(800, D)
    T, top_k = np.array([0.7, 1.0, 0.0, 1.5, 0.9], np.float32), np.array([0, 50, 0, 2000, 3], np.int32)
    top_p, min_p = np.array([0.9, 1.0, 1.0, 0.95, 0.5], np.float32), np.array([0.0, 0.02, 0.0, 0.0, 0.0], np.float32)
    sampling = m.Sampling(u, temperature=dev.upload(T), top_k=dev.upload(top_k), top_p=dev.upload(top_p), min_p=dev.upload(min_p))
    plan = m.Plan(dev)
    plan.add_gemm_quant_grouped(S, [(x, F32, W["qkv"], qkv, F32)])
    plan.add_kv_append_paged_ex(qkv, F32, width, b, cache, heads, q, m.Rope(dev.upload(table), 800, D),
                                m.HeadNorm(dev.upload(qw), dev.upload(kw), eps))
    plan.add_attention_paged(q, b, cache, o, F32, heads)
    plan.add_gemm_quant_grouped(S, [(o, F32, W["dense"], y, F32)], epilogues=[{"residual": x}])
    plan.add_gemv(y, F32, W["head"], logits, F32, S)
    plan.add_logits_process(logits, F32, S, vocab, vocab, controls, out)
    plan.add_sample(out, F32, S, vocab, vocab, sampling, token)
    plan.use_graph(True)
    seen = np.zeros((S, steps), np.int32)
    for step in range(steps):
        lens = lens + 1
        batch.lens = [int(v) for v in lens]
        b.buffers[0].upload(lens)
        xs, us = rng.standard_normal((S, hidden)).astype(np.float32), rng.random(S).astype(np.float32)
        x.upload(xs)
        u.upload(us)
        history.upload(seen)
        hlen.upload(np.full(S, step, np.int32))
        plan.run()
        got = {n: buf.download(np.float32).reshape(S, -1).astype(np.float64) for n, buf in
               (("qkv", qkv), ("o", o), ("y", y), ("logits", logits), ("out", out))}
        ref, S_ = xs.astype(np.float64) @ deq["qkv"].T, np.abs(xs.astype(np.float64)) @ np.abs(deq["qkv"]).T
        assert np.all(np.abs(got["qkv"] - ref) <= 1e-5 * S_)
        gq = q.download(np.uint16).reshape(S, heads, D)
        now = mx_ref.cache_from(cache, shape)
        for r, s, p in batch.each_row():
            at = batch.place(s, p)
            yr, t = made_rows(got["qkv"][r], heads, kv_heads, D, p, table, D, False, qw, kw, eps)
            assert close(from_bits(gq[r], BF16), yr[:heads], t[:heads], BF16) <= 1.0
            for (codes, word), (c0, w0), lo in zip(now, held, (heads, heads + kv_heads)):
                used = np.uint32(0xFFFFFFFF >> (32 - 8 * len(mx_ref.blocks(D))))
                in_8_bits(mx_ref.decode(codes[at[0], :, at[1]], word[at[0], :, at[1]] & used), yr[lo:lo + kv_heads], t[lo:lo + kv_heads])
                c0[at[0], :, at[1]], w0[at[0], :, at[1]] = codes[at[0], :, at[1]], word[at[0], :, at[1]]
        for a, z in zip(now, held):                          # nothing else was written
            assert all(np.array_equal(i, j) for i, j in zip(a, z))
        gK, gV = (mx_ref.bf16_of(*z) for z in now)
        ref, tol = attention(batch, gq, gK, gV, BF16, D ** -0.5, 2)
        assert same_or_close(got["o"].reshape(S, heads, D), ref, tol, F32) <= 1.0
        ref, S_ = got["o"] @ deq["dense"].T + xs, np.abs(got["o"]) @ np.abs(deq["dense"]).T + np.abs(xs)
        assert np.all(np.abs(got["y"] - ref) <= 1e-5 * S_)
        ref, S_ = got["y"] @ deq["head"].T, np.abs(got["y"]) @ np.abs(deq["head"]).T
        assert np.all(np.abs(got["logits"] - ref) <= 1e-5 * S_)
        ref = got["logits"].copy()
        for r in range(S):
            ids, times = np.unique(seen[r, :step], return_counts=True)
            z = ref[r, ids]
            ref[r, ids] = np.where(z > 0, z / np.float64(pen[0, 0]), z * np.float64(pen[0, 0])) - (times * np.float64(pen[0, 1]) + np.float64(pen[0, 2]))
        assert np.all(np.abs(got["out"] - ref) <= 4 * 2.0 ** -24 * (np.abs(ref) + 3.0))
        picked = token.download(np.int32)
        for r in range(S):
            want, near = pick(got["out"][r], float(T[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]), float(us[r]))
            assert picked[r] == want or near < slack(vocab), (step, r, picked[r], want, near)
        seen[:, step] = picked


def test_a_prompt_in_chunks(dev):
    """three chunks of a prompt and the tokens of two other sequences: appended, attended over, read back whole at
    the end; attention over what was read back is the same as over the cache"""
    rng = np.random.default_rng(42)
    heads, kv_heads, D, page = 8, 2, 64, 16
    width = (heads + 2 * kv_heads) * D
    full = [300, 12, 33]
    batch = Batch(rng, [1, 1, 1], full, page)
    start = [mx_ref.garbage(rng, batch, kv_heads, D) for _ in range(2)]
    cache = mx_ref.cache_on(dev, batch, *start)
    table = dev.upload(rope_table(300, 32))
    norm_w = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    norm = m.HeadNorm(dev.upload(norm_w), dev.upload(norm_w), 1e-6)
    done = np.zeros(3, int)
    kept = [np.zeros((L, 2, kv_heads, D)) for L in full]     # values as the cache holds them
    for news in ([100, 12, 0], [1, 0, 33], [199, 0, 0]):
        done += news
        batch.lens = [int(v) for v in done]
        batch.news = list(news)
        rows = batch.rows = sum(news)
        batch.start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        d = batch.device(dev)
        x = values(rng, (rows, width), BF16)
        q, o = dev.alloc(rows * heads * D * 2), dev.alloc(rows * heads * D * 4)
        dev.kv_append_paged_ex(dev.upload(x), BF16, width, d, cache, heads, q, m.Rope(table, 300, 32), norm)
        dev.attention_paged(q, d, cache, o, F32, heads)
        now = mx_ref.cache_from(cache, (batch.pages, kv_heads, page, D))
        vals = [mx_ref.decode(*z) for z in now]
        for s in range(3):
            for t in range(done[s]):
                at = batch.place(s, t)
                here = np.stack([v[at[0], :, at[1]] for v in vals])
                assert t >= done[s] - news[s] or np.array_equal(kept[s][t], here)
                kept[s][t] = here
        ref, tol = attention(batch, q.download(np.uint16).reshape(rows, heads, D), *(mx_ref.bf16_of(*z) for z in now), BF16, D ** -0.5, 2)
        assert same_or_close(o.download(np.float32).astype(np.float64).reshape(rows, heads, D), ref, tol, F32) <= 1.0
    rows = sum(full)
    batch.news, batch.rows, batch.start = full, rows, np.concatenate([[0], np.cumsum(full)]).astype(np.int32)
    d = batch.device(dev)
    out = [dev.alloc(rows * kv_heads * D * 4) for _ in range(2)]
    dev.kv_read_paged(d, cache, out[0], out[1], F32, kv_heads * D)
    for i, buf in enumerate(out):
        assert np.array_equal(buf.download(np.float32).reshape(rows, kv_heads, D), np.concatenate([z[:, i] for z in kept]))


def test_two_devices_at_once(dev):
    """two handles with work of their own in flight: workspaces and counters are the handle's"""
    other = m.Device(0)
    rng = np.random.default_rng(43)
    jobs = []
    for d, L, n in ((dev, 3000, 60000), (other, 1700, 40000)):
        batch = Batch(rng, [1, 1], [L, 900], 16, ragged=False)
        cache = mx_ref.cache_on(d, batch, *mx_ref.filled(rng, batch, 2, 64))
        q = d.upload(values(rng, (2, 8, 64), BF16))
        x = d.upload((3 * rng.standard_normal((2, n))).astype(np.float32))
        s = m.Sampling(d.upload(rng.random(2).astype(np.float32)), top_p=d.upload(np.full(2, 0.9, np.float32)))
        jobs.append((d, batch.device(d), cache, q, x, n, s, [d.alloc(2 * 8 * 64 * 4) for _ in range(12)], [d.alloc(8) for _ in range(12)]))
    for i in range(12):
        for d, b, cache, q, x, n, s, outs, toks in jobs:
            d.attention_paged(q, b, cache, outs[i], F32, 8)
            d.sample(x, F32, 2, n, n, s, toks[i])
    for d, b, cache, q, x, n, s, outs, toks in jobs:
        first, token = outs[0].download(np.uint32), toks[0].download(np.int32)
        assert all(np.array_equal(z.download(np.uint32), first) for z in outs)
        assert all(np.array_equal(z.download(np.int32), token) for z in toks) and np.all((token >= 0) & (token < n))
    del jobs, d, b, cache, q, x, s, outs, toks
    other.close()
