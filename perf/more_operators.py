"""Operators of a batch's step with an 8-bit cache and sampled tokens, as they are measured.

  append     new rows of q | k | v: each q and k head normalised, rotary positions, keys and values into their
             sequences' pages, 16-bit or 8-bit (mvlm_kv_append_paged_ex); rows that went into an 8-bit cache are read
             back as the values it holds (mvlm_kv_read_paged)
  read       positions of sequences out of their pages, in a row (mvlm_kv_read_paged)
  attention  the new rows of each sequence over its 8-bit pages, causal within the new rows: single tokens, chunks of
             a prompt, and both in one batch (mvlm_attention_paged)
  sample     a token of each row of logits by temperature, min-p, top-k, top-p and a given random number (mvlm_sample)

An 8-bit cache holds e4m3 codes and a power of two for every 32 dims of a head.  Where `own` is false, run() computes
the same with elementary torch operations in 32 bits, tokens in 64.  Calls that a program makes once a step for single
tokens are replayed from a plan, prompts are called directly.
"""
import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6                             # of the norms


# ---- the cases -------------------------------------------------------------------

def _append(name, x, cache, norm, seqs, chunks, new, cached, heads, kv_heads, dim, rot, interleaved, page):
    return {"name": name, "kind": "append", "x": x, "cache": cache, "norm": norm, "seqs": seqs, "chunks": chunks,
            "new": new, "cached_lo": cached, "cached_hi": cached, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "interleaved": interleaved, "page": page, "idle": 0}


def _read(name, out, cache, seqs, new, kv_heads, dim, page):
    return {"name": name, "kind": "read", "out": out, "cache": cache, "seqs": seqs, "chunks": seqs, "new": new,
            "cached_lo": 0, "cached_hi": 0, "heads": kv_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "idle": 0}


def _attention(name, out, seqs, chunks, new, lo, hi, heads, kv_heads, dim, page, idle=0):
    return {"name": name, "kind": "attention", "out": out, "cache": "mxfp8", "seqs": seqs, "chunks": chunks, "new": new,
            "cached_lo": lo, "cached_hi": hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "idle": idle}


def _sample(name, dtype, rows, vocab, top_k, top_p, min_p, masked):
    return {"name": name, "kind": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "masked": masked}


def listed():
    return [
        # one conversation, one token of Phi-1.5 into an 8-bit cache: the launches are what counts
        _append("append_8bit_one_token", "f32", "mxfp8", False, 1, 0, 1, 511, 32, 32, 64, 32, False, 16),
        # an image's 729 positions and some text through a model that normalises q and k, 16-bit cache
        _append("append_norm_768", "f16", "f16", True, 1, 1, 768, 0, 32, 32, 64, 32, False, 64),
        # long prompts of four users at once into an 8-bit cache, shared key heads
        _append("append_norm_8bit_4x4096", "bf16", "mxfp8", True, 4, 4, 4096, 0, 32, 8, 128, 128, False, 64),
        # an image's positions out of an 8-bit cache, for attention over contiguous keys
        _read("read_8bit_729", "f16", "mxfp8", 1, 729, 32, 64, 16),
        # long documents out of an 8-bit cache, as when a conversation moves on
        _read("read_8bit_4x16384", "bf16", "mxfp8", 4, 16384, 8, 128, 64),
        # one Phi-1.5 conversation in mid-length
        _attention("decode_8bit_1x512", "f32", 1, 0, 1, 511, 511, 32, 32, 64, 16),
        # sixteen of them, of all lengths up to the model's 2048 positions, two of the places idle
        _attention("decode_8bit_16x2047", "f32", 16, 0, 1, 30, 2046, 32, 32, 64, 16, 2),
        # few users with long documents, eight key heads shared by thirty-two
        _attention("decode_8bit_4x32768", "bf16", 4, 0, 1, 20000, 32767, 32, 8, 128, 64),
        # a chunk of a long document behind what is cached of it
        _attention("chunk_8bit_2048_on_8192", "bf16", 1, 1, 2048, 8192, 8192, 32, 8, 128, 64),
        # one conversation's token, the usual filters
        _sample("sample_1x51200", "f32", 1, 51200, 50, 0.95, 0.0, 0.0),
        # sixteen conversations, a grammar's mask on their logits, no limit on the number of tokens
        _sample("sample_16x51200", "bf16", 16, 51200, 0, 0.9, 0.0, 0.5),
        # a full server: many rows, a large vocabulary, filters of all kinds
        _sample("sample_128x128000", "f32", 128, 128000, 1000, 0.95, 0.02, 0.0),
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def _drawn(rng):
    kind = rng.choice(["append", "append", "read", "attention", "attention", "sample", "sample"])
    if kind == "sample":
        return {"kind": kind, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "rows": _log(rng, 1, 128),
                "vocab": _log(rng, 1000, 128000), "top_k": rng.choice([0, 0, 1, 20, 50, _log(rng, 2, 5000)]),
                "top_p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
    dim = rng.choice([64, 64, 72, 80, 96, 128, 128])
    kv_heads = rng.choice([2, 4, 8, 8, 16, 32])
    case = {"kind": kind, "cache": "mxfp8", "heads": kv_heads * rng.choice([1, 1, 2, 4, 8]), "kv_heads": kv_heads,
            "dim": dim, "page": rng.choice([8, 16, 32, 48, 64, 128, 256]), "idle": 0}
    if kind == "append":
        case["cache"] = rng.choice(["mxfp8", "mxfp8", "f16", "bf16"])
        case["norm"] = case["cache"] != "mxfp8" or rng.random() < 0.6
        case["x"] = rng.choice(["f32", "bf16" if case["cache"] == "mxfp8" else case["cache"]])
        case["rot"] = rng.choice([dim // 2, dim])
        case["interleaved"] = rng.random() < 0.5
    elif kind == "read":
        case["cache"] = rng.choice(["mxfp8", "mxfp8", "f16", "bf16"])
        case["out"] = rng.choice(["f32", "f16", "bf16"])
    else:
        case["out"] = rng.choice(["f32", "bf16", "bf16"])
    form = "chunk" if kind == "read" else rng.choice(["single", "chunk", "mixed"])
    if form == "single":
        case |= {"seqs": _log(rng, 1, 64), "chunks": 0, "new": 1}
        case["cached_lo"] = rng.randrange(0, 200)
        case["cached_hi"] = case["cached_lo"] + _log(rng, 1, max(2, 100000 // case["seqs"]))
        if kind == "attention" and case["seqs"] > 2 and rng.random() < 0.4:
            case["idle"] = rng.randrange(1, case["seqs"] // 2 + 1)
    else:
        chunks = rng.randrange(1, 5)
        case |= {"seqs": chunks + (rng.randrange(1, 12) if form == "mixed" else 0), "chunks": chunks,
                 "new": _log(rng, 2, (16384 if kind == "read" else 2048) // chunks)}
        case["cached_lo"] = rng.choice([0, 0, rng.randrange(0, 1000)])
        case["cached_hi"] = case["cached_lo"] + rng.choice([0, _log(rng, 1, 4000)])
    return case


def draw(rng):
    most = [max(work(c)[k] for c in listed() if c["kind"] == "attention") for k in ("bytes", "flops")]
    while True:
        case = _drawn(rng)
        w = work(case)
        padded = 0 if case["kind"] != "attention" else case["seqs"] * case["heads"] * _news(case)[0] * max(_lengths(case))
        if case["heads" if case["kind"] != "sample" else "rows"] <= 128 and w["bytes"] <= most[0] \
                and w["flops"] <= most[1] and padded <= 1 << 30:
            return case


def _news(case):
    """New rows of each sequence: chunks of unlike lengths first, single tokens behind them."""
    return [case["new"] - (37 * i) % max(1, case["new"] // 2) for i in range(case["chunks"])] + \
        [1] * (case["seqs"] - case["chunks"])


def _lengths(case):
    """Positions of each sequence with its new rows; idle places hold none."""
    span = case["cached_hi"] - case["cached_lo"]
    cached = [case["cached_hi"] - int(span * ((0.618034 * i) % 1.0)) for i in range(case["seqs"])]
    live = case["seqs"] - case["idle"]
    return [(c + n if i < live else 0) for i, (c, n) in enumerate(zip(cached, _news(case)))]


def _row_bytes(case):
    """Bytes of one head's keys at one position in the cache."""
    return case["dim"] + 4 if case["cache"] == "mxfp8" else 2 * case["dim"]


def work(case):
    if case["kind"] == "sample":
        es, n, rows = SIZE[case["dtype"]], case["vocab"], case["rows"]
        return {"bytes": rows * (n * es + 24), "flops": 20 * rows * n}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    news, lengths = _news(case), _lengths(case)
    rows, width, held = sum(news), -(-max(lengths) // case["page"]), 2 * Hk * _row_bytes(case)
    if case["kind"] == "append":
        b = rows * ((H + 2 * Hk) * D * SIZE[case["x"]] + H * D * 2 + held + case["rot"] * 4 + 4) + 8 * case["seqs"]
        if case["cache"] == "mxfp8":   # read back
            b += rows * (held + 2 * Hk * D * 2)
        return {"bytes": b, "flops": rows * (H + Hk) * (3 * case["rot"] + (4 * D if case["norm"] else 0))}
    if case["kind"] == "read":
        return {"bytes": rows * (held + 2 * Hk * D * SIZE[case["out"]] + 4) + 8 * case["seqs"], "flops": 2 * rows * Hk * D}
    pairs = sum(n * L - n * (n - 1) // 2 for n, L in zip(news, lengths) if L > 0)
    b = rows * H * D * (2 + SIZE[case["out"]]) + sum(lengths) * held + 4 * case["seqs"] * (width + 2)
    return {"bytes": b, "flops": 4 * H * D * pairs}


# ---- inputs ------------------------------------------------------------------------

class _Source:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=self.gen).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    src = _Source(seed)
    if case["kind"] == "sample":
        rows, n = case["rows"], case["vocab"]
        x = src.normal(rows, n, std=3.0)
        if case["masked"]:
            x.masked_fill_(src.uniform(rows, n) < case["masked"], -math.inf)
        t = {"x": x.to(TORCH[case["dtype"]]), "uniform": src.uniform(rows)}
        # requests have settings of their own; a row in eight or so takes the largest logit
        t["temperature"] = 0.5 + src.uniform(rows)
        t["temperature"][src.uniform(rows) < 0.12] = 0.0
        t["top_k"] = (case["top_k"] * (0.25 + src.uniform(rows))).ceil().int()
        t["top_p"] = torch.full((rows,), case["top_p"], device="cuda") ** (0.5 + src.uniform(rows))
        t["min_p"] = case["min_p"] * (0.5 + src.uniform(rows))
        return t
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    news, lengths, page = _news(case), _lengths(case), case["page"]
    width = -(-max(lengths) // page)
    need = [-(-L // page) for L in lengths]
    pages = sum(need) + 8
    order = torch.randperm(pages, device="cuda", generator=src.gen).int()
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    start = [0]
    for k in news:
        start.append(start[-1] + k)
    t = {"kv_len": _ints(lengths), "table": table}
    for name in ("k", "v"):
        x = src.normal(pages, Hk, page, D)
        if case["cache"] == "mxfp8":
            t[name], t[name + "_scale"] = _codes(x)
        else:
            t[name] = x.to(TORCH[case["cache"]])
    if case["chunks"]:
        t["row_start"] = _ints(start)
    if case["kind"] == "attention":
        t["q"] = src.normal(start[-1], H, D, dtype=torch.bfloat16)
    if case["kind"] == "append":
        t["qkv"] = src.normal(start[-1], (H + 2 * Hk) * D, dtype=TORCH[case["x"]])
        t["rope"] = _rope_table(width * page, case["rot"]).float()
        if case["norm"]:
            t["q_weight"], t["k_weight"] = 1.0 + src.normal(D, std=0.2), 1.0 + src.normal(D, std=0.2)
    return t


def _rope_table(positions, rot):
    """cos and sin of position p at 10000^(-2 i / rot), made once in 64 bits: [positions][rot / 2][2]."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1)


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if own:
        _place(state)
    return state


# ---- the plain form ------------------------------------------------------------------

def run(state):
    """One pass through an operator, and the tensors it writes."""
    if own:
        state["call"]()
        return state["out"]
    return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention,
            "sample": _plain_sample}[state["case"]["kind"]](state["case"], state["t"])


def _power(e):
    """2^e in 32 bits, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _codes(x):
    """e4m3 codes of x [..., dim] and the exponents of their blocks of 32 dims, biased by 127, four to a position."""
    D = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, 128 - D)).unflatten(-1, (4, 32))
    mant, exp = torch.frexp(blocks.abs().amax(-1))            # mant in [0.5, 1)
    e = (exp - 9 + (mant > 0.875).int()).clamp_min(-100)
    codes = (blocks * _power(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).flatten(-2)[..., :D].contiguous(), (e + 127).to(torch.uint8)


def _values(codes, scale):
    """fp32 values of codes [..., dim] with the exponents [..., 4] of their blocks."""
    powers = _power(scale.int() - 127).repeat_interleave(32, -1)[..., :codes.shape[-1]]
    return codes.view(torch.float8_e4m3fn).float() * powers


def _rows(case, t):
    """Sequence, index within its new rows, and position of each row."""
    if "row_start" not in t:
        seq = torch.arange(case["seqs"], device="cuda")
        return seq, torch.zeros_like(seq), t["kv_len"].long() - 1
    start = t["row_start"].long()
    row = torch.arange(sum(_news(case)), device="cuda")
    seq = torch.bucketize(row, start, right=True) - 1
    j = row - start[seq]
    return seq, j, t["kv_len"].long()[seq] - (start[seq + 1] - start[seq]) + j


def _rotate(x, cs, rot, interleaved):
    """x [rows][heads][dim] in 32 bits, cs [rows][rot / 2][2]."""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _norm(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _plain_append(case, t):
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    seq, _, p = _rows(case, t)
    x = t["qkv"].float().view(-1, H + 2 * Hk, D)
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    if case["norm"]:
        q, k = _norm(q, t["q_weight"]), _norm(k, t["k_weight"])
    cs = t["rope"][p]
    q, k = _rotate(q, cs, case["rot"], case["interleaved"]), _rotate(k, cs, case["rot"], case["interleaved"])
    page, slot = t["table"][seq, p // case["page"]].long(), p % case["page"]
    if case["cache"] != "mxfp8":
        cache = TORCH[case["cache"]]
        t["k"][page, :, slot], t["v"][page, :, slot] = k.to(cache), v.to(cache)
        return {"q": q.to(cache), "k": t["k"], "v": t["v"]}
    out = {"q": q.to(torch.bfloat16)}
    for name, rows in (("k", k), ("v", v)):
        t[name][page, :, slot], t[name + "_scale"][page, :, slot] = _codes(rows)
        out[name] = _values(t[name][page, :, slot], t[name + "_scale"][page, :, slot]).to(torch.bfloat16)
    return out


def _plain_read(case, t):
    seq, _, p = _rows(case, t)
    page, slot = t["table"][seq, p // case["page"]].long(), p % case["page"]
    out = {}
    for name in ("k", "v"):
        x = t[name][page, :, slot]
        x = _values(x, t[name + "_scale"][page, :, slot]) if case["cache"] == "mxfp8" else x.float()
        out[name] = x.to(TORCH[case["out"]])
    return out


def _plain_attention(case, t):
    H, Hk, D, S = case["heads"], case["kv_heads"], case["dim"], case["seqs"]
    new, L = max(_news(case)), max(_lengths(case))
    seq, j, p = _rows(case, t)
    pages = t["table"].clamp_min(0).long()
    k, v = (_values(t[n][pages], t[n + "_scale"][pages]).transpose(1, 2).reshape(S, Hk, -1, D)[:, :, :L] for n in ("k", "v"))
    q = torch.zeros(S, new, H, D, device="cuda")
    q[seq, j] = t["q"].float()
    at = torch.full((S, new), -1, dtype=torch.int64, device="cuda")
    at[seq, j] = p
    q = q.view(S, new, Hk, H // Hk, D).transpose(1, 2).reshape(S, Hk, -1, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(D)).view(S, Hk, new, H // Hk, L)
    s.masked_fill_(torch.arange(L, device="cuda") > at[:, None, :, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = s.sum(-1)
    o = torch.matmul(s.view(S, Hk, -1, L), v).view(S, Hk, new, H // Hk, D)
    o = (o / total.clamp_min(1e-30)[..., None]).transpose(1, 2).reshape(S, new, H, D)
    return [o[seq, j].to(TORCH[case["out"]])]


def _plain_sample(case, t):
    n = case["vocab"]
    x, token = torch.sort(t["x"].double(), dim=1, descending=True, stable=True)
    temperature, top_p, min_p, u = (t[k].double()[:, None] for k in ("temperature", "top_p", "min_p", "uniform"))
    rank = torch.arange(n, device="cuda")
    w = torch.where(x > -math.inf, torch.exp((x - x[:, :1]) / temperature.clamp_min(1e-30)), 0.0)
    limit = torch.where(t["top_k"] > 0, t["top_k"], n)[:, None]
    w = torch.where((w >= min_p) & (rank < limit), w, 0.0)
    before = torch.cumsum(w, 1) - w
    w = torch.where((rank == 0) | (top_p >= 1.0) | (before < top_p * w.sum(1, keepdim=True)), w, 0.0)
    sums = torch.cumsum(w, 1)
    picked = torch.where(t["temperature"][:, None] > 0, (sums <= u * sums[:, -1:]).sum(1, keepdim=True), 0)
    return [token.gather(1, picked)[:, 0].int()]


# ---- the framework's calls -------------------------------------------------------------

_device = None


class _InPlace:
    """A buffer as torch sees it.  The C ABI's handles are opaque and have no accessor for the device address, so
    it is read from the handle (the second word of mvlm_buffer); the buffer lives as long as the tensor."""

    def __init__(self, buf, count, typestr):
        import ctypes
        self.buf = buf
        address = ctypes.c_uint64.from_address(buf.handle.value + 8).value
        self.__cuda_array_interface__ = {"shape": (count,), "typestr": typestr, "data": (address, False), "version": 2}


def _view(buf, dtype, shape):
    typestr = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.int32: "<i4",
               torch.uint8: "|u1"}[dtype]
    t = torch.as_tensor(_InPlace(buf, math.prod(shape), typestr), device="cuda")
    return (t.view(torch.bfloat16) if dtype == torch.bfloat16 else t).view(shape)


def _place(state):
    """The inputs in the framework's buffers, its handles and the call, as a program holds them."""
    global _device
    import mvlm_amd as m
    if _device is None:
        torch.cuda.init()
        _device = m.Device(0)
    dev, case, t = _device, state["case"], state["t"]
    names = {"f32": m.F32, "f16": m.F16, "bf16": m.BF16, "mxfp8": m.MXFP8}

    def empty(dtype, *shape):
        buf = dev.alloc(math.prod(shape) * SIZE[dtype])
        return buf, _view(buf, TORCH[dtype], shape)

    b = {}
    for name in list(t):
        if name in ("k_scale", "v_scale"):
            continue
        size = t[name].numel() * t[name].element_size()
        if name + "_scale" in t:           # codes, then their scales, in one buffer
            pages, Hk, page, D = t[name].shape
            b[name] = dev.alloc(m.paged_kv_bytes(m.MXFP8, pages, page, Hk, D))
            whole = _view(b[name], torch.uint8, (b[name].nbytes,))
            scale = t.pop(name + "_scale")
            whole[:size].copy_(t[name].view(-1))
            whole[-scale.numel():].copy_(scale.view(-1))
            t[name] = whole
            continue
        b[name] = dev.alloc(size)
        place = _view(b[name], t[name].dtype, t[name].shape)
        place.copy_(t[name])
        t[name] = place
    torch.cuda.synchronize()
    if case["kind"] == "sample":
        rows, n = case["rows"], case["vocab"]
        out = dev.alloc(4 * rows)
        settings = m.Sampling(b["uniform"], temperature=b["temperature"], top_k=b["top_k"], top_p=b["top_p"],
                              min_p=b["min_p"])
        plan = m.Plan(dev)
        plan.add_sample(b["x"], names[case["dtype"]], rows, n, n, settings, out)
        state |= {"plan": plan, "call": plan.run, "out": [_view(out, torch.int32, (rows,))]}
        return
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows, pages = sum(_news(case)), sum(-(-L // page) for L in _lengths(case)) + 8
    cache = m.PagedKV(b["k"], b["v"], names[case["cache"]], num_pages=pages, page_size=page, kv_heads=Hk, head_dim=D)
    batch = m.PagedBatch(case["seqs"], rows, b["kv_len"], b["table"], t["table"].shape[1], row_start=b.get("row_start"))
    calls, out = [], {}
    if case["kind"] == "append":
        q, out["q"] = empty("f16" if case["cache"] == "f16" else "bf16", rows, H, D)
        rope = m.Rope(b["rope"], positions=t["rope"].shape[0], rot_dim=case["rot"], interleaved=case["interleaved"])
        norm = m.HeadNorm(b["q_weight"], b["k_weight"], EPS) if case["norm"] else None
        calls.append(("kv_append_paged_ex", (b["qkv"], names[case["x"]], (H + 2 * Hk) * D, batch, cache, H, q, rope, norm)))
        if case["cache"] != "mxfp8":
            out |= {"k": t["k"], "v": t["v"]}
    if case["kind"] == "read" or case["cache"] == "mxfp8" and case["kind"] == "append":
        form = case.get("out", "bf16")
        (k, out["k"]), (v, out["v"]) = empty(form, rows, Hk, D), empty(form, rows, Hk, D)
        calls.append(("kv_read_paged", (batch, cache, k, v, names[form], Hk * D)))
    if case["kind"] == "attention":
        o, seen = empty(case["out"], rows, H, D)
        calls.append(("attention_paged", (b["q"], batch, cache, o, names[case["out"]], H)))
        out = [seen]
    state["out"] = out
    if case["chunks"]:
        direct = [(getattr(dev, name), args) for name, args in calls]
        state["call"] = lambda: [f(*args) for f, args in direct]
        return
    plan = m.Plan(dev)
    for name, args in calls:
        getattr(plan, "add_" + name)(*args)
    if len(calls) > 1:
        plan.use_graph(True)
    state |= {"plan": plan, "call": plan.run}


# ---- from the definitions, in 64 bits ------------------------------------------------------

def _exact_codes(x):
    """The values that 8 bits hold of x [..., dim] in 64 bits: 4 significant bits of each, in units of the least power of
    two that takes the largest of its 32 dims to 448 or below."""
    out = torch.empty_like(x)
    for d in range(0, x.shape[-1], 32):
        block = x[..., d:d + 32]
        top = block.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / 448.0))
        e += (top > 448.0 * torch.exp2(e)).double() - (top <= 448.0 * torch.exp2(e - 1.0)).double()
        scale = torch.exp2(e.clamp_min(-100.0))
        y = block / scale
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
        out[..., d:d + 32] = torch.round(y / step) * step * scale
    return out


def _exact_cache(case, t, name, page):
    """[heads][slots][dim] of one page in 64 bits."""
    x = t[name][page]
    if case["cache"] != "mxfp8":
        return x.double()
    b = torch.arange(256, device="cuda").double()
    sign, exp, mant = torch.where(b >= 128, -1.0, 1.0), (b % 128).div(8, rounding_mode="floor"), b % 8
    table = sign * torch.where(exp > 0, (8.0 + mant) * 2.0 ** (exp - 10.0), mant * 2.0 ** -9)
    dims = torch.arange(x.shape[-1], device="cuda") // 32
    return table[x.long()] * 2.0 ** (t[name + "_scale"][page].double()[..., dims] - 127.0)


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "sample":
        return [torch.tensor([_exact_token(case, t, r) for r in range(case["rows"])], dtype=torch.int32)]
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    news, lengths = _news(case), _lengths(case)
    held = {s: t["table"][s, :-(-L // page)].long() for s, L in enumerate(lengths) if L > 0}
    row = 0
    if case["kind"] == "read":
        parts = {"k": [], "v": []}
        for s, (n, L) in enumerate(zip(news, lengths)):
            for name in parts:
                x = _exact_cache(case, t, name, held[s]).transpose(1, 2).reshape(-1, Hk, D)
                parts[name].append(x[L - n:L])
        return {name: torch.cat(x) for name, x in parts.items()}
    if case["kind"] == "append":
        q, keys, values, rot = [], [], [], case["rot"]
        mx = case["cache"] == "mxfp8"
        k, v = (None, None) if mx else (t["k"].double(), t["v"].double())
        for s, (n, L) in enumerate(zip(news, lengths)):
            x = t["qkv"][row:row + n].double().view(n, H + 2 * Hk, D).clone()
            if case["norm"]:
                for lo, hi, w in ((0, H, "q_weight"), (H, H + Hk, "k_weight")):
                    x[:, lo:hi] *= t[w].double() / torch.sqrt(x[:, lo:hi].square().sum(-1, keepdim=True) / D + EPS)
            p = torch.arange(L - n, L, device="cuda")
            # complex numbers turned by the table's unit vectors (its 32-bit values are the input)
            z = torch.view_as_complex(t["rope"][p].double().contiguous())[:, None]
            first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
            second = first + (1 if case["interleaved"] else rot // 2)
            turned = torch.complex(x[:, :H + Hk, first], x[:, :H + Hk, second]) * z
            x[:, :H + Hk, first], x[:, :H + Hk, second] = turned.real, turned.imag
            q.append(x[:, :H])
            if mx:
                keys.append(_exact_codes(x[:, H:H + Hk].contiguous()))
                values.append(_exact_codes(x[:, H + Hk:].contiguous()))
            else:
                for i in range(-(-L // page)):
                    lo, hi = max(i * page, L - n), min((i + 1) * page, L)
                    if lo < hi:
                        at, a, b = int(t["table"][s, i]), lo - (L - n), hi - (L - n)
                        k[at, :, lo - i * page:hi - i * page] = x[a:b, H:H + Hk].transpose(0, 1)
                        v[at, :, lo - i * page:hi - i * page] = x[a:b, H + Hk:].transpose(0, 1)
            row += n
        return {"q": torch.cat(q), "k": torch.cat(keys) if mx else k, "v": torch.cat(values) if mx else v}
    outs = []
    for s, (n, L) in enumerate(zip(news, lengths)):
        o = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
        if L > 0:
            k, v = (_exact_cache(case, t, name, held[s]) for name in ("k", "v"))
            hide = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
            for h in range(H):
                kh, vh = (x[:, h // (H // Hk)].reshape(-1, D)[:L] for x in (k, v))
                score = (t["q"][row:row + n, h].double() @ kh.T.contiguous()) / D ** 0.5
                o[:, h] = torch.softmax(score.masked_fill_(hide, -math.inf), -1) @ vh
        outs.append(o)
        row += n
    return [torch.cat(outs)]


def _exact_token(case, t, r):
    x = t["x"][r].double().cpu().numpy()
    temperature, top_p, min_p, u = (float(t[k][r]) for k in ("temperature", "top_p", "min_p", "uniform"))
    order = np.lexsort((np.arange(len(x)), -x))
    if temperature <= 0.0:
        return int(order[0])
    w = np.exp((x - x.max()) / temperature)
    kept = [i for i in order[:int(t["top_k"][r]) or len(x)] if w[i] >= min_p]
    if top_p < 1.0:
        kept = kept[:int(np.searchsorted(np.cumsum(w[kept]), top_p * math.fsum(w[kept]))) + 1]
    sums = np.cumsum(w[kept])
    return int(kept[int(np.searchsorted(sums, u * sums[-1], side="right"))])
