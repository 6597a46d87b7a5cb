"""The operators of a step over a batch of sequences with a paged cache, as they are measured.

  append     new rows of q | k | v: rotary positions on q and k, keys and values into their sequences' pages
             (mvlm_kv_append_paged)
  attention  the new rows of each sequence over its pages, causal within the new rows: single tokens, chunks of a
             prompt, and both in one batch (mvlm_attention_paged)
  logits     penalties of repeated tokens, biases and grammar masks on a batch's logits (mvlm_logits_process)

Where `own` is false, run() computes the same with elementary torch operations in 32 bits.  Calls that a program
makes once a step for single tokens are replayed from a plan, prompts are called directly.
"""
import ctypes
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases -------------------------------------------------------------------

def _append(name, x, cache, seqs, chunks, new, cached, heads, kv_heads, dim, rot, interleaved, page):
    return {"name": name, "kind": "append", "x": x, "cache": cache, "seqs": seqs, "chunks": chunks, "new": new,
            "cached_lo": cached, "cached_hi": cached, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "interleaved": interleaved, "page": page, "idle": 0}


def _attention(name, out, cache, seqs, chunks, new, lo, hi, heads, kv_heads, dim, page, idle=0):
    return {"name": name, "kind": "attention", "out": out, "cache": cache, "seqs": seqs, "chunks": chunks, "new": new,
            "cached_lo": lo, "cached_hi": hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "idle": idle}


def _logits(name, dtype, rows, vocab, history, bias, mask):
    return {"name": name, "kind": "logits", "dtype": dtype, "rows": rows, "vocab": vocab, "history": history,
            "bias": bias, "mask": mask}


def listed():
    return [
        # one conversation, one token of Phi-1.5 (32 of a head's 64 dims are rotated): the launch is what counts
        _append("append_one_token", "f32", "f16", 1, 0, 1, 511, 32, 32, 64, 32, False, 16),
        # sixteen conversations decoded together, as many rows as the quantized products take
        _append("append_16_tokens", "f32", "f16", 16, 0, 1, 1000, 32, 32, 64, 32, False, 16),
        # an image's 729 positions and some text, all new
        _append("append_prompt_768", "f16", "f16", 1, 1, 768, 0, 32, 32, 64, 32, False, 64),
        # long prompts of four users at once, shared key heads, interleaved pairs
        _append("append_prompts_4x4096", "bf16", "bf16", 4, 4, 4096, 0, 32, 8, 128, 128, True, 64),
        # one Phi-1.5 conversation in mid-length
        _attention("decode_1x512", "f32", "f16", 1, 0, 1, 511, 511, 32, 32, 64, 16),
        # sixteen of them, of all lengths up to the model's 2048 positions, two of the places idle
        _attention("decode_16x2047", "f32", "f16", 16, 0, 1, 30, 2046, 32, 32, 64, 16, 2),
        # few users with long documents, eight key heads shared by thirty-two
        _attention("decode_4x32768", "bf16", "bf16", 4, 0, 1, 20000, 32767, 32, 8, 128, 64),
        # the image and its text through one layer
        _attention("prompt_768", "f16", "f16", 1, 1, 768, 0, 0, 32, 32, 64, 64),
        # a chunk of a long document behind what is cached of it
        _attention("chunk_2048_on_8192", "bf16", "bf16", 1, 1, 2048, 8192, 8192, 32, 8, 128, 64),
        # a chunk of one prompt in the same step as eleven single tokens; pages off the tile
        _attention("mixed_256_and_11", "f16", "f16", 12, 1, 256, 100, 1700, 32, 32, 64, 48),
        # the logits of one conversation
        _logits("logits_1x51200", "f32", 1, 51200, 512, 16, True),
        # a full server: many rows, a large vocabulary, long histories
        _logits("logits_128x128000", "f32", 128, 128000, 4096, 64, True),
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def _drawn(rng):
    kind = rng.choice(["append", "attention", "attention", "logits"])
    if kind == "logits":
        return {"kind": kind, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "rows": _log(rng, 1, 128),
                "vocab": _log(rng, 1000, 128000), "history": _log(rng, 1, 4096), "bias": rng.choice([0, 1, 16, 64]),
                "mask": rng.random() < 0.6}
    dim = rng.choice([64, 64, 72, 80, 96, 128, 128])
    kv_heads = rng.choice([2, 4, 8, 8, 16, 32])
    case = {"kind": kind, "cache": rng.choice(["f16", "bf16"]), "heads": kv_heads * rng.choice([1, 1, 2, 4, 8]),
            "kv_heads": kv_heads, "dim": dim, "page": rng.choice([8, 16, 32, 48, 64, 128, 256]), "idle": 0}
    if kind == "append":
        case["x"] = rng.choice(["f32", case["cache"]])
        case["rot"] = rng.choice([dim // 2, dim])
        case["interleaved"] = rng.random() < 0.5
    else:
        case["out"] = rng.choice(["f32", case["cache"], case["cache"]])
    form = rng.choice(["single", "chunk", "mixed"])
    if form == "single":
        case |= {"seqs": _log(rng, 1, 64), "chunks": 0, "new": 1}
        case["cached_lo"] = rng.randrange(0, 200)
        case["cached_hi"] = case["cached_lo"] + _log(rng, 1, max(2, 100000 // case["seqs"]))
        if kind == "attention" and case["seqs"] > 2 and rng.random() < 0.4:
            case["idle"] = rng.randrange(1, case["seqs"] // 2 + 1)
    else:
        chunks = rng.randrange(1, 5)
        case |= {"seqs": chunks + (rng.randrange(1, 12) if form == "mixed" else 0), "chunks": chunks,
                 "new": _log(rng, 2, 2048 // chunks)}
        case["cached_lo"] = rng.choice([0, 0, rng.randrange(0, 1000)])
        case["cached_hi"] = case["cached_lo"] + rng.choice([0, _log(rng, 1, 4000)])
    return case


def draw(rng):
    most = [max(work(c)[k] for c in listed() if c["kind"] == "attention") for k in ("bytes", "flops")]
    while True:
        case = _drawn(rng)
        w = work(case)
        padded = 0 if case["kind"] != "attention" else case["seqs"] * case["heads"] * _news(case)[0] * max(_lengths(case))
        if case["heads" if case["kind"] != "logits" else "rows"] <= 128 and w["bytes"] <= most[0] \
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


def work(case):
    if case["kind"] == "logits":
        es, n, rows = SIZE[case["dtype"]], case["vocab"], case["rows"]
        b = rows * (2 * n * es + 4 * case["history"] + 8 * case["bias"] + 24) + (rows * ((n + 31) // 32) * 4 if case["mask"] else 0)
        return {"bytes": b, "flops": 4 * rows * n}
    H, Hk, D, cs = case["heads"], case["kv_heads"], case["dim"], SIZE[case["cache"]]
    news, lengths = _news(case), _lengths(case)
    rows, width = sum(news), -(-max(lengths) // case["page"])
    if case["kind"] == "append":
        b = rows * ((H + 2 * Hk) * D * (SIZE[case["x"]] + cs) + case["rot"] * 4 + 4) + 8 * case["seqs"]
        return {"bytes": b, "flops": 3 * rows * (H + Hk) * case["rot"]}
    pairs = sum(n * L - n * (n - 1) // 2 for n, L in zip(news, lengths) if L > 0)
    b = rows * H * D * (cs + SIZE[case["out"]]) + sum(lengths) * 2 * Hk * D * cs + 4 * case["seqs"] * (width + 2)
    return {"bytes": b, "flops": 4 * H * D * pairs}


# ---- inputs ------------------------------------------------------------------------

class _Source:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=self.gen).to(dtype)

    def ints(self, hi, *shape):
        return torch.randint(0, hi, shape, dtype=torch.int32, device="cuda", generator=self.gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    src = _Source(seed)
    if case["kind"] == "logits":
        rows, n, h, nb = case["rows"], case["vocab"], case["history"], case["bias"]
        t = {"x": src.normal(rows, n, dtype=TORCH[case["dtype"]], std=4.0)}
        # text repeats itself: most of a history comes from few tokens; lengths and prompts are the requests' own
        common, rare = src.ints(max(1, min(n, 300)), rows, h), src.ints(n, rows, h)
        t["history"] = torch.where(src.ints(4, rows, h) > 0, (common.long() * 7919 % n).int(), rare)
        t["history_len"] = h - src.ints(h // 2 + 1, rows)
        t["generated_from"] = (t["history_len"].float() * torch.rand(rows, device="cuda", generator=src.gen)).int()
        t["penalties"] = torch.rand(rows, 3, device="cuda", generator=src.gen) * 0.5
        t["penalties"][:, 0] += 1.0
        if nb:
            t["bias_ids"], t["bias_values"] = src.ints(n, rows, nb), src.normal(rows, nb, std=5.0)
            t["bias_len"] = nb - src.ints(nb // 2 + 1, rows)
        if case["mask"]:
            t["allowed"] = torch.randint(-2**31, 2**31, (rows, (n + 31) // 32), dtype=torch.int32, device="cuda",
                                         generator=src.gen)
        return t
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    news, lengths, page = _news(case), _lengths(case), case["page"]
    cache = TORCH[case["cache"]]
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
    t = {"kv_len": _ints(lengths), "table": table, "k": src.normal(pages, Hk, page, D, dtype=cache),
         "v": src.normal(pages, Hk, page, D, dtype=cache)}
    if case["chunks"]:
        t["row_start"] = _ints(start)
    if case["kind"] == "attention":
        t["q"] = src.normal(start[-1], H, D, dtype=cache)
        return t
    t["qkv"] = src.normal(start[-1], (H + 2 * Hk) * D, dtype=TORCH[case["x"]])
    t["rope"] = _rope_table(width * page, case["rot"]).float()
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
    return {"append": _plain_append, "attention": _plain_attention, "logits": _plain_logits}[state["case"]["kind"]](
        state["case"], state["t"])


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


def _plain_append(case, t):
    H, Hk, D, cache = case["heads"], case["kv_heads"], case["dim"], TORCH[case["cache"]]
    seq, _, p = _rows(case, t)
    x = t["qkv"].float().view(-1, H + 2 * Hk, D)
    qk = _rotate(x[:, :H + Hk], t["rope"][p], case["rot"], case["interleaved"]).to(cache)
    page, slot = t["table"][seq, p // case["page"]].long(), p % case["page"]
    t["k"][page, :, slot] = qk[:, H:]
    t["v"][page, :, slot] = x[:, H + Hk:].to(cache)
    return {"q": qk[:, :H], "k": t["k"], "v": t["v"]}


def _plain_attention(case, t):
    H, Hk, D, S = case["heads"], case["kv_heads"], case["dim"], case["seqs"]
    new, L = max(_news(case)), max(_lengths(case))
    seq, j, p = _rows(case, t)
    pages = t["table"].clamp_min(0).long()
    k = t["k"][pages].transpose(1, 2).reshape(S, Hk, -1, D)[:, :, :L].float()
    v = t["v"][pages].transpose(1, 2).reshape(S, Hk, -1, D)[:, :, :L].float()
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


def _plain_logits(case, t):
    rows, n = case["rows"], case["vocab"]
    at = torch.arange(case["history"], device="cuda")
    ids = t["history"].long()
    seen = (at < t["history_len"][:, None]).float()
    made = seen * (at >= t["generated_from"][:, None])
    c = torch.zeros(rows, n, device="cuda").scatter_add_(1, ids, seen)
    g = torch.zeros(rows, n, device="cuda").scatter_add_(1, ids, made)
    rep, freq, pres = (t["penalties"][:, i:i + 1] for i in range(3))
    x = t["x"].float()
    x = torch.where(c > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (g * freq + (g > 0).float() * pres)
    if case["bias"]:
        entry = torch.arange(case["bias"], device="cuda").expand(rows, -1)
        entry = torch.where(entry < t["bias_len"][:, None], entry, -1)
        last = torch.full((rows, n), -1, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(1, t["bias_ids"].long(), entry, "amax")
        x = x + torch.where(last >= 0, t["bias_values"].gather(1, last.clamp_min(0)), 0.0)
    if case["mask"]:
        bits = (t["allowed"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x = x.masked_fill(bits.view(rows, -1)[:, :n] == 0, -math.inf)
    return [x.to(TORCH[case["dtype"]])]


# ---- the framework's calls -------------------------------------------------------------

_device = None


class _InPlace:
    """A buffer as torch sees it.  The C ABI's handles are opaque and have no accessor for the device address, so
    it is read from the handle (the second word of mvlm_buffer); the buffer lives as long as the tensor."""

    def __init__(self, buf, count, typestr):
        self.buf = buf
        address = ctypes.c_uint64.from_address(buf.handle.value + 8).value
        self.__cuda_array_interface__ = {"shape": (count,), "typestr": typestr, "data": (address, False), "version": 2}


def _view(buf, dtype, shape):
    typestr = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.int32: "<i4"}[dtype]
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
    names = {"f32": m.F32, "f16": m.F16, "bf16": m.BF16}

    def empty(dtype, *shape):
        buf = dev.alloc(math.prod(shape) * SIZE[dtype])
        return buf, _view(buf, TORCH[dtype], shape)

    b = {}
    for name in list(t):
        b[name] = dev.alloc(t[name].numel() * t[name].element_size())
        place = _view(b[name], t[name].dtype, t[name].shape)
        place.copy_(t[name])
        t[name] = place
    torch.cuda.synchronize()
    if case["kind"] == "logits":
        rows, n = case["rows"], case["vocab"]
        out, seen = empty(case["dtype"], rows, n)
        controls = m.LogitControls(history=b["history"], history_len=b["history_len"],
                                   generated_from=b["generated_from"], history_width=case["history"],
                                   penalties=b["penalties"], bias_ids=b.get("bias_ids"),
                                   bias_values=b.get("bias_values"), bias_len=b.get("bias_len"),
                                   bias_width=case["bias"], allowed=b.get("allowed"))
        plan = m.Plan(dev)
        plan.add_logits_process(b["x"], names[case["dtype"]], rows, n, n, controls, out)
        state |= {"plan": plan, "call": plan.run, "out": [seen]}
        return
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    rows = sum(_news(case))
    cache = m.PagedKV(b["k"], b["v"], names[case["cache"]], num_pages=t["k"].shape[0], page_size=case["page"],
                      kv_heads=Hk, head_dim=D)
    batch = m.PagedBatch(case["seqs"], rows, b["kv_len"], b["table"], t["table"].shape[1], row_start=b.get("row_start"))
    if case["kind"] == "append":
        q, seen = empty(case["cache"], rows, H, D)
        rope = m.Rope(b["rope"], positions=t["rope"].shape[0], rot_dim=case["rot"], interleaved=case["interleaved"])
        args = (b["qkv"], names[case["x"]], (H + 2 * Hk) * D, batch, cache, H, q, rope)
        direct, add, out = dev.kv_append_paged, "add_kv_append_paged", {"q": seen, "k": t["k"], "v": t["v"]}
    else:
        o, seen = empty(case["out"], rows, H, D)
        args = (b["q"], batch, cache, o, names[case["out"]], H)
        direct, add, out = dev.attention_paged, "add_attention_paged", [seen]
    state["out"] = out
    if case["chunks"]:
        state["call"] = lambda: direct(*args)
        return
    plan = m.Plan(dev)
    getattr(plan, add)(*args)
    state |= {"plan": plan, "call": plan.run}


# ---- from the definitions, in 64 bits ------------------------------------------------------

def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "logits":
        return [torch.stack([_exact_row(case, t, r) for r in range(case["rows"])])]
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    news, lengths = _news(case), _lengths(case)
    outs, row = [], 0
    if case["kind"] == "append":
        k, v, rot = t["k"].double(), t["v"].double(), case["rot"]
        for s, (n, L) in enumerate(zip(news, lengths)):
            x = t["qkv"][row:row + n].double().view(n, H + 2 * Hk, D)
            p = torch.arange(L - n, L, device="cuda")
            # complex numbers turned by the table's unit vectors (its 32-bit values are the input)
            z = torch.view_as_complex(t["rope"][p].double().contiguous())[:, None]
            first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
            second = first + (1 if case["interleaved"] else rot // 2)
            turned = torch.complex(x[:, :H + Hk, first], x[:, :H + Hk, second]) * z
            x[:, :H + Hk, first], x[:, :H + Hk, second] = turned.real, turned.imag
            outs.append(x[:, :H])
            for i in range(-(-L // page)):
                lo, hi = max(i * page, L - n), min((i + 1) * page, L)
                if lo < hi:
                    at, a, b = int(t["table"][s, i]), lo - (L - n), hi - (L - n)
                    k[at, :, lo - i * page:hi - i * page] = x[a:b, H:H + Hk].transpose(0, 1)
                    v[at, :, lo - i * page:hi - i * page] = x[a:b, H + Hk:].transpose(0, 1)
            row += n
        return {"q": torch.cat(outs), "k": k, "v": v}
    for s, (n, L) in enumerate(zip(news, lengths)):
        o = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
        if L > 0:
            used = t["table"][s, :-(-L // page)].long()
            hide = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
            for h in range(H):
                kh = t["k"][used, h // (H // Hk)].double().reshape(-1, D)[:L]
                vh = t["v"][used, h // (H // Hk)].double().reshape(-1, D)[:L]
                score = (t["q"][row:row + n, h].double() @ kh.T.contiguous()) / D ** 0.5
                o[:, h] = torch.softmax(score.masked_fill_(hide, -math.inf), -1) @ vh
        outs.append(o)
        row += n
    return [torch.cat(outs)]


def _exact_row(case, t, r):
    x = t["x"][r].double()
    ids = t["history"][r, :int(t["history_len"][r])].long()
    rep, freq, pres = (float(v) for v in t["penalties"][r].double())
    known = torch.unique(ids)
    x[known] = torch.where(x[known] > 0, x[known] / rep, x[known] * rep)
    made, times = torch.unique(ids[int(t["generated_from"][r]):], return_counts=True)
    x[made] -= times.double() * freq + pres
    if case["bias"]:
        count = int(t["bias_len"][r])
        entries = dict(zip(t["bias_ids"][r, :count].tolist(), t["bias_values"][r, :count].double().tolist()))
        x[list(entries)] += torch.tensor(list(entries.values()), dtype=torch.float64, device="cuda")
    if case["mask"]:
        word = torch.arange(case["vocab"], device="cuda")
        x[(t["allowed"][r].long()[word // 32] >> (word % 32)) % 2 == 0] = -math.inf
    return x
