"""What the operators around the quantized products are timed on: the cache append with its position rotation, the
attention over the paged cache, and the rules on the logits, as an engine calls them while it serves a model.

The cache is pages of `page` tokens; a page holds K, then V, each [head][token][dim] in fp16, or in int8 rows followed
by the f32 scales of the head's rows. A sequence's pages are listed in its row of the table. Activations are 32-bit, as
the projections write them.
"""
import math
import random
import weakref

import torch

own = False

DEV = "cuda"
PAD = 64                          # readable bytes past a wrapped tensor
NONE = -1                         # a table entry without a page
EPS = 1e-6
MOST_KV = 2.4e9                   # bytes of keys and values that a pass reads
MOST_FLOPS = 7e10
MOST_LOGITS = 32 * 131072


def listed():
    return [
        # one request, one token: q and k normed and rotated, k and v into an fp16 cache
        {"name": "append_token", "op": "append", "kv": "f16", "heads": 32, "kv_heads": 4, "dim": 64, "page": 16, "seqs": 1, "new": 1,
         "len": 700, "rot": 64, "halves": True, "norm": True, "fused": False},
        # a batch of requests, one token each, into an 8-bit cache, from the rows of one q + k + v projection
        {"name": "append_batch_i8", "op": "append", "kv": "i8", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "seqs": 96, "new": 1,
         "len": 8192, "rot": 128, "halves": False, "norm": False, "fused": True},
        # prompts of several requests, of lengths of their own, a quarter of the channels rotated
        {"name": "append_prompts", "op": "append", "kv": "f16", "heads": 16, "kv_heads": 4, "dim": 256, "page": 64, "seqs": 7, "new": 1021,
         "len": 2500, "rot": 64, "halves": True, "norm": True, "fused": True},
        # decode: one request, a short context
        {"name": "attn_token", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "seqs": 1, "new": 1, "len": 517,
         "window": 0},
        # decode: one request at the end of a very long context, split over the length
        {"name": "attn_long", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "seqs": 1, "new": 1, "len": 130001,
         "window": 0},
        # decode: a batch of requests whose contexts have every length up to 16384
        {"name": "attn_batch", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "seqs": 64, "new": 1, "len": 16384,
         "window": 0},
        # the same over an 8-bit cache, wide heads, eight query heads to a key head
        {"name": "attn_batch_i8", "op": "attn", "kv": "i8", "heads": 16, "kv_heads": 2, "dim": 256, "page": 16, "seqs": 40, "new": 1, "len": 9001,
         "window": 0},
        # a draft of five tokens of each request is verified, under a sliding window
        {"name": "attn_draft", "op": "attn", "kv": "f16", "heads": 24, "kv_heads": 8, "dim": 96, "page": 16, "seqs": 24, "new": 5, "len": 4100,
         "window": 1024},
        # chunks of three prompts over what is cached of them
        {"name": "attn_prompt", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "seqs": 3, "new": 1000, "len": 3001,
         "window": 0},
        # one request before its sampler: the penalties of the last 64 tokens
        {"name": "logits_token", "op": "logits", "rows": 1, "vocab": 65536, "history": 64, "bias": 0, "masked": 0},
        # a batch: penalties over whole conversations, some biased tokens
        {"name": "logits_batch", "op": "logits", "rows": 32, "vocab": 131072, "history": 4096, "bias": 50, "masked": 0},
        # requests under grammars: most of the vocabulary is masked, for one request all of it
        {"name": "logits_grammar", "op": "logits", "rows": 48, "vocab": 50021, "history": 16000, "bias": 7, "masked": 30},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append"] * 2 + ["attn"] * 4 + ["logits"] * 2)
    if op == "logits":
        vocab = _log(rng, 1000, 200000)
        rows = _log(rng, 1, max(1, min(256, MOST_LOGITS // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "history": _log(rng, 1, min(32768, 400000 // rows)),
                "bias": rng.choice([0, _log(rng, 1, 300)]), "masked": rng.choice([0, rng.randrange(1, rows + 1)])}
    case = {"op": op, "kv": rng.choice(["f16", "f16", "i8"]), "kv_heads": rng.choice([1, 2, 3, 4, 8, 8, 16])}
    case["dim"] = rng.choice([64, 64, 96, 128, 128, 128, 256])
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 4, 5, 6, 7, 8, 8, 12, 16])
    if 3072 in (case["heads"] * case["dim"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]):
        case["heads"] = 9 * case["kv_heads"]
    case["page"] = rng.choice([16, 16, 32, 64, 128, 256])
    if op == "append":
        seqs = _log(rng, 1, 128)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(3, 4000 // seqs))
        while seqs * new * case["heads"] * case["dim"] > 7 * 1021 * 4096:
            new = max(1, new // 2)
            seqs = max(1, seqs // 2) if new == 1 else seqs
        case.update(seqs=seqs, new=new, len=new + _log(rng, 1, 30000), rot=case["dim"] // rng.choice([1, 1, 2, 4]),
                    halves=rng.random() < 0.6, norm=case["kv"] == "f16" and rng.random() < 0.5, fused=rng.random() < 0.5)
        return case
    kind = rng.choice(["token", "token", "token", "draft", "prompt"])
    seqs = _log(rng, 1, 128 if kind != "prompt" else 6)
    new = 1 if kind == "token" else rng.randrange(2, 9) if kind == "draft" else _log(rng, 16, 1024)
    length = new + _log(rng, 1, 130000 if kind != "prompt" else 4000)
    row = case["kv_heads"] * case["dim"] * (4 if case["kv"] == "f16" else 2)
    while seqs * length * row > 0.8 * MOST_KV or seqs * new * length * case["heads"] * case["dim"] * 4.0 > MOST_FLOPS:
        if seqs > 1:
            seqs //= 2
        else:
            length = max(new, length // 2)
            new = max(1, new // 2) if length == new else new
    case.update(seqs=seqs, new=new, len=length, window=0 if rng.random() < 0.7 else _log(rng, 1, 8192))
    return case


def _ragged(case):
    """The sequences' lengths and new tokens: the first has the most of both, the others any."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["new"], case["len"]))
    new = [case["new"]] + [rng.randrange(max(1, case["new"] // 3), case["new"] + 1) for _ in range(case["seqs"] - 1)]
    lens = [case["len"]] + [rng.randrange(n, case["len"] + 1) for n in new[1:]]
    return new, lens


def _seen(case):
    """Of each sequence: the cached tokens that any of its new ones sees, and the pairs of a new token and a seen one."""
    got = []
    for n, length in zip(*_ragged(case)):
        w = case["window"] or length
        first = length - n
        got.append((length - max(0, first - w + 1), sum(min(first + i + 1, w) for i in range(n))))
    return got


def work(case):
    if case["op"] == "logits":
        r, v = case["rows"], case["vocab"]
        words = sum(_counts(case))
        return {"bytes": 8.0 * r * v + 4.0 * words + 8.0 * r * case["bias"] + case["masked"] * ((v + 31) // 32 * 4) + 24.0 * r,
                "flops": 1.0 * r * v + 6.0 * words}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    row = d * 2 if case["kv"] == "f16" else d + 4
    tokens = sum(_ragged(case)[0])
    if case["op"] == "append":
        return {"bytes": 4.0 * tokens * (2 * h + 2 * kv) * d + 2.0 * tokens * kv * row + 4.0 * tokens * case["rot"] + 8.0 * tokens,
                "flops": 6.0 * tokens * (h + 2 * kv) * d}
    seen = _seen(case)
    return {"bytes": 2.0 * kv * row * sum(s for s, _ in seen) + 8.0 * tokens * h * d, "flops": 4.0 * h * d * sum(p for _, p in seen)}


# ---- inputs ------------------------------------------------------------------

def _counts(case):
    """The tokens of each row's history: the first has the most, one of several has none."""
    rng = random.Random("%d %d" % (case["rows"], case["history"]))
    n = [case["history"]] + [rng.randrange(1, case["history"] + 1) for _ in range(case["rows"] - 1)]
    if case["rows"] > 2:
        n[2] = 0
    return n


def _starts(counts):
    return torch.tensor([0] + counts).cumsum(0)


def _logits_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r, v = case["rows"], case["vocab"]
    counts = _counts(case)
    total = sum(counts)
    # words of a conversation: a few tokens are most of it
    u = torch.rand(total, device=DEV, generator=gen)
    s = {"z": 3 * torch.randn(r, v, device=DEV, generator=gen),
         "history": (v * u ** 4).to(torch.int32).clamp(max=v - 1), "history_starts": _starts(counts).to(torch.int32).to(DEV)}
    p = torch.rand(r, 3, device=DEV, generator=gen, dtype=torch.float64)
    s["penalties"] = torch.stack([1 + 0.3 * p[:, 0], 0.4 * p[:, 1], 0.5 * p[:, 2]], 1)
    s["history_row"] = torch.repeat_interleave(torch.arange(r), torch.tensor(counts)).to(DEV)
    if case["bias"]:
        b = min(case["bias"], v)
        first = torch.randint(0, v, (r, 1), device=DEV, generator=gen)
        s["bias_ids"] = ((first + torch.arange(b, device=DEV) * max(1, v // b)) % v).to(torch.int32).view(-1)
        s["bias_values"] = 4 * torch.randn(r * b, device=DEV, generator=gen)
        s["bias_starts"] = (torch.arange(r + 1, device=DEV) * b).to(torch.int32)
    if case["masked"]:
        m, words = case["masked"], (v + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (m, words), device=DEV, generator=gen, dtype=torch.int32)
        for _ in range(3):                # one token in sixteen stays
            bits &= torch.randint(-2 ** 31, 2 ** 31, (m, words), device=DEV, generator=gen, dtype=torch.int32)
        if m > 1:
            bits[1] = 0                   # a grammar that allows nothing
        rows = torch.full((r,), NONE, dtype=torch.int32)
        rows[torch.randperm(r, generator=torch.Generator().manual_seed(seed))[:m]] = torch.arange(m, dtype=torch.int32)
        s["mask"], s["mask_of"] = bits, rows.to(DEV)
    return s


def _rope(positions, rot):
    """cos and sin of every position: [positions][2][rot / 2]."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos(), a.sin()], 1).float()


def _rows(n, gen, *shape):
    """Rows of keys or values: channels with magnitudes of their own."""
    scale = torch.exp(0.4 * torch.randn(shape[-1], device=DEV, generator=gen))
    return (torch.randn(n, *shape, device=DEV, generator=gen) * scale).to(torch.float16)


def _cache(case, pages, gen):
    """Pages of earlier tokens: fp16 [pages][2][heads][page][dim], or int8 rows and their scales as bytes."""
    shape = (2, case["kv_heads"], case["page"], case["dim"])
    x = torch.cat([_rows(min(256, pages - a), gen, *shape) for a in range(0, pages, 256)])
    if case["kv"] == "f16":
        return x
    out = torch.empty(pages, *shape[:2], case["page"] * (case["dim"] + 4), dtype=torch.uint8, device=DEV)
    q, scales = _parts(out, case)
    for a in range(0, pages, 256):
        f = x[a:a + 256].float()
        top = f.abs().amax(-1)
        q[a:a + 256] = torch.round(f * (127 / top)[..., None]).to(torch.int8)
        scales[a:a + 256] = top / 127
    return out


def _parts(cache, case):
    """The int8 rows and the scales of an 8-bit cache, as views."""
    n = case["page"] * case["dim"]
    return cache[..., :n].view(torch.int8).unflatten(-1, (case["page"], case["dim"])), cache[..., n:].view(torch.float32)


def _kv_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    new, lens = _ragged(case)
    h, kv, d, pt = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tokens, width = sum(new), (case["len"] + pt - 1) // pt
    table = torch.full((case["seqs"], width), NONE, dtype=torch.int32)
    used = []
    for i, (n, length) in enumerate(zip(new, lens)):
        # an append's earlier pages are not asked for: the table has none there
        first = (length - n) // pt if case["op"] == "append" else 0
        used += [(i, p) for p in range(first, (length + pt - 1) // pt)]
    order = torch.randperm(len(used) + 3, generator=host)[:len(used)].to(torch.int32)
    at = torch.tensor(used)
    table[at[:, 0], at[:, 1]] = order
    seq = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(new))
    starts = _starts(new)
    index = torch.arange(tokens) - starts[seq]
    pos = torch.tensor(lens)[seq] - torch.tensor(new)[seq] + index
    s = {"cache": _cache(case, len(used) + 3, gen), "table": table.to(DEV), "starts": starts.to(torch.int32).to(DEV),
         "lens": torch.tensor(lens, dtype=torch.int32).to(DEV), "seq": seq.to(DEV), "index": index.to(DEV), "pos": pos.to(DEV)}
    if case["op"] == "attn":
        sharp = torch.exp(0.5 * torch.randn(h, 1, device=DEV, generator=gen))
        s["q"] = sharp * torch.randn(tokens, h, d, device=DEV, generator=gen)
        return s
    if case["fused"]:
        rows = torch.randn(tokens, h + 2 * kv, d, device=DEV, generator=gen)
        s["rows"], s["q"], s["k"], s["v"] = rows, rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
    else:
        s["q"], s["k"], s["v"] = (torch.randn(tokens, n, d, device=DEV, generator=gen) for n in (h, kv, kv))
    s["rope"] = _rope(case["len"], case["rot"])
    if case["norm"]:
        s["q_norm"], s["k_norm"] = (1 + 0.2 * torch.randn(d, device=DEV, generator=gen) for _ in range(2))
    return s


# ---- the program's side ------------------------------------------------------

_program = {}


def _context():
    """The one context of the program, on a torch stream of its own."""
    if not _program:
        import __graft_entry__
        _program["eff"] = __graft_entry__.package()
        _program["stream"] = torch.cuda.Stream()
        _program["ctx"] = _program["eff"].Context(0)
        _program["ctx"].set_stream(_program["stream"].cuda_stream)
    return _program["eff"], _program["ctx"]


def _wrap(t):
    """A tensor's memory as one of the library's buffers; the tensor is moved to memory with readable bytes after it."""
    eff, ctx = _context()
    size = t.numel() * t.element_size()
    memory = torch.empty(size + PAD, device=DEV, dtype=torch.uint8)
    view = memory[:size].view(t.dtype).view(t.shape)
    view.copy_(t)
    h = eff.ctypes.c_void_p()
    ctx._check(eff.lib().eff_buf_wrap(ctx.h, memory.data_ptr(), size, eff.ctypes.byref(h)))
    b = eff.Buffer(ctx, h, size)
    weakref.finalize(b, eff.lib().eff_buf_free, ctx.h, h)   # gives the handle back; the memory is torch's
    return view, b


def _handles(case, s):
    """The plan that a program keeps: the cache, the batch, the rows, the rules."""
    eff, ctx = _context()
    b = {}
    for key in ("z", "out", "cache", "table", "starts", "lens", "q", "k", "v", "rows", "rope", "q_norm", "k_norm", "history",
                "history_starts", "penalties", "bias_ids", "bias_values", "bias_starts", "mask", "mask_of"):
        if key in s and not (key in "qkv" and "rows" in s):
            s[key], b[key] = _wrap(s[key])
    if case["op"] == "logits":
        rules = eff.LogitsRules(**{k: b[k] for k in b if k not in ("z", "out")}, mask_count=case["masked"])
        return {"buffers": b, "rules": rules}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    pages = s["cache"].shape[0]
    cache = eff.KvCache({"f16": eff.KV_F16, "i8": eff.KV_I8}[case["kv"]], kv, d, case["page"], pages, b["cache"])
    batch = eff.KvBatch(b["table"], b["starts"], b["lens"], seqs=case["seqs"], tokens=s["seq"].numel(), table_pages=s["table"].shape[1],
                        max_new=case["new"], max_len=case["len"])
    if case["op"] == "attn":
        return {"buffers": b, "cache": cache, "batch": batch}
    if "rows" in s:
        n, at = (h + 2 * kv) * d, {"q": (b["rows"], 0), "k": (b["rows"], h * d), "v": (b["rows"], (h + kv) * d)}
        at = {**at, "q_stride": n, "k_stride": n, "v_stride": n}
    else:
        at = {key: (b[key], 0) for key in "qkv"}
    rows = eff.KvRows(**at, q_out=b["out"], q_heads=h, rope=b["rope"], rope_positions=case["len"], rope_dim=case["rot"],
                      rope_mode=eff.ROPE_HALVES if case["halves"] else eff.ROPE_PAIRS, q_norm=b.get("q_norm"), k_norm=b.get("k_norm"), eps=EPS)
    return {"buffers": b, "cache": cache, "batch": batch, "kv_rows": rows}


def prepare(case, seed):
    s = _logits_inputs(case, seed) if case["op"] == "logits" else _kv_inputs(case, seed)
    s["case"] = case
    s["out"] = torch.empty_like(s["z"]) if case["op"] == "logits" else torch.empty(s["q"].shape, device=DEV)
    if case["op"] == "append" and case["kv"] == "i8":
        s["values"] = torch.empty(_parts(s["cache"], case)[0].shape, device=DEV, dtype=torch.float16)
    if own:
        s["own"] = _handles(case, s)
    torch.cuda.synchronize()
    return s


def _own_run(s):
    _, ctx = _context()
    case, p = s["case"], s["own"]
    if case["op"] == "logits":
        ctx.logits_apply(p["buffers"]["z"], p["buffers"]["out"], case["rows"], case["vocab"], p["rules"])
        return s["out"]
    if case["op"] == "attn":
        ctx.kv_attn(p["cache"], p["batch"], p["buffers"]["q"], p["buffers"]["out"], case["heads"], case["dim"] ** -0.5, case["window"])
        return s["out"]
    ctx.kv_append(p["cache"], p["batch"], p["kv_rows"])
    if case["kv"] == "f16":
        return {"q": s["out"], "cache": s["cache"]}
    with torch.cuda.stream(_program["stream"]):
        return _values(s)


def _values(s):
    """The rotated q, and the 8-bit cache as the values it stands for."""
    q, scales = _parts(s["cache"], s["case"])
    torch.mul(q, scales[..., None], out=s["values"])
    return {"q": s["out"], "cache": s["values"]}


# ---- plain forms -------------------------------------------------------------

def _turn(x, s):
    """Norm and rotation of rows [tokens][heads][dim]."""
    case, r = s["case"], s["case"]["rot"]
    c, t = s["rope"][s["pos"]].unbind(1)
    c, t = c[:, None], t[:, None]
    if case["halves"]:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * c - b * t, a * t + b * c], -1)
    else:
        a, b = x[..., :r:2], x[..., 1:r:2]
        y = torch.stack([a * c - b * t, a * t + b * c], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _append(s):
    case, pt = s["case"], s["case"]["page"]
    q, k, v = s["q"], s["k"], s["v"]
    if case["norm"]:
        q, k = _normed(q, s["q_norm"]), _normed(k, s["k_norm"])
    s["out"] = _turn(q, s)
    kv = torch.stack([_turn(k, s), v], 1)                         # [tokens][2][heads][dim]
    page, slot = s["table"][s["seq"], s["pos"] // pt].long(), s["pos"] % pt
    if case["kv"] == "f16":
        s["cache"][page, :, :, slot] = kv.to(torch.float16)
        return {"q": s["out"], "cache": s["cache"]}
    rows, scales = _parts(s["cache"], case)
    top = kv.abs().amax(-1)
    rows[page, :, :, slot] = torch.round(kv * torch.where(top > 0, 127 / top, top)[..., None]).to(torch.int8)
    scales[page, :, :, slot] = top * (1 / 127)
    return _values(s)


def _attn(s):
    case = s["case"]
    n, h, kv, d, pt = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    new, g = case["new"], h // kv
    pages = s["table"].clamp(min=0).long()
    if case["kv"] == "f16":
        x = s["cache"][pages].float()                             # [seqs][pages][2][heads][page][dim]
    else:
        rows, scales = _parts(s["cache"], case)
        x = rows[pages].float() * scales[pages][..., None]
    k, v = x.permute(2, 0, 3, 1, 4, 5).flatten(3, 4).unbind(0)    # [seqs][heads][length][dim]
    at = torch.arange(k.shape[2], device=DEV)
    q = torch.zeros(n, new, h, d, device=DEV)
    q[s["seq"], s["index"]] = s["q"]
    q = q.view(n, new, kv, g, d).permute(0, 2, 1, 3, 4).reshape(n, kv, new * g, d)
    pos = torch.full((n, new), -1, device=DEV)
    pos[s["seq"], s["index"]] = s["pos"]
    seen = at <= pos[..., None]
    if case["window"]:
        seen &= at > pos[..., None] - case["window"]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, kv, new, g, -1) * d ** -0.5
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    v = torch.where((at < s["lens"][:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.view(n, kv, new * g, -1), v).view(n, kv, new, g, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    s["out"] = o.permute(0, 2, 1, 3, 4).reshape(n, new, h, d)[s["seq"], s["index"]]
    return s["out"]


def _logits(s):
    z, v = s["z"], s["case"]["vocab"]
    count = torch.zeros(z.numel(), device=DEV).scatter_add_(0, s["history_row"] * v + s["history"], torch.ones_like(s["history"], dtype=torch.float32))
    count = count.view(z.shape)
    repeat, frequency, presence = s["penalties"].float().t()[..., None]
    y = torch.where(z > 0, z / repeat, z * repeat) - (frequency * count + presence)
    y = torch.where(count > 0, y, z)
    if "bias_ids" in s:
        y.view(z.shape).scatter_add_(1, s["bias_ids"].long().view(z.shape[0], -1), s["bias_values"].view(z.shape[0], -1))
    if "mask" in s:
        at = torch.arange(v, device=DEV)
        allowed = (s["mask"][s["mask_of"].clamp(min=0).long()][:, at >> 5] >> (at & 31)) & 1
        y = y.masked_fill((allowed == 0) & (s["mask_of"] >= 0)[:, None], -math.inf)
    s["out"] = y
    return y


def run(s):
    if own:
        return _own_run(s)
    return {"append": _append, "attn": _attn, "logits": _logits}[s["case"]["op"]](s)


# ---- in 64 bits --------------------------------------------------------------

def _exact_append(case, s):
    r, pt = case["rot"], case["page"]
    angles = s["rope"].double()[s["pos"]]
    c, t = angles[:, 0, None], angles[:, 1, None]

    def turned(x, w):
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * w.double()
        z = torch.complex(*((x[..., :r // 2], x[..., r // 2:r]) if case["halves"] else (x[..., 0:r:2], x[..., 1:r:2])))
        z = z * torch.complex(c, t)
        y = x.clone()
        if case["halves"]:
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        return y

    k, v = turned(s["k"], s.get("k_norm")), s["v"].double()
    if case["kv"] == "f16":
        cache = s["cache"].double()
    else:
        q, scales = _parts(s["cache"], case)
        cache = q.double() * scales.double()[..., None]
        k, v = (torch.round(x * 127 / x.abs().amax(-1, keepdim=True)) * x.abs().amax(-1, keepdim=True) / 127 for x in (k, v))
    table = s["table"].tolist()
    for i, (seq, pos) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
        page = cache[table[seq][pos // pt]]
        page[0, :, pos % pt], page[1, :, pos % pt] = k[i], v[i]
    return {"q": turned(s["q"], s.get("q_norm")), "cache": cache}


def _exact_attn(case, s):
    new, lens = _ragged(case)
    kv, d, pt = case["kv_heads"], case["dim"], case["page"]
    out, at = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64), 0
    for i, (n, length) in enumerate(zip(new, lens)):
        pages = s["table"][i, :(length + pt - 1) // pt].long()
        first = length - n
        for j in range(kv):
            if case["kv"] == "f16":
                k, v = s["cache"][pages, :, j].double().transpose(0, 1).reshape(2, -1, d)[:, :length]
            else:
                q, scales = _parts(s["cache"], case)
                k, v = (q[pages, :, j].double() * scales[pages, :, j].double()[..., None]).transpose(0, 1).reshape(2, -1, d)[:, :length]
            heads = slice(j * case["heads"] // kv, (j + 1) * case["heads"] // kv)
            for a in range(0, n, 128):
                m = min(128, n - a)
                x = s["q"][at + a:at + a + m, heads].double()
                pos, t = first + a + torch.arange(m, device=DEV)[:, None, None], torch.arange(length, device=DEV)
                hidden = t > pos
                if case["window"]:
                    hidden = hidden | (t <= pos - case["window"])
                w = torch.softmax((x @ k.t().contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                out[at + a:at + a + m, heads] = w @ v
        at += n
    return out


def _exact_logits(case, s):
    y, v = s["z"].double(), case["vocab"]
    row = s["history_row"] * v + s["history"].long()
    count = torch.bincount(row, minlength=y.numel()).view(y.shape)
    repeat, frequency, presence = (s["penalties"][:, i, None] for i in range(3))
    penal = torch.where(y > 0, y / repeat, y * repeat) - frequency * count - presence
    y = torch.where(count > 0, penal, y)
    for i in range(case["rows"]):
        if case["bias"]:
            a, b = s["bias_starts"][i:i + 2].tolist()
            y[i, s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        m = int(s["mask_of"][i]) if case["masked"] else NONE
        if m >= 0:
            bits = torch.stack([(s["mask"][m] >> j) & 1 for j in range(32)], 1).view(-1)[:v]
            y[i, bits == 0] = -math.inf
    return y


def exact(case, seed):
    s = _logits_inputs(case, seed) if case["op"] == "logits" else _kv_inputs(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "logits": _exact_logits}[case["op"]](case, s)
