"""What the operators of drafted, forked and packed requests are timed on: the cache append with positions of several
axes, attention for trees of drafts, with capped or biased scores and masks of documents and prefixes, and the copies
and compactions of cache pages, as an engine calls them while it serves a model.

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
MOST_KV = 8.5e8                   # keys and values that a pass reads
MOST_FLOPS = 4.9e10
MOST_MOVED = {"f16": 3.2e8, "i8": 2e7}   # bytes of the caches of all layers that a copy or a compaction is given
MOST_ROWS = 5 * 1531 * 2048       # values of q that an append is given


def listed():
    return [
        # one request, one token of a model with positions of time, height and width, q and k normed
        {"name": "append_token", "op": "append", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "seqs": 1, "new": 1,
         "len": 900, "rot": 128, "halves": True, "norm": True, "fused": False, "axes": 3, "mixed": False},
        # prompts with images: text at one position on all axes, patches at their row and column; axes dealt out pair by pair
        {"name": "append_images", "op": "append", "kv": "f16", "heads": 16, "kv_heads": 2, "dim": 128, "page": 64, "seqs": 5, "new": 1531,
         "len": 2600, "rot": 128, "halves": True, "norm": True, "fused": True, "axes": 3, "mixed": True},
        # trees of drafts of a batch, each draft at the position of its depth, into an 8-bit cache
        {"name": "append_drafts_i8", "op": "append", "kv": "i8", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "seqs": 48, "new": 25,
         "len": 8192, "rot": 64, "halves": False, "norm": False, "fused": True, "axes": 1, "mixed": False},
        # one request's tree of drafts over a short context
        {"name": "tree_one", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "seqs": 1, "new": 26, "len": 1026,
         "window": 0, "cap": 0.0, "bias": False, "mask": "tree"},
        # the trees of a batch over contexts of every length up to 16384
        {"name": "tree_batch", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "seqs": 16, "new": 32, "len": 16384,
         "window": 0, "cap": 0.0, "bias": False, "mask": "tree"},
        # small trees over an 8-bit cache, wide heads, under a sliding window
        {"name": "tree_batch_i8", "op": "attn", "kv": "i8", "heads": 16, "kv_heads": 2, "dim": 256, "page": 16, "seqs": 40, "new": 6, "len": 9001,
         "window": 4096, "cap": 0.0, "bias": False, "mask": "tree"},
        # decode: a batch whose scores are capped, wide heads
        {"name": "cap_batch", "op": "attn", "kv": "f16", "heads": 16, "kv_heads": 8, "dim": 256, "page": 32, "seqs": 48, "new": 1, "len": 8192,
         "window": 0, "cap": 50.0, "bias": False, "mask": ""},
        # decode: one request at the end of a long context, a bias of each head's own slope times the distance
        {"name": "bias_long", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 32, "dim": 128, "page": 64, "seqs": 1, "new": 1, "len": 20001,
         "window": 0, "cap": 0.0, "bias": True, "mask": ""},
        # prompts into which several documents were packed: a token sees its own document
        {"name": "documents", "op": "attn", "kv": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "seqs": 2, "new": 2500, "len": 2500,
         "window": 0, "cap": 0.0, "bias": False, "mask": "documents"},
        # forking: each request's last page, as far as it is filled, for all layers
        {"name": "fork", "op": "fork", "kv": "f16", "layers": 32, "kv_heads": 8, "dim": 128, "page": 32, "count": 30},
        # after verification: the accepted drafts of each request move up, for all layers
        {"name": "keep_batch", "op": "keep", "kv": "f16", "layers": 32, "kv_heads": 8, "dim": 128, "page": 16, "seqs": 24, "new": 32, "len": 4096,
         "kept": 7},
        # the same for one request and a small model with an 8-bit cache
        {"name": "keep_one_i8", "op": "keep", "kv": "i8", "layers": 16, "kv_heads": 2, "dim": 64, "page": 16, "seqs": 1, "new": 16, "len": 700,
         "kept": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _row(case):
    """Bytes of one token's row of a head."""
    return case["dim"] * 2 if case["kv"] == "f16" else case["dim"] + 4


def draw(rng):
    op = rng.choice(["append"] * 2 + ["attn"] * 5 + ["fork"] + ["keep"] * 2)
    case = {"op": op, "kv": rng.choice(["f16", "f16", "i8"]), "kv_heads": rng.choice([1, 2, 3, 4, 8, 8, 16])}
    case["dim"] = rng.choice([64, 64, 96, 128, 128, 128, 256])
    case["page"] = rng.choice([16, 16, 32, 64, 128, 256])
    if op in ("fork", "keep"):
        whole = 2 * case["kv_heads"] * _row(case) * case["page"]
        case["layers"] = rng.randrange(1, min(60, int(MOST_MOVED[case["kv"]] / whole / 8)) + 1)
        whole *= case["layers"]
        if op == "fork":
            case["count"] = _log(rng, 1, max(1, min(300, int(MOST_MOVED[case["kv"]] / whole / 2) - 1)))
            return case
        new = rng.randrange(2, 65)
        each = whole * (new // case["page"] + 2)
        case.update(seqs=_log(rng, 1, max(1, min(64, int(MOST_MOVED[case["kv"]] / each)))), new=new, len=new + _log(rng, 1, 30000), kept=rng.randrange(1, min(new, 12) + 1))
        return case
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 4, 5, 6, 7, 8, 8, 12, 16])
    if op == "append":
        axes = rng.choice([1, 1, 2, 3, 3])
        seqs = _log(rng, 1, 128)
        new = 1 if rng.random() < 0.3 else _log(rng, 2, 64 if axes == 1 else max(3, 4000 // seqs))
        while seqs * new * case["heads"] * case["dim"] > MOST_ROWS:
            new = max(1, new // 2)
            seqs = max(1, seqs // 2) if new == 1 else seqs
        case.update(seqs=seqs, new=new, len=new + _log(rng, 1, 30000), rot=case["dim"] // rng.choice([1, 1, 2, 4]), halves=rng.random() < 0.6,
                    norm=case["kv"] == "f16" and rng.random() < 0.5, fused=rng.random() < 0.5, axes=axes, mixed=axes > 1 and rng.random() < 0.5)
        return case
    kind = rng.choice(["tree", "tree", "token", "token", "prompt"])
    seqs = _log(rng, 1, 64 if kind == "token" else 32 if kind == "tree" else 6)
    new = 1 if kind == "token" else rng.randrange(2, 65) if kind == "tree" else _log(rng, 16, 2500)
    length = new + _log(rng, 8, 2000 if kind == "prompt" else 60000)
    while 2.0 * seqs * length * case["kv_heads"] * case["dim"] > MOST_KV or seqs * new * length * case["heads"] * case["dim"] * 4.0 > MOST_FLOPS:
        if seqs > 1:
            seqs //= 2
        else:
            length = max(new, length // 2)
            new = max(1, new // 2) if length == new else new
    mask = "tree" if kind == "tree" else "" if kind == "token" else rng.choice(["documents", "prefix", ""])
    cap = rng.choice([0.0, 20.0, 30.0, 50.0])
    bias = rng.random() < (0.3 if cap else 0.6 if not mask else 0.2)
    window = max(new, _log(rng, 16, 8192)) if mask in ("tree", "") and rng.random() < 0.3 else 0
    case.update(seqs=seqs, new=new, len=length, window=window, cap=cap if cap or bias or mask else 50.0, bias=bias, mask=mask)
    return case


def _ragged(case):
    """The sequences' lengths and new tokens: the first has the most of both, the others any."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["new"], case["len"]))
    new = [case["new"]] + [rng.randrange(max(1, case["new"] // 3), case["new"] + 1) for _ in range(case["seqs"] - 1)]
    lens = [case["len"]] + [rng.randrange(n, case["len"] + 1) for n in new[1:]]
    return new, lens


# ---- what new tokens see, and where they are ------------------------------------

def _trees(case):
    """The parent of each draft, of each sequence: the first has none, the others one of those before them."""
    rng = random.Random("tree %d %d" % (case["seqs"], case["new"]))
    return [[-1] + [max(0, i - 1 - int(rng.expovariate(0.4))) for i in range(1, n)] for n in _ragged(case)[0]]


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _tree_bits(parents, words):
    """Of each draft: a bit for each draft that it sees, its ancestors and itself, in words of 32."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return [[(r >> 32 * w & 0xFFFFFFFF) - (1 << 32 if r >> 32 * w & 1 << 31 else 0) for w in range(words)] for r in rows]


def _ranges(case):
    """Of each sequence, of each new token: the first cached position that it sees, and the one behind the last."""
    rng = random.Random("ranges %d %d" % (case["seqs"], case["len"]))
    got = []
    for n, length in zip(*_ragged(case)):
        pos = range(length - n, length)
        if case["mask"] == "prefix":              # the first part of a prompt sees all of itself
            prefix = rng.randrange(1, length + 1)
            got.append([(0, max(p + 1, prefix)) for p in pos])
            continue
        starts, at = [], 0                        # documents, from the beginning of the cache
        while at < length:
            size = _log(rng, 30, 900)
            starts += [at] * size
            at += size
        got.append([(starts[p], p + 1) for p in pos])
    return got


def _turns(case):
    """Of each sequence: the positions of its new tokens on each axis, [axis][token]."""
    rng = random.Random("turns %d %d" % (case["seqs"], case["len"]))
    got = []
    for i, (n, length) in enumerate(zip(*_ragged(case))):
        if case["axes"] == 1:                     # drafts: the position of their depth
            got.append([[length - n + d for d in _depths(_trees(case)[i])]])
            continue
        at, p = [], length - n                    # text and images in turn
        while len(at) < n:
            at += [(p + k,) * 3 for k in range(rng.randrange(1, 150))]
            p = at[-1][0] + 1
            rows, columns = rng.randrange(4, 33), rng.randrange(4, 33)
            at += [(p, p + y, p + x) for y in range(rows) for x in range(columns)]
            p += max(rows, columns)
        got.append([[min(x[a], length - 1) for x in at[:n]] for a in range(case["axes"])])
    return got


def _pair_axes(case):
    """The axis of each pair of the rotated channels: dealt out one by one, or side by side."""
    pairs, axes = case["rot"] // 2, case["axes"]
    return [i % axes for i in range(pairs)] if case["mixed"] else [min(axes - 1, i * 3 * axes // (pairs * 3 + 1)) for i in range(pairs)]


def _seen(case):
    """Of each sequence: the cached tokens that any of its new ones sees, and the pairs of a new token and a seen one."""
    got = []
    for i, (n, length) in enumerate(zip(*_ragged(case))):
        first, w = length - n, case["window"] or length
        if case["mask"] == "tree":
            d = _depths(_trees(case)[i])
            got.append((n + min(first, w - 1), sum(x + 1 + max(0, min(first, w - 1 - x)) for x in d)))
        elif case["mask"]:
            r = _ranges(case)[i]
            got.append((max(b for _, b in r) - min(a for a, _ in r), sum(b - a for a, b in r)))
        else:
            got.append((length - max(0, first - w + 1), sum(min(first + j + 1, w) for j in range(n))))
    return got


def work(case):
    kv, d = case["kv_heads"], case["dim"]
    row = _row(case)
    if case["op"] == "fork":
        moved = sum(t for _, t in _fork(case)) * case["layers"] * 2 * kv * row
        return {"bytes": 2.0 * moved + 12.0 * case["count"], "flops": 0.0}
    if case["op"] == "keep":
        paths = _kept(case)
        moved = sum(i != k for p in paths for i, k in enumerate(p)) * case["layers"] * 2 * kv * row
        return {"bytes": 2.0 * moved + 4.0 * sum(map(len, paths)) + 16.0 * case["seqs"], "flops": 0.0}
    h, tokens = case["heads"], sum(_ragged(case)[0])
    if case["op"] == "append":
        return {"bytes": 4.0 * tokens * (2 * h + 2 * kv) * d + 2.0 * tokens * kv * row + 4.0 * tokens * (case["rot"] + case["axes"]) + 8.0 * tokens,
                "flops": 6.0 * tokens * (h + 2 * kv) * d}
    seen = _seen(case)
    pairs = sum(p for _, p in seen)
    masks = {"tree": (case["new"] + 31) // 32, "": 0}.get(case["mask"], 2) * 4.0 * tokens
    return {"bytes": 2.0 * kv * row * sum(s for s, _ in seen) + 8.0 * tokens * h * d + masks,
            "flops": 4.0 * h * d * pairs + h * pairs * (10.0 * (case["cap"] > 0) + 2.0 * case["bias"])}


# ---- inputs ------------------------------------------------------------------

def _starts(counts):
    return torch.tensor([0] + counts).cumsum(0)


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


def _fork(case):
    """The filled tokens of each page to copy; every fourth page is full."""
    rng = random.Random("fork %d %d" % (case["count"], case["page"]))
    return [(i, case["page"] if i % 4 == 3 else rng.randrange(1, case["page"] + 1)) for i in range(case["count"])]


def _kept(case):
    """Of each sequence, the accepted drafts: a path from the root of its tree; of one of several, none."""
    rng = random.Random("kept %d %d" % (case["seqs"], case["new"]))
    got = []
    for s, parents in enumerate(_trees(case)):
        path, most = [0], rng.randrange(1, case["kept"] + 1) if s else case["kept"]
        while len(path) < most:
            after = [i for i, p in enumerate(parents) if p == path[-1]]
            if not after:
                break
            path.append(rng.choice(after))
        got.append([] if s == 2 else path)
    return got


def _pages(case, seed):
    """A table of shuffled pages for the tokens of every sequence that the pass reads or writes."""
    host = torch.Generator().manual_seed(seed)
    new, lens = _ragged(case)
    pt = case["page"]
    table = torch.full((case["seqs"], (case["len"] + pt - 1) // pt), NONE, dtype=torch.int32)
    used = []
    for i, (n, length) in enumerate(zip(new, lens)):
        # the pages ahead of the new tokens are attention's alone
        first = 0 if case["op"] == "attn" else (length - n) // pt
        used += [(i, p) for p in range(first, (length + pt - 1) // pt)]
    at = torch.tensor(used)
    table[at[:, 0], at[:, 1]] = torch.randperm(len(used) + 3, generator=host)[:len(used)].to(torch.int32)
    seq = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(new))
    starts = _starts(new)
    index = torch.arange(sum(new)) - starts[seq]
    pos = torch.tensor(lens)[seq] - torch.tensor(new)[seq] + index
    return len(used) + 3, {"table": table.to(DEV), "starts": starts.to(torch.int32).to(DEV), "lens": torch.tensor(lens, dtype=torch.int32).to(DEV),
                           "seq": seq.to(DEV), "index": index.to(DEV), "pos": pos.to(DEV)}


def _moved_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "fork":
        n = case["count"]
        s, pages = {}, 2 * n + 1
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
        s["copies"] = torch.stack([order[:n], order[n:2 * n], torch.tensor([t for _, t in _fork(case)])], 1).to(torch.int32).to(DEV)
    else:
        pages, s = _pages(case, seed)
        paths = _kept(case)
        kept = torch.zeros(s["seq"].numel(), dtype=torch.int32)
        for a, p in zip(s["starts"].tolist(), paths):
            kept[a:a + len(p)] = torch.tensor(p, dtype=torch.int32)
        s["kept"], s["counts"] = kept.to(DEV), torch.tensor([len(p) for p in paths], dtype=torch.int32).to(DEV)
        s["new_lens"] = torch.empty_like(s["lens"])
    s["cache"] = _cache(case, pages * case["layers"], gen).unflatten(0, (case["layers"], pages))
    return s


def _kv_inputs(case, seed):
    if case["op"] in ("fork", "keep"):
        return _moved_inputs(case, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    pages, s = _pages(case, seed)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    tokens = s["seq"].numel()
    s["cache"] = _cache(case, pages, gen)
    if case["op"] == "attn":
        sharp = torch.exp(0.5 * torch.randn(h, 1, device=DEV, generator=gen))
        s["q"] = sharp * torch.randn(tokens, h, d, device=DEV, generator=gen)
        if case["bias"]:                          # slopes halve from head to head, eight heads to a power of two
            s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, h + 1, dtype=torch.float64) / h)).float().to(DEV)
        if case["mask"] == "tree":
            words = (case["new"] + 31) // 32
            s["tree"] = torch.tensor([r for p in _trees(case) for r in _tree_bits(p, words)], dtype=torch.int32).to(DEV)
        elif case["mask"]:
            s["ranges"] = torch.tensor([r for x in _ranges(case) for r in x], dtype=torch.int32).to(DEV)
        return s
    if case["fused"]:
        rows = torch.randn(tokens, h + 2 * kv, d, device=DEV, generator=gen)
        s["rows"], s["q"], s["k"], s["v"] = rows, rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
    else:
        s["q"], s["k"], s["v"] = (torch.randn(tokens, n, d, device=DEV, generator=gen) for n in (h, kv, kv))
    s["rope"] = _rope(case["len"], case["rot"])
    at = _turns(case)
    s["turns"] = torch.tensor([[p for x in at for p in x[a]] for a in range(case["axes"])], dtype=torch.int32).to(DEV)
    s["pair_axes"] = torch.tensor(_pair_axes(case)).to(DEV)
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


def _buffer(address, size):
    """Memory of torch's as one of the library's buffers."""
    eff, ctx = _context()
    h = eff.ctypes.c_void_p()
    ctx._check(eff.lib().eff_buf_wrap(ctx.h, address, size, eff.ctypes.byref(h)))
    b = eff.Buffer(ctx, h, size)
    weakref.finalize(b, eff.lib().eff_buf_free, ctx.h, h)   # gives the handle back; the memory is torch's
    return b


def _wrap(t):
    """A tensor, moved to memory with readable bytes after it, and that memory as a buffer."""
    size = t.numel() * t.element_size()
    memory = torch.empty(size + PAD, device=DEV, dtype=torch.uint8)
    view = memory[:size].view(t.dtype).view(t.shape)
    view.copy_(t)
    return view, _buffer(memory.data_ptr(), size)


def _handles(case, s):
    """The plan that a program keeps: the caches, the batch, the rows, the rules."""
    eff, _ = _context()
    b = {}
    for key in ("out", "cache", "table", "starts", "lens", "q", "k", "v", "rows", "rope", "turns", "q_norm", "k_norm", "slopes", "tree", "ranges",
                "copies", "kept", "counts", "new_lens"):
        if key in s and not (key in "qkv" and "rows" in s):
            s[key], b[key] = _wrap(s[key])
    t, kv, d, page = {"f16": eff.KV_F16, "i8": eff.KV_I8}[case["kv"]], case["kv_heads"], case["dim"], case["page"]
    p = {"buffers": b}
    if case["op"] in ("fork", "keep"):
        each = s["cache"][0].numel() * s["cache"].element_size()
        p["layers"] = eff.KvLayers(eff.KvCache(t, kv, d, page, s["cache"].shape[1], _buffer(s["cache"].data_ptr() + i * each, each))
                                   for i in range(case["layers"]))
    if case["op"] == "fork":
        return p
    p["batch"] = eff.KvBatch(b["table"], b["starts"], b["lens"], seqs=case["seqs"], tokens=s["seq"].numel(), table_pages=s["table"].shape[1],
                             max_new=case["new"], max_len=case["len"])
    if case["op"] == "keep":
        return p
    h = case["heads"]
    p["cache"] = eff.KvCache(t, kv, d, page, s["cache"].shape[0], b["cache"])
    if case["op"] == "attn":
        p["rules"] = eff.KvRules(cap=case["cap"], slopes=b.get("slopes"), ranges=b.get("ranges"), tree=b.get("tree"),
                                 tree_words=s["tree"].shape[1] if "tree" in s else 0)
        return p
    if "rows" in s:
        n, at = (h + 2 * kv) * d, {"q": (b["rows"], 0), "k": (b["rows"], h * d), "v": (b["rows"], (h + kv) * d)}
        at = {**at, "q_stride": n, "k_stride": n, "v_stride": n}
    else:
        at = {key: (b[key], 0) for key in "qkv"}
    p["rows"] = eff.KvRows(**at, q_out=b["out"], q_heads=h, rope=b["rope"], rope_positions=case["len"], rope_dim=case["rot"],
                           rope_mode=eff.ROPE_HALVES if case["halves"] else eff.ROPE_PAIRS, q_norm=b.get("q_norm"), k_norm=b.get("k_norm"), eps=EPS)
    p["turns"] = eff.KvTurns(b["turns"], _pair_axes(case), axes=case["axes"])
    return p


def prepare(case, seed):
    s = _kv_inputs(case, seed)
    s["case"] = case
    if "q" in s:
        s["out"] = torch.empty(s["q"].shape, device=DEV)
    if case["op"] != "attn" and case["kv"] == "i8":
        s["values"] = torch.empty(_parts(s["cache"], case)[0].shape, device=DEV, dtype=torch.float16)
    if own:
        s["own"] = _handles(case, s)
    torch.cuda.synchronize()
    return s


def _own_run(s):
    _, ctx = _context()
    case, p = s["case"], s["own"]
    b = p["buffers"]
    if case["op"] == "attn":
        ctx.kv_attn(p["cache"], p["batch"], b["q"], b["out"], case["heads"], case["dim"] ** -0.5, case["window"], rules=p["rules"])
    elif case["op"] == "append":
        ctx.kv_append(p["cache"], p["batch"], p["rows"], turns=p["turns"])
    elif case["op"] == "fork":
        ctx.kv_copy(p["layers"], b["copies"], case["count"])
    else:
        ctx.kv_keep(p["layers"], p["batch"], b["kept"], b["counts"], b["new_lens"])
    if case["op"] == "attn" or case["kv"] == "f16":
        return _outputs(s)
    with torch.cuda.stream(_program["stream"]):
        return _outputs(s)


def _outputs(s):
    """What a pass gives; an 8-bit cache that it wrote as the values it stands for."""
    if s["case"]["op"] == "attn":
        return s["out"]
    cache = s["cache"]
    if s["case"]["kv"] == "i8":
        q, scales = _parts(cache, s["case"])
        cache = torch.mul(q, scales[..., None], out=s["values"])
    return {"cache": cache, **{k: s[k] for k in ("out", "new_lens") if k in s}}


# ---- plain forms -------------------------------------------------------------

def _turn(x, s):
    """Norm and rotation of rows [tokens][heads][dim], each pair by the position on its axis."""
    case, r = s["case"], s["case"]["rot"]
    at = s["turns"].long()[s["pair_axes"]].t()                    # [tokens][pairs]
    pair = torch.arange(r // 2, device=DEV)
    c, t = s["rope"][at, 0, pair][:, None], s["rope"][at, 1, pair][:, None]
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
        return _outputs(s)
    rows, scales = _parts(s["cache"], case)
    top = kv.abs().amax(-1)
    rows[page, :, :, slot] = torch.round(kv * torch.where(top > 0, 127 / top, top)[..., None]).to(torch.int8)
    scales[page, :, :, slot] = top * (1 / 127)
    return _outputs(s)


def _visible(s, at):
    """Of each sequence and new token: its position, the keys' positions and which of them it sees."""
    case = s["case"]
    n, new = case["seqs"], case["new"]
    place = torch.full((n, new), -1, device=DEV)
    place[s["seq"], s["index"]] = s["pos"]
    first = (s["lens"] - (s["starts"][1:] - s["starts"][:-1])).long()          # of each sequence's new tokens
    if case["mask"] == "tree":
        bits = torch.zeros(n, new, s["tree"].shape[1], device=DEV, dtype=torch.int32)
        bits[s["seq"], s["index"]] = s["tree"]
        j = torch.arange(new, device=DEV)
        among = (bits[:, :, j // 32] >> (j % 32) & 1).bool()                   # [seqs][new][new]
        pos = first[:, None] + among.sum(-1) - 1
        j = at - first[:, None]                                                # of each cached token, which new one it is
        key = torch.where(j < 0, at, pos.gather(1, j.clamp(0, new - 1)))
        seen = torch.where((j < 0)[:, None], torch.ones_like(j, dtype=torch.bool)[:, None],
                           among.gather(2, j.clamp(0, new - 1)[:, None].expand(n, new, -1)))
        seen &= (at < s["lens"][:, None])[:, None] & (place >= 0)[..., None]
        if case["window"]:
            seen &= key[:, None] > pos[..., None] - case["window"]
        return pos, key, seen
    pos, key = place, at.expand(n, -1)
    if case["mask"]:
        r = torch.zeros(n, new, 2, device=DEV, dtype=torch.int32)
        r[s["seq"], s["index"]] = s["ranges"]
        return pos, key, (at >= r[..., :1]) & (at < r[..., 1:])
    seen = at <= pos[..., None]
    if case["window"]:
        seen &= at > pos[..., None] - case["window"]
    return pos, key, seen


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
    pos, key, seen = _visible(s, at)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, kv, new, g, -1) * d ** -0.5
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    if case["bias"]:
        far = (pos[..., None] - key[:, None]).abs()               # [seqs][new][length]
        score = score - s["slopes"].view(kv, 1, g, 1) * far[:, None, :, None]
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    v = torch.where((at < s["lens"][:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.view(n, kv, new * g, -1), v).view(n, kv, new, g, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    s["out"] = o.permute(0, 2, 1, 3, 4).reshape(n, new, h, d)[s["seq"], s["index"]]
    return s["out"]


def _move(s, page, slot, to_page, to_slot):
    """Rows of all layers and heads from their places to others."""
    for x in (s["cache"],) if s["case"]["kv"] == "f16" else _parts(s["cache"], s["case"]):
        x[:, to_page, :, :, to_slot] = x[:, page, :, :, slot]


def _fork_pages(s):
    pt = s["case"]["page"]
    page, to, tokens = (x[:, None].expand(-1, pt) for x in s["copies"].long().unbind(1))
    slot = torch.arange(pt, device=DEV).expand(page.shape)
    # a token behind the filled ones takes the first one's place, with its value
    slot = torch.where(slot < tokens, slot, torch.zeros_like(slot))
    _move(s, page.reshape(-1), slot.reshape(-1), to.reshape(-1), slot.reshape(-1))
    return _outputs(s)


def _keep(s):
    pt = s["case"]["page"]
    n = s["starts"][1:] - s["starts"][:-1]
    s["new_lens"] = s["lens"] - n + s["counts"]
    first = (s["lens"] - n).long()[s["seq"]]
    # the drafts behind the kept ones stay where they are
    kept = torch.where(s["index"] < s["counts"][s["seq"]], s["kept"].long(), s["index"])
    a, b = first + kept, first + s["index"]
    _move(s, s["table"][s["seq"], a // pt].long(), a % pt, s["table"][s["seq"], b // pt].long(), b % pt)
    return _outputs(s)


def run(s):
    if own:
        return _own_run(s)
    return {"append": _append, "attn": _attn, "fork": _fork_pages, "keep": _keep}[s["case"]["op"]](s)


# ---- in 64 bits --------------------------------------------------------------

def _whole(cache, case):
    """A cache's values."""
    if case["kv"] == "f16":
        return cache.double()
    q, scales = _parts(cache, case)
    return q.double() * scales.double()[..., None]


def _exact_append(case, s):
    r, pt = case["rot"], case["page"]
    turns = torch.tensor([[p for x in _turns(case) for p in x[a]] for a in range(case["axes"])], device=DEV)
    z = torch.complex(s["rope"][:, 0].double(), s["rope"][:, 1].double())                  # [positions][pairs]
    unit = torch.stack([z[turns[a], i] for i, a in enumerate(_pair_axes(case))], 1)[:, None]

    def turned(x, w):
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * w.double()
        u = torch.complex(*((x[..., :r // 2], x[..., r // 2:r]) if case["halves"] else (x[..., 0:r:2], x[..., 1:r:2]))) * unit
        y = x.clone()
        if case["halves"]:
            y[..., :r // 2], y[..., r // 2:r] = u.real, u.imag
        else:
            y[..., 0:r:2], y[..., 1:r:2] = u.real, u.imag
        return y

    k, v = turned(s["k"], s.get("k_norm")), s["v"].double()
    cache = _whole(s["cache"], case)
    if case["kv"] == "i8":
        k, v = (torch.round(x * 127 / x.abs().amax(-1, keepdim=True)) * x.abs().amax(-1, keepdim=True) / 127 for x in (k, v))
    table = s["table"].tolist()
    for i, (seq, pos) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
        page = cache[table[seq][pos // pt]]
        page[0, :, pos % pt], page[1, :, pos % pt] = k[i], v[i]
    return {"cache": cache, "out": turned(s["q"], s.get("q_norm"))}


def _exact_attn(case, s):
    new, lens = _ragged(case)
    kv, d, pt = case["kv_heads"], case["dim"], case["page"]
    g, w = case["heads"] // kv, case["window"]
    out, start = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64), 0
    for i, (n, length) in enumerate(zip(new, lens)):
        pages, first = s["table"][i, :(length + pt - 1) // pt].long(), length - n
        t = torch.arange(length, device=DEV)
        keys, pos = t, first + torch.arange(n, device=DEV)
        if case["mask"] == "tree":
            parents = _trees(case)[i]
            pos = first + torch.tensor(_depths(parents), device=DEV)
            keys = torch.cat([t[:first], pos])
            hidden = torch.ones(n, length, dtype=torch.bool)
            hidden[:, :first] = False
            for j, p in enumerate(parents):
                if p >= 0:
                    hidden[j] = hidden[p]
                hidden[j, first + j] = False
            hidden = hidden.to(DEV)
        elif case["mask"]:
            r = torch.tensor(_ranges(case)[i], device=DEV)
            hidden = (t < r[:, :1]) | (t >= r[:, 1:])
        else:
            hidden = t > pos[:, None]
        if w:
            hidden = hidden | (keys <= pos[:, None] - w)
        far = (pos[:, None] - keys).abs().double()
        x = s["cache"][pages] if case["kv"] == "f16" else None
        for j in range(kv):
            if x is None:
                q, scales = _parts(s["cache"], case)
                k, v = (q[pages, :, j].double() * scales[pages, :, j].double()[..., None]).transpose(0, 1).reshape(2, -1, d)[:, :length]
            else:
                k, v = x[:, :, j].double().transpose(0, 1).reshape(2, -1, d)[:, :length]
            for a in range(0, n, 128):
                rows = slice(a, min(n, a + 128))
                of = slice(start + a, start + rows.stop)
                z = s["q"][of, j * g:(j + 1) * g].double() @ k.t().contiguous() / math.sqrt(d)          # [tokens][group][length]
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                if case["bias"]:
                    z = z - far[rows, None] * s["slopes"][j * g:(j + 1) * g, None].double()
                out[of, j * g:(j + 1) * g] = torch.softmax(z.masked_fill(hidden[rows, None], -math.inf), -1) @ v
        start += n
    return out


def _exact_moved(case, s):
    cache, pt = _whole(s["cache"], case), case["page"]
    before = cache.clone()
    if case["op"] == "fork":
        for a, b, n in s["copies"].tolist():
            cache[:, b, :, :, :n] = before[:, a, :, :, :n]
        return {"cache": cache}
    table, left = s["table"].tolist(), []
    for i, (path, n, length) in enumerate(zip(_kept(case), *_ragged(case))):
        for j, k in enumerate(path):
            a, b = length - n + k, length - n + j
            cache[:, table[i][b // pt], :, :, b % pt] = before[:, table[i][a // pt], :, :, a % pt]
        left.append(length - n + len(path))
    return {"cache": cache, "new_lens": torch.tensor(left, dtype=torch.int32, device=DEV)}


def exact(case, seed):
    s = _kv_inputs(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "fork": _exact_moved, "keep": _exact_moved}[case["op"]](case, s)
