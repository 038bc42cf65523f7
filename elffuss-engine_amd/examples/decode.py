"""Greedy decoding of a batch of requests: prompts of different lengths, then one token of each request a step.

    python elffuss-engine_amd/examples/decode.py

A model of one attention layer with random quantized weights (embedding, norm, q + k + v, output projection, head).
Every step runs on the device, the token's row of the embedding to the top-k of its processed logits:

    gather_norm -> qmatmul (q, k, v) -> kv_append -> kv_attn -> qmatmul -> qmatmul (head) -> logits_apply -> topk

The prompts go through the same calls as one ragged batch. The steps after them are one recording, replayed with the
next ids, lengths and histories.
"""
import importlib.util
import os
import sys

import numpy as np


def package():
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("elffuss_amd", os.path.join(here, "elffuss_amd.py"))
    sys.modules["elffuss_amd"] = eff = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(eff)
    return eff


class Model:
    """Sizes and weights: {name: (type, rows, k, bytes)}."""

    def __init__(self, eff, embed=512, heads=8, kv_heads=2, dim=64, vocab=5000, kv=None, page=16, seed=1):
        self.embed, self.heads, self.kv_heads, self.dim, self.vocab = embed, heads, kv_heads, dim, vocab
        self.kv, self.page = eff.KV_F16 if kv is None else kv, page
        qkv = (heads + 2 * kv_heads) * dim
        shapes = {"embedding": ("Q8_0", vocab, embed), "qkv": ("Q4_K", qkv, embed), "out": ("Q6_K", embed, heads * dim),
                  "head": ("Q6_K", vocab, embed)}
        self.weights = {n: (t, r, k, eff.quantize(t, eff.fill_normal(seed + i, 3 * k ** -0.5, r * k)))
                        for i, (n, (t, r, k)) in enumerate(shapes.items())}
        rng = np.random.default_rng(seed)
        self.norms = {n: (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
                      for n, d in (("norm", embed), ("q_norm", dim), ("k_norm", dim))}
        self.freqs = 10000.0 ** (-np.arange(0, dim, 2) / dim)
        self.eps, self.scale = 1e-6, dim ** -0.5


class Decoder:
    """The device's side of `requests` requests of up to max_len tokens."""

    def __init__(self, eff, ctx, model, requests, max_len, rules):
        self.eff, self.ctx, self.m, self.n, self.max_len, self.rules = eff, ctx, model, requests, max_len, rules
        m, up = model, ctx.upload
        self.w = {n: (t, up(data), r, k) for n, (t, r, k, data) in m.weights.items()}
        self.norms = {n: up(x) for n, x in m.norms.items()}
        self.rope = ctx.rope_table(m.freqs, max_len)
        per = -(-max_len // m.page)
        self.table_pages, pages = per, requests * per
        self.cache = eff.KvCache(m.kv, m.kv_heads, m.dim, m.page, pages,
                                 ctx.alloc(pages * eff.kv_page_bytes(m.kv, m.kv_heads, m.dim, m.page)))
        # any page serves any request: dealt out in turn here
        self.table = up((np.arange(per)[None] * requests + np.arange(requests)[:, None]).astype(np.uint32))
        self.lens = up(np.zeros(requests, np.uint32))
        self.last, self.logits = ctx.alloc(4 * requests * m.embed), ctx.alloc(4 * requests * m.vocab)
        self.chosen = [ctx.alloc(eff.lib().eff_topk_out_bytes()) for _ in range(requests)]
        self.history, self.history_starts = ctx.alloc(4 * requests * max_len), up(np.zeros(requests + 1, np.uint32))
        at = {"history": self.history, "history_starts": self.history_starts,
              "penalties": up(np.tile(np.array(rules["penalties"], np.float64), (requests, 1)))}
        if rules.get("mask") is not None:
            at.update(mask=up(rules["mask"]), mask_of=up(np.asarray(rules["mask_of"], np.uint32)), mask_count=len(rules["mask"]))
        self.logits_rules = eff.LogitsRules(**at)

    def layer(self, tokens, starts, max_new):
        """Buffers of a call of `tokens` new tokens, and the call up to the output projection."""
        ctx, eff, m = self.ctx, self.eff, self.m
        qkv = self.w["qkv"][2]
        ids = ctx.alloc(4 * tokens)
        x, nrm, y = (ctx.alloc(4 * tokens * m.embed) for _ in range(3))
        rows, q, o = ctx.alloc(4 * tokens * qkv), ctx.alloc(4 * tokens * m.heads * m.dim), ctx.alloc(4 * tokens * m.heads * m.dim)
        batch = eff.KvBatch(self.table, ctx.upload(np.asarray(starts, np.uint32)), self.lens, seqs=self.n, tokens=tokens,
                            table_pages=self.table_pages, max_new=max_new, max_len=self.max_len)
        k0, v0 = m.heads * m.dim, (m.heads + m.kv_heads) * m.dim
        kv_rows = eff.KvRows(q=(rows, 0), k=(rows, k0), v=(rows, v0), q_stride=qkv, k_stride=qkv, v_stride=qkv, q_heads=m.heads,
                             q_out=q, rope=self.rope, rope_positions=self.max_len, rope_dim=m.dim, rope_mode=eff.ROPE_HALVES,
                             q_norm=self.norms["q_norm"], k_norm=self.norms["k_norm"], eps=m.eps)

        def run():
            t, w, _, _ = self.w["embedding"]
            ctx.gather_norm(t, w, ids, self.norms["norm"], m.eps, x, nrm, m.embed, tokens)
            self.product("qkv", nrm, rows, tokens)
            ctx.kv_append(self.cache, batch, kv_rows)
            ctx.kv_attn(self.cache, batch, q, o, m.heads, m.scale)
            self.product("out", o, y, tokens)
        return ids, y, run

    def product(self, name, x, y, tokens):
        t, w, rows, k = self.w[name]
        self.ctx.qmatmul(t, w, x, y, rows, k, tokens)

    def choose(self, x):
        """The head of each request's last row, the rules, and the best token of each."""
        m = self.m
        self.product("head", x, self.logits, self.n)
        self.ctx.logits_apply(self.logits, self.logits, self.n, m.vocab, self.logits_rules)
        for r in range(self.n):
            self.ctx.topk(self.logits, r * m.vocab, m.vocab, 1, out=self.chosen[r])

    def read(self):
        logits = self.logits.read(np.float32).reshape(self.n, self.m.vocab)
        return logits, [int(self.eff.parse_topk(c.read(np.uint32))["ids"][0]) for c in self.chosen]

    def put(self, lens, histories):
        """What the next call reads: the lengths, and the ids that the penalties count."""
        self.lens.write(np.asarray(lens, np.uint32))
        self.history.write(np.array([i for h in histories for i in h] or [0], np.uint32))
        self.history_starts.write(np.concatenate([[0], np.cumsum([len(h) for h in histories])]).astype(np.uint32))


def decode(eff, ctx, model, prompts, steps, rules):
    """The tokens of `steps` steps of each prompt, and the processed logits of each step [steps][requests][vocab]."""
    if not prompts or not all(len(p) for p in prompts) or steps < 1:
        raise ValueError("decode: prompts of one token or more, and a step or more")   # the first step reads a prompt's last row
    n, max_len = len(prompts), max(len(p) for p in prompts) + steps
    d = Decoder(eff, ctx, model, n, max_len, rules)
    sequences, logits = [list(p) for p in prompts], []
    # the prompts, as one ragged batch
    starts = np.concatenate([[0], np.cumsum([len(p) for p in prompts])])
    ids, y, run = d.layer(int(starts[-1]), starts, max(len(p) for p in prompts))
    ids.write(np.array([i for p in prompts for i in p], np.uint32))
    d.put([len(s) for s in sequences], sequences)
    run()
    for r in range(n):
        ctx.copy(d.last, y, 4 * model.embed, 4 * model.embed * r, 4 * model.embed * (int(starts[r + 1]) - 1))
    d.choose(d.last)
    # one token of each request a step: run once as it is, then recorded
    ids, y, run = d.layer(n, np.arange(n + 1), 1)
    graph = None
    for step in range(steps):
        z, chosen = d.read()
        logits.append(z)
        for s, i in zip(sequences, chosen):
            s.append(i)
        if step + 1 == steps:
            break
        ids.write(np.array(chosen, np.uint32))
        d.put([len(s) for s in sequences], sequences)
        if step == 0:
            run()
            d.choose(y)
        elif graph is None:
            ctx.graph_begin()
            run()
            d.choose(y)
            graph = ctx.graph_end()
            graph.launch()
        else:
            graph.launch()
    if graph:
        graph.destroy()
    return [s[len(p):] for s, p in zip(sequences, prompts)], np.stack(logits)


def main():
    eff = package()
    model = Model(eff)
    rng = np.random.default_rng(7)
    prompts = [list(rng.integers(0, model.vocab, n)) for n in (37, 5, 120, 1)]
    allowed = rng.integers(0, 2 ** 32, (1, (model.vocab + 31) // 32), dtype=np.uint32)
    rules = {"penalties": (1.1, 0.2, 0.1), "mask": allowed, "mask_of": [0xFFFFFFFF, 0, 0xFFFFFFFF, 0xFFFFFFFF]}
    with eff.Context(0) as ctx:
        tokens, _ = decode(eff, ctx, model, prompts, 12, rules)
        stats = ctx.stats()
    for p, t in zip(prompts, tokens):
        print(f"{len(p):4d} tokens -> {t}")
    print({k: stats[k] for k in ("gather", "kv_append", "kv_attn", "logits", "topk")})


if __name__ == "__main__":
    main()
