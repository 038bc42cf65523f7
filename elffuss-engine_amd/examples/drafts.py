"""Several answers to each prompt, decoded by trees of drafts: the model checks a tree of guessed tokens at once.

    python elffuss-engine_amd/examples/drafts.py

The model is that of decode.py. Each prompt goes through it once; its answers share its full pages, and its last one is
copied for each (kv_copy). A step then takes a tree of drafts of every answer: node 0 is the answer's last token, which is
not in the cache yet, and the others guess what follows their parent. All of them are appended, turned by the position of
their depth (kv_append with turns), and see their ancestors and what is cached (kv_attn with a tree):

    gather_norm -> qmatmul (q, k, v) -> kv_append -> kv_attn -> qmatmul -> qmatmul (head) -> logits_apply -> topk

From node 0 on, where the best token of a node is a child's, the child is accepted; the accepted nodes' keys and values
move up (kv_keep) and the others are overwritten by the next step. The tokens are those of decoding one at a time.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from decode import Decoder, Model, package  # noqa: E402


def repeat(sequence, nodes):
    """A tree from the sequence itself: what followed its last token before, the latest times first; a chain for each."""
    tokens, parents = [sequence[-1]], [-1]
    for i in range(len(sequence) - 2, -1, -1):
        if sequence[i] != sequence[-1]:
            continue
        at = 0
        for t in sequence[i + 1:i + 4]:
            if len(tokens) == nodes:
                return tokens, parents
            child = next((j for j, p in enumerate(parents) if p == at and tokens[j] == t), None)
            if child is None:
                child = len(tokens)
                tokens.append(t)
                parents.append(at)
            at = child
    return tokens, parents


class Drafting(Decoder):
    """The device's side: requests of which each step brings up to `nodes` drafts."""

    def __init__(self, eff, ctx, model, requests, max_len, rules, nodes):
        super().__init__(eff, ctx, model, requests, max_len, rules)
        m, rows, up = model, requests * nodes, ctx.upload
        self.nodes, self.words, self.rows = nodes, (nodes + 31) // 32, rows
        self.pages = np.arange(self.table_pages)[None] * requests + np.arange(requests)[:, None]
        self.layers = eff.KvLayers([self.cache])
        self.z = ctx.alloc(4 * rows * m.vocab)
        self.best = [ctx.alloc(eff.lib().eff_topk_out_bytes()) for _ in range(rows)]
        self.seen, self.seen_starts = ctx.alloc(4 * rows * max_len), up(np.zeros(rows + 1, np.uint32))
        at = {"history": self.seen, "history_starts": self.seen_starts, "penalties": up(np.tile(np.array(rules["penalties"], np.float64), (rows, 1)))}
        if rules.get("mask") is not None:
            at.update(mask=up(rules["mask"]), mask_of=up(np.repeat(np.asarray(rules["mask_of"], np.uint32), nodes)), mask_count=len(rules["mask"]))
        self.rows_rules = eff.LogitsRules(**at)
        # what a step's append, attention and compaction read
        self.at, self.tree = ctx.alloc(4 * rows), ctx.alloc(4 * rows * self.words)
        self.kept, self.counts, self.left = ctx.alloc(4 * rows), ctx.alloc(4 * requests), ctx.alloc(4 * requests)
        self.turns, self.rules_of_tree = eff.KvTurns(self.at), eff.KvRules(tree=self.tree, tree_words=self.words)

    def fork(self, source, others, length):
        """`others` begin as `source` does: its full pages are theirs, the rest of its `length` tokens is copied."""
        full, rest = divmod(length, self.m.page)
        for r in others:
            self.pages[r, :full] = self.pages[source, :full]
        self.table.write(self.pages.astype(np.uint32))
        if rest and others:
            copies = [[self.pages[source, full], self.pages[r, full], rest] for r in others]
            self.ctx.kv_copy(self.layers, self.ctx.upload(np.array(copies, np.uint32)), len(copies))

    def step(self):
        """Buffers of a step, and the step: the drafts' logits and the best token of each."""
        ids, y, run = self.layer(self.rows, np.arange(self.n + 1) * self.nodes, self.nodes, turns=self.turns, rules=self.rules_of_tree)

        def whole():
            run()
            self.product("head", y, self.z, self.rows)
            self.ctx.logits_apply(self.z, self.z, self.rows, self.m.vocab, self.rows_rules)
            for r in range(self.rows):
                self.ctx.topk(self.z, r * self.m.vocab, self.m.vocab, 1, out=self.best[r])
        return ids, self.batch, whole

    def put_trees(self, ids, lens, trees, histories):
        """What a step reads: ids, positions and trees of the drafts, lengths, and the ids that each draft's penalties count."""
        at, bits = np.zeros((self.n, self.nodes), np.uint32), np.zeros((self.n, self.nodes, self.words), np.uint32)
        tokens, paths = np.zeros((self.n, self.nodes), np.uint32), []
        for r, (t, parents) in enumerate(trees):
            seen = []
            for i in range(self.nodes):
                # places without a draft hold one that sees itself and that nobody sees
                p = parents[i] if i < len(t) else -1
                seen.append((seen[p] if p >= 0 else []) + [i])
                tokens[r, i] = t[i] if i < len(t) else 0
                at[r, i] = lens[r] + len(seen[i]) - 1
                for j in seen[i]:
                    bits[r, i, j // 32] |= np.uint32(1 << j % 32)
                paths.append(histories[r][:-1] + [int(tokens[r, j]) for j in seen[i]])
        ids.write(tokens)
        self.at.write(at)
        self.tree.write(bits)
        self.lens.write((np.asarray(lens) + self.nodes).astype(np.uint32))
        self.seen.write(np.array([i for h in paths for i in h], np.uint32))
        self.seen_starts.write(np.concatenate([[0], np.cumsum([len(h) for h in paths])]).astype(np.uint32))

    def keep(self, batch, accepted):
        """The accepted drafts' keys and values move up behind the tokens before them; the lengths with them."""
        kept = np.zeros((self.n, self.nodes), np.uint32)
        for r, path in enumerate(accepted):
            kept[r, :len(path)] = path
        self.kept.write(kept)
        self.counts.write(np.array([len(p) for p in accepted], np.uint32))
        self.ctx.kv_keep(self.layers, batch, self.kept, self.counts, self.left)
        return self.left.read(np.uint32).tolist()


def decode_drafts(eff, ctx, model, prompts, answers, tokens, rules, nodes=8, draft=repeat):
    """`answers` continuations of `tokens` tokens of each prompt, their logits [answer][token][vocab], and the steps taken.

    rules["mask_of"] has an entry for each answer (prompts times answers), so that they may differ; draft(sequence,
    nodes) gives a tree's tokens, the sequence's last first, and parents, each before its children."""
    if not prompts or not all(len(p) for p in prompts) or answers < 1 or tokens < 1 or nodes < 1:
        raise ValueError("decode_drafts: prompts of one token or more, and an answer, a token and a node or more")
    n, most = len(prompts) * answers, max(len(p) for p in prompts) + tokens + 2 * nodes
    d = Drafting(eff, ctx, model, n, most, rules, nodes)
    sequences, logits = [list(p) for p in prompts for _ in range(answers)], [[] for _ in range(n)]
    # the prompts, each in the place of its first answer
    new = [len(p) if a == 0 else 0 for p in prompts for a in range(answers)]
    starts = np.concatenate([[0], np.cumsum(new)])
    ids, y, run = d.layer(int(starts[-1]), starts, max(new))
    ids.write(np.array([i for p in prompts for i in p], np.uint32))
    d.put([len(s) for s in sequences], sequences)
    run()
    for r in range(n):
        last = int(starts[r // answers * answers + 1]) - 1
        ctx.copy(d.last, y, 4 * model.embed, 4 * model.embed * r, 4 * model.embed * last)
        if r % answers == 0:
            d.fork(r, list(range(r + 1, r + answers)), len(sequences[r]))
    d.choose(d.last)
    z, chosen = d.read()
    for r in range(n):
        logits[r].append(z[r])
        sequences[r].append(chosen[r])
    lens, goal = [len(s) - 1 for s in sequences], [len(p) + tokens for p in prompts for _ in range(answers)]
    ids, batch, step = d.step()
    graph, steps = None, 0
    while any(len(s) < g for s, g in zip(sequences, goal)):
        trees = [draft(s, nodes) for s in sequences]
        d.put_trees(ids, lens, trees, sequences)
        if steps == 0:
            step()
        elif graph is None:
            ctx.graph_begin()
            step()
            graph = ctx.graph_end()
            graph.launch()
        else:
            graph.launch()
        steps += 1
        z = d.z.read(np.float32).reshape(n, nodes, model.vocab)
        best = np.array([eff.parse_topk(b.read(np.uint32))["ids"][0] for b in d.best]).reshape(n, nodes)
        accepted = []
        for r, (t, parents) in enumerate(trees):
            path = []
            node = 0 if len(sequences[r]) < goal[r] else None   # an answer that is complete stays as it is
            while node is not None:
                path.append(node)
                logits[r].append(z[r, node])
                sequences[r].append(int(best[r, node]))
                if len(sequences[r]) == goal[r]:
                    break
                node = next((i for i, p in enumerate(parents) if p == node and t[i] == best[r, node]), None)
            accepted.append(path)
        lens = d.keep(batch, accepted)
    if graph:
        graph.destroy()
    return [s[len(prompts[r // answers]):] for r, s in enumerate(sequences)], [np.stack(x) for x in logits], steps


def main():
    eff = package()
    model = Model(eff)
    rng = np.random.default_rng(7)
    prompts = [list(map(int, rng.integers(0, model.vocab, n))) for n in (37, 120)]
    # few tokens are allowed, so that they come again and the drafts have something to repeat
    allowed = np.zeros((3, (model.vocab + 31) // 32), np.uint32)
    for row in allowed:
        np.bitwise_or.at(row, (i := rng.integers(0, model.vocab, 6)) // 32, np.uint32(1) << (i % 32).astype(np.uint32))
    rules = {"penalties": (1.0, 0.0, 0.0), "mask": allowed, "mask_of": [0, 1, 2, 0, 1, 2]}
    with eff.Context(0) as ctx:
        tokens, _, steps = decode_drafts(eff, ctx, model, prompts, 3, 24, rules)
        stats = ctx.stats()
    for i, t in enumerate(tokens):
        print(f"prompt {i // 3}, answer {i % 3}: {t}")
    print(f"{len(tokens[0])} tokens of each answer in {steps + 1} steps")
    print({k: stats[k] for k in ("kv_append", "kv_attn", "kv_copy", "kv_keep")})


if __name__ == "__main__":
    main()
