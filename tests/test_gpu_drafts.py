"""The example that runs forking, appending, attention and compaction together over trees of drafts (examples/drafts.py):
the tokens of every answer are those of decoding one at a time, and its logits those of the same model in 64 bits without
a cache, within what test_gpu_decode derives for them."""
import importlib.util
import os
import sys

import numpy as np
import pytest

from kv_reference import F16, I8
from test_gpu_decode import ROOT, reference


def example():
    here = os.path.join(ROOT, "elffuss-engine_amd", "examples")
    spec = importlib.util.spec_from_file_location("drafts_example", os.path.join(here, "drafts.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    sys.path.remove(here)
    return m


def guesses(rng, truth, right):
    """Trees that hold the sequence's continuation in part, among wrong guesses: a node continues it with chance `right`."""
    def draft(sequence, nodes):
        ahead = next((t[len(sequence):] for t in truth if t[:len(sequence)] == sequence), [])
        tokens, parents, on = [sequence[-1]], [-1], 0
        while len(tokens) < nodes:
            if on < len(ahead) and rng.random() < right:
                parents.append(0 if on == 0 else last)
                tokens.append(ahead[on])
                last, on = len(tokens) - 1, on + 1
            else:
                parents.append(int(rng.integers(0, len(tokens))))
                tokens.append(int(rng.integers(0, 1000)))
        return tokens, parents
    return draft


@pytest.mark.gpu
@pytest.mark.parametrize("kv,limit", [(F16, 2e-3), (I8, 2e-2)])
@pytest.mark.parametrize("nodes,right", [(1, 0.0), (7, 0.6), (40, 0.3)])
def test_drafts_example(ctx, eff, orc, kv, limit, nodes, right):
    ex = example()
    m = ex.Model(eff, kv=kv)
    rng = np.random.default_rng(nodes)
    prompts = [list(map(int, rng.integers(0, m.vocab, n))) for n in (37, 16, 1)]
    answers, count = 2, 9
    mask = rng.integers(0, 2 ** 32, (2, (m.vocab + 31) // 32), dtype=np.uint32)
    rules = {"penalties": (1.2, 0.1, 0.3), "mask": mask, "mask_of": [0, 7, 7, 1, 0, 1]}
    # one at a time: each prompt once for each of its answers
    one, _ = sys.modules["decode"].decode(eff, ctx, m, [p for p in prompts for _ in range(answers)], count, rules)
    truth = [p + t for p, t in zip([p for p in prompts for _ in range(answers)], one)]
    before = ctx.stats()
    tokens, logits, steps = ex.decode_drafts(eff, ctx, m, prompts, answers, count, rules, nodes, guesses(rng, truth, right))
    after = ctx.stats()
    assert tokens == one
    assert after["kv_copy"] > before["kv_copy"] and after["kv_keep"] - before["kv_keep"] == steps
    assert steps == count - 1 if nodes == 1 else steps < count - 1
    want = reference(eff, orc, m, [p for p in prompts for _ in range(answers)], tokens, rules)
    for r in range(len(tokens)):
        for step in range(count):
            a, b = logits[r][step].astype(np.float64), want[step, r]
            seen = np.isfinite(b)
            assert np.array_equal(seen, np.isfinite(a))
            assert np.linalg.norm(a[seen] - b[seen]) <= limit * np.linalg.norm(b[seen]), (r, step)


def test_trees_that_repeat():
    """The example's own drafts."""
    ex = example()
    assert ex.repeat([5, 1, 2, 3, 4, 1, 9, 1], 6) == ([1, 9, 1, 2, 3, 4], [-1, 0, 1, 0, 3, 4])
    assert ex.repeat([5], 3) == ([5], [-1])


@pytest.mark.parametrize("prompts,answers,tokens,nodes", [([], 1, 3, 2), ([[1], []], 1, 3, 2), ([[1]], 0, 3, 2), ([[1]], 1, 0, 2), ([[1]], 1, 1, 0)])
def test_refusals(prompts, answers, tokens, nodes):
    with pytest.raises(ValueError, match="decode_drafts"):
        example().decode_drafts(None, None, None, prompts, answers, tokens, {}, nodes)
