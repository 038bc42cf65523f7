"""The example that runs the operators together (examples/decode.py): its processed logits against the same model in 64
bits over the dequantized weights, without a cache, at every step.

Tolerance. The products and the attention are f32-accurate (1e-5 relative each, five in a row, and the norm after the
first passes it on); int8 pages round every key and value by up to 1/254 of the row's maximum, independently, which a
mean over the tokens seen and the output projection do not enlarge: 0.02 of the logits' norm. The fp16 pages round by
2^-11: 0.002."""
import importlib.util
import os

import numpy as np
import pytest

from kv_reference import F16, I8, turn

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("decode_example", os.path.join(ROOT, "elffuss-engine_amd", "examples", "decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def reference(eff, orc, m, prompts, tokens, rules):
    """The processed logits of every step, from the whole sequence each time."""
    w = {n: orc.dequant(orc.NAMES[t], data, r * k // eff.geometry(t)[0]).reshape(r, k).astype(np.float64)
         for n, (t, r, k, data) in m.weights.items()}
    out = []
    for step in range(len(tokens[0])):
        rows = []
        for i, p in enumerate(prompts):
            seq = list(p) + tokens[i][:step]
            x = w["embedding"][seq]
            x = x / np.sqrt((x * x).mean(1, keepdims=True) + m.eps) * m.norms["norm"]
            qkv = (x @ w["qkv"].T).reshape(len(seq), -1, m.dim)
            pos = np.arange(len(seq))
            a = pos[:, None] * m.freqs
            rope = np.stack([np.cos(a), np.sin(a)], 1)
            q = turn(qkv[-1:, :m.heads], pos[-1:], rope, m.dim, True, m.norms["q_norm"], m.eps)[0]
            k = turn(qkv[:, m.heads:m.heads + m.kv_heads], pos, rope, m.dim, True, m.norms["k_norm"], m.eps)
            v, g = qkv[:, m.heads + m.kv_heads:], m.heads // m.kv_heads
            o = []
            for h in range(m.heads):
                s = k[:, h // g] @ q[h] * m.scale
                s = np.exp(s - s.max())
                o.append(s @ v[:, h // g] / s.sum())
            z = w["head"] @ (w["out"] @ np.concatenate(o))
            rep, freq, pres = rules["penalties"]
            ids, c = np.unique(seq, return_counts=True)
            z[ids] = np.where(z[ids] > 0, z[ids] / rep, z[ids] * rep) - (freq * c + pres)
            j = rules["mask_of"][i]
            if j < len(rules["mask"]):
                z[np.unpackbits(rules["mask"][j].view(np.uint8), bitorder="little")[:m.vocab] == 0] = -np.inf
            rows.append(z)
        out.append(rows)
    return np.array(out)


@pytest.mark.parametrize("kv,limit", [(F16, 2e-3), (I8, 2e-2)])
def test_decode_example(ctx, eff, orc, kv, limit):
    ex = example()
    m = ex.Model(eff, kv=kv)
    rng = np.random.default_rng(kv)
    prompts = [list(map(int, rng.integers(0, m.vocab, n))) for n in (37, 5, 130, 1, 16)]
    mask = rng.integers(0, 2 ** 32, (2, (m.vocab + 31) // 32), dtype=np.uint32)
    rules = {"penalties": (1.2, 0.1, 0.3), "mask": mask, "mask_of": [1, 7, 0, 7, 7]}
    before = ctx.stats()
    tokens, logits = ex.decode(eff, ctx, m, prompts, 10, rules)
    after = ctx.stats()
    assert all(after[k] - before[k] >= 3 for k in ("gather", "kv_append", "kv_attn", "logits", "topk"))
    want = reference(eff, orc, m, prompts, tokens, rules)
    for step in range(10):
        for i in range(len(prompts)):
            a, b = logits[step, i].astype(np.float64), want[step, i]
            seen = np.isfinite(b)
            assert np.array_equal(seen, np.isfinite(a))
            assert np.linalg.norm(a[seen] - b[seen]) <= limit * np.linalg.norm(b[seen]), (step, i)
            assert tokens[i][step] == int(np.argmax(a)) and np.isfinite(b[tokens[i][step]])
