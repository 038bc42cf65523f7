"""The JavaScript host's calls with positions, rules, copies and drafts that stay on the GPU (tests/js/shim_rules.js),
checked here in 64 bits and byte by byte."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from kv_reference import F16, I8, Batch, decode, encode
from kv_rules_reference import attend_rules, random_tree, row_bytes, tree_mask, tree_words, turn_at
from test_gpu_kv_attn import check
from test_gpu_kv_turns import TURN

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skip(reason="of several runs of these calls in node one ended in a segmentation fault of the process, and its cause is not known: "
                         "the host refuses them (KV_REGLAS_ENCENDIDO in index.js), which tests/test_js_rules.py checks")
@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
@pytest.mark.parametrize("t", [F16, I8])
def test_js_shim_rules(tmp_path, t):
    rng = np.random.default_rng(t)
    heads, q_heads, dim, page = 2, 6, 64, 16
    b = Batch(rng, [9, 4], [70, 33], page, spare=3)
    first, _ = encode(t, rng.standard_normal((b.pages, 2, heads, page, dim)).astype(np.float32))
    q, k, v = (rng.standard_normal((b.tokens, n, dim)).astype(np.float32) for n in (q_heads, heads, heads))
    masks = [tree_mask(random_tree(rng, n)) for n in b.new]
    axis = [i % 2 for i in range(dim // 2)]
    at = rng.integers(0, 90, (2, b.tokens)).astype(np.uint32)
    ranges = np.sort(rng.integers(0, 33, (b.tokens, 2)), 1).astype(np.uint32)
    slopes = (0.5 ** np.arange(1, q_heads + 1)).astype(np.float32)
    kept = [[0, 3, 8], [2]]
    entries = np.zeros(b.tokens, np.uint32)
    for s, x in enumerate(kept):
        entries[b.starts[s]:b.starts[s] + len(x)] = x
    freqs = 10000.0 ** (-np.arange(0, dim, 2) / dim)
    for name, x in {"cache": first, "table": b.table, "starts": b.starts.astype(np.uint32), "lens": np.array(b.lens, np.uint32), "q": q, "k": k,
                    "v": v, "at": at, "ranges": ranges, "slopes": slopes, "tree": tree_words(masks, 1), "kept": entries,
                    "counts": np.array([3, 1], np.uint32)}.items():
        np.ascontiguousarray(x).tofile(tmp_path / f"{name}.bin")
    copies = [int(b.table[0, 0]), int(b.spare[0]), 16, int(b.table[0, 4]), int(b.spare[1]), 6]
    meta = {"tipo": "F16" if t == F16 else "I8", "cabezas": heads, "cabezasQ": q_heads, "dim": dim, "pagina": page, "paginas": b.pages,
            "secuencias": 2, "tokens": b.tokens, "paginasTabla": b.table_pages, "maxNuevos": 9, "maxLargo": 70, "escala": 0.125, "freqs": freqs.tolist(),
            "posiciones": 90, "ejes": 2, "eje": axis, "tope": 6.0, "palabras": 1, "copias": copies}
    (tmp_path / "meta.json").write_text(json.dumps(meta))
    r = subprocess.run(["node", os.path.join(HERE, "js", "shim_rules.js"), str(tmp_path)], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stderr
    out = json.loads((tmp_path / "out.json").read_text())
    a = np.arange(90)[:, None] * freqs
    rope = np.stack([np.cos(a), np.sin(a)], 1).astype(np.float32)
    want = turn_at(q, at, axis, rope, dim, False)
    got = np.array(out["q"], np.float32).reshape(q.shape)
    assert (np.abs(got - want) <= TURN * np.abs(want).max(-1, keepdims=True)).all()
    data = np.array(out["cache"], np.uint8)
    values = decode(t, data, b.pages, heads, dim, page)
    for y, rules in (("y", {"masks": masks, "cap": 6.0, "slopes": slopes}), ("z", {"ranges": ranges})):
        check(np.array(out[y], np.float32).reshape(q.shape), attend_rules(values, b, got, q_heads, 0.125, **rules), values)
    for layer, x in enumerate((data, first.ravel())):
        rows = row_bytes(t, x, b.pages, heads, dim, page)
        for c in np.reshape(copies, (-1, 3)):
            rows[c[1], :, :, :c[2]] = rows[c[0], :, :, :c[2]]
        assert np.array_equal(row_bytes(t, np.array(out["copied"][layer], np.uint8), b.pages, heads, dim, page), rows)
        old = rows.copy()
        for s, x in enumerate(kept):
            for i, j in enumerate(x):
                p, o = (b.lens[s] - b.new[s] + n for n in (i, j))
                rows[b.table[s, p // page], :, :, p % page] = old[b.table[s, o // page], :, :, o % page]
        assert np.array_equal(row_bytes(t, np.array(out["kept"][layer], np.uint8), b.pages, heads, dim, page), rows)
    assert out["lens"] == [70 - 9 + 3, 33 - 4 + 1]
    assert out["stats"]["kvCopy"] == 1 and out["stats"]["kvKeep"] == 2
