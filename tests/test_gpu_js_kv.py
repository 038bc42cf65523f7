"""The JavaScript host's createKvOps and createLogitsOps on the GPU (tests/js/shim_kv.js), checked here in 64 bits."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from kv_reference import F16, I8, Batch, attend, decode, encode, turn
from test_gpu_logits import expected, inputs

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
@pytest.mark.parametrize("t", [F16, I8])
def test_js_shim_kv(tmp_path, t):
    rng = np.random.default_rng(t)
    heads, q_heads, dim, page, window = 2, 6, 64, 16, 40
    b = Batch(rng, [1, 5, 1], [70, 5, 33], page)
    data, _ = encode(t, rng.standard_normal((b.pages, 2, heads, page, dim)).astype(np.float32))
    rows = rng.standard_normal((b.tokens, (q_heads + 2 * heads) * dim)).astype(np.float32)
    qn, kn = ((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
    freqs = 10000.0 ** (-np.arange(0, dim, 2) / dim)
    z, h, pen, bias, mask, mask_of = inputs(rng, 3, 5003, 60, 8, 2)
    starts = lambda x: np.concatenate([[0], np.cumsum([len(i) for i in x])]).astype(np.uint32)   # noqa: E731
    flat = lambda x, d: np.array([i for r in x for i in r], d)                                   # noqa: E731
    for name, x in {"cache": data, "table": b.table, "starts": b.starts.astype(np.uint32), "lens": np.array(b.lens, np.uint32),
                    "rows": rows, "qn": qn, "kn": kn, "logits": z, "history": flat(h, np.uint32), "hstarts": starts(h),
                    "pen": np.ascontiguousarray(pen), "bids": flat([[i for i, _ in r] for r in bias], np.uint32),
                    "bvals": flat([[v for _, v in r] for r in bias], np.float32), "bstarts": starts(bias), "mask": mask,
                    "maskof": mask_of}.items():
        np.ascontiguousarray(x).tofile(tmp_path / f"{name}.bin")
    meta = {"tipo": "F16" if t == F16 else "I8", "cabezas": heads, "cabezasQ": q_heads, "dim": dim, "pagina": page, "paginas": b.pages,
            "secuencias": 3, "tokens": b.tokens, "paginasTabla": b.table_pages, "maxNuevos": 5, "maxLargo": 70, "ventana": window,
            "escala": 0.125, "freqs": freqs.tolist(), "filas": 3, "vocab": 5003, "mascaras": 2}
    (tmp_path / "meta.json").write_text(json.dumps(meta))
    r = subprocess.run(["node", os.path.join(HERE, "js", "shim_kv.js"), str(tmp_path)], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stderr
    out = json.loads((tmp_path / "out.json").read_text())
    a = np.arange(70)[:, None] * freqs
    rope = np.stack([np.cos(a), np.sin(a)], 1).astype(np.float32)
    x = rows.reshape(b.tokens, -1, dim)
    q = turn(x[:, :q_heads], b.positions(), rope, dim, True, qn, 1e-5)
    got = np.array(out["q"]).reshape(q.shape)
    assert np.abs(got - q).max() <= 2.0 ** -20 * np.abs(q).max()
    values = decode(t, np.array(out["cache"], np.uint8), b.pages, heads, dim, page)
    k = turn(x[:, q_heads:q_heads + heads], b.positions(), rope, dim, True, kn, 1e-5)
    for i, (s, pos) in enumerate(zip(b.seq(), b.positions())):
        v = values[b.table[s, pos // page], 0, :, pos % page]
        assert np.abs(v - k[i]).max() <= np.abs(k[i]).max() * (2.0 ** -11 if t == F16 else 1 / 250)
    want = attend(values, b.table, b.starts, b.lens, got, q_heads, 0.125, window, page)
    y = np.array(out["y"]).reshape(want.shape)
    assert (np.linalg.norm(y - want, axis=-1) <= 1e-5 * np.linalg.norm(want, axis=-1) + 1e-6 * np.abs(values).max()).all()
    want = expected(z, 0, h, pen, bias, mask, mask_of)
    assert np.array_equal(np.array(out["logits"], np.uint32).reshape(z.shape), want.view(np.uint32))
    assert out["stats"]["kvAppend"] >= 3 and out["stats"]["kvAttn"] >= 3 and out["stats"]["logits"] == 3
