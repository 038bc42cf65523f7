"""The softmax weights of eff_kv_attn themselves: values that are unit vectors, so that a row's output is its weights.

Tolerance. Keys and queries are such that every score is exact, and at most 0.5 (of log2) below its row's largest. What
is left, as relative errors of a weight: its exponent's rounding (2^-26 ln 2 where it is computed next to 0), the scale's
(2^-23 of 0.5, ln 2), the exponential's last place, the two fp16 parts (2^-23 at most, 2^-24 in the mean), the sum and the
division (2^-24 each). Their root of the mean square is below 1.2e-7; exponents near 14, whose last place is 2^-20, would
alone make it 1.9e-7.
"""
import numpy as np
import pytest

from kv_reference import F16, I8, Batch, attend, encode
from test_gpu_kv_attn import launch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_weights_of_a_short_context(ctx, eff, t, dim):
    rng = np.random.default_rng(dim)
    seqs, n = 16, 32
    b = Batch(rng, [1] * seqs, [n] * seqs, 16)
    rows = np.zeros((b.pages, 2, 1, 16, dim), np.float32)
    for s in range(seqs):
        for a in range(n):
            page, slot = b.table[s, a // 16], a % 16
            rows[page, 0, 0, slot, 3] = np.float16(0.34 * rng.random() + 0.01)
            rows[page, 1, 0, slot, a] = 1
    data, values = encode(t, rows)
    q = np.zeros((seqs, 16, dim), np.float32)
    q[:, :, 3] = np.float16(0.5 + 0.5 * rng.random((seqs, 16)))
    got = launch(eff, ctx, t, 1, dim, b, data, q, 16, 1.0)[:, :, :n]
    want = attend(values, b.table, b.starts, b.lens, q, 16, 1.0, 0, 16)[:, :, :n]
    assert np.sqrt(((got / want - 1) ** 2).mean()) <= 1.2e-7
