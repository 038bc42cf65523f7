"""Capped scores of very large queries over very small int8 keys, and the other way round: what the cap sees is their
product, not the size of either."""
import numpy as np
import pytest

from kv_reference import I8, Batch, encode
from kv_rules_reference import attend_rules
from test_gpu_kv_attn import check
from test_gpu_kv_rules import launch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [1e-6, 1.0, 40.0])
@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e20, 1e30, 1e37])
@pytest.mark.parametrize("group", [1, 40])
def test_queries_and_keys_of_any_size(ctx, eff, cap, size, group):
    scores = np.array([-300.0, -15.0, -0.5, 0.0, 0.25, 3.0, 15.0, 150.0])
    n = len(scores)
    b = Batch(np.random.default_rng(1), [1] * n, [2] * n, 16)
    rows = np.zeros((b.pages, 2, 1, 16, 64), np.float32)
    key = np.float32(127 * 2.0 ** -126 * (1e37 / size))      # at 1e37 the smallest scale that is a normal number
    for s in range(n):
        # the first key: its score is q's first value times it; the second's is 0
        rows[b.table[s, 0], 0, 0, 0, 0] = key
        rows[b.table[s, 0], 1, 0, 0, 0] = 1.0
    data, values = encode(I8, rows)
    q = np.zeros((n, group, 64), np.float32)
    q[:, :, 0] = (scores / 15 * size)[:, None]
    scale = 15 / (float(size) * float(key))
    got = launch(eff, ctx, I8, 1, 64, b, data, q, group, scale, cap=cap)
    check(got, attend_rules(values, b, q, group, scale, cap=cap), values)
