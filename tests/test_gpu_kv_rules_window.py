"""A window over a tree of drafts leaves out cached tokens ahead of them, and no draft whose bit is set: nor one that has
no bits of its own, whose position is the one before the first draft's, at the smallest window that a tree may have."""
import numpy as np
import pytest

from kv_reference import F16, I8, Batch
from kv_rules_reference import attend_rules
from test_gpu_kv_attn import check, make
from test_gpu_kv_rules import launch, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("n,group", [(3, 2), (8, 4), (40, 4)])
@pytest.mark.parametrize("slopes", [False, True])
def test_window_of_all_drafts(ctx, eff, t, dim, n, group, slopes):
    rng = np.random.default_rng(n)
    heads, first = 2, 100
    b = Batch(rng, [n], [first + n], 16)
    data, values = make(rng, t, heads, dim, b)
    q = rng.standard_normal((n, heads * group, dim)).astype(np.float32)
    mask = rng.random((n, n)) < 0.5
    mask[1] = False       # a draft without bits
    mask[-1] = True       # one that sees all of them: with its window of n, nothing else
    rules = {"masks": [mask], "slopes": slopes_of(heads * group) if slopes else None}
    got = launch(eff, ctx, t, heads, dim, b, data, q, heads * group, dim ** -0.5, n, **rules)
    # each row alone, without a window, over the tokens ahead that its own window leaves
    for i in range(n):
        ahead = n - int(mask[i].sum())
        one = Batch(rng, [n], [ahead + n], 16)
        rows = np.zeros((one.pages, *values.shape[1:]))
        for new, old in enumerate(range(first - ahead, first + n)):
            rows[one.table[0, new // 16], :, :, new % 16] = values[b.table[0, old // 16], :, :, old % 16]
        want = attend_rules(rows, one, q, heads * group, dim ** -0.5, **rules)
        check(got[i:i + 1], want[i:i + 1], values)
