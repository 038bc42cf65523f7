"""eff_kv_attn: a key that is not finite, and a score past f32, are seen in the rows that see them, whatever the score's sign."""
import numpy as np
import pytest

from kv_reference import F16, I8, Batch, encode
from test_gpu_kv_attn import launch

pytestmark = pytest.mark.gpu

# heads, group, new, lens: a tile each (one of a single token), shared tiles, the kernel of many rows
FORMS = [(2, 4, [1, 3, 1], [1, 515, 70]), (1, 8, [1], [20011]), (8, 8, [500, 33], [1100, 200])]


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", FORMS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_key(ctx, eff, t, dim, heads, group, new, lens, bad):
    """In int8 the row's scale, as the append writes it for a row with an infinity; in fp16 one value."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, new, lens, 32)
    data, _ = encode(t, rng.standard_normal((b.pages, 2, heads, 32, dim)).astype(np.float32))
    rows = data.reshape(b.pages, 2, heads, -1)
    for s, (n, length) in enumerate(zip(new, lens)):
        at = (length - n) // 2                # every new token of the sequence sees it
        page, slot = b.table[s, at // 32], at % 32
        if t == F16:
            rows[page, 0, :, slot * dim * 2:(slot + 1) * dim * 2].view(np.float16)[:, 7] = bad
        else:
            rows[page, 0, :, 32 * dim:].view(np.float32)[:, slot] = bad
    q = rng.standard_normal((b.tokens, heads * group, dim)).astype(np.float32)
    # halves of fp16 exactly: nothing is left for a second part, whose product could hide the first's sign
    for x in (q, q.astype(np.float16).astype(np.float32), np.abs(q), -np.abs(q)):
        got = launch(eff, ctx, t, heads, dim, b, data, x, heads * group, dim ** -0.5)
        assert not np.isfinite(got).all(-1).any()


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", FORMS)
@pytest.mark.parametrize("scale", [1e30, -1e30, 1e18, -1e18])
def test_scores_past_f32(ctx, eff, t, dim, heads, group, new, lens, scale):
    """Finite keys, queries and scale whose scores are not: no finite answer, zeros least of all."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, new, lens, 32)
    data, _ = encode(t, (1 + rng.random((b.pages, 2, heads, 32, dim))).astype(np.float32))
    q = (1e20 * (1 + rng.random((b.tokens, heads * group, dim)))).astype(np.float32)
    got = launch(eff, ctx, t, heads, dim, b, data, q, heads * group, scale)
    assert not np.isfinite(got).all(-1).any()
