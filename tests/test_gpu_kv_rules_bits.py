"""Attention under a cap: a row's bits do not depend on cached bytes that it does not see, nor on the other rows of its
tile. Ordinary scores, of which a wave computes the capped form by a polynomial alone, beside keys that take the scores
of rows which see them, or of nobody, far past the cap."""
import numpy as np
import pytest

from kv_reference import F16, I8, Batch
from test_gpu_kv_attn import make
from test_gpu_kv_rules import any_masks, launch, slopes_of, trees

pytestmark = pytest.mark.gpu


def loud(t, data, b, heads, dim, where):
    """The cache's bytes with the keys at `where` [pages][page] 3000 large, of either sign."""
    d = data.reshape(b.pages, 2, heads, -1).copy()
    rng = np.random.default_rng(0)
    for p, slot in zip(*np.nonzero(where)):
        sign = rng.choice([-1, 1], (heads, dim))
        if t == F16:
            d[p, 0, :, 2 * slot * dim:2 * (slot + 1) * dim] = (3000 * sign).astype(np.float16).view(np.uint8)
        else:
            d[p, 0, :, slot * dim:(slot + 1) * dim] = (127 * sign).astype(np.int8).view(np.uint8)
            at = b.page * dim + 4 * slot
            d[p, 0, :, at:at + 4] = np.frombuffer(np.float32(3000 / 127).tobytes(), np.uint8)
    return d.reshape(b.pages, -1)


def places(b, s, at):
    """The cache's places of sequence s at the positions `at`, [pages][page]."""
    got = np.zeros((b.pages, b.page), bool)
    at = np.asarray(at, int)
    got[b.table[s, at // b.page], at % b.page] = True
    return got


# tiles of 16 rows, whole and shared, and of 64, whole and shared
SHAPES = [(2, 4, [1, 3], [40, 500]), (1, 4, [2, 1], [9000, 300]), (4, 4, [700], [900]), (8, 4, [20, 17, 3], [3100, 2900, 50])]


def ranges_of(b):
    """Every token sees 20 cached ones or fewer, the third of them first."""
    return np.array([(length // 3, min(length, length // 3 + 20)) for n, length in zip(b.new, b.lens) for _ in range(n)])


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", SHAPES)
@pytest.mark.parametrize("name", ["", "ranges", "tree"])
def test_what_nobody_sees(ctx, eff, t, dim, heads, group, new, lens, name):
    rng = np.random.default_rng(dim)
    b = Batch(rng, new, lens, 32)
    data, _ = make(rng, t, heads, dim, b)
    q = rng.standard_normal((b.tokens, heads * group, dim)).astype(np.float32)
    rules = {"cap": 40.0, "slopes": None if name else slopes_of(heads * group)}
    unseen = np.ones((b.pages, b.page), bool)
    if name == "ranges":
        rules["ranges"] = ranges_of(b)
        seen = [np.arange(length // 3, min(length, length // 3 + 20)) for length in lens]
    elif name == "tree":
        rules["masks"] = any_masks(rng, b)
        seen = [np.concatenate([np.arange(length - n), length - n + np.flatnonzero(m.any(0))]) for n, length, m in zip(new, lens, rules["masks"])]
    else:
        seen = [np.arange(length) for length in lens]
    for s, at in enumerate(seen):
        unseen &= ~places(b, s, at)
    assert unseen.any()
    want = launch(eff, ctx, t, heads, dim, b, data, q, heads * group, dim ** -0.5, **rules)
    got = launch(eff, ctx, t, heads, dim, b, loud(t, data, b, heads, dim, unseen), q, heads * group, dim ** -0.5, **rules)
    assert np.isfinite(want).all() and want.any()
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", SHAPES)
@pytest.mark.parametrize("tree", [False, True])
def test_what_others_see(ctx, eff, t, dim, heads, group, new, lens, tree):
    """The last new token's key: the rows of the tokens before it, and of the other sequences, keep their bits."""
    rng = np.random.default_rng(dim + 1)
    b = Batch(rng, new, lens, 32)
    data, _ = make(rng, t, heads, dim, b)
    q = rng.standard_normal((b.tokens, heads * group, dim)).astype(np.float32)
    rules = {"cap": 40.0}
    s = int(np.argmax(new))
    last = int(b.starts[s]) + new[s] - 1
    sees = np.zeros(b.tokens, bool)
    sees[last] = True
    if tree:
        rules["masks"] = trees(rng, b)
        sees[b.starts[s]:last + 1] = rules["masks"][s][:, -1]
    want = launch(eff, ctx, t, heads, dim, b, data, q, heads * group, dim ** -0.5, **rules)
    got = launch(eff, ctx, t, heads, dim, b, loud(t, data, b, heads, dim, places(b, s, [lens[s] - 1])), q, heads * group, dim ** -0.5, **rules)
    assert (got[sees] != want[sees]).any()
    assert np.array_equal(got[~sees].view(np.uint32), want[~sees].view(np.uint32))
