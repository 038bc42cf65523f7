"""eff_kv_attn over int8 rows whose scales a caller wrote: of either sign, and of very different sizes.

Tolerance. A score of magnitude |s| (below 30 here) is off by about |s| 2^-22 and its weight by the same relative amount,
7e-6 at most, and a weight times a scale keeps 22 bits of the largest such product: the weighted mean moves by less than
1e-5 of the weighted mean of the values' magnitudes, column by column.
"""
import numpy as np
import pytest

from kv_reference import I8, Batch, attend, decode, encode
from test_gpu_kv_attn import launch

pytestmark = pytest.mark.gpu

# heads, group, new, lens: a tile each, shared tiles, the kernel of many rows
FORMS = [(2, 4, [1, 3], [70, 515]), (1, 8, [1], [20011]), (8, 8, [500, 33], [1100, 200])]


def near(got, values, b, q, q_heads, scale):
    want = attend(values, b.table, b.starts, b.lens, q, q_heads, scale, 0, b.page)
    sizes = values.copy()
    sizes[:, 1] = np.abs(sizes[:, 1])
    limit = 1e-5 * np.linalg.norm(attend(sizes, b.table, b.starts, b.lens, q, q_heads, scale, 0, b.page), axis=-1)
    err = np.linalg.norm(got - want, axis=-1)
    worst = np.unravel_index(np.argmax(err / limit), err.shape)
    assert np.isfinite(got).all()
    assert (err <= limit).all(), f"row {worst}: off by {err[worst]:.3g}, {limit[worst]:.3g} allowed"


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", FORMS)
@pytest.mark.parametrize("signs", ["all", "mixed", "large"])
def test_negative_scales(ctx, eff, dim, heads, group, new, lens, signs):
    """Scales of K and V below zero: all of them, one in two, or one in two of V and these eight times as large."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, new, lens, 32)
    data, _ = encode(I8, rng.standard_normal((b.pages, 2, heads, 32, dim)).astype(np.float32))
    scales = data.reshape(b.pages, 2, heads, -1)[..., 32 * dim:].view(np.float32)
    down = rng.integers(0, 2, scales.shape) == 1
    if signs == "all":
        scales *= -1
    elif signs == "mixed":
        scales[down] *= -1
    else:
        scales[:, 1][down[:, 1]] *= -8
    q = rng.standard_normal((b.tokens, heads * group, dim)).astype(np.float32)
    got = launch(eff, ctx, I8, heads, dim, b, data, q, heads * group, dim ** -0.5)
    near(got, decode(I8, data, b.pages, heads, dim, 32), b, q, heads * group, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", FORMS)
@pytest.mark.parametrize("where", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("size", [1e7, 1e12])
def test_large_scale_of_a_small_weight(ctx, eff, dim, heads, group, new, lens, where, size):
    """A value far larger than the others whose token has e^-60 of the others' weight: it takes no bits from them. Before,
    among and after them."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, new, lens, 32)
    rows = rng.standard_normal((b.pages, 2, heads, 32, dim)).astype(np.float32)
    along = np.sign(rng.standard_normal(dim)).astype(np.float32)
    for s, (n, length) in enumerate(zip(new, lens)):
        at = int(where * (length - n))        # seen by all of the sequence's new tokens
        page, slot = b.table[s, at // 32], at % 32
        rows[page, 0, :, slot] = -along
        rows[page, 1, :, slot] *= size
    data, values = encode(I8, rows)
    # scores of about -60 there, within 4 of 0 elsewhere
    q = (60 * dim ** -0.5 * along + 0.01 * rng.standard_normal((b.tokens, heads * group, dim))).astype(np.float32)
    rows_k = data.reshape(b.pages, 2, heads, -1)[:, 0]
    keep = {(b.table[s, int(where * (n - m)) // 32], int(where * (n - m)) % 32) for s, (m, n) in enumerate(zip(new, lens))}
    scales = rows_k[..., 32 * dim:].view(np.float32)
    for p in range(b.pages):
        for slot in range(32):
            if (p, slot) not in keep:
                scales[p, :, slot] *= 0.02
    got = launch(eff, ctx, I8, heads, dim, b, data, q, heads * group, dim ** -0.5)
    near(got, decode(I8, data, b.pages, heads, dim, 32), b, q, heads * group, dim ** -0.5)
