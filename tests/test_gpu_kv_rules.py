"""Attention with rules on its scores and on what is seen (eff_kv_attn_rules) on the GPU against softmax in 64 bits.

Tolerance. As in test_gpu_kv_attn a score s (below 30 in size here) is off by |s| 2^-22 of q's 22 bits, and here by three
roundings of its size (2^-24 each) on top: 1.2e-5 at most, and a weight by as much of itself. A cap gives at most
cap * 2^-23 (the exponential form, from 0.625 of the cap on; 6e-6 at 50) instead, a distance the rounding of slope times
distance, 2^-24 of a bias that leaves a weight (below 30: 2e-6). The weighted mean of values moves by less than that
times their size, and the errors of different tokens are independent: REL is 1e-5 of the row's norm, plus 1e-6 of the
largest value for rows whose values cancel.
"""
import ctypes
import threading

import numpy as np
import pytest

from kv_reference import F16, I8, NO_PAGE, Batch, encode, page_bytes
from kv_rules_reference import attend_rules, random_tree, tree_mask, tree_words
from test_gpu_kv_attn import check, make

pytestmark = pytest.mark.gpu


def slopes_of(heads):
    return (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)


def launch(eff, ctx, t, heads, dim, b, data, q, q_heads, scale, window=0, cap=0.0, slopes=None, ranges=None, masks=None, words=None, **more):
    cb, qb = ctx.upload(data), ctx.upload(q.astype(np.float32))
    out = ctx.upload(np.full(q.shape, 7, np.float32))
    rules = {"cap": cap}
    if slopes is not None:
        rules["slopes"] = ctx.upload(np.asarray(slopes, np.float32))
    if ranges is not None:
        rules["ranges"] = ctx.upload(np.asarray(ranges, np.uint32))
    if masks is not None:
        words = words or (max(max(b.new), more.get("max_new") or 1) + 31) // 32
        rules.update(tree=ctx.upload(tree_words(masks, words)), tree_words=words)
    batch = b.upload(eff, ctx, **more)
    rules = eff.KvRules(**rules)
    ctx.kv_attn(eff.KvCache(t, heads, dim, b.page, b.pages, cb), batch, qb, out, q_heads, scale, window, rules=rules)
    got = out.read(np.float32).reshape(q.shape)
    for x in [cb, qb, out] + batch.buffers + rules.buffers:
        x.free()
    return got


def run(eff, ctx, seed, t, heads, group, dim, page, new, lens, window=0, sharp=1.0, dirty=np.nan, cap=0.0, slopes=False, ranges=None, masks=None,
        words=None, **more):
    rng = np.random.default_rng(seed)
    b = Batch(rng, new, lens, page)
    data, values = make(rng, t, heads, dim, b, dirty)
    q = (sharp * rng.standard_normal((b.tokens, heads * group, dim))).astype(np.float32)
    scale = dim ** -0.5
    rules = {"cap": cap, "slopes": slopes_of(heads * group) if slopes else None, "ranges": ranges(rng, b) if ranges else None,
             "masks": masks(rng, b) if masks else None}
    got = launch(eff, ctx, t, heads, dim, b, data, q, heads * group, scale, window, words=words, **rules, **more)
    check(got, attend_rules(values, b, q, heads * group, scale, window, **rules), values)


def trees(rng, b):
    return [tree_mask(random_tree(rng, n)) if n else np.zeros((0, 0), bool) for n in b.new]


def any_masks(rng, b):
    """Any bits: drafts that nobody sees, that do not see themselves, rows without a bit."""
    got = [rng.random((n, n)) < 0.5 for n in b.new]
    for m in got:
        if len(m) > 1:
            m[:, len(m) // 2] = False
            m[len(m) // 3] = False
    return got


def documents(rng, b):
    got = []
    for n, length in zip(b.new, b.lens):
        starts, at = [], 0
        while at < length:
            size = int(rng.integers(1, 200))
            starts += [at] * size
            at += size
        got += [(starts[p] if p >= 0 else 0, max(p, 0) + 1) for p in range(length - n, length)]
    return np.array(got, np.int64).reshape(-1, 2)


def prefix(rng, b):
    got = []
    for n, length in zip(b.new, b.lens):
        k = int(rng.integers(0, length + 2))
        got += [(0, max(p + 1, k)) for p in range(length - n, length)]
    return np.array(got, np.int64).reshape(-1, 2).clip(0)


def any_ranges(rng, b):
    """Any ranges: empty ones, reversed ones, some past the end."""
    got = []
    for n, length in zip(b.new, b.lens):
        r = rng.integers(0, length + 2, (n, 2))
        r.sort(1)
        kind = rng.integers(0, 8, n)
        r[kind == 0] = r[kind == 0][:, ::-1]
        r[kind == 1, 1] = 0xFFFFFFFF
        r[kind == 2] = 5
        r[kind == 3] = (0x90000000, 0xFFFFFFFF)
        got.append(r)
    return np.concatenate(got)


MASKS = {"tree": trees, "any tree": any_masks}
RANGES = {"documents": documents, "prefix": prefix, "any range": any_ranges}
SHAPES = [(2, 4, [1, 1, 1], [1, 50, 900]), (3, 5, [6, 40, 0, 1], [500, 40, 30, 77]), (1, 16, [1, 33, 64, 7], [300, 33, 170, 1300]),
          (2, 1, [1, 2, 100], [2600, 33, 333])]


def rules_of(name):
    return {"masks": MASKS[name]} if name in MASKS else {"ranges": RANGES[name]} if name in RANGES else {}


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", SHAPES)
@pytest.mark.parametrize("name", ["tree", "any tree", "documents", "prefix", "any range"])
def test_masks(ctx, eff, t, dim, heads, group, new, lens, name):
    run(eff, ctx, dim + group, t, heads, group, dim, 16, new, lens, **rules_of(name))


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens", SHAPES)
@pytest.mark.parametrize("cap,slopes,sharp", [(2.0, False, 3.0), (0.0, True, 1.0), (20.0, True, 5.0)])
def test_scores(ctx, eff, t, dim, heads, group, new, lens, cap, slopes, sharp):
    run(eff, ctx, dim + group, t, heads, group, dim, 32, new, lens, cap=cap, slopes=slopes, sharp=sharp)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("name", ["tree", "any tree", "documents", "prefix", "any range", ""])
@pytest.mark.parametrize("dim,heads,group,new,lens", [(128, 2, 8, [30, 5], [9000, 400]), (64, 1, 4, [1, 70], [40001, 300])])
def test_masks_and_scores(ctx, eff, t, name, dim, heads, group, new, lens):
    run(eff, ctx, dim, t, heads, group, dim, 64, new, lens, cap=10.0, slopes=True, sharp=2.0, **rules_of(name))


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("name", ["tree", "any tree", ""])
@pytest.mark.parametrize("window", [40, 41, 63, 100, 5000])
def test_windows(ctx, eff, t, name, window):
    run(eff, ctx, window, t, 2, 3, 64, 16, [40, 1, 8], [700, 900, 8], window, slopes=True, cap=30.0, **rules_of(name))
    run(eff, ctx, window, t, 1, 4, 128, 16, [4, 1, 8], [700, 9000, 8], window, words=3, **rules_of(name) or {"cap": 30.0})


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("name", ["tree", "any tree", "documents", "prefix", "any range", ""])
@pytest.mark.parametrize("heads,group,new,lens", [(4, 4, [700], [900]), (8, 3, [400, 129, 1], [403, 1000, 2000])])
def test_many_rows(ctx, eff, t, dim, name, heads, group, new, lens):
    run(eff, ctx, dim, t, heads, group, dim, 32, new, lens, **rules_of(name) or {"cap": 20.0, "slopes": True})


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("name", ["any tree", "documents", "any range", ""])
def test_many_rows_of_int8(ctx, eff, dim, name):
    """Enough tiles of 64 rows for pages that are converted on the way."""
    run(eff, ctx, dim, I8, 16, 2, dim, 32, [800, 1, 500], [850, 300, 500], **rules_of(name) or {"cap": 20.0, "slopes": True})


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("group,new,lens", [(4, [1, 3], [50, 900]), (4, [30, 9], [3000, 1200]), (1, [900, 700], [900, 700])])
def test_rows_behind_the_last_sequence(ctx, eff, t, group, new, lens):
    """Tokens of a padded batch that belong to no sequence: their rows stay as they were."""
    rng = np.random.default_rng(group)
    b = Batch(rng, new, lens, 16)
    data, values = make(rng, t, 16, 64, b)
    tokens = b.tokens + 5
    q = rng.standard_normal((tokens, 16 * group, 64)).astype(np.float32)
    out = ctx.upload(np.full(q.shape, 7, np.float32))
    masks = trees(rng, b)
    words = (max(new) + 31) // 32
    tree = np.concatenate([tree_words(masks, words), np.full((5, words), 0xFFFFFFFF, np.uint32)])
    mine = b.upload(eff, ctx)
    batch = eff.KvBatch(*mine.buffers, seqs=2, tokens=tokens, table_pages=b.table_pages, max_new=max(new), max_len=max(lens))
    ctx.kv_attn(eff.KvCache(t, 16, 64, 16, b.pages, ctx.upload(data)), batch, ctx.upload(q), out, 16 * group, 0.125,
                rules=eff.KvRules(tree=ctx.upload(tree), tree_words=words))
    got = out.read(np.float32).reshape(q.shape)
    assert (got[b.tokens:] == 7).all()
    check(got[:b.tokens], attend_rules(values, b, q[:b.tokens], 16 * group, 0.125, masks=masks), values)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("name", ["tree", "any tree", "any range", ""])
def test_shared_tiles(ctx, eff, dim, name):
    """Tiles of 64 rows that several workgroups share, of sequences of any length: joins of a few and of one."""
    rng = np.random.default_rng(dim)
    new, lens = [20, 17, 0, 1, 9, 20, 3, 20], [3100, 2900, 50, 1, 9, 20, 2000, 1111]
    more = rules_of(name) or {"cap": 20.0, "slopes": True}
    run(eff, ctx, dim, F16, 8, 4, dim, 64, new, lens, **more)
    if name in ("tree", ""):
        run(eff, ctx, dim, F16, 8, 6, dim, 32, new, lens, 1500, **more)
        new = [int(n) for n in rng.integers(1, 9, 70)]      # more sequences than a wave has lanes
        run(eff, ctx, dim, F16, 4, 4, dim, 16, new, [n + int(m) for n, m in zip(new, rng.integers(0, 1400, 70))], **more)


@pytest.mark.parametrize("dim,heads,group,new,length", [(64, 2, 16, 8, 50021), (128, 1, 32, 9, 40001), (256, 1, 24, 12, 33000), (96, 4, 8, 13, 20000)])
def test_joins_in_two_steps(ctx, eff, dim, heads, group, new, length):
    """More workgroups to a tile of 64 rows than are joined at once."""
    run(eff, ctx, dim, F16, heads, group, dim, 64, [new], [length], masks=trees)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("name", ["tree", "documents", ""])
def test_lengths(ctx, eff, t, name):
    """More sequences than a wave has lanes, of every length; whole tiles, shared ones, shares that go on."""
    rng = np.random.default_rng(1)
    more = rules_of(name) or {"cap": 30.0}
    lens = [2300] + [int(n) for n in rng.integers(0, 400, 75)]
    for dim, group, new in ((64, 4, 1), (128, 2, 6), (96, 3, 20)):
        run(eff, ctx, dim, t, 4, group, dim, 16, [min(new, n) for n in lens], lens, **more)
    lens = [2300, 129] + [int(n) for n in rng.integers(300, 1300, 22)]
    run(eff, ctx, 3, t, 32, 2, 64, 64, [1] * 24, lens, **more)
    run(eff, ctx, 4, t, 2, 8, 256, 64, [5, 1], [20011, 300], **more)
    run(eff, ctx, 5, t, 2, 16, 64, 16, [1, 2], [16000, 9000], **more)
    lens = [900, 0, 1, 511, 512, 513] + [int(n) for n in rng.integers(1, 900, 11)]
    for heads in (8, 12):
        run(eff, ctx, heads, t, heads, 4, 128, 32, [min(2, n) for n in lens], lens, **more)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("new,lens", [([1], [700]), ([40, 3], [700, 20])])
def test_bounds_above_the_sizes(ctx, eff, t, new, lens):
    """The bounds of a recording, far above the sizes; more words than the trees have."""
    run(eff, ctx, 6, t, 2, 4, 128, 16, new, lens, masks=trees, max_new=300, max_len=len(lens) and 16 * -(-max(lens) // 16))
    run(eff, ctx, 7, t, 2, 4, 64, 16, new, lens, 400, masks=trees, max_new=256, words=11)
    run(eff, ctx, 8, t, 2, 4, 64, 16, new, lens, ranges=documents, max_new=300)


def test_more_new_tokens_than_length(ctx, eff):
    """Drafts without a position: zeros, and nobody sees them."""
    for more in ({"masks": any_masks}, {"ranges": any_ranges}, {"cap": 20.0, "slopes": True}):
        run(eff, ctx, 2, F16, 2, 2, 64, 16, [9, 4], [5, 30], **more)


def test_missing_pages(ctx, eff):
    rng = np.random.default_rng(5)
    b = Batch(rng, [20, 3], [100, 64], 16)
    b.table[0, 2], b.table[0, 5], b.table[1, 0] = NO_PAGE, b.pages, NO_PAGE
    data, values = make(rng, F16, 2, 64, Batch(rng, [20, 3], [100, 64], 16))
    q = rng.standard_normal((b.tokens, 6, 64)).astype(np.float32)
    for more in ({"masks": any_masks(rng, b)}, {"ranges": documents(rng, b)}, {"slopes": slopes_of(6), "cap": 9.0}):
        got = launch(eff, ctx, F16, 2, 64, b, data, q, 6, 0.1, **more)
        check(got, attend_rules(values, b, q, 6, 0.1, **more), values)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", [0, 1])
@pytest.mark.parametrize("new,group", [(12, 1), (20, 4), (130, 16)])
def test_not_finite(ctx, eff, t, dim, bad, where, new, group):
    """A draft's key or value that is not finite reaches the rows that see it, under a cap too, and no others."""
    rng = np.random.default_rng(new)
    b = Batch(rng, [new], [new + 70], 32)
    rows = rng.standard_normal((b.pages, 2, 2, 32, dim)).astype(np.float32)
    masks = trees(rng, b)
    j = new // 2
    at = 70 + j
    data, values = encode(t, rows)
    page, slot = b.table[0, at // 32], at % 32
    d = data.reshape(b.pages, 2, 2, -1)
    if t == F16:
        d[page, where, 0, 2 * (slot * dim + 3):2 * (slot * dim + 3) + 2] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    else:
        o = 32 * dim + 4 * slot
        d[page, where, 0, o:o + 4] = np.frombuffer(np.float32(bad).tobytes(), np.uint8)
    q = rng.standard_normal((new, 2 * group, dim)).astype(np.float32)
    for cap in (0.0, 5.0):
        want = attend_rules(values, b, q, 2 * group, dim ** -0.5, cap=cap, masks=masks)
        got = launch(eff, ctx, t, 2, dim, b, data.reshape(b.pages, -1), q, 2 * group, dim ** -0.5, cap=cap, masks=masks)
        sees = masks[0][:, j]
        hit = np.zeros((new, 2 * group), bool)
        hit[sees, :group] = True
        bad_rows = ~np.isfinite(got).all(-1)
        assert np.array_equal(bad_rows, hit)
        check(np.where(hit[..., None], 0, got), np.where(hit[..., None], 0, want), values)


@pytest.mark.parametrize("cap,sharp", [(1e-6, 1.0), (0.01, 1.0), (1.0, 1e-20), (30.0, 1e4), (1e6, 1.0), (5.0, 30.0)])
def test_sizes_of_caps(ctx, eff, cap, sharp):
    """From scores far past the cap to scores far below it."""
    run(eff, ctx, 3, F16, 2, 4, 64, 16, [1, 5], [300, 60], cap=cap, sharp=sharp)


def test_cap_in_itself(ctx, eff):
    """Two keys of known scores: the weights' ratio gives the capped score, over the polynomial and the exponential form."""
    scores = np.concatenate([np.linspace(-40, 40, 161), [1e-4, -1e-3, 1e3, -1e3]])
    n = len(scores)
    b = Batch(np.random.default_rng(1), [1] * n, [2] * n, 16)
    rows = np.zeros((b.pages, 2, 1, 16, 64), np.float32)
    for s in range(n):
        rows[b.table[s, 0], 0, 0, 0, 0] = 1.0      # the first key: its score is q's first value; the second's is 0
        rows[b.table[s, 0], 1, 0, 0, 0] = 1.0
    data, values = encode(F16, rows)
    q = np.zeros((n, 1, 64), np.float32)
    q[:, 0, 0] = scores
    got = launch(eff, ctx, F16, 1, 64, b, data, q, 1, 1.0, cap=8.0)[:, 0, 0].astype(np.float64)
    x = 8 * np.tanh(q[:, 0, 0].astype(np.float64) / 8)
    want = 1 / (1 + np.exp(-x))
    # x to 8 * 2^-23 + 2^-22 of itself, a weight w / (1 + w) moves by at most a quarter of that, and rounds three times
    assert (np.abs(got - want) <= (8 * 2.0 ** -23 + 8 * 2.0 ** -22) / 4 + 4 * 2.0 ** -24).all()


def test_far_ranges(ctx, eff):
    """Ranges far from the row: biases of thousands, of which only the differences count."""
    b = Batch(np.random.default_rng(2), [3], [30000], 64)
    rng = np.random.default_rng(3)
    data, values = make(rng, F16, 1, 64, b)
    q = rng.standard_normal((3, 2, 64)).astype(np.float32)
    ranges = np.array([[0, 300], [5, 17000], [100, 110]])
    slopes = np.array([0.5, 0.01], np.float32)
    got = launch(eff, ctx, F16, 1, 64, b, data, q, 2, 0.125, ranges=ranges, slopes=slopes)
    check(got, attend_rules(values, b, q, 2, 0.125, ranges=ranges, slopes=slopes), values)


def test_as_without_rules(ctx, eff):
    """Empty rules, a chain of drafts, ranges of all before: what eff_kv_attn says."""
    rng = np.random.default_rng(4)
    b = Batch(rng, [5, 1, 40], [300, 20, 700], 16)
    data, values = make(rng, F16, 2, 128, b)
    q = rng.standard_normal((b.tokens, 8, 128)).astype(np.float32)
    qb, out = ctx.upload(q), ctx.alloc(q.nbytes)
    ctx.kv_attn(eff.KvCache(F16, 2, 128, 16, b.pages, ctx.upload(data)), b.upload(eff, ctx), qb, out, 8, 0.1)
    want = out.read(np.float32).reshape(q.shape)
    assert np.array_equal(launch(eff, ctx, F16, 2, 128, b, data, q, 8, 0.1), want)
    chains = [np.tri(n, dtype=bool) for n in b.new]
    before = np.concatenate([[(0, p + 1) for p in range(length - n, length)] for n, length in zip(b.new, b.lens)])
    for more in ({"masks": chains}, {"ranges": before}):
        check(launch(eff, ctx, F16, 2, 128, b, data, q, 8, 0.1, **more), want.astype(np.float64), values)


def test_strides(ctx, eff):
    rng = np.random.default_rng(6)
    b = Batch(rng, [7, 2], [50, 90], 16)
    data, values = make(rng, F16, 2, 64, b)
    x = rng.standard_normal((b.tokens, 300)).astype(np.float32)
    q = x[:, 12:268].reshape(b.tokens, 4, 64)
    masks = trees(rng, b)
    out = ctx.alloc(q.nbytes)
    rules = eff.KvRules(tree=ctx.upload(tree_words(masks, 1)), tree_words=1, cap=30.0)
    ctx.kv_attn(eff.KvCache(F16, 2, 64, 16, b.pages, ctx.upload(data)), b.upload(eff, ctx), ctx.upload(x), out, 4, 0.125, q_offset=12, q_stride=300,
                rules=rules)
    check(out.read(np.float32).reshape(q.shape), attend_rules(values, b, q, 4, 0.125, cap=30.0, masks=masks), values)


def test_same_bits(ctx, eff):
    """The same call gives the same bits, whichever workgroup joins last."""
    rng = np.random.default_rng(7)
    for t, heads, group, dim, new, lens in ((F16, 2, 4, 128, [20, 3], [9000, 5000]), (I8, 1, 16, 64, [1], [33000]), (F16, 4, 2, 256, [300], [3000]),
                                               (F16, 8, 4, 128, [20, 17, 3], [9000, 5000, 2000])):
        b = Batch(rng, new, lens, 64)
        data, _ = make(rng, t, heads, dim, b)
        q = rng.standard_normal((b.tokens, heads * group, dim)).astype(np.float32)
        masks = trees(rng, b)
        cb, qb, out = ctx.upload(data), ctx.upload(q), ctx.alloc(q.nbytes)
        cache, batch = eff.KvCache(t, heads, dim, 64, b.pages, cb), b.upload(eff, ctx)
        words = (max(new) + 31) // 32
        rules = eff.KvRules(tree=ctx.upload(tree_words(masks, words)), tree_words=words, cap=40.0, slopes=ctx.upload(slopes_of(heads * group)))
        first = None
        for _ in range(20):
            ctx.kv_attn(cache, batch, qb, out, heads * group, 0.1, rules=rules)
            got = out.read(np.uint8)
            assert first is None or np.array_equal(got, first)
            first = got


def test_recorded(ctx, eff):
    """A recorded call takes the next step's lengths, trees and rows; two recordings share the context's scratch."""
    rng = np.random.default_rng(8)
    new, lens = [22, 4], [5000, 300]
    b = Batch(rng, new, lens, 64)
    data, values = make(rng, F16, 8, 128, b)
    q = rng.standard_normal((b.tokens, 32, 128)).astype(np.float32)
    cb, qb, out = ctx.upload(data), ctx.upload(q), ctx.alloc(q.nbytes)
    cache, batch, tb = eff.KvCache(F16, 8, 128, 64, b.pages, cb), b.upload(eff, ctx), ctx.alloc(b.tokens * 4)
    rules = [eff.KvRules(tree=tb, tree_words=1), eff.KvRules(cap=20.0, slopes=ctx.upload(slopes_of(32)))]
    graphs = []
    for r in rules:
        ctx.kv_attn(cache, batch, qb, out, 32, 0.1, rules=r)
        ctx.graph_begin()
        ctx.kv_attn(cache, batch, qb, out, 32, 0.1, rules=r)
        graphs.append(ctx.graph_end())
    for step in range(4):
        b.lens = [5000 - 1600 * step, 300 - 50 * step]
        masks = trees(rng, b)
        batch.buffers[2].write(np.array(b.lens, np.uint32))
        tb.write(tree_words(masks, 1))
        for g, r, more in zip(graphs, rules, ({"masks": masks}, {"cap": 20.0, "slopes": slopes_of(32)})):
            g.launch()
            got = out.read(np.float32).reshape(q.shape)
            check(got, attend_rules(values, b, q, 32, 0.1, **more), values)
            ctx.kv_attn(cache, batch, qb, out, 32, 0.1, rules=r)
            assert np.array_equal(out.read(np.float32).reshape(q.shape), got)
    for g in graphs:
        g.destroy()


def test_streams(ctx, eff):
    """Calls on two streams of one context in turn, without a wait of the host between them."""
    rng = np.random.default_rng(9)
    hip = ctypes.CDLL("libamdhip64.so.7")
    side = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(side), 1) == 0
    b = Batch(rng, [20, 1], [9000, 4000], 64)
    data, _ = make(rng, F16, 2, 128, b)
    masks = trees(rng, b)
    with eff.Context(0) as c:
        q = c.upload(rng.standard_normal((b.tokens, 8, 128)).astype(np.float32))
        cache, batch, rules = eff.KvCache(F16, 2, 128, 64, b.pages, c.upload(data)), b.upload(eff, c), eff.KvRules(tree=c.upload(tree_words(masks, 1)), tree_words=1)
        outs = [c.alloc(q.size) for _ in range(12)]
        for i, o in enumerate(outs):
            c.set_stream(side.value if i % 2 else None)
            c.kv_attn(cache, batch, q, o, 8, 0.1, rules=rules)
        c.set_stream(None)
        got = [o.read(np.uint8) for o in outs]
        assert got[0].any() and all(np.array_equal(got[0], g) for g in got)
        c.sync()
    assert hip.hipStreamDestroy(side) == 0


def test_two_threads(eff):
    """Two contexts on threads of their own at once: the bits of each alone."""
    def work(seed, times):
        rng = np.random.default_rng(seed)
        b = Batch(rng, [20, 17, 3], [5000, 3000, 900], 64)
        data, _ = make(rng, F16, 8, 64, b)
        q, masks = rng.standard_normal((b.tokens, 32, 64)).astype(np.float32), trees(rng, b)
        with eff.Context(0) as c:
            out, qb, cache, batch = c.alloc(q.nbytes), c.upload(q), eff.KvCache(F16, 8, 64, 64, b.pages, c.upload(data)), b.upload(eff, c)
            rules = eff.KvRules(tree=c.upload(tree_words(masks, 1)), tree_words=1, cap=30.0)
            got = []
            for _ in range(times):
                c.kv_attn(cache, batch, qb, out, 32, 0.125, rules=rules)
                got.append(out.read(np.uint8))
            return got
    want, got = [work(s, 1)[0] for s in (1, 2)], [None, None]

    def thread(i):
        got[i] = work(i + 1, 10)
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert all(g is not None and all(np.array_equal(x, w) for x in g) for g, w in zip(got, want))


def test_far_pages(ctx, eff):
    """Pages whose bytes lie past 4 GiB, and drafts there."""
    heads, dim, page = 8, 256, 256
    each = page_bytes(F16, heads, dim, page)
    pages = (5 << 30) // each + 1
    cb = ctx.alloc(pages * each)
    rng = np.random.default_rng(3)
    b = Batch(rng, [6], [page + 9], page, spare=0)
    rows = rng.standard_normal((2, 2, heads, page, dim)).astype(np.float32)
    data, values = encode(F16, rows)
    h = ctypes.c_void_p()
    assert eff.lib().eff_buf_wrap(ctx.h, cb.ptr + (pages - 2) * each, 2 * each, ctypes.byref(h)) == eff.OK
    last = eff.Buffer(ctx, h, 2 * each)
    last.write(data)
    q = rng.standard_normal((6, heads, dim)).astype(np.float32)
    masks = trees(rng, b)
    batch = b.upload(eff, ctx)
    batch.buffers[0].write(b.table + np.uint32(pages - 2))
    out = ctx.alloc(q.nbytes)
    ctx.kv_attn(eff.KvCache(F16, heads, dim, page, pages, cb), batch, ctx.upload(q), out, heads, 0.06,
                rules=eff.KvRules(tree=ctx.upload(tree_words(masks, 1)), tree_words=1))
    check(out.read(np.float32).reshape(q.shape), attend_rules(values, b, q, heads, 0.06, masks=masks), values)
    cb.free()


def test_refusals(ctx, eff):
    b = Batch(np.random.default_rng(9), [40, 1], [50, 30], 16)
    cb = ctx.alloc(b.pages * page_bytes(F16, 2, 64, 16))
    q, out = ctx.alloc(b.tokens * 4 * 64 * 4), ctx.alloc(b.tokens * 4 * 64 * 4)
    tree, ranges, slopes = ctx.alloc(b.tokens * 2 * 4), ctx.alloc(b.tokens * 8), ctx.alloc(16)
    batch, cache = b.upload(eff, ctx), eff.KvCache(F16, 2, 64, 16, b.pages, cb)
    before = ctx.stats()["kv_attn"]

    def call(code, window=0, q_heads=4, **rules):
        with pytest.raises(eff.EffError) as e:
            ctx.kv_attn(cache, batch, q, out, q_heads, 0.1, window, rules=eff.KvRules(**rules))
        assert e.value.code == code and "kv attn" in str(e.value)

    for cap in (-1.0, np.nan, np.inf, 1e-7, 2e6, -0.5e-7):
        call(eff.E_INVALID, cap=cap)
    call(eff.E_INVALID, ranges=ranges, tree=tree, tree_words=2)
    call(eff.E_INVALID, window=50, ranges=ranges)
    call(eff.E_BOUNDS, tree=tree, tree_words=1)
    call(eff.E_BOUNDS, tree=tree, tree_words=0)
    call(eff.E_BOUNDS, tree=tree, tree_words=3)
    call(eff.E_BOUNDS, tree=tree, tree_words=0xFFFFFFFF)
    call(eff.E_SHAPE, window=39, tree=tree, tree_words=2)
    call(eff.E_BOUNDS, ranges=tree.ctx.alloc(b.tokens * 8 - 4))
    call(eff.E_BOUNDS, slopes=ctx.alloc(12))
    call(eff.E_INVALID, slopes=out)
    call(eff.E_INVALID, ranges=out)
    call(eff.E_INVALID, tree=out, tree_words=2)
    call(eff.E_SHAPE, q_heads=5, cap=1.0)
    assert ctx.stats()["kv_attn"] == before
    assert eff.lib().eff_kv_attn_rules(None, None, None, None, 0, 0, None, 1, 1.0, 0, None) == eff.E_INVALID
    rules = eff.KvRules(tree=tree, tree_words=2)
    tree.free()
    with pytest.raises(eff.EffError):
        ctx.kv_attn(cache, batch, q, out, 4, 0.1, rules=rules)


def test_one_long_tile_among_many_empty_ones(ctx, eff):
    """The bound of the tiles far above those that there are: one sequence has new tokens and a long context."""
    n = 400
    new, lens = [0] * n, [1] * n
    new[77], lens[77] = 40, 70001
    run(eff, ctx, 5, F16, 1, 2, 64, 256, new, lens, masks=trees)
