"""Appending with positions of their own (eff_kv_append_at) on the GPU, against 64 bits. The tolerances are those of
test_gpu_kv_append: TURN of a row's largest value for what is turned, and the rounding of the stored type."""
import ctypes

import numpy as np
import pytest

from kv_reference import F16, I8, Batch, decode, page_bytes
from kv_rules_reference import random_tree, tree_mask, turn_at
from test_gpu_kv_append import EPS, TURN, rope_of

pytestmark = pytest.mark.gpu


def sections(pairs, axes):
    return [min(axes - 1, i * axes // pairs) for i in range(pairs)]


def dealt(pairs, axes):
    return [i % axes for i in range(pairs)]


def run(eff, ctx, seed, t, q_heads, heads, dim, page, new, lens, rope_dim, halves, axis, at=None, norm=False, positions=None, in_place=False):
    """One call, every row checked; `at` [axes][tokens], positions of the rope table."""
    rng = np.random.default_rng(seed)
    b = Batch(rng, new, lens, page)
    axes, positions = max(axis) + 1, positions or 700
    if at is None:
        at = rng.integers(0, positions, (axes, b.tokens))
    at = np.asarray(at, np.uint32)
    x = [(3 * rng.standard_normal((b.tokens, n, dim))).astype(np.float32) for n in (q_heads, heads, heads)]
    old = rng.integers(0, 256, (b.pages, page_bytes(t, heads, dim, page)), dtype=np.uint8)
    cb, bufs = ctx.upload(old), [ctx.upload(r) for r in x]
    q_out = bufs[0] if in_place else ctx.upload(np.full(x[0].shape, 5, np.float32))
    rb, rope = rope_of(ctx, eff, positions, rope_dim)
    w = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None for _ in range(2)]
    rows = eff.KvRows(q=bufs[0], k=bufs[1], v=bufs[2], q_heads=q_heads, q_out=q_out, rope=rb, rope_positions=positions, rope_dim=rope_dim,
                      rope_mode=eff.ROPE_HALVES if halves else eff.ROPE_PAIRS, q_norm=None if w[0] is None else ctx.upload(w[0]),
                      k_norm=None if w[1] is None else ctx.upload(w[1]), eps=EPS)
    ctx.kv_append(eff.KvCache(t, heads, dim, page, b.pages, cb), b.upload(eff, ctx), rows, turns=eff.KvTurns(ctx.upload(at), axis, axes=axes))
    q, got = q_out.read(np.float32).reshape(x[0].shape), cb.read(np.uint8)
    values, pos, seq = decode(t, got, b.pages, heads, dim, page), b.positions(), b.seq()
    want_q, want_k = (turn_at(r, at, axis, rope, rope_dim, halves, n, EPS) for r, n in zip(x, w))
    there = pos >= 0
    for g, want in ((q, want_q),):
        good = np.isfinite(want).all((1, 2)) & there
        assert (np.abs(g - want)[good] <= TURN * np.abs(want[good]).max(-1, keepdims=True)).all()
        assert np.array_equal(np.isnan(g[there]), np.isnan(want[there])) and not g[~there].any()
    for i in np.flatnonzero(there):
        for j, want in enumerate((want_k[i], x[2][i].astype(np.float64))):
            v = values[b.table[seq[i], pos[i] // page], j, :, pos[i] % page]
            if not np.isfinite(want).all():
                bad = np.isnan(want) if t == F16 else np.isnan(want).any(-1, keepdims=True) & np.ones(want.shape, bool)
                assert np.array_equal(np.isnan(v), bad)
                continue
            top = np.abs(want).max(-1, keepdims=True)
            limit = TURN * top + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if t == F16 else top / 254 + 2.0 ** -22 * top)
            assert (np.abs(v - want) <= limit).all(), (i, j)
    return q, got


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("axes,deal", [(1, sections), (3, sections), (3, dealt), (4, dealt)])
def test_axes(ctx, eff, t, dim, halves, axes, deal):
    run(eff, ctx, dim + axes, t, 5, 2, dim, 16, [1, 7, 0, 20], [30, 7, 9, 33], dim, halves, deal(dim // 2, axes), norm=t == F16)


@pytest.mark.parametrize("rope_dim", [4, 20, 64, 100])
@pytest.mark.parametrize("halves", [False, True])
def test_part_of_the_channels(ctx, eff, rope_dim, halves):
    run(eff, ctx, rope_dim, F16, 3, 1, 128, 32, [40, 1], [50, 2000], rope_dim, halves, dealt(rope_dim // 2, 2), in_place=True)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim,heads", [(64, 16), (96, 11), (128, 8), (256, 4)])
def test_many_tokens(ctx, eff, t, dim, heads):
    """Enough values for four rows a thread."""
    tokens = 2048 * 4096 // (dim * heads * 6) + 1
    run(eff, ctx, dim, t, 4 * heads, heads, dim, 64, [tokens], [tokens + 5], dim, True, dealt(dim // 2, 3))


def test_depths_of_a_tree(ctx, eff):
    """Drafts turned by the position of their depth, into places of their own."""
    rng = np.random.default_rng(1)
    new, lens = [25, 1, 9], [325, 1, 9]
    depths = [tree_mask(random_tree(rng, n)).sum(1) - 1 for n in new]
    at = np.concatenate([length - n + d for n, length, d in zip(new, lens, depths)])[None]
    run(eff, ctx, 1, F16, 4, 2, 64, 16, new, lens, 64, True, [0] * 32, at)


@pytest.mark.parametrize("t", [F16, I8])
def test_positions_of_the_cache(ctx, eff, t):
    """One axis with the cached positions: the bits of the call without positions."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [3, 40], [10, 300], 16)
    x = [rng.standard_normal((b.tokens, n * 128)).astype(np.float32) for n in (4, 2, 2)]
    rope, _ = rope_of(ctx, eff, 300, 128)
    got = []
    for turns in (None, eff.KvTurns(ctx.upload(b.positions().astype(np.uint32)))):
        cb, q_out = ctx.alloc(b.pages * page_bytes(t, 2, 128, 16)), ctx.alloc(x[0].nbytes)
        rows = eff.KvRows(q=ctx.upload(x[0]), k=ctx.upload(x[1]), v=ctx.upload(x[2]), q_heads=4, q_out=q_out, rope=rope, rope_positions=300,
                          rope_dim=128)
        ctx.kv_append(eff.KvCache(t, 2, 128, 16, b.pages, cb), b.upload(eff, ctx), rows, turns=turns)
        got.append((q_out.read(np.uint8), cb.read(np.uint8)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


@pytest.mark.parametrize("t", [F16, I8])
def test_positions_past_the_table(ctx, eff, t):
    """Such a pair is NaN, and no other value of an fp16 row; a table of one position, shorter than the cache."""
    at = np.array([[0, 6, 7, 0xFFFFFFFF, 3, 0x80000000], [0, 0, 6, 1, 2, 9]])
    run(eff, ctx, 5, t, 2, 2, 64, 16, [6], [400], 64, False, dealt(32, 2), at, positions=7)
    run(eff, ctx, 6, t, 2, 2, 64, 16, [3], [90], 32, True, [0] * 16, [[0, 1, 0]], positions=1)


def test_more_new_tokens_than_length(ctx, eff):
    run(eff, ctx, 7, F16, 2, 1, 64, 16, [5, 2], [3, 9], 64, True, dealt(32, 3))


@pytest.mark.parametrize("tokens", [3, 900])
def test_rows_behind_the_last_sequence(ctx, eff, tokens):
    """Tokens of a padded batch that belong to no sequence: their rows stay as they were, and the cache."""
    rng = np.random.default_rng(tokens)
    b = Batch(rng, [tokens], [tokens + 40], 64)
    x = [rng.standard_normal((tokens + 4, n, 128)).astype(np.float32) for n in (16, 2, 2)]
    at = rng.integers(0, 50, (1, tokens + 4)).astype(np.uint32)
    rb, rope = rope_of(ctx, eff, 50, 128)
    old = rng.integers(0, 256, b.pages * page_bytes(F16, 2, 128, 64), dtype=np.uint8)
    cb, q_out = ctx.upload(old), ctx.upload(np.full(x[0].shape, 5, np.float32))
    mine = b.upload(eff, ctx)
    batch = eff.KvBatch(*mine.buffers, seqs=1, tokens=tokens + 4, table_pages=b.table_pages, max_new=tokens, max_len=tokens + 40)
    ctx.kv_append(eff.KvCache(F16, 2, 128, 64, b.pages, cb), batch,
                  eff.KvRows(q=ctx.upload(x[0]), k=ctx.upload(x[1]), v=ctx.upload(x[2]), q_heads=16, q_out=q_out, rope=rb, rope_positions=50,
                             rope_dim=128), turns=eff.KvTurns(ctx.upload(at)))
    got, want = q_out.read(np.float32).reshape(x[0].shape), turn_at(x[0], at, [0] * 64, rope, 128, False)
    assert (got[tokens:] == 5).all() and (np.abs(got - want)[:tokens] <= TURN * np.abs(want[:tokens]).max(-1, keepdims=True)).all()
    values, before = (decode(F16, d, b.pages, 2, 128, 64).view(np.uint64) for d in (cb.read(np.uint8), old))
    written = np.zeros((b.pages, 64), bool)
    for pos in b.positions():
        written[b.table[0, pos // 64], pos % 64] = True
    assert np.array_equal(values.transpose(0, 3, 1, 2, 4)[~written], before.transpose(0, 3, 1, 2, 4)[~written])


def test_recorded(ctx, eff):
    """A recorded append takes the next step's positions."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [2], [40], 16)
    x = rng.standard_normal((2, 1, 64)).astype(np.float32)
    rb, rope = rope_of(ctx, eff, 50, 64)
    cb, q_out, k, pos = ctx.alloc(b.pages * page_bytes(F16, 1, 64, 16)), ctx.alloc(x.nbytes), ctx.upload(x), ctx.alloc(2 * 2 * 4)
    args = (eff.KvCache(F16, 1, 64, 16, b.pages, cb), b.upload(eff, ctx),
            eff.KvRows(q=k, k=k, v=k, q_heads=1, q_out=q_out, rope=rb, rope_positions=50, rope_dim=64), eff.KvTurns(pos, dealt(32, 2), axes=2))
    ctx.kv_append(*args)
    ctx.graph_begin()
    ctx.kv_append(*args)
    g = ctx.graph_end()
    for _ in range(4):
        at = rng.integers(0, 50, (2, 2)).astype(np.uint32)
        pos.write(at)
        g.launch()
        want = turn_at(x, at, dealt(32, 2), rope, 64, False)
        assert np.abs(q_out.read(np.float32).reshape(x.shape) - want).max() <= TURN * np.abs(want).max()
        ctx.sync()
    g.destroy()


def test_refusals(ctx, eff):
    b = Batch(np.random.default_rng(9), [1, 1], [40, 30], 16)
    cb = ctx.alloc(b.pages * page_bytes(F16, 2, 64, 16))
    x, qo, rope, pos = ctx.alloc(2 * 256 * 4), ctx.alloc(2 * 256 * 4), ctx.alloc(40 * 64 * 4), ctx.alloc(2 * 3 * 4)
    k, v = ctx.alloc(2 * 128 * 4), ctx.alloc(2 * 128 * 4)
    batch, cache = b.upload(eff, ctx), eff.KvCache(F16, 2, 64, 16, b.pages, cb)
    before = ctx.stats()["kv_append"]

    def call(code, turns, **change):
        rows = {**dict(q=x, k=k, v=v, q_heads=4, q_out=qo, rope=rope, rope_positions=40, rope_dim=64), **change}
        with pytest.raises(eff.EffError) as e:
            ctx.kv_append(cache, batch, eff.KvRows(**rows), turns=turns)
        assert e.value.code == code and "kv append" in str(e.value)

    good = eff.KvTurns(pos, dealt(32, 3), axes=3)
    call(eff.E_INVALID, good, rope=None, rope_dim=0)
    call(eff.E_BOUNDS, good, rope_positions=0)
    call(eff.E_BOUNDS, good, rope_positions=41)
    for axes in (0, 5):
        call(eff.E_SHAPE, eff.KvTurns(pos, [0] * 32, axes=axes))
    with pytest.raises(eff.EffError):
        eff.KvTurns(pos, axes=2)
    call(eff.E_INVALID, eff.KvTurns(pos, dealt(32, 3), axes=2))
    call(eff.E_INVALID, eff.KvTurns(pos, [0] * 31 + [1], axes=1))
    call(eff.E_INVALID, eff.KvTurns(None, axes=1))
    call(eff.E_BOUNDS, eff.KvTurns(pos, dealt(32, 4), axes=4))
    call(eff.E_INVALID, eff.KvTurns(qo, dealt(32, 3), axes=3))                       # written and read
    call(eff.E_INVALID, eff.KvTurns(cb, dealt(32, 3), axes=3))
    for axis in ([0] * 129, [-1], [256]):
        with pytest.raises(eff.EffError):
            eff.KvTurns(pos, axis)
    # an axis past the turned pairs is not looked at
    assert ctx.stats()["kv_append"] == before
    ctx.kv_append(cache, batch, eff.KvRows(k=k, v=v, rope=rope, rope_positions=3, rope_dim=32), turns=eff.KvTurns(pos, [0] * 16 + [9] * 16, axes=1))
    assert ctx.stats()["kv_append"] == before + 1
    assert eff.lib().eff_kv_append_at(None, None, None, None, ctypes.addressof(good.c)) == eff.E_INVALID
    pos.free()
    with pytest.raises(eff.EffError):
        ctx.kv_append(cache, batch, eff.KvRows(k=k, v=v, rope=rope, rope_positions=40, rope_dim=64), turns=good)
