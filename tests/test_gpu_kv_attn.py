"""Attention over the paged cache (eff_kv_attn) on the GPU against softmax in 64 bits.

Tolerance. q is kept to 22 bits and every product summed in f32, so a score of magnitude |s| (below 30 here) is off by
about |s| 2^-22 and a weight by the same relative amount, 7e-6 at most; the weighted mean of values then moves by less
than that times their size, and the errors of different tokens are independent. REL is 1e-5 of the row's norm, plus
1e-6 of the largest value for rows whose values cancel.
"""
import numpy as np
import pytest

from kv_reference import F16, I8, NO_PAGE, Batch, attend, encode, page_bytes

pytestmark = pytest.mark.gpu

REL, ABS = 1e-5, 1e-6


def make(rng, t, heads, dim, b, dirty=None):
    """A cache's bytes and values; the bytes that belong to no cached token are `dirty` where given."""
    rows = rng.standard_normal((b.pages, 2, heads, b.page, dim)).astype(np.float32)
    rows *= np.exp(0.4 * rng.standard_normal(dim)).astype(np.float32)
    data, values = encode(t, rows)
    if dirty is not None:
        used = np.zeros((b.pages, b.page), bool)
        for s, n in enumerate(b.lens):
            for a in range(0, n, b.page):
                used[b.table[s, a // b.page], :n - a] = True
        d = data.reshape(b.pages, 2, heads, -1).copy()
        for p in range(b.pages):
            for slot in np.flatnonzero(~used[p]):
                if t == F16:
                    d[p, :, :, slot * dim * 2:(slot + 1) * dim * 2] = np.frombuffer(np.float16(dirty).tobytes(), np.uint8)[None].repeat(dim, 0).ravel()
                else:
                    d[p, :, :, slot * dim:(slot + 1) * dim] = 0x7F
                    d[p, :, :, b.page * dim + 4 * slot:b.page * dim + 4 * slot + 4] = np.frombuffer(np.float32(dirty).tobytes(), np.uint8)
        data = d.reshape(b.pages, -1)
    return data, values


def launch(eff, ctx, t, heads, dim, b, data, q, q_heads, scale, window=0, **more):
    """One call; out as [tokens][q_heads][dim]."""
    cb, qb = ctx.upload(data), ctx.upload(q.astype(np.float32))
    out = ctx.upload(np.full(q.shape, 7, np.float32))
    cache = eff.KvCache(t, heads, dim, b.page, b.pages, cb)
    batch = b.upload(eff, ctx, **more)
    ctx.kv_attn(cache, batch, qb, out, q_heads, scale, window)
    got = out.read(np.float32).reshape(q.shape)
    for x in [cb, qb, out] + batch.buffers:
        x.free()
    return got


def check(got, want, values):
    got, want = got.astype(np.float64), want
    err = np.linalg.norm(got - want, axis=-1)
    limit = REL * np.linalg.norm(want, axis=-1) + ABS * np.abs(values).max()
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - limit), err.shape)
    assert (err <= limit).all(), f"row {worst}: off by {err[worst]:.3g}, {limit[worst]:.3g} allowed"


def run(eff, ctx, seed, t, heads, group, dim, page, new, lens, window=0, sharp=1.0, dirty=np.nan, **more):
    rng = np.random.default_rng(seed)
    b = Batch(rng, new, lens, page)
    data, values = make(rng, t, heads, dim, b, dirty)
    q = (sharp * rng.standard_normal((b.tokens, heads * group, dim))).astype(np.float32)
    scale = dim ** -0.5
    got = launch(eff, ctx, t, heads, dim, b, data, q, heads * group, scale, window, **more)
    check(got, attend(values, b.table, b.starts, b.lens, q, heads * group, scale, window, page), values)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,page", [(1, 1, 16), (2, 4, 32), (3, 5, 16), (2, 16, 64), (1, 23, 256)])
def test_one_token(ctx, eff, t, dim, heads, group, page):
    lens = [1, 15, 16, 17, 31, 32, 33, 65, 127, 128, 257, 700]
    run(eff, ctx, dim + group, t, heads, group, dim, page, [1] * len(lens), lens)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("lens", [[5000], [1], [40001], [1, 9000, 30, 1200], list(range(1, 90))])
def test_one_token_lengths(ctx, eff, t, lens):
    run(eff, ctx, len(lens), t, 2, 2, 64, 16, [1] * len(lens), lens)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("new,lens", [([5, 2, 3], [5, 700, 64]), ([40], [40]), ([1, 33, 1, 7], [300, 33, 17, 130]),
                                      ([65, 100], [65, 333])])
def test_new_tokens(ctx, eff, t, dim, new, lens):
    run(eff, ctx, sum(new), t, 2, 3, dim, 32, new, lens)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("heads,group,new", [(2, 1, 70), (1, 4, 130), (4, 7, 21)])
def test_prompt_heads(ctx, eff, t, heads, group, new):
    run(eff, ctx, new, t, heads, group, 128, 16, [new, new // 2], [new, 3 * new])


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens,window", [
    (4, 4, [700], [700], 0), (8, 3, [400, 129], [403, 1000], 0), (2, 8, [333, 1, 300], [2000, 50, 300], 0),
    (4, 5, [600], [900], 100), (16, 1, [2100, 2100], [2100, 2222], 0)])
def test_long_prompts(ctx, eff, t, dim, heads, group, new, lens, window):
    """Enough rows for the kernel of many rows, with one and two row tiles to a wave."""
    run(eff, ctx, dim, t, heads, group, dim, 32, new, lens, window)


@pytest.mark.parametrize("t", [F16, I8])
def test_long_prompt_in_a_batch(ctx, eff, t):
    """Prompts and decoding requests together: each goes to its kernel."""
    new, lens = [1, 900, 0, 5, 1, 16, 17, 300, 1], [3000, 900, 10, 77, 0, 16, 2000, 5000, 1]
    run(eff, ctx, 21, t, 4, 4, 64, 16, new, lens)
    run(eff, ctx, 22, t, 4, 4, 128, 64, new, lens, 500, max_new=4000, max_len=5001)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("window", [1, 7, 16, 33, 100, 5000])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 50, 900]), ([6, 40], [500, 40])])
def test_window(ctx, eff, t, window, new, lens):
    run(eff, ctx, window, t, 2, 4, 64, 16, new, lens, window)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim,group,new,window", [(64, 4, 1, 0), (96, 3, 6, 0), (128, 8, 5, 0), (64, 1, 3, 150), (256, 2, 1, 0)])
def test_uneven_lengths(ctx, eff, t, dim, group, new, window):
    """More sequences than a wave has lanes, nearly all short beside the longest: workgroups go on from tile to tile."""
    rng = np.random.default_rng(dim + new)
    lens = [2300] + [int(n) for n in rng.integers(0, 400, 75)]
    lens[40], lens[63], lens[64] = 1500, 128, 129
    run(eff, ctx, group, t, 8, group, dim, 16, [min(new, n) for n in lens], lens, window)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group,new,window", [(1, 1, 0), (4, 1, 200), (3, 6, 0)])
def test_whole_tiles(ctx, eff, t, dim, group, new, window):
    """Enough short tiles for a workgroup each: of eight waves where they are few."""
    rng = np.random.default_rng(dim + group)
    lens = [900, 0, 1, 511, 512, 513] + [int(n) for n in rng.integers(1, 900, 11)]
    for heads in (8, 12):
        run(eff, ctx, dim, t, heads, group, dim, 32, [min(new, n) for n in lens], lens, window)
    run(eff, ctx, dim, t, 3, group, dim, 16, [new], [599], window)


def test_long_shares(ctx, eff):
    """Sequences that take several workgroups each, which begin and end within tiles."""
    rng = np.random.default_rng(1)
    lens = [2300, 129] + [int(n) for n in rng.integers(300, 1300, 22)]
    run(eff, ctx, 1, F16, 32, 2, 64, 64, [1] * 24, lens)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim,heads,group,new,lens,window", [
    (256, 2, 8, [1], [20011], 0), (128, 1, 16, [1], [33000], 0), (64, 2, 16, [1, 2], [16000, 9000], 0),
    (128, 2, 8, [5, 1], [19000, 17000], 18001), (96, 1, 5, [1], [40001], 0)])
def test_many_workgroups_to_a_tile(ctx, eff, t, dim, heads, group, new, lens, window):
    """More of their sums than are joined at once."""
    run(eff, ctx, dim, t, heads, group, dim, 64, new, lens, window)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("where", [0, 1])
def test_not_finite_in_a_long_tile(ctx, eff, bad, where):
    """A key or value that is not finite, in one of many workgroups' tokens: the rows that see it are not finite."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [2], [20000], 64)
    rows = rng.standard_normal((b.pages, 2, 1, 64, 128)).astype(np.float32)
    rows[b.table[0, 7000 // 64], where, 0, 7000 % 64, 5] = bad
    q = np.abs(rng.standard_normal((2, 16, 128))).astype(np.float32)
    out = launch(eff, ctx, F16, 1, 128, b, encode(F16, rows)[0], q, 16, 0.1)
    assert not np.isfinite(out).all(-1).any()


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("lens", [[1], [700], [20, 5, 300]])
def test_length_bound(ctx, eff, t, lens):
    """The bound of the lengths far above them, as a recording has it."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [1] * len(lens), lens, 16, table_pages=4096)
    data, values = make(rng, t, 2, 128, b, np.nan)
    q = rng.standard_normal((b.tokens, 8, 128)).astype(np.float32)
    got = launch(eff, ctx, t, 2, 128, b, data, q, 8, 128 ** -0.5, max_len=65536)
    check(got, attend(values, b.table, b.starts, b.lens, q, 8, 128 ** -0.5, 0, 16), values)


def test_mixed_batch(ctx, eff):
    """A prompt among decoding requests, one with no new token, one without a token at all; bounds above the sizes."""
    new, lens = [1, 1, 90, 0, 1, 0, 1, 3], [40, 1, 200, 77, 513, 0, 16, 3]
    run(eff, ctx, 8, F16, 2, 4, 128, 16, new, lens, max_new=1000, max_len=513)
    run(eff, ctx, 9, I8, 1, 8, 64, 16, [1] * 70 + [120] + [1] * 70, [33] * 70 + [300] + list(range(1, 71)))


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("new", [1, 20, 600])
def test_what_is_not_seen(ctx, eff, t, new):
    """NaN, infinities or zeros at the places that no token sees: the same bits."""
    rng = np.random.default_rng(new)
    b = Batch(rng, [new, new], [new + 5, new + 333], 64, spare=3)
    q = rng.standard_normal((b.tokens, 8, 128)).astype(np.float32)
    got = []
    for dirty in (np.nan, np.inf, -np.inf, 0.0):
        data, values = make(np.random.default_rng(1), t, 2, 128, b, dirty)
        got.append(launch(eff, ctx, t, 2, 128, b, data, q, 8, 0.1, 100))
    check(got[0], attend(values, b.table, b.starts, b.lens, q, 8, 0.1, 100, 64), values)
    for g in got[1:]:
        assert np.array_equal(got[0].view(np.uint32), g.view(np.uint32))


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", [0, 1])
@pytest.mark.parametrize("new,group", [(40, 4), (700, 16)])
def test_later_tokens_do_not_reach_earlier_rows(ctx, eff, t, bad, where, new, group):
    """A key (where = 0) or value (1) that is not finite: rows before it are not changed, rows that see it are not finite."""
    rng = np.random.default_rng(3)
    length, at = new + 10, new - 9
    b = Batch(rng, [new], [length], 16)
    rows = rng.standard_normal((b.pages, 2, 1, 16, 64)).astype(np.float32)
    q = rng.standard_normal((new, group, 64)).astype(np.float32)
    clean, _ = encode(t, rows)
    data = clean.copy().reshape(b.pages, 2, -1)
    page, slot = b.table[0, at // 16], at % 16
    if t == F16:
        data[page, where, slot * 128 + 6:slot * 128 + 8] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    else:
        data[page, where, 16 * 64 + 4 * slot:16 * 64 + 4 * slot + 4] = np.frombuffer(np.float32(bad).tobytes(), np.uint8)
    a = launch(eff, ctx, t, 1, 64, b, clean, q, group, 0.1)
    g = launch(eff, ctx, t, 1, 64, b, data.reshape(b.pages, -1), q, group, 0.1)
    before = at - (length - new)          # new tokens before position `at`
    assert np.array_equal(a[:before].view(np.uint32), g[:before].view(np.uint32))
    if where == 1 or not np.isinf(bad):
        assert not np.isfinite(g[before:]).all(axis=-1).any()


def test_missing_pages(ctx, eff):
    """Tokens on pages that the table does not have are not seen; where none is left the row is zeros."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [1, 3, 1, 2], [100, 90, 64, 40], 16)
    b.table[0, 2] = NO_PAGE
    b.table[1, :4] = b.pages          # any number past the cache
    b.table[2, :] = NO_PAGE
    b.table[3, 2] = 0x80000000
    for t in (F16, I8):
        data, values = make(rng, t, 2, 64, b)
        q = rng.standard_normal((b.tokens, 6, 64)).astype(np.float32)
        got = launch(eff, ctx, t, 2, 64, b, data, q, 6, 0.2)
        check(got, attend(values, b.table, b.starts, b.lens, q, 6, 0.2, 0, 16), values)
        assert not got[4].any()


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,new,lens,window", [
    (8, 8, [500, 33], [1100, 200], 0), (4, 16, [450, 1, 300], [1500, 50, 300], 100), (16, 1, [1500, 700], [1500, 1222], 0),
    (7, 3, [1301], [1301], 0)])
def test_many_rows(ctx, eff, t, dim, heads, group, new, lens, window):
    """Enough rows for the kernel of many rows, of int8 too; all sequences in one launch."""
    run(eff, ctx, dim, t, heads, group, dim, 32, new, lens, window)


@pytest.mark.parametrize("t", [F16, I8])
def test_many_rows_in_a_batch(ctx, eff, t):
    """Prompts and decoding requests together, in two launches."""
    new, lens = [1, 900, 0, 5, 1, 16, 17, 300, 1], [3000, 900, 10, 77, 0, 16, 2000, 5000, 1]
    run(eff, ctx, 31, t, 8, 4, 64, 16, new, lens)
    run(eff, ctx, 32, t, 8, 4, 128, 64, new, lens, 500, max_new=4000, max_len=5001)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("bad", [np.nan, -np.inf])
@pytest.mark.parametrize("where", [0, 1])
def test_later_tokens_of_many_rows(ctx, eff, t, bad, where):
    test_later_tokens_do_not_reach_earlier_rows(ctx, eff, t, bad, where, 1650, 16)


@pytest.mark.parametrize("t", [F16, I8])
def test_what_many_rows_do_not_see(ctx, eff, t):
    test_what_is_not_seen(ctx, eff, t, 1800)


def test_more_new_tokens_than_length(ctx, eff):
    """New tokens without a position, and sequences of length 0: zeros."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [4, 1, 30], [2, 0, 11], 16)
    data, values = make(rng, F16, 1, 64, b)
    q = rng.standard_normal((b.tokens, 2, 64)).astype(np.float32)
    got = launch(eff, ctx, F16, 1, 64, b, data, q, 2, 0.2)
    check(got, attend(values, b.table, b.starts, b.lens, q, 2, 0.2, 0, 16), values)
    assert not got[:2].any() and not got[4:5].any() and not got[5:24].any()


@pytest.mark.parametrize("sharp", [1e-30, 1e-3, 30.0, 1e4])
@pytest.mark.parametrize("t", [F16, I8])
def test_query_sizes(ctx, eff, t, sharp):
    """From scores that are all alike to one token that takes everything."""
    rng = np.random.default_rng(7)
    b = Batch(rng, [1, 5], [300, 90], 16)
    data, values = make(rng, t, 1, 128, b)
    q = (sharp * rng.standard_normal((b.tokens, 4, 128))).astype(np.float32)
    q[0, 0] = 0
    q[1, 1, :5] = 0
    got = launch(eff, ctx, t, 1, 128, b, data, q, 4, 0.09)
    x = np.abs(np.einsum("thd,psd->th", np.abs(q).astype(np.float64), np.abs(values[:, 0, 0]))).max() / values[:, 0, 0, :, 0].size
    want = attend(values, b.table, b.starts, b.lens, q, 4, 0.09, 0, 16)
    # a score's error grows with it: 2^-22 of sum |q k| scale, twice (its own, and the largest score's)
    tol = max(REL, 2 * 0.09 * x * 128 ** 0.5 * 2.0 ** -22)
    err = np.linalg.norm(got - want, axis=-1)
    assert np.isfinite(got).all() and (err <= tol * np.linalg.norm(want, axis=-1) + ABS * np.abs(values).max()).all()


def test_small_weights_of_a_long_context(ctx, eff):
    """One token that outweighs each of 30000 others by e^9 and all of them together by little."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [1], [30001], 64)
    for t in (F16, I8):
        rows = rng.standard_normal((b.pages, 2, 1, 64, 64)).astype(np.float32)
        rows[:, 0] *= 0.01
        rows[b.table[0, 100], 0, 0, 9] = 1
        data, values = encode(t, rows)
        q = np.full((1, 1, 64), 9 / 64, np.float32)
        got = launch(eff, ctx, t, 1, 64, b, data, q, 1, 1.0)
        check(got, attend(values, b.table, b.starts, b.lens, q, 1, 1.0, 0, 64), values)


def test_value_scales(ctx, eff):
    """int8 rows whose scales span 10^16: large values beside small ones, in either order."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [1, 1], [200, 200], 16)
    rows = rng.standard_normal((b.pages, 2, 1, 16, 64)).astype(np.float32)
    for s in range(2):
        size = 10.0 ** np.linspace(-8, 8, 200)[::1 - 2 * s]
        for p in range(200):
            rows[b.table[s, p // 16], 1, 0, p % 16] *= size[p]
    data, values = encode(I8, rows)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    got = launch(eff, ctx, I8, 1, 64, b, data, q, 2, 0.1)
    want = attend(values, b.table, b.starts, b.lens, q, 2, 0.1, 0, 16)
    assert (np.linalg.norm(got - want, axis=-1) <= REL * np.linalg.norm(want, axis=-1)).all()


def test_strides(ctx, eff):
    """q inside rows of a fused projection, at an offset."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [3, 1], [60, 9], 16)
    data, values = make(rng, F16, 2, 64, b)
    rows = rng.standard_normal((b.tokens, 4 + 8 * 64 + 12)).astype(np.float32)
    q = rows[:, 4:4 + 512].reshape(-1, 8, 64)
    cb, qb, out = ctx.upload(data), ctx.upload(rows), ctx.alloc(b.tokens * 512 * 4)
    batch = b.upload(eff, ctx)
    ctx.kv_attn(eff.KvCache(F16, 2, 64, 16, b.pages, cb), batch, qb, out, 8, 0.125, 0, 4, 528)
    check(out.read(np.float32).reshape(-1, 8, 64), attend(values, b.table, b.starts, b.lens, q, 8, 0.125, 0, 16), values)


def test_far_pages(ctx, eff):
    """A cache past 2^32 bytes: pages at both ends and in the middle."""
    rng = np.random.default_rng(11)
    page, heads, dim = 1024, 8, 128
    size = page_bytes(F16, heads, dim, page)
    pages = 5 * 2 ** 30 // size
    cb = ctx.alloc(pages * size)
    ids = [pages - 1, 0, pages // 2, pages - 2]
    rows = rng.standard_normal((4, 2, heads, page, dim)).astype(np.float32)
    data, values = encode(F16, rows)
    for i, p in enumerate(ids):
        cb.write(data[i], p * size)
    lens = [4000, 1500]
    table = np.array([ids, [ids[3], ids[0], 7, 7]], np.uint32)
    starts = np.array([0, 1, 2])
    q = rng.standard_normal((2, 16, dim)).astype(np.float32)
    bufs = [ctx.upload(x.astype(np.uint32)) for x in (table, starts, np.array(lens))]
    batch = eff.KvBatch(*bufs, seqs=2, tokens=2, table_pages=4, max_new=1, max_len=4000)
    qb, out = ctx.upload(q), ctx.alloc(q.nbytes)
    ctx.kv_attn(eff.KvCache(F16, heads, dim, page, pages, cb), batch, qb, out, 16, 0.09)
    got = out.read(np.float32).reshape(q.shape)
    near = np.array([[0, 1, 2, 3], [3, 0, 0, 0]], np.uint32)
    check(got, attend(values, near, starts, lens, q, 16, 0.09, 0, page), values)
    cb.free()


def test_same_bits(ctx, eff):
    """The same call twice, split and not: the same bits; other calls in between do not matter."""
    rng = np.random.default_rng(12)
    b = Batch(rng, [1, 1, 1], [20000, 9000, 400], 64)
    data, _ = make(rng, F16, 2, 128, b)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    first = launch(eff, ctx, F16, 2, 128, b, data, q, 8, 0.09)
    run(eff, ctx, 13, I8, 4, 4, 64, 16, [1] * 9, [3000] * 9)
    for _ in range(4):
        assert np.array_equal(first.view(np.uint32), launch(eff, ctx, F16, 2, 128, b, data, q, 8, 0.09).view(np.uint32))


@pytest.mark.parametrize("t,heads,group,dim,lens", [
    (F16, 8, 2, 64, [2300] + list(range(1, 380, 5))), (I8, 2, 8, 256, [20000]), (I8, 8, 4, 128, [2300] + [700] * 70)])
def test_same_bits_shared(ctx, eff, t, heads, group, dim, lens):
    """Tiles that workgroups share, in one order of joining: the same bits again and again."""
    rng = np.random.default_rng(13)
    b = Batch(rng, [1] * len(lens), lens, 64)
    data, _ = make(rng, t, heads, dim, b)
    q = rng.standard_normal((len(lens), heads * group, dim)).astype(np.float32)
    cb, qb, out = ctx.upload(data), ctx.upload(q), ctx.alloc(q.nbytes)
    cache, batch = eff.KvCache(t, heads, dim, 64, b.pages, cb), b.upload(eff, ctx)
    got = []
    for _ in range(6):
        out.write(np.full(q.shape, 9, np.float32))
        ctx.kv_attn(cache, batch, qb, out, heads * group, 0.1)
        got.append(out.read(np.uint32).copy())
    assert all(np.array_equal(got[0], g) for g in got[1:])
    for x in [cb, qb, out] + batch.buffers:
        x.free()


def test_recorded(ctx, eff):
    """A recorded call takes the next steps' lengths and pages; each replay gives the eager call's bits."""
    rng = np.random.default_rng(14)
    t, heads, dim, page, q_heads = F16, 2, 64, 16, 8
    b = Batch(rng, [1, 1], [2000, 60], page, table_pages=200)
    data, values = make(rng, t, heads, dim, b)
    q = rng.standard_normal((2, q_heads, dim)).astype(np.float32)
    cb, qb, out = ctx.upload(data), ctx.upload(q), ctx.alloc(q.nbytes)
    cache, batch = eff.KvCache(t, heads, dim, page, b.pages, cb), b.upload(eff, ctx, max_len=3200)
    def call():
        ctx.kv_attn(cache, batch, qb, out, q_heads, 0.125)
    call()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()
    assert g.nodes >= 1
    for step, lens in enumerate([[2000, 60], [1, 64], [1333, 7], [2000, 0]]):
        x = rng.standard_normal(q.shape).astype(np.float32)
        qb.write(x)
        batch.buffers[2].write(np.array(lens, np.uint32))
        out.write(np.full(q.shape, 9, np.float32))
        g.launch()
        got = out.read(np.float32).reshape(q.shape)
        check(got, attend(values, b.table, b.starts, lens, x, q_heads, 0.125, 0, page), values)
        out.write(np.full(q.shape, 9, np.float32))
        call()
        assert np.array_equal(got.view(np.uint32), out.read(np.uint32).reshape(q.shape)), step
        ctx.sync()
    g.destroy()


def test_streams(ctx, eff):
    """Two contexts on streams of their own, calls in turn: neither disturbs the other."""
    rng = np.random.default_rng(15)
    b = Batch(rng, [1] * 4, [9000, 5000, 100, 7000], 32)
    data, values = make(rng, F16, 2, 128, b)
    q = rng.standard_normal((4, 8, 128)).astype(np.float32)
    want = attend(values, b.table, b.starts, b.lens, q, 8, 0.09, 0, 32)
    with eff.Context(0) as other:
        made = []
        for c in (ctx, other):
            bufs = [c.upload(data), c.upload(q), c.alloc(q.nbytes)]
            made.append((c, bufs, eff.KvCache(F16, 2, 128, 32, b.pages, bufs[0]), b.upload(eff, c)))
        for _ in range(8):
            for c, bufs, cache, batch in made:
                c.kv_attn(cache, batch, bufs[1], bufs[2], 8, 0.09)
        for c, bufs, _, _ in made:
            check(bufs[2].read(np.float32).reshape(q.shape), want, values)
        for c, bufs, _, batch in made:
            for x in bufs + batch.buffers:
                x.free()


def test_refusals(ctx, eff):
    rng = np.random.default_rng(16)
    b = Batch(rng, [1, 1], [40, 30], 16)
    data, _ = make(rng, F16, 2, 64, b)
    cb, qb, out = ctx.upload(data), ctx.alloc(2 * 8 * 64 * 4), ctx.alloc(2 * 8 * 64 * 4)
    bufs = b.upload(eff, ctx).buffers
    good = dict(seqs=2, tokens=2, table_pages=b.table_pages, max_new=1, max_len=40)

    def call(code, t=F16, heads=2, dim=64, page=16, pages=b.pages, buf=cb, arrays=bufs, q=qb, o=out, q_heads=8, scale=0.1, window=0,
             off=0, stride=0, **change):
        with pytest.raises(eff.EffError) as e:
            ctx.kv_attn(eff.KvCache(t, heads, dim, page, pages, buf), eff.KvBatch(*arrays, **{**good, **change}), q, o, q_heads,
                        scale, window, off, stride)
        assert e.value.code == code and "kv attn" in str(e.value)

    before = ctx.stats()["kv_attn"]
    call(eff.E_TYPE, t=8)
    for change in (dict(dim=80), dict(page=24), dict(page=8), dict(page=2048), dict(heads=0), dict(q_heads=7), dict(q_heads=0)):
        call(eff.E_SHAPE, **change)
    for change in (dict(seqs=0), dict(max_new=0), dict(max_len=0), dict(table_pages=0), dict(pages=0), dict(scale=float("nan")),
                   dict(scale=float("inf")), dict(off=1), dict(stride=514), dict(stride=256), dict(o=qb)):
        call(eff.E_INVALID, **change)
    for change in (dict(pages=b.pages + 1), dict(tokens=3), dict(seqs=3), dict(max_len=16 * b.table_pages + 1), dict(off=4),
                   dict(stride=516), dict(table_pages=b.table_pages + 1)):
        call(eff.E_BOUNDS, **change)
    with pytest.raises(eff.EffError) as e:
        ctx._check(eff.lib().eff_kv_attn(ctx.h, None, None, qb.handle, 0, 0, out.handle, 8, 0.1, 0))
    assert e.value.code == eff.E_INVALID
    assert eff.lib().eff_kv_attn(None, None, None, None, 0, 0, None, 8, 0.1, 0) == eff.E_INVALID
    # no new token: nothing runs
    ctx.kv_attn(eff.KvCache(F16, 2, 64, 16, b.pages, cb), eff.KvBatch(*bufs, **{**good, "tokens": 0}), qb, out, 8, 0.1)
    assert ctx.stats()["kv_attn"] == before
