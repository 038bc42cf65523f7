"""Appending to the paged cache (eff_kv_append) and the rotation's table (eff_rope_table) on the GPU, against 64 bits.

Tolerances. A rotated value is two f32 products and their difference: 2^-23 of the pair's size; the norm adds its sum,
square root and two products, 2^-21 of the value: TURN = 2^-20 of the largest value of the row. An fp16 row then has
half a unit in the last place (2^-11 of the value, 2^-25 below the normal range), an int8 row half a step and the
scale's two roundings (2^-22).
"""
import numpy as np
import pytest

from kv_reference import F16, I8, NO_PAGE, Batch, decode, page_bytes, turn

pytestmark = pytest.mark.gpu

TURN = 2.0 ** -20
EPS = 1e-5


def rope_of(ctx, eff, positions, rope_dim, base=10000.0, scale=1.0):
    f = base ** (-np.arange(0, rope_dim, 2) / rope_dim)
    buf = ctx.rope_table(f, positions, scale)
    return buf, buf.read(np.float32).reshape(positions, 2, rope_dim // 2)


@pytest.mark.parametrize("n,positions,scale", [(32, 300, 1.0), (1, 7, 0.5), (128, 1000, 1.1), (256, 3, 1.0)])
def test_rope_table(ctx, eff, n, positions, scale):
    f = 10000.0 ** (-np.arange(n) / n)
    got = ctx.rope_table(f, positions, scale).read(np.float32).reshape(positions, 2, n)
    a = np.arange(positions)[:, None] * f
    want = np.stack([np.cos(a), np.sin(a)], 1) * np.float64(np.float32(scale))
    assert np.abs(got - want).max() <= 2.0 ** -24 * max(1, scale) * 1.01


def test_rope_table_far(ctx, eff):
    """Position 10^6: the angle is reduced in 64 bits."""
    f = np.array([1.0, 0.37, 1e-4])
    got = ctx.rope_table(f, 1000001).read(np.float32).reshape(-1, 2, 3)[-1]
    assert np.abs(got - np.stack([np.cos(1e6 * f), np.sin(1e6 * f)])).max() < 2.0 ** -23


def run(eff, ctx, seed, t, q_heads, heads, dim, page, new, lens, rope_dim=0, halves=False, norm=False, layout="apart", table=None,
        edit=None, place=True):
    rng = np.random.default_rng(seed)
    b = Batch(rng, new, lens, page)
    if table is not None:
        table(b)
    size = [q_heads * dim, heads * dim, heads * dim]
    rows = [(3 * rng.standard_normal((b.tokens, n))).astype(np.float32) for n in size]
    if edit:
        edit(rows)
    old = rng.integers(0, 256, (b.pages, page_bytes(t, heads, dim, page)), dtype=np.uint8)
    cb, qo = ctx.upload(old), ctx.upload(np.full((b.tokens, max(1, size[0])), 5, np.float32))
    names = "qkv" if q_heads else "kv"
    if layout == "fused":                 # one buffer, with a gap before and after
        pad = [rng.standard_normal((b.tokens, n)).astype(np.float32) for n in (8, 4)]
        buf = ctx.upload(np.concatenate([pad[0]] + rows + [pad[1]], 1))
        at, off = {}, 8
        for name, n in zip("qkv", size):
            at[name], at[name + "_stride"] = (buf, off), sum(size) + 12
            off += n
        at = {k: v for k, v in at.items() if k[0] in names}
    else:
        at = {name: ctx.upload(r) for name, r in zip("qkv", rows) if name in names}
        if layout == "in place":
            qo = at["q"]
    if q_heads:
        at.update(q_heads=q_heads, q_out=qo)
    rope = None
    if rope_dim:
        rb, rope = rope_of(ctx, eff, max(lens) + 3, rope_dim)
        at.update(rope=rb, rope_positions=max(lens) + 3, rope_dim=rope_dim, rope_mode=eff.ROPE_HALVES if halves else eff.ROPE_PAIRS)
    w = [None, None]
    if norm:
        w = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
        at.update(q_norm=ctx.upload(w[0]), k_norm=ctx.upload(w[1]), eps=EPS)
    ctx.kv_append(eff.KvCache(t, heads, dim, page, b.pages, cb), b.upload(eff, ctx), eff.KvRows(**at))
    got = cb.read(np.uint8).reshape(old.shape)
    q = qo.read(np.float32)[:b.tokens * size[0]].reshape(b.tokens, q_heads, dim)
    if not place:
        return b, rows, old, got, q
    pos, seq = b.positions(), b.seq()
    x = [r.reshape(b.tokens, -1, dim) for r in rows]
    k = turn(x[1], pos, rope, rope_dim, halves, w[1], EPS)
    if q_heads:
        want = turn(x[0], pos, rope, rope_dim, halves, w[0], EPS)
        assert (np.abs(q - want) <= TURN * np.abs(want).max(-1, keepdims=True)).all()
    values, before = decode(t, got, b.pages, heads, dim, page), decode(t, old, b.pages, heads, dim, page)
    written = np.zeros((b.pages, page), bool)
    for i in range(b.tokens):
        p, slot = b.table[seq[i], pos[i] // page], pos[i] % page
        if p >= b.pages:
            continue
        written[p, slot] = True
        for j, want in enumerate((k[i], x[2][i].astype(np.float64))):
            v, top = values[p, j, :, slot], np.abs(want).max(-1, keepdims=True)
            limit = TURN * top + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if t == F16 else top / 254 + 2.0 ** -22 * top)
            assert (np.abs(v - want) <= limit).all(), (i, j)
    # the other tokens of the cache keep their bytes
    a, c = (d.reshape(b.pages, 2, heads, -1) for d in (old, got))
    for s in range(page):
        n = 2 * dim if t == F16 else dim
        keep = ~written[:, s]
        assert np.array_equal(a[keep, :, :, s * n:(s + 1) * n], c[keep, :, :, s * n:(s + 1) * n])
        if t == I8:
            at = page * dim + 4 * s
            assert np.array_equal(a[keep, :, :, at:at + 4], c[keep, :, :, at:at + 4])
    assert before.shape == values.shape
    return b, rows, old, got, q


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_decode(ctx, eff, t, dim, halves, norm):
    run(eff, ctx, dim, t, 12, 3, dim, 16, [1] * 5, [1, 16, 17, 300, 4001], dim, halves, norm)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("rope_dim,halves", [(0, False), (4, True), (20, False), (32, True), (96, True)])
@pytest.mark.parametrize("layout", ["apart", "fused", "in place"])
def test_prompts(ctx, eff, t, rope_dim, halves, layout):
    run(eff, ctx, rope_dim, t, 5, 2, 96, 32, [33, 1, 0, 70], [33, 64, 10, 200], rope_dim, halves, rope_dim == 32, layout)


def test_keys_alone(ctx, eff):
    run(eff, ctx, 1, F16, 0, 4, 64, 16, [3, 9], [3, 40], 64, True)


def test_many_sequences(ctx, eff):
    """More sequences than a wave has lanes, some without a new token, at both ends."""
    rng = np.random.default_rng(2)
    new = [0, 0] + list(rng.integers(0, 4, 200)) + [0]
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 60, len(new)))]
    run(eff, ctx, 2, I8, 2, 1, 64, 16, new, lens, 32, True)


def test_missing_pages(ctx, eff):
    """Tokens whose page the table does not have are dropped; their q rows are made all the same."""
    def table(b):
        b.table[0, 1] = NO_PAGE
        b.table[1, :] = b.pages
    for t in (F16, I8):
        run(eff, ctx, 3, t, 4, 2, 64, 16, [20, 5], [40, 9], 64, True, table=table)


def test_more_new_tokens_than_length(ctx, eff):
    """The first new tokens have no position: not cached, their q rows zeros."""
    b, rows, old, got, q = run(eff, ctx, 4, F16, 2, 1, 64, 16, [5, 1], [2, 0], place=False)
    assert not q[:3].any() and q[3:5].any() and not q[5].any()
    page = got[b.table[0, 0]].view(np.float16).reshape(2, 16, 64)
    assert np.array_equal(page[1, :2], rows[2][3:5].astype(np.float16))
    other = [p for p in range(b.pages) if p != b.table[0, 0]]
    assert np.array_equal(got[other], old[other])


def test_rows_of_zeros(ctx, eff):
    def edit(rows):
        for r in rows:
            r[:2] = 0
    run(eff, ctx, 5, I8, 2, 2, 128, 16, [4], [9], 128, edit=edit)
    run(eff, ctx, 5, I8, 2, 2, 128, 16, [4], [9], 128, norm=True, edit=edit)


@pytest.mark.parametrize("size", [1e-30, 1e-35, 3e-36, 1e-36, 1e-38, 1e-42])
def test_smallest_int8_rows(ctx, eff, size):
    """Rows whose largest value is next to the smallest numbers: rounded, or zeros below 2^-119; zeros stay zeros."""
    def edit(rows):
        rows[2][:] = np.linspace(-size, size, 64, dtype=np.float32)[None]
        rows[2][:, 7] = 0
    b, rows, _, got, _ = run(eff, ctx, 8, I8, 1, 1, 64, 16, [2], [2], 0, edit=edit, place=False)
    v = decode(I8, got, b.pages, 1, 64, 16)[b.table[0, 0], 1, 0, :2]
    assert (v[:, 7] == 0).all()
    step = np.float64(size) / 254 + 2.0 ** -149 * 127 if size > 2.0 ** -119 else size * 1.01
    assert (np.abs(v - rows[2]) <= step * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_finite(ctx, eff, bad):
    """In int8 the whole row is not finite; in fp16 the value is; other rows are as ever."""
    def edit(rows):
        rows[2][1, 70] = bad              # v of token 1, head 1
    for t in (F16, I8):
        b, rows, _, got, _ = run(eff, ctx, 6, t, 2, 2, 64, 16, [3], [3], 0, edit=edit, place=False)
        v = decode(t, got, b.pages, 2, 64, 16)[b.table[0, 0], 1]
        with np.errstate(invalid="ignore"):
            assert not np.isfinite(v[1, 1] if t == I8 else v[1, 1, 6]).any()
        assert np.isfinite(v[0, :3]).all() and np.isfinite(v[1, [0, 2]]).all()


def test_fp16_range(ctx, eff):
    """Values past fp16 become infinities, below it subnormals or zeros."""
    def edit(rows):
        rows[2][:] = np.array([1e30, -70000, 65504, 1e-6, 6e-8, 1e-9, 65519.9, 65520], np.float32).repeat(8)[None]
    b, rows, _, got, _ = run(eff, ctx, 7, F16, 1, 1, 64, 16, [1], [1], 0, edit=edit, place=False)
    with np.errstate(over="ignore"):
        want = rows[2][0].astype(np.float16)
    assert np.array_equal(got[b.table[0, 0]].view(np.float16).reshape(2, 16, 64)[1, 0], want)


def test_far_pages(ctx, eff):
    """A page past 2^32 bytes."""
    page, heads, dim = 1024, 8, 128
    size = page_bytes(F16, heads, dim, page)
    pages = 5 * 2 ** 30 // size
    cb = ctx.alloc(pages * size)
    k, v = (np.random.default_rng(s).standard_normal((1, heads * dim)).astype(np.float32) for s in (1, 2))
    bufs = [ctx.upload(np.array(x, np.uint32)) for x in ([[pages - 1]], [0, 1], [1000])]
    batch = eff.KvBatch(*bufs, seqs=1, tokens=1, table_pages=1, max_new=1, max_len=1024)
    ctx.kv_append(eff.KvCache(F16, heads, dim, page, pages, cb), batch, eff.KvRows(k=ctx.upload(k), v=ctx.upload(v)))
    got = cb.read(np.float16, size // 2, (pages - 1) * size).reshape(2, heads, page, dim)
    assert np.array_equal(got[0, :, 999], k.reshape(heads, dim).astype(np.float16))
    assert np.array_equal(got[1, :, 999], v.reshape(heads, dim).astype(np.float16))
    got[:, :, 999] = 0
    assert not got.any()
    cb.free()


def test_recorded(ctx, eff):
    """A recorded append takes the next step's rows, lengths and pages."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [1, 1], [40, 3], 16)
    cb, k, v = ctx.alloc(b.pages * page_bytes(I8, 2, 64, 16)), ctx.alloc(2 * 128 * 4), ctx.alloc(2 * 128 * 4)
    cache, batch, rows = eff.KvCache(I8, 2, 64, 16, b.pages, cb), b.upload(eff, ctx), eff.KvRows(k=k, v=v)
    ctx.kv_append(cache, batch, rows)
    ctx.graph_begin()
    ctx.kv_append(cache, batch, rows)
    g = ctx.graph_end()
    other = ctx.alloc(cb.size)
    for lens in ([40, 3], [17, 1], [33, 2]):
        x = rng.standard_normal((2, 2, 128)).astype(np.float32)
        k.write(x[0])
        v.write(x[1])
        batch.buffers[2].write(np.array(lens, np.uint32))
        g.launch()
        got = cb.read()
        ctx.copy(other, cb, cb.size)
        ctx.kv_append(eff.KvCache(I8, 2, 64, 16, b.pages, other), batch, rows)
        assert np.array_equal(got, other.read())
        vals = decode(I8, got, b.pages, 2, 64, 16)
        for s in range(2):
            at = vals[b.table[s, (lens[s] - 1) // 16], 0, :, (lens[s] - 1) % 16]
            assert np.abs(at - x[0, s].reshape(2, 64)).max() <= np.abs(x[0, s]).max() / 253
        ctx.sync()
    g.destroy()


def test_refusals(ctx, eff):
    b = Batch(np.random.default_rng(9), [1, 1], [40, 30], 16)
    size = page_bytes(F16, 2, 64, 16)
    assert eff.kv_page_bytes(F16, 2, 64, 16) == size and eff.kv_page_bytes(I8, 2, 64, 16) == page_bytes(I8, 2, 64, 16)
    for bad in ((8, 2, 64, 16), (F16, 0, 64, 16), (F16, 2, 65, 16), (F16, 2, 64, 17), (F16, 2, 64, 8), (I8, 2, 512, 16)):
        assert eff.kv_page_bytes(*bad) == 0
    cb, x, qo, rope, w = ctx.alloc(b.pages * size), ctx.alloc(2 * 256 * 4), ctx.alloc(2 * 256 * 4), ctx.alloc(40 * 64 * 4), ctx.alloc(256)
    k, v = ctx.alloc(2 * 128 * 4), ctx.alloc(2 * 128 * 4)
    batch = b.upload(eff, ctx)
    before = ctx.stats()["kv_append"]

    def call(code, cache=None, **change):
        rows = {**dict(q=x, k=k, v=v, q_heads=4, q_out=qo, rope=rope, rope_positions=40, rope_dim=64, q_norm=w, k_norm=w), **change}
        with pytest.raises(eff.EffError) as e:
            ctx.kv_append(cache or eff.KvCache(F16, 2, 64, 16, b.pages, cb), batch, eff.KvRows(**rows))
        assert e.value.code == code and "kv append" in str(e.value)

    call(eff.E_TYPE, eff.KvCache(2, 2, 64, 16, b.pages, cb))
    call(eff.E_BOUNDS, eff.KvCache(F16, 2, 64, 16, b.pages + 1, cb))
    for change in (dict(rope_dim=66), dict(rope_dim=128), dict(rope_dim=6)):
        call(eff.E_SHAPE, **change)
    for change in (dict(k=None), dict(v=None), dict(q_heads=0), dict(q=None), dict(q_out=None), dict(rope=None), dict(rope_mode=2),
                   dict(q=(x, 2)), dict(k_stride=130), dict(k_stride=64), dict(q_out=k, q_heads=2), dict(q=(x, 0), q_out=x, q_heads=2, q_stride=256)):
        call(eff.E_INVALID, **change)
    for change in (dict(rope_positions=39), dict(rope_positions=41), dict(q_heads=5), dict(k=(k, 4)), dict(v_stride=132), dict(q_norm=ctx.alloc(16))):
        call(eff.E_BOUNDS, **change)
    assert ctx.stats()["kv_append"] == before
    assert eff.lib().eff_kv_append(None, None, None, None) == eff.E_INVALID
    for f, n, positions in ((None, 4, 4), (w, 0, 4), (w, 257, 4), (w, 4, 0)):
        rc = eff.lib().eff_rope_table(ctx.h, np.zeros(257).ctypes.data if f else None, n, positions, 1.0, rope.handle)
        assert rc in (eff.E_INVALID, eff.E_SHAPE)
    with pytest.raises(eff.EffError) as e:
        ctx.rope_table(np.ones(4), 1000, out=w)
    assert e.value.code == eff.E_BOUNDS
