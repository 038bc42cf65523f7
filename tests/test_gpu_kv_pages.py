"""Copies of pages and drafts that stay (eff_kv_copy, eff_kv_keep) on the GPU: bytes against bytes, in every layer; what
the calls do not name keeps its bytes."""
import ctypes

import numpy as np
import pytest

from kv_reference import F16, I8, NO_PAGE, Batch, page_bytes
from kv_rules_reference import random_tree, row_bytes, tree_mask

pytestmark = pytest.mark.gpu


def layers_of(eff, ctx, rng, t, layers, heads, dim, page, pages):
    """Caches of random bytes: their description, and the bytes [layers][...]."""
    data = rng.integers(0, 256, (layers, pages * page_bytes(t, heads, dim, page)), dtype=np.uint8)
    return eff.KvLayers([eff.KvCache(t, heads, dim, page, pages, ctx.upload(x)) for x in data]), data


def read(caches, t, heads, dim, page, pages):
    return [row_bytes(t, c.buffers[0].read(np.uint8), pages, heads, dim, page) for c in caches.caches]


def free(*x):
    for b in x:
        b.free()


# ---- copies --------------------------------------------------------------------

def copy(eff, ctx, seed, t, layers, heads, dim, page, pages, copies):
    rng = np.random.default_rng(seed)
    caches, data = layers_of(eff, ctx, rng, t, layers, heads, dim, page, pages)
    cb = ctx.upload(np.array(copies, np.uint32).reshape(-1, 3))
    ctx.kv_copy(caches, cb, len(copies))
    for d, got in zip(data, read(caches, t, heads, dim, page, pages)):
        want = row_bytes(t, d, pages, heads, dim, page)
        old = want.copy()
        for a, b, n in copies:
            if a < pages and b < pages:
                want[b, :, :, :n] = old[a, :, :, :n]
        assert np.array_equal(got, want)
    free(cb, *caches.buffers)


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("layers,heads,page", [(1, 1, 16), (3, 2, 64), (2, 5, 256)])
def test_copy(ctx, eff, t, dim, layers, heads, page):
    copies = [(0, 7, page), (1, 8, 1), (2, 9, page - 1), (3, 10, 5), (3, 11, 0), (4, 12, page + 9), (5, 13, 0xFFFFFFFF), (5, 14, 3)]
    copy(eff, ctx, dim, t, layers, heads, dim, page, 16, copies)


@pytest.mark.parametrize("t", [F16, I8])
def test_copy_of_no_page(ctx, eff, t):
    """Numbers past the cache copy nothing; a page onto itself keeps its bytes."""
    copy(eff, ctx, 1, t, 2, 2, 64, 16, 6, [(NO_PAGE, 1, 16), (0, NO_PAGE, 16), (6, 2, 4), (3, 6, 4), (4, 4, 9), (0, 5, 8)])


@pytest.mark.parametrize("t", [F16, I8])
def test_many_copies(ctx, eff, t):
    rng = np.random.default_rng(2)
    order = rng.permutation(1000)
    copy(eff, ctx, 2, t, 2, 3, 96, 16, 1000, [(int(a), int(b), int(n)) for a, b, n in zip(order[:450], order[450:900], rng.integers(0, 17, 450))])


def test_copies_of_large_pages(ctx, eff):
    """Runs that end inside a workgroup's part."""
    for t in (F16, I8):
        copy(eff, ctx, 3, t, 1, 3, 96, 1024, 4, [(0, 2, 1000), (1, 3, 77)])


@pytest.mark.parametrize("layers", [64, 65, 130])
def test_copies_of_many_layers(ctx, eff, layers):
    copy(eff, ctx, layers, I8, layers, 1, 64, 16, 3, [(0, 2, 7)])


# ---- drafts that stay ------------------------------------------------------------

def keep(eff, ctx, seed, t, layers, heads, dim, page, new, lens, kept, counts=None, table=None, max_new=None, max_len=None, lens_too=True):
    """kept: of each sequence its list; counts: as the call has them, where they are others."""
    rng = np.random.default_rng(seed)
    b = Batch(rng, new, lens, page)
    if table is not None:
        table(b)
    counts = [len(k) for k in kept] if counts is None else counts
    caches, data = layers_of(eff, ctx, rng, t, layers, heads, dim, page, b.pages)
    entries = rng.integers(0, 2 ** 32, b.tokens, dtype=np.uint32)
    for s, k in enumerate(kept):
        entries[b.starts[s]:b.starts[s] + len(k)] = k
    batch, kb, cb = b.upload(eff, ctx, max_new=max_new, max_len=max_len), ctx.upload(entries), ctx.upload(np.array(counts, np.uint32))
    lb = ctx.upload(np.full(len(new), 77, np.uint32)) if lens_too else None
    ctx.kv_keep(caches, batch, kb, cb, lb)
    for d, got in zip(data, read(caches, t, heads, dim, page, b.pages)):
        want = row_bytes(t, d, b.pages, heads, dim, page)
        old = want.copy()
        for s, (n, length) in enumerate(zip(new, lens)):
            first = length - n
            for i in range(min(counts[s], n)):
                k = int(entries[b.starts[s] + i])
                if not i <= k < n or first + i < 0:
                    continue
                p = [int(b.table[s, (first + j) // page]) for j in (k, i)]
                if max(p) < b.pages:
                    want[p[1], :, :, (first + i) % page] = old[p[0], :, :, (first + k) % page]
        assert np.array_equal(got, want)
    if lens_too:
        assert lb.read(np.uint32).tolist() == [max(0, length - n + min(c, n)) for n, length, c in zip(new, lens, counts)]
        free(lb)
    free(kb, cb, *caches.buffers, *batch.buffers)


def paths(rng, new):
    got = []
    for n in new:
        m = tree_mask(random_tree(rng, n)) if n else np.zeros((0, 0), bool)
        got.append([int(j) for j in np.flatnonzero(m[rng.integers(0, n)])] if n else [])
    return got


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("layers,heads,page", [(1, 1, 16), (3, 2, 32), (2, 5, 64)])
def test_keep(ctx, eff, t, dim, layers, heads, page):
    rng = np.random.default_rng(dim)
    new = [25, 1, 0, 9, 64, 16, 2]
    keep(eff, ctx, dim, t, layers, heads, dim, page, new, [125, 1, 7, 9, 500, 47, 33], paths(rng, new))


@pytest.mark.parametrize("t", [F16, I8])
@pytest.mark.parametrize("n,stay", [(2, [1]), (40, list(range(1, 40))), (40, list(range(40))), (33, [0, 32]), (30, []), (200, list(range(5, 195))),
                                    (300, list(range(0, 300, 2))), (70, [0] + list(range(2, 70)))])
def test_lists(ctx, eff, t, n, stay):
    """Places that are read after others are written: each takes what was there before the call."""
    keep(eff, ctx, n, t, 2, 2, 128, 16, [n, 3], [n + 21, 3], [stay, [0, 2]])


@pytest.mark.parametrize("t", [F16, I8])
def test_entries_that_move_nothing(ctx, eff, t):
    """Below their place, past the new tokens, more than there are, the same twice."""
    keep(eff, ctx, 4, t, 1, 2, 64, 16, [6, 6, 4, 5, 3], [30, 6, 20, 25, 9], [[0, 0, 5], [2, 6, 4], [3, 3, 3, 3], [4, 0xFFFFFFFF, 4], [1, 2]],
         counts=[3, 3, 0xFFFFFFFF, 3, 7])


def test_without_pages_and_positions(ctx, eff):
    def table(b):
        b.table[0, 1] = NO_PAGE           # of the places, then of the tokens
        b.table[1, 2] = b.pages
    keep(eff, ctx, 5, F16, 2, 1, 64, 16, [20, 20, 5], [40, 50, 3], [[0, 5, 12, 19], [0, 1, 15, 18], [1, 3, 4]], table=table)
    keep(eff, ctx, 6, F16, 1, 1, 64, 16, [8], [20], [[0, 3, 7]], lens_too=False)


def test_bounds_above_the_sizes(ctx, eff):
    keep(eff, ctx, 7, I8, 2, 3, 96, 32, [5, 1] * 40, [60, 1] * 40, [[0, 2, 4], [0]] * 40, max_new=600, max_len=64)


@pytest.mark.parametrize("layers", [64, 65, 200])
def test_keep_in_many_layers(ctx, eff, layers):
    keep(eff, ctx, layers, F16, layers, 1, 64, 16, [9, 4], [20, 4], [[0, 4, 8], [1, 3]])


def test_keep_recorded(ctx, eff):
    """A recorded call takes the next step's lists; its lengths are the next call's."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [8, 8], [24, 40], 16)
    caches, data = layers_of(eff, ctx, rng, F16, 3, 2, 64, 16, b.pages)
    batch, kb, cb, lb = b.upload(eff, ctx), ctx.alloc(4 * 16), ctx.alloc(8), ctx.alloc(8)
    ctx.kv_keep(caches, batch, kb, cb, lb)
    ctx.graph_begin()
    ctx.kv_keep(caches, batch, kb, cb, lb)
    g = ctx.graph_end()
    for _ in range(4):
        lists = [sorted(rng.choice(8, rng.integers(0, 9), replace=False).tolist()) for _ in range(2)]
        entries = np.zeros((2, 8), np.uint32)
        for s, k in enumerate(lists):
            entries[s, :len(k)] = k
        for c, d in zip(caches.caches, data):
            c.buffers[0].write(d)
        kb.write(entries)
        cb.write(np.array([len(k) for k in lists], np.uint32))
        g.launch()
        assert lb.read(np.uint32).tolist() == [16 + len(lists[0]), 32 + len(lists[1])]
        for d, got in zip(data, read(caches, F16, 2, 64, 16, b.pages)):
            want = row_bytes(F16, d, b.pages, 2, 64, 16)
            old = want.copy()
            for s, k in enumerate(lists):
                for i, j in enumerate(k):
                    a, c = b.lens[s] - 8 + j, b.lens[s] - 8 + i
                    want[b.table[s, c // 16], :, :, c % 16] = old[b.table[s, a // 16], :, :, a % 16]
            assert np.array_equal(got, want)
        ctx.sync()
    g.destroy()


def test_far_pages(ctx, eff):
    """Pages whose bytes lie past 4 GiB."""
    t, heads, dim, page = F16, 8, 256, 256
    each = page_bytes(t, heads, dim, page)
    pages = (5 << 30) // each + 2
    cb = ctx.alloc(pages * each)
    rng = np.random.default_rng(3)
    rows = rng.integers(0, 256, (2, each), dtype=np.uint8)
    caches = eff.KvLayers([eff.KvCache(t, heads, dim, page, pages, cb)])
    h = [ctypes.c_void_p() for _ in range(3)]
    for x, p in zip(h, (0, pages - 1, pages - 2)):
        assert eff.lib().eff_buf_wrap(ctx.h, cb.ptr + p * each, each, ctypes.byref(x)) == eff.OK
    first, last, other = (eff.Buffer(ctx, x, each) for x in h)
    first.write(rows[0])
    last.write(rows[1])
    other.write(rows[1])
    ctx.kv_copy(caches, ctx.upload(np.array([0, pages - 2, page], np.uint32)), 1)
    assert np.array_equal(other.read(), rows[0])
    # a sequence of two pages, the second far behind the first
    up = lambda *x: ctx.upload(np.array(x, np.uint32))   # noqa: E731
    batch = eff.KvBatch(up(0, pages - 1), up(0, 4), up(page + 2), seqs=1, tokens=4, table_pages=2, max_new=4, max_len=2 * page)
    ctx.kv_keep(caches, batch, up(0, 3, 0, 0), up(2))
    a, b = (row_bytes(t, x, 1, heads, dim, page)[0] for x in (first.read(), last.read()))
    old = [row_bytes(t, x, 1, heads, dim, page)[0] for x in rows]
    assert np.array_equal(b, old[1]) and np.array_equal(a[:, :, page - 1], old[1][:, :, 1]) and np.array_equal(a[:, :, :page - 1], old[0][:, :, :page - 1])
    cb.free()


def test_refusals(ctx, eff):
    rng = np.random.default_rng(4)
    b = Batch(rng, [2, 2], [20, 9], 16)
    caches, _ = layers_of(eff, ctx, rng, F16, 2, 2, 64, 16, b.pages)
    one, two = caches.caches
    batch, x, y, lens = b.upload(eff, ctx), ctx.upload(np.zeros(12, np.uint32)), ctx.upload(np.zeros(4, np.uint32)), ctx.alloc(8)
    before = ctx.stats()
    L = eff.KvLayers

    def call(code, f):
        with pytest.raises(eff.EffError) as e:
            f()
        assert e.value.code == code and "kv " in str(e.value), str(e.value)

    other = [eff.KvCache(I8, 2, 64, 16, 2, one.buffers[0]), eff.KvCache(F16, 1, 64, 16, b.pages, one.buffers[0]),
             eff.KvCache(F16, 2, 64, 16, b.pages - 1, one.buffers[0])]
    big = eff.KvCache(F16, 2, 64, 16, b.pages + 1, one.buffers[0])
    for o in other:
        call(eff.E_SHAPE, lambda: ctx.kv_copy(L([two, o]), x, 1))
        call(eff.E_SHAPE, lambda: ctx.kv_keep(L([two, o]), batch, x, y, lens))
    for f in (lambda c: ctx.kv_copy(c, x, 1), lambda c: ctx.kv_keep(c, batch, x, y, lens)):
        call(eff.E_INVALID, lambda: f(L([])))
        call(eff.E_INVALID, lambda: f(L([one, two, one])))                            # one layer twice
        call(eff.E_BOUNDS, lambda: f(L([big])))
        call(eff.E_TYPE, lambda: f(L([eff.KvCache(2, 2, 64, 16, 1, one.buffers[0])])))
    half = ctypes.c_void_p()
    size = one.buffers[0].size
    whole = ctx.alloc(2 * size)
    assert eff.lib().eff_buf_wrap(ctx.h, whole.ptr + size // 2 // 16 * 16, size, ctypes.byref(half)) == eff.OK
    shifted = eff.KvCache(F16, 2, 64, 16, b.pages, eff.Buffer(ctx, half, size))
    call(eff.E_INVALID, lambda: ctx.kv_copy(L([shifted, eff.KvCache(F16, 2, 64, 16, b.pages, whole)]), x, 1))
    call(eff.E_BOUNDS, lambda: ctx.kv_copy(caches, x, 5))
    call(eff.E_INVALID, lambda: ctx.kv_copy(caches, two.buffers[0], 1))
    cut = eff.KvBatch(*batch.buffers, seqs=2, tokens=13, table_pages=b.table_pages, max_new=2, max_len=20)
    call(eff.E_BOUNDS, lambda: ctx.kv_keep(caches, cut, x, y, lens))
    call(eff.E_BOUNDS, lambda: ctx.kv_keep(caches, batch, x, ctx.alloc(4), lens))
    call(eff.E_BOUNDS, lambda: ctx.kv_keep(caches, batch, x, y, ctx.alloc(4)))
    for bad in (x, y, *batch.buffers, two.buffers[0]):
        call(eff.E_INVALID, lambda: ctx.kv_keep(caches, batch, x, y, bad))           # new_lens over what is read
    for bad in (one.buffers[0], two.buffers[0]):
        call(eff.E_INVALID, lambda: ctx.kv_keep(caches, batch, bad, y))
        call(eff.E_INVALID, lambda: ctx.kv_keep(caches, batch, x, bad))
    after = ctx.stats()
    assert all(before[k] == after[k] for k in ("kv_copy", "kv_keep"))
    ctx.kv_copy(caches, x, 0)
    assert ctx.stats()["kv_copy"] == before["kv_copy"]
    assert eff.lib().eff_kv_copy(None, None, 1, None, 0) == eff.E_INVALID
    assert eff.lib().eff_kv_keep(None, None, 1, None, None, None, None) == eff.E_INVALID
    assert eff.lib().eff_kv_copy(ctx.h, None, 1, x.handle, 1) == eff.E_INVALID
    one.buffers[0].free()
    with pytest.raises(eff.EffError):
        ctx.kv_copy(caches, x, 1)
