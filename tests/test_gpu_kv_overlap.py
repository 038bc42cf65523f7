"""eff_kv_append and eff_kv_attn refuse to write over what they read, and take buffers that only touch. Every call here
is refused by the host, or its buffers are apart."""
import ctypes

import numpy as np
import pytest

from kv_reference import F16, page_bytes

pytestmark = pytest.mark.gpu


def part(eff, ctx, buf, offset, size):
    """`size` bytes of a buffer from `offset` on, as a buffer of its own."""
    h = ctypes.c_void_p()
    assert eff.lib().eff_buf_wrap(ctx.h, buf.ptr + offset, size, ctypes.byref(h)) == eff.OK
    return eff.Buffer(ctx, h, size)


HEADS, DIM, PAGE, PAGES, TOKENS, Q_HEADS, LEN = 2, 64, 16, 3, 2, 4, 16
CACHE = PAGES * page_bytes(F16, HEADS, DIM, PAGE)
SIZES = {"cache": CACHE, "q": TOKENS * Q_HEADS * DIM * 4, "k": TOKENS * HEADS * DIM * 4, "v": TOKENS * HEADS * DIM * 4,
         "q_out": TOKENS * Q_HEADS * DIM * 4, "rope": LEN * DIM * 4, "q_norm": DIM * 4, "k_norm": DIM * 4, "table": 16, "starts": 16,
         "lens": 16}


def calls(eff, ctx, at):
    """The two calls with their buffers at the given offsets of one allocation."""
    whole = ctx.alloc(1 << 20)
    b = {n: part(eff, ctx, whole, at[n], SIZES[n]) for n in SIZES}
    for n, x in (("table", [0, 1]), ("starts", [0, 1, 2]), ("lens", [3, 9])):
        b[n].write(np.array(x, np.uint32))
    cache = eff.KvCache(F16, HEADS, DIM, PAGE, PAGES, b["cache"])
    batch = eff.KvBatch(b["table"], b["starts"], b["lens"], seqs=2, tokens=TOKENS, table_pages=1, max_new=1, max_len=LEN)
    rows = eff.KvRows(q=b["q"], k=b["k"], v=b["v"], q_heads=Q_HEADS, q_out=b["q_out"], rope=b["rope"], rope_positions=LEN, rope_dim=DIM,
                      q_norm=b["q_norm"], k_norm=b["k_norm"])
    return (whole, lambda: ctx.kv_append(cache, batch, rows),
            lambda: ctx.kv_attn(cache, batch, b["q"], b["q_out"], Q_HEADS, 0.1))


def apart():
    at, end = {}, 0
    for n, size in SIZES.items():
        at[n], end = end, end + (size + 15) // 16 * 16
    return at


def test_side_by_side(ctx, eff):
    whole, append, attn = calls(eff, ctx, apart())
    append()
    attn()
    ctx.sync()
    whole.free()


@pytest.mark.parametrize("written", ["cache", "q_out"])
@pytest.mark.parametrize("end", ["first", "last"])
def test_overlaps(ctx, eff, written, end):
    """The first or the last 16 bytes of what is written over the other end of each thing that is read."""
    for read in SIZES:
        if read == written:
            continue
        at = apart()
        # what is read moves past everything else, and what is written to one end of it
        at[read] = 1 << 19
        at[written] = at[read] + SIZES[read] - 16 if end == "first" else at[read] - SIZES[written] + 16
        whole, append, attn = calls(eff, ctx, at)
        before = ctx.stats()
        with pytest.raises(eff.EffError) as e:
            append()
        assert e.value.code == eff.E_INVALID and "overlap" in str(e.value), read
        if {read, written} <= {"cache", "q_out", "q", "table", "starts", "lens"} and "q_out" in (read, written):
            with pytest.raises(eff.EffError) as e:
                attn()
            assert e.value.code == eff.E_INVALID and "overlap" in str(e.value), read
        after = ctx.stats()
        assert all(before[k] == after[k] for k in ("kv_append", "kv_attn"))
        # touching is not overlapping
        at[written] += 16 if end == "first" else -16
        whole.free()
        whole, append, attn = calls(eff, ctx, at)
        append()
        attn()
        ctx.sync()
        whole.free()


def test_no_tokens(ctx, eff):
    """A call without new tokens writes nothing."""
    x = ctx.alloc(CACHE)
    t = [ctx.upload(np.array(v, np.uint32)) for v in ([0], [0, 0], [0])]
    batch = eff.KvBatch(*t, seqs=1, tokens=0, table_pages=1, max_new=1, max_len=16)
    cache = eff.KvCache(F16, HEADS, DIM, PAGE, PAGES, x)
    ctx.kv_append(cache, batch, eff.KvRows(k=x, v=x))
    ctx.kv_attn(cache, batch, x, x, Q_HEADS, 0.1)


def test_one_token_in_place(ctx, eff):
    """q turned within a fused row: a single token's q is its buffer's first floats whatever the stride."""
    rng = np.random.default_rng(1)
    fused = (Q_HEADS + 2 * HEADS) * DIM
    row = rng.standard_normal(fused).astype(np.float32)
    x, kept = ctx.upload(row), ctx.upload(row)
    rope, other = ctx.rope_table(1e4 ** (-np.arange(0, DIM, 2) / DIM), LEN), ctx.alloc(Q_HEADS * DIM * 4)
    b = [ctx.upload(np.array(v, np.uint32)) for v in ([1], [0, 1], [5])]
    batch = eff.KvBatch(*b, seqs=1, tokens=1, table_pages=1, max_new=1, max_len=LEN)
    got = []
    for rows, q_out in ((kept, other), (x, x)):
        buf = ctx.alloc(CACHE)
        ctx.kv_append(eff.KvCache(F16, HEADS, DIM, PAGE, PAGES, buf), batch,
                      eff.KvRows(q=rows, k=(rows, Q_HEADS * DIM), v=(rows, (Q_HEADS + HEADS) * DIM), q_stride=fused, k_stride=fused,
                                 v_stride=fused, q_heads=Q_HEADS, q_out=q_out, rope=rope, rope_positions=LEN, rope_dim=DIM))
        got.append((q_out.read(np.float32, Q_HEADS * DIM), buf.read()))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1]) and got[0][1].any()
    assert not np.array_equal(got[0][0], row[:Q_HEADS * DIM])
    assert np.array_equal(x.read(np.float32)[Q_HEADS * DIM:], row[Q_HEADS * DIM:])
