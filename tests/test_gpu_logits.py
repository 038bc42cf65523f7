"""Rules on the logits of a batch (eff_logits_apply) on the GPU: every bit as numpy's 64-bit numbers rounded to f32 give it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def expected(z, stride, history, penalties, bias, mask, mask_of):
    """The rules in f64, rounded to f32 after each; history: a list of ids a row, bias: a list of (id, value) a row."""
    out = z.copy()
    rows, vocab = z.shape
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                ids, count = np.unique([i for i in history[r] if i < vocab], return_counts=True)
                for i, c in zip(ids.astype(int), count):
                    rep, freq, pres = penalties[r]
                    x = out[r, i]
                    if rep != 1:
                        x = np.float32(np.float64(x) / rep if x > 0 else np.float64(x) * rep)
                    out[r, i] = np.float32(np.float64(x) - (freq * np.float64(c) + pres))
            if bias is not None:
                for i, value in {i: v for i, v in bias[r]}.items():
                    if i < vocab:
                        out[r, i] += np.float32(value)
            if mask is not None and mask_of[r] < len(mask):
                bits = np.unpackbits(mask[mask_of[r]].view(np.uint8), bitorder="little")[:vocab]
                out[r, bits == 0] = -np.inf
    return out


def ragged(ctx, lists, dtype=np.uint32):
    flat = np.array([x for row in lists for x in row], dtype)
    return ctx.upload(flat), ctx.upload(np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.uint32))


def run(eff, ctx, z, stride=0, history=None, penalties=None, bias=None, mask=None, mask_of=None, in_place=False, offset=None):
    rows, vocab = z.shape
    stride = stride or vocab
    full = np.full((rows, stride), 3, np.float32)
    full[:, :vocab] = z
    src = ctx.upload(full.ravel()[:(rows - 1) * stride + vocab])
    dst = src if in_place else ctx.upload(np.full(src.size // 4, 8, np.float32))
    at = {}
    if history is not None:
        at["history"], at["history_starts"] = ragged(ctx, history)
        at["penalties"] = ctx.upload(np.asarray(penalties, np.float64))
    if bias is not None:
        at["bias_ids"], at["bias_starts"] = ragged(ctx, [[i for i, _ in row] for row in bias])
        at["bias_values"] = ragged(ctx, [[v for _, v in row] for row in bias], np.float32)[0]
    if mask is not None:
        at.update(mask=ctx.upload(mask), mask_of=ctx.upload(np.asarray(mask_of, np.uint32)), mask_count=len(mask))
    ctx.logits_apply(src, dst, rows, vocab, eff.LogitsRules(**at), stride if stride != vocab else 0)
    got = np.empty((rows, stride), np.float32)
    got.ravel()[:src.size // 4] = dst.read(np.float32)
    want = expected(z, stride, history, penalties, bias, mask, mask_of)
    same = (got[:, :vocab].view(np.uint32) == want.view(np.uint32)) | (np.isnan(got[:, :vocab]) & np.isnan(want))
    assert same.all(), np.argwhere(~same)[:5]
    gap = got[:-1, vocab:]
    assert (gap == (3 if in_place else 8)).all()
    return got[:, :vocab]


def inputs(rng, rows, vocab, history=50, bias=0, masks=0):
    z = (4 * rng.standard_normal((rows, vocab))).astype(np.float32)
    h = [list((vocab * rng.random(n) ** 3).astype(int)) for n in rng.integers(0, history + 1, rows)]
    pen = np.stack([1 + rng.random(rows), rng.random(rows) - 0.3, rng.random(rows) - 0.3], 1)
    b = [[(int(i), float(np.float32(v))) for i, v in zip(rng.integers(0, vocab, n), rng.standard_normal(n))]
         for n in rng.integers(0, bias + 1, rows)] if bias else None
    m = rng.integers(0, 2 ** 32, (masks, (vocab + 31) // 32), dtype=np.uint32) if masks else None
    mo = rng.integers(0, masks + 2, rows).astype(np.uint32) if masks else None
    return z, h, pen, b, m, mo


def test_quotients_between_two_numbers(ctx, eff):
    """Repeats for which a logit over the repeat lies next to the middle of two f32 numbers, and the smallest quotients."""
    rng = np.random.default_rng(5)
    rows = 4000
    z = np.exp(rng.uniform(-3, 3, (rows, 4))).astype(np.float32)
    low = rng.uniform(0.3, 30, rows).astype(np.float32)
    middle = (low.astype(np.float64) + np.nextafter(low, np.float32(np.inf)).astype(np.float64)) / 2
    repeat = z[:, 0].astype(np.float64) / middle
    for step in range(-3, 4):
        at = np.arange(rows) % 7 == step + 3
        repeat[at] += step * np.spacing(repeat[at])
    z[:, 1] *= np.float32(1e-38)
    z[:, 2] *= -1
    run(eff, ctx, z, history=[[0, 1, 2, 3]] * rows, penalties=[[x, 0, 0] for x in repeat])
    run(eff, ctx, z, history=[[0, 1, 2, 3, 3]] * rows, penalties=[[x, 0.25, 0.5] for x in 10.0 ** rng.uniform(-120, 120, rows)])


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (2, 33), (3, 1000), (5, 4096), (2, 4097), (4, 50021), (1, 200003), (70, 300)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules(ctx, eff, rows, vocab, in_place):
    rng = np.random.default_rng(rows * vocab)
    z, h, pen, b, m, mo = inputs(rng, rows, vocab, 80, 9, 3)
    run(eff, ctx, z, 0, h, pen, b, m, mo, in_place)
    run(eff, ctx, z, vocab + 5, h, pen, b, m, mo, in_place)


@pytest.mark.parametrize("which", ["history", "bias", "mask", "none"])
def test_one_rule(ctx, eff, which):
    rng = np.random.default_rng(1)
    z, h, pen, b, m, mo = inputs(rng, 6, 9001, 300, 20, 2)
    at = {"history": dict(history=h, penalties=pen), "bias": dict(bias=b), "mask": dict(mask=m, mask_of=mo), "none": {}}[which]
    for in_place in (False, True):
        run(eff, ctx, z, in_place=in_place, **at)


def test_long_history(ctx, eff):
    """70000 ids of one row, most of them a few tokens; others have none."""
    rng = np.random.default_rng(2)
    z, _, pen, *_ = inputs(rng, 4, 32000)
    h = [[], list((32000 * rng.random(70000) ** 8).astype(int)), [31999] * 66000, [0]]
    run(eff, ctx, z, 0, h, pen)


def test_ids_past_the_vocabulary(ctx, eff):
    rng = np.random.default_rng(3)
    z, _, pen, *_ = inputs(rng, 2, 5000)
    far = [5000, 5001, 2 ** 31, 2 ** 32 - 1, 9000]
    run(eff, ctx, z, 0, [far + [7], far], pen, [[(i, 1.0) for i in far], [(4999, 2.0), (6000, 1.0)]])


def test_repeated_biases(ctx, eff):
    """Of several values of one id the last counts."""
    rng = np.random.default_rng(4)
    z = rng.standard_normal((2, 700)).astype(np.float32)
    b = [[(5, 1.0), (6, 2.0), (5, -3.0), (5, 0.5)], [(699, float(i)) for i in range(1000)]]
    got = run(eff, ctx, z, bias=b)
    assert got[1, 699] == z[1, 699] + np.float32(999)


def test_masks_that_leave_nothing(ctx, eff):
    """A mask of zeros: the row is -inf; one of ones: the row is as it was; NaN and infinities that are masked go too."""
    rng = np.random.default_rng(5)
    z = rng.standard_normal((4, 777)).astype(np.float32)
    z[0, ::3], z[1, ::5], z[2, ::7], z[3, 5] = np.nan, np.inf, -np.inf, np.nan
    m = np.stack([np.zeros(25, np.uint32), np.full(25, 2 ** 32 - 1, np.uint32)])
    got = run(eff, ctx, z, mask=m, mask_of=[0, 0, 1, 0xFFFFFFFF])
    assert (got[:2] == -np.inf).all()


def test_values_that_are_not_finite(ctx, eff):
    z = np.array([[np.nan, np.inf, -np.inf, 0.0, -0.0, 3e38, -3e38, 1e-45, -1e-45, 1]], np.float32)
    for pen in ([1.5, 0, 0], [0.5, 0.25, -1], [1.0, 0.0, 0.0], [np.inf, 0, 0], [1.0, 1e300, 0], [1.0, 0.0, np.nan], [0.0, 0, 0]):
        run(eff, ctx, z, 0, [list(range(10)) * 2], [pen], [[(1, 1.0), (2, np.inf), (9, np.nan)]])


def test_sampler_penalties(ctx, eff):
    """Without a frequency: what the sampler does to a Float32Array with its window (repeat, then presence)."""
    rng = np.random.default_rng(6)
    z = (5 * rng.standard_normal((1, 3000))).astype(np.float32)
    window = list(rng.integers(0, 3000, 64))
    want = z[0].copy()
    for i in set(window):
        want[i] = np.float64(want[i]) / 1.1 if want[i] > 0 else np.float64(want[i]) * 1.1
        want[i] = np.float64(want[i]) - 0.3
    got = run(eff, ctx, z, 0, [window], [[1.1, 0.0, 0.3]])
    assert np.array_equal(got[0], want)


def test_recorded(ctx, eff):
    rng = np.random.default_rng(7)
    z, h, pen, b, m, mo = inputs(rng, 3, 6000, 40, 0, 2)
    src, dst = ctx.upload(z), ctx.alloc(z.nbytes)
    hb, hs = ctx.alloc(4 * 200), ctx.alloc(16)
    rules = eff.LogitsRules(history=hb, history_starts=hs, penalties=ctx.upload(pen), mask=ctx.upload(m), mask_of=ctx.upload(mo), mask_count=2)
    ctx.logits_apply(src, dst, 3, 6000, rules)
    ctx.graph_begin()
    ctx.logits_apply(src, dst, 3, 6000, rules)
    g = ctx.graph_end()
    for step in range(4):
        z, h, *_ = inputs(rng, 3, 6000, 40)
        src.write(z)
        hb.write(np.array([x for row in h for x in row] + [0], np.uint32))
        hs.write(np.concatenate([[0], np.cumsum([len(x) for x in h])]).astype(np.uint32))
        dst.write(np.zeros_like(z))
        g.launch()
        got = dst.read(np.uint32).reshape(z.shape)
        assert np.array_equal(got, expected(z, 0, h, pen, None, m, mo).view(np.uint32)), step
        ctx.logits_apply(src, dst, 3, 6000, rules)
        assert np.array_equal(got, dst.read(np.uint32).reshape(z.shape))
        ctx.sync()
    g.destroy()


def test_then_topk(ctx, eff):
    """A row of the result is what the top-k reads."""
    rng = np.random.default_rng(8)
    z, h, pen, b, m, mo = inputs(rng, 3, 40000, 100, 5, 1)
    src, dst = ctx.upload(z), ctx.alloc(z.nbytes)
    at = dict(zip(("history", "history_starts"), ragged(ctx, h)))
    ctx.logits_apply(src, dst, 3, 40000, eff.LogitsRules(penalties=ctx.upload(pen), **at))
    want = expected(z, 0, h, pen, None, None, None)
    for r in range(3):
        top = eff.parse_topk(ctx.topk(dst, r * 40000, 40000, 40).read(np.uint32))
        order = np.lexsort((np.arange(40000), -want[r].astype(np.float64)))[:40]
        assert np.array_equal(top["ids"], order)


def test_refusals(ctx, eff):
    z, small = ctx.alloc(4 * 300), ctx.alloc(16)
    starts, pen = ctx.upload(np.zeros(4, np.uint32)), ctx.alloc(72)
    before = ctx.stats()["logits"]

    def call(code, rows=3, vocab=100, stride=0, src=z, dst=z, **rules):
        with pytest.raises(eff.EffError) as e:
            ctx.logits_apply(src, dst, rows, vocab, eff.LogitsRules(**rules), stride)
        assert e.value.code == code and "logits" in str(e.value)

    call(eff.E_SHAPE, vocab=0)
    call(eff.E_INVALID, stride=99)
    call(eff.E_BOUNDS, vocab=101)
    call(eff.E_BOUNDS, stride=101)
    call(eff.E_BOUNDS, dst=small)
    call(eff.E_INVALID, history=small)
    call(eff.E_INVALID, history=small, history_starts=starts)
    call(eff.E_BOUNDS, history=small, history_starts=ctx.alloc(12), penalties=pen)
    call(eff.E_BOUNDS, history=small, history_starts=starts, penalties=ctx.alloc(48))
    call(eff.E_INVALID, bias_ids=small, bias_values=small)
    call(eff.E_INVALID, mask=small, mask_count=1)
    call(eff.E_BOUNDS, mask=ctx.alloc(12), mask_of=starts, mask_count=1)
    call(eff.E_BOUNDS, mask=small, mask_of=ctx.alloc(8), mask_count=1)
    assert eff.lib().eff_logits_apply(None, None, None, 0, 0, 0, None) == eff.E_INVALID
    ctx.logits_apply(z, z, 0, 100, eff.LogitsRules())
    assert ctx.stats()["logits"] == before
