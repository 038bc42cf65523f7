"""The batch's operators from two host threads at once, and from one context whose stream changes between calls: the bits
of the calls made alone. Attention's tiles are shared by workgroups here, whose counters and sums lie in the context's
scratch; a call on a new stream has to find them as the one before left them."""
import ctypes
import threading

import numpy as np
import pytest

from kv_reference import F16, I8, Batch, page_bytes

pytestmark = pytest.mark.gpu

# type, key heads, group, dim, lengths: shares that end with a tile, shares that go on, a join in two steps
CASES = [(F16, 2, 8, 128, [9000, 5000, 100]), (I8, 8, 2, 64, [2300] + list(range(1, 380, 5))), (F16, 1, 16, 128, [33000])]


def made(eff, ctx, seed):
    """The buffers of every case, and its step: append, attention, rules."""
    steps = []
    for t, heads, group, dim, lens in CASES:
        rng = np.random.default_rng(seed)
        n = len(lens)
        b = Batch(rng, [1] * n, lens, 64)
        kv = rng.standard_normal(b.pages * page_bytes(F16, heads, dim, 64) // 2).astype(np.float16)
        data = kv.view(np.uint8)
        if t == I8:     # any bytes are int8; scales of their own size
            data = rng.integers(0, 256, (b.pages, 2, heads, 64 * (dim + 4)), dtype=np.uint8)
            data[..., 64 * dim:].view(np.float32)[:] = (0.01 + 0.01 * rng.random((b.pages, 2, heads, 64))).astype(np.float32)
        up = ctx.upload
        fused = (heads * group + 2 * heads) * dim
        x = up(rng.standard_normal(n * fused).astype(np.float32))
        q, y = ctx.alloc(n * heads * group * dim * 4), ctx.alloc(n * heads * group * dim * 4)
        cache, batch = eff.KvCache(t, heads, dim, 64, b.pages, up(data)), b.upload(eff, ctx)
        rope = ctx.rope_table(1e4 ** (-np.arange(0, dim, 2) / dim), max(lens))
        rows = eff.KvRows(q=x, k=(x, heads * group * dim), v=(x, (heads * group + heads) * dim), q_stride=fused, k_stride=fused, v_stride=fused,
                          q_heads=heads * group, q_out=q, rope=rope, rope_positions=max(lens), rope_dim=dim)
        rules = eff.LogitsRules(history=up(np.arange(5 * n, dtype=np.uint32)), history_starts=up(5 * np.arange(n + 1, dtype=np.uint32)),
                                penalties=up(np.tile([1.1, 0.2, 0.1], n)))
        z = ctx.alloc(n * heads * group * dim * 4)

        def step(cache=cache, batch=batch, rows=rows, q=q, y=y, z=z, rules=rules, n=n, h=heads * group, d=dim, keep=(x, rope)):
            ctx.kv_append(cache, batch, rows)
            ctx.kv_attn(cache, batch, q, y, h, d ** -0.5)
            ctx.logits_apply(y, z, n, h * d, rules)
            return y, z, cache.buffers[0]
        steps.append(step)
    return steps


def read(out):
    return [b.read(np.uint8) for b in out]


def alone(eff, seed):
    with eff.Context(0) as c:
        return [read(step()) for step in made(eff, c, seed)]


def test_two_threads(eff):
    want = [alone(eff, s) for s in (1, 2)]
    got, errors = [[], []], []

    def work(i):
        try:
            with eff.Context(0) as c:
                steps = made(eff, c, i + 1)
                for _ in range(5):
                    got[i].append([read(step()) for step in steps])
        except Exception as e:   # raised below
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and not any(t.is_alive() for t in threads)
    for i in range(2):
        for outs in got[i]:
            assert all(np.array_equal(a, b) for x, y in zip(outs, want[i]) for a, b in zip(x, y))


def test_streams_in_turn(eff):
    """Two streams of one context: each call behind the one before, without a wait of the host between them."""
    want = alone(eff, 3)
    hip = ctypes.CDLL("libamdhip64.so.7")   # the runtime the library already loaded
    side = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(side), 1) == 0
    with eff.Context(0) as c:
        steps = made(eff, c, 3)
        for turn in range(12):
            c.set_stream(side.value if turn % 2 else None)
            outs = [step() for step in steps]
        c.set_stream(None)
        assert all(np.array_equal(a, b) for x, y in zip([read(o) for o in outs], want) for a, b in zip(x, y))
        c.sync()
    assert hip.hipStreamDestroy(side) == 0
