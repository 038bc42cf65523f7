"""Descriptions of a call's buffers (KvCache, KvBatch, KvRows, LogitsRules) after one of the buffers was given back: an
error, as with every other call, and not the freed handle."""
import numpy as np
import pytest


class NoContext:
    """What Buffer.free() needs of a context: the library does nothing without one."""
    h = None

    def _check(self, rc):
        return rc


def made(eff):
    new = lambda: eff.Buffer(NoContext(), 0x1000, 64)   # noqa: E731
    b = new()
    yield "buf", b, eff.KvCache(eff.KV_F16, 1, 64, 16, 1, b)
    for name in ("table", "starts", "lens"):
        x = {n: new() for n in ("table", "starts", "lens")}
        yield name, x[name], eff.KvBatch(**x, seqs=1, tokens=1, table_pages=1, max_new=1, max_len=1)
    for name in ("q", "k", "v", "q_out", "rope", "q_norm", "k_norm"):
        x = {n: new() for n in ("q", "k", "v", "q_out", "rope", "q_norm", "k_norm")}
        b = x[name]
        x["k"] = (x["k"], 64)
        yield name, b, eff.KvRows(**x, q_heads=1)
    for name in ("history", "history_starts", "penalties", "bias_ids", "bias_values", "bias_starts", "mask", "mask_of"):
        x = {n: new() for n in ("history", "history_starts", "penalties", "bias_ids", "bias_values", "bias_starts", "mask", "mask_of")}
        yield name, x[name], eff.LogitsRules(**x, mask_count=1)


@pytest.mark.parametrize("give_back", ["free", "retire"])
def test_freed_buffer(eff, give_back):
    seen = 0
    for name, buffer, described in list(made(eff)):
        assert described.ref and getattr(described.c, name) == 0x1000
        getattr(buffer, give_back)()
        for _ in range(2):
            with pytest.raises(eff.EffError) as e:
                described.ref
            assert e.value.code == eff.E_INVALID and name in str(e.value)
        seen += 1
    assert seen == 19


def test_other_buffers_freed(eff):
    """Only a description's own buffers matter to it; one without buffers has nothing to lose."""
    b, other = (eff.Buffer(NoContext(), 0x1000, 64) for _ in range(2))
    cache, none = eff.KvCache(eff.KV_F16, 1, 64, 16, 1, b), eff.LogitsRules()
    at = cache.ref, none.ref
    other.free()
    assert (cache.ref, none.ref) == at and cache.c.buf == 0x1000


@pytest.mark.gpu
def test_calls_after_free(ctx, eff):
    up = lambda x, d=np.uint32: ctx.upload(np.array(x, d))   # noqa: E731
    x = [ctx.alloc(4 * 64) for _ in range(4)]

    def refused(call):
        with pytest.raises(eff.EffError) as e:
            call()
        assert e.value.code == eff.E_INVALID

    cache = eff.KvCache(eff.KV_F16, 1, 64, 16, 1, ctx.alloc(eff.kv_page_bytes(eff.KV_F16, 1, 64, 16)))
    batch = eff.KvBatch(up([0]), up([0, 1]), up([1]), seqs=1, tokens=1, table_pages=1, max_new=1, max_len=16)
    rows = eff.KvRows(k=x[0], v=x[1], k_norm=x[2])
    rules = eff.LogitsRules(history=up([1]), history_starts=up([0, 1]), penalties=up([1, 0, 0], np.float64))
    before = ctx.stats()
    for _ in range(2):
        ctx.kv_append(cache, batch, rows)
        ctx.kv_attn(cache, batch, x[3], x[0], 1, 0.1)
        ctx.logits_apply(x[1], x[1], 1, 64, rules)
    x[2].retire()
    refused(lambda: ctx.kv_append(cache, batch, rows))
    rules.buffers[0].free()
    refused(lambda: ctx.logits_apply(x[1], x[1], 1, 64, rules))
    batch.buffers[1].free()
    refused(lambda: ctx.kv_attn(cache, batch, x[3], x[0], 1, 0.1))
    after = ctx.stats()
    assert all(after[k] - before[k] == 2 for k in ("kv_append", "kv_attn", "logits"))
