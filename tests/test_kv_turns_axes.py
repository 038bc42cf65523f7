"""KvTurns on the CPU: axes that are named for fewer pairs than turn are an error, not axis 0 for the rest."""
import pytest


class NoLibrary:
    """What Context.kv_append needs of a context: its handle, and a look at what the library says."""
    h = None

    def _check(self, rc):
        self.rc = rc


def append(eff, axis, axes, rope_dim):
    b = eff.Buffer(None, 0x1000, 64)
    c = NoLibrary()
    rows = eff.KvRows(k=b, v=b, rope=b, rope_positions=1, rope_dim=rope_dim)
    cache, batch = eff.KvCache(eff.KV_F16, 1, 64, 16, 1, b), eff.KvBatch(b, b, b, seqs=1, tokens=1, table_pages=1, max_new=1, max_len=1)
    eff.Context.kv_append(c, cache, batch, rows, turns=eff.KvTurns(b, axis, axes=axes))
    return c.rc


@pytest.mark.parametrize("axis,axes,rope_dim", [([0] * 16 + [1] * 15, 2, 64), ([0], 1, 64), ([0, 1, 2], 3, 8)])
def test_fewer_axes_than_pairs(eff, axis, axes, rope_dim):
    with pytest.raises(eff.EffError) as e:
        append(eff, axis, axes, rope_dim)
    assert e.value.code == eff.E_INVALID and "KvTurns" in str(e.value)


@pytest.mark.parametrize("axis,axes,rope_dim", [((), 1, 64), ([0] * 16 + [1] * 16, 2, 64), ([0] * 128, 1, 64), ([0, 1], 2, 4), ([0], 1, 0)])
def test_axes_of_all_pairs(eff, axis, axes, rope_dim):
    """These reach the library, which has no context here."""
    assert append(eff, axis, axes, rope_dim) == eff.E_INVALID
