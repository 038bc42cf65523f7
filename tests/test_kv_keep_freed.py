"""kv_keep on the CPU: lengths that were given back are an error, not left out."""
import pytest


class NoLibrary:
    h = None

    def _check(self, rc):
        self.rc = rc


@pytest.mark.parametrize("give_back", ["free", "retire"])
def test_freed_lengths(eff, give_back):
    c = NoLibrary()
    b, lens = (eff.Buffer(c, 0x1000, 64) for _ in range(2))
    layers = eff.KvLayers([eff.KvCache(eff.KV_F16, 1, 64, 16, 1, b)])
    batch = eff.KvBatch(b, b, b, seqs=1, tokens=1, table_pages=1, max_new=1, max_len=1)
    for new_lens in (None, lens):
        eff.Context.kv_keep(c, layers, batch, b, b, new_lens)   # reaches the library, which has no context here
        assert c.rc == eff.E_INVALID
    getattr(lens, give_back)()
    with pytest.raises(eff.EffError) as e:
        eff.Context.kv_keep(c, layers, batch, b, b, lens)
    assert e.value.code == eff.E_INVALID and "new_lens" in str(e.value)
