"""eff_logits_apply refuses to write over what its rules read, and takes buffers that only touch."""
import numpy as np
import pytest

from test_gpu_kv_overlap import part

pytestmark = pytest.mark.gpu

ROWS, VOCAB = 3, 100
SIZES = {"history_starts": 16, "penalties": 72, "bias_starts": 16, "mask": 32, "mask_of": 12}


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("end", ["first", "last"])
def test_overlaps(ctx, eff, name, end):
    """The first bytes of what is read under out's last ones, or its last under out's first; then side by side."""
    whole, z = ctx.alloc(1 << 16), ctx.alloc(ROWS * VOCAB * 4)
    size, out = SIZES[name], ROWS * VOCAB * 4
    rules = {n: part(eff, ctx, whole, 256 * i, s) for i, (n, s) in enumerate(SIZES.items())}
    rules["mask_of"].write(np.array([0, 7, 1], np.uint32))
    rules.update({n: part(eff, ctx, whole, 4096 + 256 * i, 64) for i, n in enumerate(("history", "bias_ids", "bias_values"))})

    def call(read, written):
        rules[name] = part(eff, ctx, whole, read, size)
        ctx.logits_apply(z, part(eff, ctx, whole, written, out), ROWS, VOCAB, eff.LogitsRules(**rules, mask_count=2))

    before = ctx.stats()["logits"]
    with pytest.raises(eff.EffError) as e:
        call(8192 + out - 16, 8192) if end == "first" else call(8192, 8192 + (size - 1) // 16 * 16)
    assert e.value.code == eff.E_INVALID and "overlap" in str(e.value) and ctx.stats()["logits"] == before
    call(8192 + out, 8192) if end == "first" else call(8192, 8192 + (size + 15) // 16 * 16)
    ctx.sync()
    whole.free()
