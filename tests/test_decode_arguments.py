"""The decoding example's arguments, without a device: what it cannot decode is an error before anything is made."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("prompts,steps", [([], 3), ([[1, 2], []], 3), ([[]], 1), ([[1]], 0)])
def test_refusals(prompts, steps):
    spec = importlib.util.spec_from_file_location("decode_example", os.path.join(ROOT, "elffuss-engine_amd", "examples", "decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    with pytest.raises(ValueError, match="prompt|step"):
        m.decode(None, None, None, prompts, steps, {})
