"""The JavaScript host's calls that are switched off, on the GPU (tests/js/shim_rules_off.js): through the addon too they
end in an error before anything reaches the library."""
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
def test_js_rules_switched_off():
    r = subprocess.run(["node", os.path.join(HERE, "js", "shim_rules_off.js")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "shim_rules_off ok" in r.stdout
