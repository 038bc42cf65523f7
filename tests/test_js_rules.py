"""The JavaScript host's positions, rules, copies and drafts that stay on the CPU: what they refuse
(tests/js/shim_rules_cpu.js, no device calls)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
def test_js_shim_rules_cpu(eff):
    r = subprocess.run(["node", os.path.join(HERE, "js", "shim_rules_cpu.js")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "shim_rules_cpu ok" in r.stdout
