"""The JS layer's routing and 8-bit routines through the addon, against float64 in tests/js/experts.mjs."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(NODE is None, reason="node is not installed")]


def test_results():
    env = dict(os.environ)
    env.pop("WGBLAS_HIP_ADDON", None)
    res = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "experts.mjs")], cwd=ROOT, env=env, capture_output=True,
                         text=True, timeout=100)
    assert res.returncode == 0 and "5 passed, 0 failed" in res.stdout, res.stdout + res.stderr
