"""The JS layer's routing and 8-bit routines: their refusals on a host-memory stand-in for the addon's memory calls."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")


@pytest.mark.skipif(NODE is None, reason="node is not installed")
def test_refusals():
    env = dict(os.environ, WGBLAS_HIP_ADDON=os.path.join(ROOT, "tests", "js", "stub_addon.cjs"))
    res = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "experts.mjs"), "refusals"], cwd=ROOT, env=env,
                         capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "1 passed, 0 failed" in res.stdout, res.stdout + res.stderr


def test_addon_binds_the_calls_the_routines_make():
    text = open(os.path.join(ROOT, "wgblas_amd", "csrc", "napi_addon.cc")).read()
    for name in ("fp8Quantize", "fp8Dequantize", "fp8Gemm", "route", "routeGrad", "routeOrder", "routeGather", "routeCombine",
                 "routeCombineGrad"):
        assert '{"%s", ' % name in text
