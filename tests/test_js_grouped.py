"""The JS layer's grouped and 4-bit routines (sgemmGrouped, sgemmGroupedK,
Mxfp4Matrix, mxfp4Gemm, mxfp4GemmGrouped) through a host-memory stand-in for the
addon's calls; the kernels behind the C ABI are the pytest GPU suites' part."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")


@pytest.mark.skipif(NODE is None, reason="node is not installed")
def test_js_grouped_routines():
    env = dict(os.environ, WGBLAS_HIP_ADDON=os.path.join(ROOT, "tests", "js", "grouped_addon.cjs"))
    res = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "grouped.mjs")], cwd=ROOT, env=env, capture_output=True,
                         text=True, timeout=120)
    assert res.returncode == 0 and "7 passed, 0 failed" in res.stdout, res.stdout + res.stderr


def test_addon_binds_the_calls_the_routines_make():
    text = open(os.path.join(ROOT, "wgblas_amd", "csrc", "napi_addon.cc")).read()
    for name in ("gemmGrouped", "gemmGroupedK", "mxfp4Quantize", "mxfp4Dequantize", "mxfp4Gemm"):
        assert '{"%s", ' % name in text
