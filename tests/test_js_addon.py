"""The grouped and 4-bit routines of the JavaScript layer through the real
addon and library on the CPU: node runs with a stand-in for the HIP runtime
(tests/native/ragged_runtime.cc) that lists every kernel's arguments. The same
calls through the Python binding, on operands of the same sizes allocated in the
same order, have to give the same list: the order and the types of what the
addon hands on are right. No kernel runs."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from tests.test_host_side import PRELUDE
from tests.test_ragged_host_side import runtime  # noqa: F401  (fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")
ADDON = os.path.join(ROOT, "wgblas_amd", "lib", "wgblas_hip.node")
BYTES = 160  # of the products' argument block

# addon_calls.mjs in the binding's terms; sizes are bytes of the allocations in their order
PYTHON = """
runtime.standin_arguments({bytes})
runtime.standin_clear()
ctx, out = wg.Context(0), []
F32 = wg.F32

def room(*sizes):
    return [ctx.empty(n, "uint8") for n in sizes]

def free(*buffers):
    for b in buffers:
        b.free()

A, B, off, C = room(600, 320, 32, 240)
ctx.gemm_grouped(F32, 1, 3, 5, 10, 7, 1.5, A, 9, 50, B, 8, off, 0.5, C, 6)
A, B, off, C = room(604, 324, 32, 244)
ctx.gemm_grouped(F32, 0, 3, 5, 10, 7, -2.0, A, 6, 51, B, 8, off, 0.0, C, 6)
A, B, C = room(608, 328, 248)
off, = room(32)
ctx.gemm_grouped(F32, 1, 3, 5, 10, 7, 1.0, A, 9, 50, B, 8, off, 1.0, C, 6)
A, B, off, C = room(220, 308, 24, 392)
ctx.gemm_grouped_k(F32, 2, 4, 6, 11, 0.25, A, 5, B, 7, off, -1.0, C, 8, 49)
wc, ws, x = room(12 * 128, 12 * 8, 12 * 131 * 4)
ctx.mxfp4_quantize(F32, 0, 130, 12, x, 131, wc, ws, 256)
xc, xs, x = room(9 * 128, 9 * 8, 1300 * 4)
ctx.mxfp4_quantize(F32, 1, 130, 9, x, 10, xc, xs, 256)
back, = room(130 * 12 * 4)
ctx.mxfp4_dequantize(F32, 130, 12, wc, ws, 256, back, 130)
C, = room(9 * 13 * 4)
ctx.mxfp4_gemm(12, 9, 130, 2.0, wc, ws, 256, xc, xs, 256, 0.75, C, 13, F32)
off, C = room(32, 9 * 5 * 4)
ctx.mxfp4_gemm_grouped(3, 4, 9, 130, 3.0, wc, ws, 256, 4 * 256, xc, xs, 256, off, 0.125, C, 5, F32)
print(json.dumps(runtime.standin_log().decode().splitlines()))
"""


def steps(lines):
    """Allocations, launches and their arguments."""
    return [line for line in lines if line.split()[0] in ("malloc", "at", "launch", "arguments")]


@pytest.mark.skipif(NODE is None, reason="node is not installed")
def test_the_addon_hands_on_what_the_binding_does(runtime, tmp_path):  # noqa: F811
    if not os.path.exists(ADDON):
        pytest.fail("the addon is not built: python -m wgblas_amd.build")
    log = str(tmp_path / "log")
    preload = ":".join([runtime] + [p for p in [os.environ.get("LD_PRELOAD")] if p])
    env = dict(os.environ, LD_PRELOAD=preload, STANDIN_ARGUMENTS=str(BYTES), STANDIN_LOG=log)
    env.pop("WGBLAS_HIP_ADDON", None)
    res = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "addon_calls.mjs")], cwd=ROOT, env=env, capture_output=True,
                         text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    script = PRELUDE.format(runtime=runtime) + PYTHON.replace("{bytes}", str(BYTES))
    py = subprocess.run([sys.executable, "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert py.returncode == 0, py.stderr
    with open(log) as file:
        got = steps(file.read().splitlines())
    want = steps(json.loads(py.stdout))
    assert sum("ragged_kernel" in line for line in want) == 6 and sum("quantize" in line for line in want) == 3
    assert got == want
