"""Which kernels an 8-bit product takes, asked of the library through the stand-in for the HIP runtime
(tests/native/ragged_runtime.cc), which runs none: for the tests that hold a kernel to what it computes."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from tests.test_host_side import PRELUDE

HERE = os.path.dirname(os.path.abspath(__file__))

SCRIPT = """
import re
from wgblas_amd import BF16, F16, F32, NO_TRANS
ctx = wg.Context(0)
TYPES = dict(f32=F32, f16=F16, bf16=BF16)

def run(k):
    return max(128, (k + 127) // 128 * 128)

def kernels(trans, block, ct, sizes, m, k, extra=0):
    "Of each launch: '256', 'fold', 'few', or the sides of its tiles."
    length, columns = (m, k) if trans == NO_TRANS else (k, m)
    n, lda, ldsa = sum(sizes) + extra, run(length), (columns + block - 1) // block
    a = (lda, block, P, ldsa), (P, run(k), P, n)
    if len(sizes) == 1:
        f = lambda: ctx.fp8_gemm(trans, m, n, k, 1.0, P, *a[0], *a[1], 0.0, P, m, TYPES[ct])
    else:
        f = lambda: ctx.fp8_gemm_grouped(trans, len(sizes), m, n, k, 1.0, P, lda, lda * columns, block, P, ldsa, lda // 128 * ldsa,
                                         *a[1], P, 0.0, P, m, TYPES[ct])
    log, error = calls(f)
    assert error is None, error
    out = []
    for line in log:
        word = line.split()
        if word[0] == "launch":
            name = word[5]
            out.append("fold" if "FoldKernel" in name else "256" if "Fp8Large" in name else "few" if "Fp8Skinny" in name else
                       "x".join(re.search("Fp8KernelI.*?Li([0-9]+)ELi([0-9]+)E", name).groups()))
    return out
"""


def of(cases, where):
    """The kernels of each (trans, block, ct, sizes, m, k, columns of no group), one group: a dense product; `where`: a folder for the stand-in's library."""
    gxx, hipcc = shutil.which("g++"), shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "include")
    if gxx is None or not os.path.exists(os.path.join(include, "hip", "hip_runtime_api.h")):
        pytest.skip("g++ or the HIP headers are not available")
    so = os.path.join(str(where), "ragged_runtime.so")
    subprocess.run([gxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", include,
                    os.path.join(HERE, "native", "ragged_runtime.cc"), "-o", so], check=True)
    script = PRELUDE.format(runtime=so) + SCRIPT + f"print(json.dumps([kernels(*c) for c in {list(cases)!r}]))"
    res = subprocess.run([sys.executable, "-c", script], cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    return json.loads(res.stdout)
