"""The host side of routing and of the 8-bit products without a GPU, through the stand-in for the HIP runtime that runs no
kernel: refused arguments, empty sizes, the workspace."""
import shutil
import subprocess
import sys
import json
import os

import pytest

from tests.test_host_side import PRELUDE

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

CALLS = """
from wgblas_amd import BF16, F16, F32, NO_TRANS, SIGMOID, SOFTMAX, TRANS
ctx = wg.Context(0)

def call(name, **change):
    "A good call with some arguments changed."
    arguments = dict(GOOD[name])
    assert set(change) <= set(arguments), change
    arguments.update(change)
    return calls(lambda: getattr(ctx, name)(*arguments.values()))

GOOD = {
    "route": dict(type=F32, scoring=SOFTMAX, experts=64, n=5, topk=8, logits=P, ldl=64, bias=None, groups=8, top_groups=2,
                  best=2, renorm=1, scale=1.0, ids=P, weights=P),
    "route_grad": dict(type=BF16, scoring=SIGMOID, experts=64, n=5, topk=8, logits=P, ldl=64, ids=P, renorm=0, scale=1.0,
                       dweights=P, dlogits=P, ldd=64),
    "route_order": dict(experts=64, n=5, topk=8, ids=P, offsets=P, places=P, pairs=P),
    "route_gather": dict(type=F16, d=100, n=5, topk=2, X=P, ldx=100, places=P, weights=None, Y=P, ldy=100),
    "route_combine": dict(type=F16, d=100, n=5, topk=2, Y=P, ldy=100, places=P, weights=None, beta=0.0, C=P, ldc=100,
                          ctype=F32),
    "route_combine_grad": dict(type=F16, d=100, n=5, topk=2, dC=P, lddc=100, Y=P, ldy=100, places=P, weights=P, dY=P,
                               lddy=100, dweights=P),
    "fp8_quantize": dict(type=BF16, trans=TRANS, block=1, k=300, n=20, X=P, ldx=20, codes=P, ld=384, scales=P, lds=20),
    "fp8_dequantize": dict(type=BF16, block=128, k=300, n=200, codes=P, ld=384, scales=P, lds=2, X=P, ldx=300),
    "fp8_gemm": dict(transA=TRANS, m=200, n=20, k=300, alpha=1.0, A=P, lda=384, blockA=128, scaleA=P, ldsa=2, B=P, ldb=384,
                     scaleB=P, ldsb=20, beta=0.0, C=P, ldc=200, ctype=F32),
    "fp8_gemm_grouped": dict(transA=NO_TRANS, groups=3, m=200, n=20, k=300, alpha=1.0, A=P, lda=256, strideA=256 * 300,
                             blockA=128, scaleA=P, ldsa=3, strideScaleA=6, B=P, ldb=384, scaleB=P, ldsb=20, offsets=P,
                             beta=0.0, C=P, ldc=200, ctype=BF16),
}

def launches(log):
    return [line for line in log if "launch" in line]
"""


@pytest.fixture(scope="module")
def child(tmp_path_factory):
    gxx, hipcc = shutil.which("g++"), shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "include")
    if gxx is None or not os.path.exists(os.path.join(include, "hip", "hip_runtime_api.h")):
        pytest.skip("g++ or the HIP headers are not available")
    so = str(tmp_path_factory.mktemp("runtime") / "ragged_runtime.so")
    subprocess.run([gxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", include,
                    os.path.join(HERE, "native", "ragged_runtime.cc"), "-o", so], check=True)

    def run(script):
        res = subprocess.run([sys.executable, "-c", PRELUDE.format(runtime=so) + CALLS + script], cwd=ROOT,
                             capture_output=True, text=True, timeout=300)
        assert res.returncode == 0, res.stderr
        return json.loads(res.stdout)

    return run


REFUSED = {
    "route": [dict(type=3), dict(scoring=2), dict(experts=0), dict(experts=1025, ldl=2000, groups=1, top_groups=1),
              dict(n=-1), dict(topk=0), dict(topk=65), dict(topk=17), dict(n=2 ** 31 // 8), dict(n=2 ** 24, topk=1), dict(ldl=63), dict(groups=0),
              dict(groups=7), dict(groups=128, experts=128, ldl=128), dict(top_groups=0), dict(top_groups=9), dict(best=0),
              dict(best=3), dict(logits=None), dict(ids=None), dict(weights=None)],
    "route_grad": [dict(type=-1), dict(scoring=-1), dict(experts=7), dict(n=-2), dict(topk=70), dict(ldl=8), dict(ldd=8),
                   dict(logits=None), dict(ids=None), dict(dweights=None), dict(dlogits=None)],
    "route_order": [dict(experts=0), dict(experts=2000), dict(n=-1), dict(topk=0), dict(topk=65), dict(n=2 ** 30),
                    dict(ids=None), dict(offsets=None), dict(places=None), dict(pairs=None)],
    "route_gather": [dict(type=5), dict(d=-1), dict(d=2 ** 31, ldx=2 ** 31, ldy=2 ** 31), dict(n=-1), dict(topk=0),
                     dict(topk=65), dict(n=2 ** 31), dict(n=2 ** 24, topk=1), dict(ldx=99), dict(ldy=99), dict(X=None), dict(places=None), dict(Y=None)],
    "route_combine": [dict(type=5), dict(ctype=2), dict(d=-1), dict(n=-1), dict(topk=0), dict(ldy=99), dict(ldc=99),
                      dict(Y=None), dict(places=None), dict(C=None)],
    "route_combine_grad": [dict(type=5), dict(d=-1), dict(n=-1), dict(topk=65), dict(lddc=99), dict(ldy=99), dict(lddy=99),
                           dict(dC=None), dict(Y=None), dict(places=None), dict(weights=None), dict(dY=None),
                           dict(dweights=None)],
    "fp8_quantize": [dict(type=3), dict(trans=2), dict(block=64), dict(k=-1), dict(n=-1), dict(n=2 ** 31), dict(n=2 ** 26, lds=2 ** 26),
                     dict(ldx=19),
                     dict(ld=300), dict(ld=256), dict(ld=2 ** 23 + 128), dict(lds=19), dict(lds=2 ** 29), dict(X=None),
                     dict(codes=None), dict(scales=None), "codes=P + 8", "scales=P + 2"],
    "fp8_dequantize": [dict(type=3), dict(block=0), dict(k=-1), dict(ld=320), dict(lds=1), dict(ldx=299), dict(X=None),
                       dict(codes=None), dict(scales=None)],
    "fp8_gemm": [dict(transA=2), dict(m=-1), dict(n=-1), dict(k=-1), dict(lda=300), dict(lda=256), dict(blockA=2),
                 dict(blockA=1, transA=0, lda=256, ldsa=400), dict(ldsa=1), dict(blockA=1, ldsa=199), dict(ldb=256),
                 dict(ldsb=19), dict(ldc=199), dict(ctype=3), dict(A=None), dict(scaleA=None), dict(B=None),
                 dict(scaleB=None), dict(C=None), "A=P + 4", "B=P + 4", "scaleA=P + 1", "scaleB=P + 1"],
    "fp8_gemm_grouped": [dict(groups=-1), dict(groups=2 ** 20 + 1), dict(lda=128), dict(strideA=256 * 300 - 16),
                         dict(strideA=256 * 300 + 8), dict(strideScaleA=5), dict(ldsa=2), dict(offsets=None), dict(C=None),
                         dict(k=2 ** 31, strideA=256 * 2 ** 31)],
}


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused_before_any_launch(child, name):
    changes = ", ".join(f"dict({c})" if isinstance(c, str) else repr(c) for c in REFUSED[name])
    got = child(f"""
out = [call({name!r}, **c) for c in [{changes}]]
log, error = call({name!r})
print(json.dumps([[[len(launches(l)), e] for l, e in out], len(launches(log)), error]))
""")
    for change, (count, error) in zip(REFUSED[name], got[0]):
        assert error and "status -1" in error, (change, error)
        assert count == 0, change
    assert got[1] >= 1 and got[2] is None  # the call that all of them change


def test_empty_sizes_launch_nothing(child):
    """No tokens, no columns, no rows: nothing to do, and no pointer is needed. The order of no pairs has boundaries."""
    got = child("""
nothing = dict(logits=None, ids=None, weights=None)
out = [call("route", n=0, **nothing), call("route_grad", n=0, logits=None, ids=None, dweights=None, dlogits=None),
       call("route_gather", n=0, X=None, places=None, Y=None), call("route_gather", d=0, X=None, Y=None),
       call("route_combine", n=0, Y=None, places=None, C=None), call("route_combine_grad", n=0, dC=None, Y=None, dY=None),
       call("fp8_quantize", k=0, X=None, codes=None, scales=None), call("fp8_quantize", n=0, ldx=1, X=None, codes=None),
       call("fp8_dequantize", n=0, X=None), call("fp8_gemm", m=0, A=None, C=None), call("fp8_gemm", n=0, B=None, C=None),
       call("fp8_gemm_grouped", groups=0, offsets=None, C=None)]
order = call("route_order", n=0, ids=None, places=None, pairs=None)
print(json.dumps([[[len(launches(l)), e] for l, e in out], [len(launches(order[0])), order[1]]]))
""")
    assert got[0] == [[0, None]] * len(got[0])
    assert got[1] == [1, None]


def test_order_of_few_pairs_is_one_launch_without_workspace(child):
    got = child("""
few = call("route_order", n=128)
many = call("route_order", n=129)
print(json.dumps([few, many]))
""")
    (few, e1), (many, e2) = got
    assert e1 is None and e2 is None
    assert sum("launch" in line for line in few) == 1 and not any("alloc" in line for line in few)
    assert sum("launch" in line for line in many) == 2
