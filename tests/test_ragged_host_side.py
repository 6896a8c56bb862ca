"""The host side of the grouped and 4-bit products without a GPU, through a
stand-in for the HIP runtime (tests/native/ragged_runtime.cc) that runs no
kernel and keeps a list of what was asked of it: the context's workspace, the
kernels' LDS sizes, which tiles a call takes."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from tests.test_host_side import PRELUDE

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

CALLS = """
from wgblas_amd import BF16, F16, F32, NO_TRANS, TRANS
ctx = wg.Context(0)

def columns(m, n, k, groups=1, t=BF16, trans=TRANS, pad=0, on=None, A=P):
    lda = (k if trans == TRANS else m) + pad
    (on or ctx).gemm_grouped(t, trans, groups, m, n, k, 1.0, A, lda, lda * (m if trans == TRANS else k), P + (1 << 30), k + pad,
                             P, 0.0, P, m)

def ragged_k(m, n, k, groups=1, t=BF16, pad=0, on=None):
    (on or ctx).gemm_grouped_k(t, groups, m, n, k, 1.0, P, m + pad, P + (1 << 30), n + pad, P, 0.0, P, m, m * n, F32)

def of(log, kind):
    return [line.split()[1] for line in log if line.split()[0] == kind]
"""


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    gxx, hipcc = shutil.which("g++"), shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "include")
    if gxx is None or not os.path.exists(os.path.join(include, "hip", "hip_runtime_api.h")):
        pytest.skip("g++ or the HIP headers are not available")
    so = str(tmp_path_factory.mktemp("runtime") / "ragged_runtime.so")
    subprocess.run([gxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", include,
                    os.path.join(HERE, "native", "ragged_runtime.cc"), "-o", so], check=True)
    return so


@pytest.fixture(scope="module")
def child(runtime):
    def run(script):
        res = subprocess.run([sys.executable, "-c", PRELUDE.format(runtime=runtime) + CALLS + script], cwd=ROOT,
                             capture_output=True, text=True, timeout=300)
        assert res.returncode == 0, res.stderr
        return json.loads(res.stdout)

    return run


def test_a_workspace_that_a_graph_holds_is_kept_when_it_grows(child):
    """A captured call records the workspace's address. A later call that needs a larger one may not free it: replays
    would write into memory that is someone else's by then. It goes with the context."""
    got = child("""
small, large = (lambda: columns(1501, 1700, 801)), (lambda: columns(4001, 4100, 4097))
log, error = calls(small)
assert error is None and len(of(log, "at")) == 1, (log, error)
first = of(log, "at")[0]
runtime.standin_capture(1)
captured, error = calls(small)
assert error is None, error
runtime.standin_capture(0)
grown, error = calls(large)
assert error is None, error
second = of(grown, "at")[0]
again, error = calls(lambda: columns(8001, 8100, 8097))
gone, error = calls(ctx.close)
print(json.dumps([first, second, of(captured, "at"), of(captured, "free"), of(grown, "free"), of(again, "free"), of(gone, "free")]))
""")
    first, second, *rest = got
    assert rest[:2] == [[], []]
    assert first not in rest[2]  # the graph's
    assert rest[3] == [second]  # no graph holds this one
    assert first in rest[4] and second not in rest[4]


def test_a_captured_call_may_not_grow_the_workspace(child):
    """It is refused before it asks for anything that would end the capture."""
    got = child("""
runtime.standin_capture(1)
log, error = calls(lambda: columns(1501, 1700, 801))
runtime.standin_capture(0)
print(json.dumps([log, error, calls(lambda: columns(1501, 1700, 801))[1]]))
""")
    log, error, after = got
    assert error and "captur" in error, error
    assert not any(line.split()[0] in ("launch", "malloc", "synchronize", "free") for line in log), log
    assert after is None


def test_every_device_gets_the_kernels_lds_size(child):
    """The kernels use more LDS than a launch has by default, which is allowed for each device by itself; where that
    fails, the next call tries again."""
    got = child("""
second, out = wg.Context(1), []
runtime.standin_attributes(0)
out.append(calls(lambda: columns(4096, 4096, 1024)))
runtime.standin_attributes(1)
for on in (ctx, second, ctx, second):
    out.append(calls(lambda: columns(4096, 4096, 1024, on=on)))
print(json.dumps(out))
""")
    failed, *rest = got
    assert failed[1] and not any(line.startswith("launch") for line in failed[0]), failed
    seen = set()
    for (log, error), device in zip(rest, "0101"):
        assert error is None, error
        for line in log:
            word = line.split()
            if word[0] == "attribute":
                assert word[1] == device and (device, word[3]) not in seen, log
                seen.add((device, word[3]))
            elif word[0] == "launch" and "ragged_kernel" in word[5]:
                assert (device, word[5]) in seen, (log, seen)
    assert len(seen) >= 2 and len(seen) % 2 == 0


def test_no_memory_for_the_workspace_is_no_error(child):
    """What it is for only makes a call faster: copies of operands at odd leading dimensions, and the sums of tiles that
    are cut along k. Without it the operands are loaded through registers, the tiles are not cut."""
    got = child("""
out = []
for limit in (1 << 20, 1 << 50):
    runtime.standin_memory(ctypes.c_size_t(limit))
    for call in (lambda: columns(1501, 1700, 801), lambda: ragged_k(1501, 1701, 8001), lambda: columns(2048, 8448, 4096, groups=2)):
        log, error = calls(call)
        out.append([error, [line.split() for line in log if line.startswith("launch")], of(log, "out_of_memory")])
print(json.dumps(out))
""")
    for (error, launches, failed), odd in zip(got, (True, True, False) * 2):
        assert error is None, error
        kernels = [line[5] for line in launches]
        assert all(int(line[1]) > 0 for line in launches)
        if failed:
            assert not any("align" in name or "Fold" in name for name in kernels), kernels
        else:
            assert any(("align" if odd else "Fold") in name for name in kernels), kernels
        assert any("ragged_kernel" in name for name in kernels)
    assert all(failed for _, _, failed in got[:3]) and not any(failed for _, _, failed in got[3:])


TILES = """
import re

def tiles(f):
    "Of each product launch of f: its kind and the sides of its tiles."
    log, error = calls(f)
    assert error is None, error
    out = []
    for line in log:
        word = line.split()
        if word[0] != "launch":
            continue
        if "FoldKernel" in word[5]:
            out.append("fold")
        elif "TurnKernel" in word[5]:
            out.append("256")
        elif "SkinnyKernel" in word[5]:
            out.append("few")
        elif "ragged_kernel" in word[5]:
            out.append("x".join(re.search("6KernelI.*?Li([0-9]+)ELi([0-9]+)E", word[5]).groups()))
        else:
            out.append(re.search("align|quantize", word[5]).group(0))
    return out

def mxfp4(m, n, k, groups=0, ct=BF16):
    ld = (k + 127) // 128 * 128
    if groups:
        ctx.mxfp4_gemm_grouped(groups, m, n, k, 1.0, P, P, ld, m * ld, P, P, ld, P, 0.0, P, m, ct)
    else:
        ctx.mxfp4_gemm(m, n, k, 1.0, P, P, ld, P, P, ld, 0.0, P, m, ct)
"""


def test_small_products_take_small_tiles(child):
    """One to three tiles of 256 x 256 would leave nearly all CUs idle for as long as one of them takes."""
    got = child(TILES + """
out = {}
for m, n in ((256, 256), (512, 256), (256, 768), (200, 180), (40, 50)):
    for k in (512, 4096, 8192):
        out[f"columns {m} {n} {k}"] = tiles(lambda: columns(m, n, k))
        out[f"no-transpose {m} {n} {k}"] = tiles(lambda: columns(m, n, k, trans=NO_TRANS, t=F16))
        out[f"ragged k {m} {n} {k}"] = tiles(lambda: ragged_k(m, n, k))
        out[f"mxfp4 {m} {n} {k}"] = tiles(lambda: mxfp4(m, n, k))
print(json.dumps(out))
""")
    assert len(got) == 60
    for case, kinds in got.items():
        assert kinds == ["64x64"], (case, kinds)


def test_small_operands_are_not_moved_on_a_false_estimate(child):
    """At odd leading dimensions the copies cost a launch (about 3 us), which products this small do not get back."""
    got = child(TILES + """
print(json.dumps([tiles(lambda: columns(m, n, k, pad=1)) for m, n, k in ((64, 64, 256), (256, 64, 256), (200, 180, 128))]))
""")
    assert got == [["64x64"]] * 3


def test_the_cases_of_the_256_tiles_take_them(child):
    """tests/test_gpu_ragged_turns.py holds the 256 x 256 kernel to what it computes: all its cases have to reach it."""
    from tests import test_gpu_ragged_turns as cases

    mxfp4 = [(m, sum(sizes), k, len(sizes)) for m, k, sizes, _ in cases.MXFP4]
    columns = [(m, sum(sizes), k, len(sizes)) for m, k, sizes, _ in cases.COLUMNS]
    ragged_k = [(m, n, sum(sizes), len(sizes)) for m, n, sizes, _ in cases.K]
    got = child(TILES + f"""
print(json.dumps([
    [tiles(lambda: mxfp4(*c, ct=ct)) for c in {mxfp4} for ct in (BF16, F32)],
    [tiles(lambda: columns(*c, t=t, trans=trans)) for c in {columns} for t in (BF16, F16) for trans in (NO_TRANS, TRANS)],
    [tiles(lambda: ragged_k(*c, t=t)) for c in {ragged_k} for t in (BF16, F16)]]))
""")
    for rows, listed, each in zip(got, (cases.MXFP4, cases.COLUMNS, cases.K), (2, 4, 2)):
        assert len(rows) == each * len(listed)
        for i, kinds in enumerate(rows):
            assert "256" in kinds and ("fold" in kinds) == listed[i // each][3], (listed[i // each], kinds)
