"""The copies that stage 8-bit operands (wgblas_amd/csrc/copy_plan.h), compiled for the host: every read of every tile shape
and layout stays inside small matrices, and each code comes from its own address."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_copies_stay_inside_the_matrix(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "copy_plan_fp8_check")
    subprocess.run([gxx, "-O1", "-std=c++17", "-Wno-unknown-pragmas", os.path.join(HERE, "native", "copy_plan_fp8_check.cc"),
                    "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    lines = out.splitlines()
    assert len(lines) == 7, out
    for line in lines:
        name, result = line.split(": ", 1)
        assert result.split()[0] == "ok" and int(result.split()[1]) > 100, out
