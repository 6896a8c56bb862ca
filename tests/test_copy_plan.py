"""The copies that stage operands of the grouped and 4-bit products
(wgblas_amd/csrc/copy_plan.h), compiled for the host with g++ from the same
source the kernels include: for every tile shape and layout, over small
matrices, each read stays inside the matrix and each element comes from its own
address. Row-contiguous matrices of 1 to 3 rows are among them, whose k-rows are
closer together than a copy is long."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_copies_stay_inside_the_matrix(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "copy_plan_check")
    subprocess.run([gxx, "-O1", "-std=c++17", "-Wno-unknown-pragmas", os.path.join(HERE, "native", "copy_plan_check.cc"),
                    "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    lines = out.splitlines()
    assert len(lines) == 16, out
    for line in lines:
        name, result = line.split(": ", 1)
        assert result.split()[0] == "ok" and int(result.split()[1]) > 1000, out
