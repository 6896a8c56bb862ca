"""Grouped products of operands with 1 to 9 rows, k-rows of a row-contiguous one a few bytes apart: k around whole
k-tiles (32 of fp32, 64 of 16-bit values), where copies of 16 bytes reach over several k-rows and the last ones have to
be loaded by element (tests/test_copy_plan.py checks the addresses)."""
import pytest

from tests.test_gpu_grouped import run_columns, run_k
from wgblas_amd import NO_TRANS

pytestmark = pytest.mark.gpu

KS = {"f32": (32, 33, 34, 35, 36, 65, 66, 97), "f16": (64, 65, 66, 67, 70, 72, 129, 131), "bf16": (64, 65, 66, 67, 70, 72, 129, 131)}


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 1, 2])
@pytest.mark.parametrize("m", [1, 2, 3, 5, 9])
def test_columns(ctx, t, m, pad):
    for k in KS[t]:
        run_columns(ctx, t, t, NO_TRANS, m, k, [5, 0, 40], (pad, 0, 0), seed=k)  # few columns a group
        run_columns(ctx, t, "f32", NO_TRANS, m, k, [300], (pad, 0, 0), seed=k)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 1, 2])
@pytest.mark.parametrize("m,n", [(1, 1), (2, 3), (1, 200), (200, 1), (3, 140), (5, 9)])
def test_k(ctx, t, m, n, pad):
    for k in KS[t]:
        run_k(ctx, t, "f32", m, n, [7, k], (pad, pad, 0), seed=k)
