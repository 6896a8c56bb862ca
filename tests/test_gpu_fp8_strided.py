"""Quantising along the strided axis, more values than the caches hold, at whole dwords (past the caches) and between them:
bit for bit as the definition."""
import numpy as np
import pytest

from tests import fp8 as F
from tests import ragged as R
from wgblas_amd import TRANS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("block", [1, 128])
def test_strided_past_the_caches(ctx, t, block):
    n, k = 4222, 4100
    rng = np.random.default_rng(9)
    stored = R.encode(rng.standard_normal((n, k)), t)
    code, scale = F.quantize(R.decode(stored, t), block)
    code = np.where(code == 0x80, 0, code)
    for pad, first in ((0, 0), (2, 0), (1, 0), (0, 1)):  # `first`: an element that X starts behind
        host = np.zeros(1 + k * (n + pad), stored.dtype)
        host[first:first + k * (n + pad)].reshape(k, n + pad)[:, :n] = stored.T
        dX, codes, scales = ctx.upload(host), ctx.empty((n, F.runs(k)), np.uint8), ctx.empty(scale.shape, np.float32)
        ctx.fp8_quantize(R.TYPES[t], TRANS, block, k, n, dX.ptr + 2 * first, n + pad, codes, F.runs(k), scales, scale.shape[1])
        got = codes.to_host()
        assert np.array_equal(scales.to_host(), scale), (pad, first)
        assert np.array_equal(np.where(got == 0x80, 0, got), code), (pad, first)
        for d in (dX, codes, scales):
            d.free()
