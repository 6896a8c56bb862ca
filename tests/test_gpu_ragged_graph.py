"""Grouped and 4-bit products in a captured graph: the workspace that the graph was captured with (aligned copies, the
sums of tiles cut along k) stays its own when later calls of the context need a larger one. Every replay gives the eager
result, bit for bit."""
import ctypes

import numpy as np
import pytest

from tests import ragged as R
from tests.test_gpu_ragged_large import values16
from wgblas_amd import NO_TRANS, TRANS

pytestmark = pytest.mark.gpu


def test_replays_after_the_workspace_grew():
    from wgblas_amd import Context

    hip = ctypes.CDLL("libamdhip64.so")

    def check(status):
        assert status == 0, f"HIP status {status}"

    rng = np.random.default_rng(1)
    bf16 = R.TYPES["bf16"]
    # k odd: both operands move to the workspace; 8 tiles of 256 past a round, cut along k: their sums are there too
    m, k, sizes = 2045, 2101, [8000, 300]
    n, off = sum(sizes), R.boundaries(sizes)
    with Context(0) as c:
        stream = ctypes.c_void_p(c.stream)
        A, B, x4 = (c.upload(values16(rng, s, "bf16")) for s in ((2, m, k), (n, k), (n, 2304)))
        offsets, C, W = c.upload(off), c.empty((n, m), np.float32), c.empty((2, 2048, k), np.float32)
        codes, scales = c.empty((n, 1152), np.uint8), c.empty((n, 72), np.uint8)

        def products():
            c.gemm_grouped(bf16, TRANS, 2, m, n, k, 1.0, A, k, m * k, B, k, offsets, 0.0, C, m, R.TYPES["f32"])
            c.mxfp4_quantize(bf16, NO_TRANS, 2304, n, x4, 2304, codes, scales, 2304)
            c.gemm_grouped_k(bf16, 2, k, 2048, n, 1.0, B, k, x4, 2304, offsets, 0.0, W, k, 2048 * k, R.TYPES["f32"])

        products()
        c.synchronize()
        graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
        check(hip.hipStreamBeginCapture(stream, 1))  # thread-local mode
        try:
            products()
        finally:
            check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        check(hip.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, ctypes.c_size_t(0)))
        for replay in range(4):
            if replay == 1:  # needs a workspace about three times as large
                big, out = c.upload(values16(rng, (6001, 6001), "bf16")), c.empty((6001, 6001), np.float32)
                one = c.upload(np.array([0, 6001], np.int64))
                c.gemm_grouped(bf16, TRANS, 1, 6001, 6001, 6001, 1.0, big, 6001, 6001 * 6001, big, 6001, one, 0.0, out, 6001,
                               R.TYPES["f32"])
            c.h2d(B.ptr, values16(rng, (n, k), "bf16"))
            products()
            c.synchronize()
            eager = [buf.to_host() for buf in (C, W, codes, scales)]
            for buf in (C, W):
                c.h2d(buf.ptr, np.full(buf.shape, np.nan, np.float32))
            check(hip.hipGraphLaunch(executable, stream))
            c.synchronize()
            for buf, want in zip((C, W, codes, scales), eager):
                assert (buf.to_host().view(np.uint8) == want.view(np.uint8)).all(), replay
        check(hip.hipGraphExecDestroy(executable))
        check(hip.hipGraphDestroy(graph))
