"""FP8 products on the 256 x 256 kernel, with and without a rest that is cut along k: cut rows, columns and k, last tiles of
each number of used column blocks, several tiles a block, empty groups, C's own terms, all of C's types. A sample of rows
over all columns against float64 products, within tests/test_gpu_fp8.py's bounds, and the same bits from call to call. That
the cases take these kernels is checked on the CPU (tests/test_fp8_tiles_host_side.py)."""
import ctypes

import numpy as np
import pytest

from tests import fp8 as F
from tests import ragged as R
from tests.test_gpu_fp8 import DROPPED
from wgblas_amd import NO_TRANS, TRANS

pytestmark = pytest.mark.gpu

# columns of the groups (one: a dense product), m, k, whether the rest is cut along k
CASES = [([3847], 4001, 1100, False),  # one round; k ends inside a k-tile
         ([4096], 4090, 129, False),  # two k-tiles, one value in the second
         ([3847], 4001, 100, False),  # one k-tile
         ([12000], 4090, 140, False),  # three tiles a block
         ([7900], 2040, 1150, False),
         ([63, 65, 127, 129, 191, 193, 255, 2023], 4090, 1100, False),  # 1 to 4 used column blocks
         ([3000, 0, 1, 2555, 1944], 4090, 700, False),  # two rounds
         ([1300, 0, 1, 2047, 300, 5000], 2040, 6200, True),
         ([4150], 4000, 6300, True),
         ([2800], 6240, 6200, True)]
EXTRA = 3  # columns of no group behind those of groups
# layout, block of A, type of C, alpha, beta, padding
FORMS = [(TRANS, 128, "f32", -0.75, 0.5, 3), (TRANS, 128, "f16", 1.0, 0.0, 0), (TRANS, 128, "bf16", 0.5, -1.0, 1),
         (TRANS, 1, "bf16", 1.0, 0.0, 0), (TRANS, 1, "f16", 0.5, 0.25, 2), (NO_TRANS, 128, "f32", 1.0, 0.0, 0),
         (NO_TRANS, 128, "bf16", -0.5, 0.75, 2), (NO_TRANS, 128, "f16", 0.5, 0.0, 1)]
CALLS = [(*case, *form) for case in CASES for form in (FORMS[::3] + FORMS[2:6:3] if case[3] else FORMS)]


def codes_of(rng, columns, length):
    """(columns, whole runs of 128) codes of magnitudes from 2^-3 to 8, zeros past `length`."""
    c = rng.integers(0, 256, (columns, F.runs(length)), dtype=np.uint8)
    c = (c & 0x87) | (((c >> 3) % 6 + 4) << 3)
    c[:, length:] = 0
    return c.astype(np.uint8)


def scales_of(rng, columns, length, block, lds):
    s = np.full((F.runs(length) // 128, lds), np.nan, np.float32)
    s[:, :(columns + block - 1) // block] = rng.uniform(0.1, 0.4, (len(s), (columns + block - 1) // block))
    return s


def sample(rng, m):
    edges = [r for r in (0, 15, 16, 127, 128, 255, 256, m // 256 * 256 - 1, m // 256 * 256, m - 1) if 0 <= r < m]
    return np.unique(np.concatenate([edges, rng.choice(m, 50, replace=False)]))


@pytest.mark.parametrize("sizes,m,k,cut,trans,block,ct,alpha,beta,pad", CALLS)
def test_product(ctx, sizes, m, k, cut, trans, block, ct, alpha, beta, pad):
    rng = np.random.default_rng(m + k)
    groups, off, extra = len(sizes), R.boundaries(sizes), 0 if len(sizes) == 1 else EXTRA
    n = int(off[-1]) + extra
    length, columns = (m, k) if trans == NO_TRANS else (k, m)
    lda, ldsa, ldb, ldsb, ldc = F.runs(length), (columns + block - 1) // block + pad, F.runs(k), n + pad, m + pad
    A = np.stack([codes_of(rng, columns, length) for _ in range(groups)])
    SA = np.stack([scales_of(rng, columns, length, block, ldsa) for _ in range(groups)])
    B, SB = codes_of(rng, n, k), scales_of(rng, n, k, 1, ldsb)
    C0 = R.encode(rng.standard_normal((n, ldc)) if beta else np.full((n, ldc), np.nan), ct)
    dA, dSA, dB, dSB, d_off = (ctx.upload(x) for x in (A, SA, B, SB, off))
    out = []
    for _ in range(2):
        dC = ctx.upload(C0)
        if groups == 1:
            ctx.fp8_gemm(trans, m, n, k, alpha, dA, lda, block, dSA, ldsa, dB, ldb, dSB, ldsb, beta, dC, ldc, R.TYPES[ct])
        else:
            ctx.fp8_gemm_grouped(trans, groups, m, n, k, alpha, dA, lda, columns * lda, block, dSA, ldsa, SA[0].size, dB, ldb, dSB,
                                 ldsb, d_off, beta, dC, ldc, R.TYPES[ct])
        out.append(dC.to_host())
        dC.free()
    for d in (dA, dSA, dB, dSB, d_off):
        d.free()
    got = out[0]
    assert np.array_equal(got.view(np.uint8), out[1].view(np.uint8))
    # columns of no group and the padding are left as they were
    assert np.array_equal(got[off[-1]:].view(np.uint8), C0[off[-1]:].view(np.uint8))
    assert got[:, m:].tobytes() == C0[:, m:].tobytes()
    rows = sample(rng, m)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        if trans == TRANS:
            scale = SA[g][:, rows // block].T.repeat(128, axis=1)[:, :k]
            W = (F.VALUES[A[g][rows, :k]] * scale).T
        else:
            scale = SA[g][rows // 128][:, np.arange(k) // 128].T
            W = F.VALUES[A[g][:, rows]] * scale
        x = F.VALUES[B[lo:hi, :k]] * SB[:, lo:hi].T.astype(np.float64).repeat(128, axis=1)[:, :k]
        R.assert_product(R.decode(got[lo:hi, rows], ct), x @ W, np.abs(x) @ np.abs(W), k + DROPPED[ct] * 2.0 ** 23, ct, alpha, beta,
                         R.decode(C0[lo:hi, rows], ct))


CAPTURED = ([4150], 4000, 6300, True)  # its rest is cut along k: sums in the workspace


@pytest.mark.parametrize("trans,block", [(TRANS, 128), (TRANS, 1), (NO_TRANS, 128)])
def test_replays_with_sums_in_the_workspace(trans, block):
    """A captured product's partial sums' workspace stays its own when a later call grows the context's."""
    from wgblas_amd import BF16, Context

    hip = ctypes.CDLL("libamdhip64.so")

    def check(status):
        assert status == 0, f"HIP status {status}"

    (n,), m, k, _ = CAPTURED
    rng = np.random.default_rng(4)
    length, columns = (m, k) if trans == NO_TRANS else (k, m)
    lda, cols, ldb = F.runs(length), (columns + block - 1) // block, F.runs(k)
    with Context(0) as c:
        A, SA = c.upload(codes_of(rng, columns, length)), c.upload(scales_of(rng, columns, length, block, cols))
        B, SB, C = c.empty((n, ldb), np.uint8), c.empty((ldb // 128, n), np.float32), c.empty((n, m), np.uint16)
        X = c.empty((n, k), np.float32)

        def product():
            c.fp8_quantize(R.TYPES["f32"], NO_TRANS, 1, k, n, X, k, B, ldb, SB, n)
            c.fp8_gemm(trans, m, n, k, 1.0, A, lda, block, SA, cols, B, ldb, SB, n, 0.0, C, m, BF16)

        c.fill_normal(X, 2)
        product()
        c.synchronize()
        stream = ctypes.c_void_p(c.stream)
        graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
        check(hip.hipStreamBeginCapture(stream, 1))  # thread-local mode
        try:
            product()
        finally:
            check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        check(hip.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, ctypes.c_size_t(0)))
        for replay in range(4):
            if replay == 1:  # both operands moved to a workspace of 150 MB
                big, out = c.upload(R.encode(rng.standard_normal((6001, 6001)), "bf16")), c.empty((6001, 6001), np.float32)
                one = c.upload(np.array([0, 6001], np.int64))
                c.gemm_grouped(BF16, TRANS, 1, 6001, 6001, 6001, 1.0, big, 6001, 6001 * 6001, big, 6001, one, 0.0, out, 6001,
                               R.TYPES["f32"])
            c.fill_normal(X, 10 + replay)
            product()
            eager = C.to_host()
            c.h2d(C.ptr, np.zeros((n, m), np.uint16))
            check(hip.hipGraphLaunch(executable, stream))
            c.synchronize()
            assert np.array_equal(C.to_host(), eager), replay
        check(hip.hipGraphExecDestroy(executable))
        check(hip.hipGraphDestroy(graph))
