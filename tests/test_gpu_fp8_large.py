"""FP8 products of sizes that take the large tiles: ragged groups, cut rows, columns and k, rests shared along k, and C's
own terms; against the float64 products of tests/test_gpu_fp8.py's bounds."""
import numpy as np
import pytest

from tests import fp8 as F
from tests import ragged as R
from tests.test_gpu_fp8 import FORMS, check_product, operand
from wgblas_amd import TRANS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trans,block", FORMS)
@pytest.mark.parametrize("ct", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(2048, 2048, 512), (4000, 2077, 400), (2305, 4099, 129)])
def test_dense(ctx, trans, block, ct, m, n, k):
    check_product(ctx, trans, block, ct, [n], m, k, pad=1, dense=True)


@pytest.mark.parametrize("trans,block", FORMS)
@pytest.mark.parametrize("ct", ["f16", "f32"])
@pytest.mark.parametrize("sizes,m,k", [([1100, 0, 300, 17, 1, 900], 2100, 520), ([257] * 9, 2048, 256),
                                       ([63, 65, 127, 129, 191, 193, 255, 2000], 1800, 300)])
def test_grouped(ctx, trans, block, ct, sizes, m, k):
    """Last tiles of a group with each number of used column blocks, groups smaller than a tile, an empty one."""
    check_product(ctx, trans, block, ct, sizes, m, k, pad=2, extra=5)


@pytest.mark.parametrize("trans,block", FORMS)
@pytest.mark.parametrize("ct", ["f32", "bf16"])
def test_rest_along_k(ctx, trans, block, ct):
    """264 tiles of 256 x 256: eight past a round, whose k is shared."""
    check_product(ctx, trans, block, ct, [2816], 6144, 2000, dense=True)


@pytest.mark.parametrize("trans,block", FORMS)
@pytest.mark.parametrize("ct", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes,m,k", [([1500, 700], 2051, 260), ([2816], 6100, 640)])
def test_alpha_and_beta(ctx, trans, block, ct, sizes, m, k):
    check_product(ctx, trans, block, ct, sizes, m, k, alpha=-0.5, beta=0.75)


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("ct", ["f32", "bf16"])
@pytest.mark.parametrize("n,beta", [(1, 0.5), (5, 0.0), (16, -1.0), (17, 0.25), (32, 0.0)])
@pytest.mark.parametrize("m,k", [(100, 3000), (2000, 640), (4101, 1100)])
def test_few_columns(ctx, block, ct, n, beta, m, k):
    check_product(ctx, TRANS, block, ct, [n], m, k, pad=1, alpha=1.25, beta=beta, dense=True)


@pytest.mark.parametrize("trans,block", FORMS)
@pytest.mark.parametrize("m,n,k", [(300, 40, 1000), (2048, 2100, 700)])
def test_the_same_bits_again(ctx, trans, block, m, n, k):
    """Sums have one order: a second call, and one of another context, give the same bits."""
    from wgblas_amd import Context

    rng = np.random.default_rng(3)
    (dA, dSA), lda, ldsa, _, _, _ = operand(rng, ctx, trans, block, 1, m, k, 0)
    codes, scales, _ = F.random_matrix(rng, n, k, 1)
    dB, dSB = F.to_device(ctx, codes, scales, F.runs(k), n)

    def run(c):
        dC = c.empty((n, m), np.float32)
        c.fp8_gemm(trans, m, n, k, 1.0, dA, lda, block, dSA, ldsa, dB, F.runs(k), dSB, n, 0.0, dC, m, R.TYPES["f32"])
        return dC.to_host().view(np.uint32)

    first = run(ctx)
    ctx.synchronize()
    with Context(0) as other:
        assert np.array_equal(first, run(other))
    assert np.array_equal(first, run(ctx))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("trans", [0, TRANS])
@pytest.mark.parametrize("block", [1, 128])
def test_conversion_past_the_caches(ctx, t, trans, block):
    """More than 32 MB of values, odd rows and leading dimensions: bit for bit as the definition."""
    n, k, pad = 4200, 4100, 3
    rng = np.random.default_rng(9)
    stored = R.encode(rng.standard_normal((n, k)), t)
    rows = stored.T if trans == TRANS else stored
    host = np.zeros((rows.shape[0], rows.shape[1] + pad), stored.dtype)
    host[:, :rows.shape[1]] = rows
    code, scale = F.quantize(R.decode(stored, t), block)
    dX, ld, lds = ctx.upload(host), F.runs(k), scale.shape[1]
    codes, scales = ctx.empty((n, ld), np.uint8), ctx.empty(scale.shape, np.float32)
    ctx.fp8_quantize(R.TYPES[t], trans, block, k, n, dX, host.shape[1], codes, ld, scales, lds)
    got = codes.to_host()
    assert np.array_equal(scales.to_host(), scale)
    assert np.array_equal(np.where(got == 0x80, 0, got), np.where(code == 0x80, 0, code))
    want = R.encode(F.values(code, scale, block)[:, :k], t)
    for odd in (0, 1):  # at whole dwords and between them
        ldx = k + pad + odd
        back = ctx.upload(np.zeros((n, ldx), want.dtype))
        ctx.fp8_dequantize(R.TYPES[t], block, k, n, codes, ld, scales, lds, back, ldx)
        out = back.to_host()
        assert np.array_equal(R.decode(out[:, :k], t), R.decode(want, t)) and not out[:, k:].any()
        back.free()
    for d in (dX, codes, scales):
        d.free()


@pytest.mark.parametrize("trans,block", FORMS)
def test_replays_with_sums_in_the_workspace(trans, block):
    """A captured product whose rest is cut along k: its partial sums' workspace stays its own when a later call grows it."""
    import ctypes

    from wgblas_amd import BF16, NO_TRANS, Context

    hip = ctypes.CDLL("libamdhip64.so")

    def check(status):
        assert status == 0, f"HIP status {status}"

    rng = np.random.default_rng(4)
    m, n, k = 6144, 2816, 640
    rows, cols = (k, m) if trans == TRANS else (m, k)
    with Context(0) as c:
        W, X = c.empty((cols, rows), np.float32), c.empty((n, k), np.float32)
        c.fill_normal(W, 1)
        A, SA = c.empty((cols, rows), np.uint8), c.empty((rows // 128, (cols + block - 1) // block), np.float32)
        c.fp8_quantize(R.TYPES["f32"], NO_TRANS, block, rows, cols, W, rows, A, rows, SA, SA.shape[1])
        B, SB, C = c.empty((n, k), np.uint8), c.empty((k // 128, n), np.float32), c.empty((n, m), np.uint16)

        def product():
            c.fp8_quantize(R.TYPES["f32"], NO_TRANS, 1, k, n, X, k, B, k, SB, n)
            c.fp8_gemm(trans, m, n, k, 1.0, A, rows, block, SA, SA.shape[1], B, k, SB, n, 0.0, C, m, BF16)

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
