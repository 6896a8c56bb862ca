"""Routing, rows and 8-bit matrices whose columns lie farther apart than 32-bit offsets reach: the bits of the same calls on
dense matrices. Only the columns themselves are written or read of the large allocations."""
import numpy as np
import pytest

from tests import fp8 as F
from tests import ragged as R
from wgblas_amd import NO_TRANS, SOFTMAX, TRANS

pytestmark = pytest.mark.gpu

BF16, F32 = R.TYPES["bf16"], R.TYPES["f32"]
FAR = 1 << 26  # elements between columns: 70 of them pass 2^32


def columns(ctx, buffer, n, ld, rows, dtype):
    out = np.empty((n, rows), dtype)
    for j in range(n):
        ctx.d2h(out[j], buffer.ptr + j * ld * out.itemsize)
    return out


def test_rows_and_router(ctx):
    rng = np.random.default_rng(1)
    n, topk, d = 35, 2, 64
    rows = n * topk
    places = rng.permutation(rows).astype(np.int32).reshape(n, topk)
    w = rng.standard_normal((n, topk)).astype(np.float32)
    x = R.encode(rng.standard_normal((n, d)), "bf16")
    dX, dP, dW = ctx.upload(x), ctx.upload(places), ctx.upload(w)
    far, near = ctx.empty(rows * FAR, np.uint16), ctx.empty((rows, d), np.uint16)
    for y, ld in ((far, FAR), (near, d)):
        ctx.route_gather(BF16, d, n, topk, dX, d, dP, dW, y, ld)
    assert np.array_equal(columns(ctx, far, rows, FAR, d, np.uint16), near.to_host())
    out = []
    for y, ld in ((far, FAR), (near, d)):
        c, dw = ctx.empty((n, d), np.float32), ctx.empty((n, topk), np.float32)
        ctx.route_combine(BF16, d, n, topk, y, ld, dP, dW, 0.0, c, d, F32)
        out.append([c.to_host()])
        ctx.route_combine_grad(BF16, d, n, topk, dX, d, y, ld, dP, dW, y, ld, dw)
        out[-1].append(dw.to_host())
    assert all(np.array_equal(a, b) for a, b in zip(*out))
    assert np.array_equal(columns(ctx, far, rows, FAR, d, np.uint16), near.to_host())
    # 8 bits, along the contiguous axis
    codes = [ctx.empty((rows, 128), np.uint8) for _ in range(2)]
    scales = [ctx.empty((1, rows), np.float32) for _ in range(2)]
    for y, ld, c, s in ((far, FAR, codes[0], scales[0]), (near, d, codes[1], scales[1])):
        ctx.fp8_quantize(BF16, NO_TRANS, 1, d, rows, y, ld, c, 128, s, rows)
    assert np.array_equal(codes[0].to_host(), codes[1].to_host()) and np.array_equal(scales[0].to_host(), scales[1].to_host())
    ctx.fp8_dequantize(BF16, 1, d, rows, codes[0], 128, scales[0], rows, far, FAR)
    ctx.fp8_dequantize(BF16, 1, d, rows, codes[1], 128, scales[1], rows, near, d)
    assert np.array_equal(columns(ctx, far, rows, FAR, d, np.uint16), near.to_host())
    # and along the strided one: rows of k far apart
    codes = [ctx.empty((d, 128), np.uint8) for _ in range(2)]
    scales = [ctx.empty((1, d), np.float32) for _ in range(2)]
    for y, ld, c, s in ((far, FAR, codes[0], scales[0]), (near, d, codes[1], scales[1])):
        ctx.fp8_quantize(BF16, TRANS, 1, rows, d, y, ld, c, 128, s, d)
    assert np.array_equal(codes[0].to_host(), codes[1].to_host()) and np.array_equal(scales[0].to_host(), scales[1].to_host())
    # the router on those columns as logits
    ids = [ctx.empty((rows, 4), np.int32) for _ in range(2)]
    weights = [ctx.empty((rows, 4), np.float32) for _ in range(2)]
    dlogits = ctx.empty((rows, d), np.uint16)
    for y, ld, i, v in ((far, FAR, ids[0], weights[0]), (near, d, ids[1], weights[1])):
        ctx.route(BF16, SOFTMAX, d, rows, 4, y, ld, None, 1, 1, 1, 1, 1.0, i, v)
    assert np.array_equal(ids[0].to_host(), ids[1].to_host()) and np.array_equal(weights[0].to_host(), weights[1].to_host())
    ctx.route_grad(BF16, SOFTMAX, d, rows, 4, near, d, ids[1], 1, 1.0, weights[1], dlogits, d)
    ctx.route_grad(BF16, SOFTMAX, d, rows, 4, far, FAR, ids[0], 1, 1.0, weights[0], far, FAR)
    assert np.array_equal(columns(ctx, far, rows, FAR, d, np.uint16), dlogits.to_host())
    for b in (dX, dP, dW, far, near):
        b.free()


@pytest.mark.parametrize("ct", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k,ldb,ldc", [(300, 600, 256, 1 << 23, 300), (257, 70, 130, 256, FAR)])
def test_products(ctx, ct, m, n, k, ldb, ldc):
    rng = np.random.default_rng(2)
    ca, sa, _ = F.random_matrix(rng, m, k, 1)
    x = ctx.upload(R.encode(rng.standard_normal((n, k)), "bf16"))
    A, SA = F.to_device(ctx, ca, sa, F.runs(k), m)
    out = []
    for b, c in ((ldb, ldc), (F.runs(k), m)):
        B, SB, C = ctx.empty(n * b, np.uint8), ctx.empty((F.runs(k) // 128, n), np.float32), ctx.empty(n * c, R.STORE[ct])
        ctx.fp8_quantize(BF16, NO_TRANS, 1, k, n, x, k, B, b, SB, n)
        ctx.fp8_gemm(TRANS, m, n, k, 1.0, A, F.runs(k), 1, SA, m, B, b, SB, n, 0.0, C, c, R.TYPES[ct])
        out.append(columns(ctx, C, n, c, m, R.STORE[ct]))
        for v in (B, SB, C):
            v.free()
    assert np.array_equal(out[0].view(np.uint8), out[1].view(np.uint8))
    # A's columns far apart: what was B's matrix, read as rows of op(A)
    ids = []
    for a in (ldb, F.runs(k)):
        W, SW, C = ctx.empty(n * a, np.uint8), ctx.empty((F.runs(k) // 128, n), np.float32), ctx.empty((m, n), R.STORE[ct])
        ctx.fp8_quantize(BF16, NO_TRANS, 1, k, n, x, k, W, a, SW, n)
        ctx.fp8_gemm(TRANS, n, m, k, 1.0, W, a, 1, SW, n, A, F.runs(k), SA, m, 0.0, C, n, R.TYPES[ct])
        ids.append(C.to_host())
        for v in (W, SW, C):
            v.free()
    assert np.array_equal(ids[0].view(np.uint8), ids[1].view(np.uint8))
    for v in (x, A, SA):
        v.free()
