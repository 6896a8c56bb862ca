"""MXFP4: conversion bit for bit against the format's definition in float64,
products against float64 products of the values the codes stand for."""
import numpy as np
import pytest

from tests import ragged as R
from wgblas_amd import NO_TRANS, TRANS, WgblasError

pytestmark = pytest.mark.gpu

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def runs(k):
    return (k + 127) // 128 * 128


def quantize(x):
    """The definition: x (n, k) float64 -> codes (n, runs(k)) 0..15 and scale bytes (n, runs(k) / 32)."""
    n, k = x.shape
    full = np.zeros((n, runs(k)))
    full[:, :k] = x
    blocks = full.reshape(n, -1, 32)
    top = np.abs(blocks).max(axis=2)
    bad = ~np.isfinite(blocks).all(axis=2)
    e = np.where(bad | (top == 0), 0, np.frexp(np.where(bad, 1.0, top))[1] - 1) - 2
    byte = np.where(bad, 255, np.where(top == 0, 0, np.maximum(e + 127, 0)))
    v = np.where(bad[:, :, None], 0.0, blocks) * np.exp2(127.0 - np.minimum(byte, 254))[:, :, None]
    dist = np.abs(np.abs(v)[..., None] - LEVELS)
    near = dist.min(axis=-1, keepdims=True)
    # of two equally near codes the even one
    order = np.where(dist == near, np.arange(8) % 2, 2)
    code = order.argmin(axis=-1) + 8 * np.signbit(v)
    code = np.where(bad[:, :, None], 0, code)
    return code.reshape(n, -1).astype(np.uint8), byte.astype(np.uint8)


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def values(code, byte):
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127.0))
    return v * np.repeat(s, 32, axis=1)


def to_device(ctx, code, byte, ld):
    """Codes and scales with leading dimension ld; what is past the last run of 128 is junk no call may read."""
    n = code.shape[0]
    c = np.full((n, ld // 2), 0x77, np.uint8)
    s = np.full((n, ld // 32), 0xFF, np.uint8)
    c[:, :code.shape[1] // 2] = pack(code)
    s[:, :byte.shape[1]] = byte
    return ctx.upload(c), ctx.upload(s)


def inputs(kind, rng, n, k, t):
    if kind == "normal":
        x = rng.standard_normal((n, k))
    elif kind == "wide":  # blocks of very different sizes, outliers in them
        x = rng.standard_normal((n, k)) * np.exp2(rng.integers(-20, 12, (n, 1 + (k - 1) // 32)).repeat(32, 1)[:, :k])
        x[rng.random((n, k)) < 0.02] *= 100.0 if t != "f16" else 4.0
    elif kind == "ties":  # every midpoint between codes, both signs, each in blocks of every scale
        mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        x = np.where(rng.random((n, k)) < 0.5, -1, 1) * rng.choice(mid, (n, k))
        x = x * np.exp2(rng.integers(-8, 8, (n, 1)))
    elif kind == "small":  # near and below the smallest normal numbers
        low = {"f32": -149, "f16": -24, "bf16": -133}[t]
        x = rng.integers(-9, 10, (n, k)) * np.exp2(rng.integers(low, low + 12, (n, 1)).astype(np.float64))
    elif kind == "large":
        top = {"f32": 3.4e38, "f16": 65504.0, "bf16": 3.38e38}[t]
        x = rng.uniform(-1, 1, (n, k)) * top
    else:  # special
        x = rng.standard_normal((n, k))
        x[rng.random((n, k)) < 0.01] = np.inf
        x[rng.random((n, k)) < 0.01] = np.nan
        x[rng.random((n, k)) < 0.01] = -np.inf
        x[::3] = 0.0
        x[1::3] = -0.0
    return x


@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "small", "large", "special"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("n,k,pad", [(1, 1, 0), (1, 32, 0), (3, 33, 1), (17, 257, 2), (130, 128, 0), (5, 1000, 3),
                                     (257, 96, 1), (64, 640, 8)])
def test_conversion_is_exact(ctx, kind, t, trans, n, k, pad):
    rng = np.random.default_rng(k + n)
    with np.errstate(over="ignore"):
        x = inputs(kind, rng, n, k, t)
        stored = R.encode(x, t)
    x = R.decode(stored, t)
    rows = stored.T if trans == TRANS else stored
    host = R.encode(np.full((rows.shape[0], rows.shape[1] + pad), np.nan), t)
    host[:, :rows.shape[1]] = rows
    ld = runs(k) + (128 if pad else 0)
    codes, scales = ctx.upload(np.full((n, ld // 2), 0xAB, np.uint8)), ctx.upload(np.full((n, ld // 32), 0xCD, np.uint8))
    dX = ctx.upload(host)
    ctx.mxfp4_quantize(R.TYPES[t], trans, k, n, dX, host.shape[1], codes, scales, ld)
    code, byte = quantize(x)
    got_c, got_s = codes.to_host(), scales.to_host()
    assert np.array_equal(got_s[:, :byte.shape[1]], byte)
    assert np.array_equal(got_c[:, :code.shape[1] // 2], pack(code))
    # nothing past the last run of 128 is written
    assert (got_c[:, code.shape[1] // 2:] == 0xAB).all() and (got_s[:, byte.shape[1]:] == 0xCD).all()
    want = values(code, byte)[:, :k]
    for out in ("f32", "f16", "bf16"):
        back = ctx.upload(R.encode(np.full((n, k + pad), 7.0), out))
        ctx.mxfp4_dequantize(R.TYPES[out], k, n, codes, scales, ld, back, k + pad)
        got = back.to_host()
        with np.errstate(over="ignore"):
            exact = R.decode(R.encode(want, out), out)
        assert np.array_equal(R.decode(got[:, :k], out), exact, equal_nan=True), out
        assert (R.decode(got[:, k:], out) == 7.0).all()
        back.free()
    for d in (dX, codes, scales):
        d.free()


def test_dequantize_every_code_and_scale(ctx):
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 8))  # a run of 128 codes a column
    byte = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 4, axis=1)
    c, s = to_device(ctx, code, byte, 128)
    out = ctx.empty((256, 128), np.float32)
    ctx.mxfp4_dequantize(R.TYPES["f32"], 128, 256, c, s, 128, out, 128)
    with np.errstate(over="ignore"):
        assert np.array_equal(out.to_host(), values(code, byte).astype(np.float32), equal_nan=True)


def random_packed(rng, n, k, spread=6):
    code = np.zeros((n, runs(k)), np.uint8)
    code[:, :k] = rng.integers(0, 16, (n, k))
    byte = np.zeros((n, runs(k) // 32), np.uint8)
    used = (k + 31) // 32
    byte[:, :used] = rng.integers(127 - spread, 127 + spread, (n, used))
    return code, byte


def run_product(ctx, ct, m, k, sizes, grouped=True, alpha=1.0, beta=0.0, pads=(0, 0, 0), spare=0, seed=0):
    rng = np.random.default_rng(seed)
    off = R.boundaries(sizes)
    n, groups = int(off[-1]) + spare, len(sizes)
    lda, ldb, ldc = max(128, runs(k)) + 128 * pads[0], max(128, runs(k)) + 128 * pads[1], m + pads[2]
    ca, sa = random_packed(rng, groups * m, k)
    cb, sb = random_packed(rng, n, k)
    if spare:
        sb[n - spare:] = 255
    C0 = R.encode(np.full((n, ldc), np.nan) if beta == 0.0 else rng.standard_normal((n, ldc)), ct)
    dA, dSA = to_device(ctx, ca, sa, lda)
    dB, dSB = to_device(ctx, cb, sb, ldb)
    dC, dO = ctx.upload(C0), ctx.upload(off)
    if grouped:
        ctx.mxfp4_gemm_grouped(groups, m, n, k, alpha, dA, dSA, lda, m * lda, dB, dSB, ldb, dO, beta, dC, ldc, R.TYPES[ct])
    else:
        ctx.mxfp4_gemm(m, n, k, alpha, dA, dSA, lda, dB, dSB, ldb, beta, dC, ldc, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dSA, dB, dSB, dC, dO):
        d.free()
    A, B = values(ca, sa)[:, :k].reshape(groups, m, k), values(cb, sb)[:, :k]
    C64 = R.decode(C0, ct)[:, :m]
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if lo < hi:
            exact, absdot = B[lo:hi] @ A[g].T, np.abs(B[lo:hi]) @ np.abs(A[g]).T
            R.assert_product(R.decode(got[lo:hi, :m], ct), exact, absdot, k, ct, alpha, beta, C64[lo:hi])
    es = got.dtype.itemsize
    raw, raw0 = got.view(np.uint8).reshape(n, -1), C0.view(np.uint8).reshape(n, -1)
    assert np.array_equal(raw[:, m * es:], raw0[:, m * es:])
    assert np.array_equal(raw[int(off[-1]):], raw0[int(off[-1]):])
    return got


GROUPS = {
    "empty_ends": [0, 7, 0, 0, 130, 1, 0],
    "skewed": [3, 0, 300, 1, 17],
    "many": [1, 2, 0, 5] * 20,
    "long": [700, 515],
    "tiny": [1, 1, 2, 1, 0, 1, 3, 1],
}


@pytest.mark.parametrize("ct", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes", sorted(GROUPS))
@pytest.mark.parametrize("m,k", [(136, 200), (1, 1), (257, 128), (40, 1111), (128, 512), (300, 320)])
def test_grouped_products(ctx, ct, sizes, m, k):
    run_product(ctx, ct, m, k, GROUPS[sizes], seed=m + k, spare=3)


@pytest.mark.parametrize("ct", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 16, 17, 33, 100, 300, 513])
@pytest.mark.parametrize("m,k", [(1, 1), (264, 256), (1000, 777), (520, 2048), (17, 4096)])
def test_products(ctx, ct, n, m, k):
    run_product(ctx, ct, m, k, [n], grouped=False, seed=n + m)


@pytest.mark.parametrize("alpha,beta", [(1.5, 0.5), (-0.25, 1.0), (0.0, 0.5), (0.0, 0.0)])
@pytest.mark.parametrize("sizes", ["skewed", "tiny", "long"])
def test_alpha_beta_and_strides(ctx, alpha, beta, sizes):
    run_product(ctx, "f32", 200, 300, GROUPS[sizes], alpha=alpha, beta=beta, pads=(1, 2, 3))
    run_product(ctx, "bf16", 200, 300, [sum(GROUPS[sizes])], grouped=False, alpha=alpha, beta=beta, pads=(1, 2, 3))
    run_product(ctx, "bf16", 30, 0, GROUPS[sizes], alpha=alpha, beta=beta)


def test_a_block_that_is_nan_shows_in_its_products_only(ctx):
    rng = np.random.default_rng(3)
    for n in (5, 60, 300):
        m, k = 150, 400
        ca, sa = random_packed(rng, m, k)
        cb, sb = random_packed(rng, n, k)
        sa[7, 3], sb[2, 12] = 255, 255
        dA, dSA = to_device(ctx, ca, sa, runs(k))
        dB, dSB = to_device(ctx, cb, sb, runs(k))
        dC = ctx.upload(np.zeros((n, m), np.float32))
        ctx.mxfp4_gemm(m, n, k, 1.0, dA, dSA, runs(k), dB, dSB, runs(k), 0.0, dC, m, R.TYPES["f32"])
        want = np.ones((n, m), bool)
        want[2], want[:, 7] = False, False
        assert np.array_equal(np.isfinite(dC.to_host()), want)


def test_scales_far_from_one(ctx):
    """Scales whose product leaves fp32's range on the way but not in the result's."""
    rng = np.random.default_rng(4)
    m, n, k = 40, 20, 256
    for ea, eb in ((1, 253), (253, 1), (0, 254), (60, 190)):
        ca, sa = random_packed(rng, m, k)
        cb, sb = random_packed(rng, n, k)
        sa[:], sb[:] = ea, eb
        dA, dSA = to_device(ctx, ca, sa, k)
        dB, dSB = to_device(ctx, cb, sb, k)
        dC = ctx.upload(np.zeros((n, m), np.float32))
        ctx.mxfp4_gemm(m, n, k, 1.0, dA, dSA, k, dB, dSB, k, 0.0, dC, m, R.TYPES["f32"])
        A, B = values(ca, sa), values(cb, sb)
        R.assert_product(dC.to_host().astype(np.float64), B @ A.T, np.abs(B) @ np.abs(A).T, k, "f32")


def test_scales_past_32_bits(ctx):
    """Expert weights 2^33 elements apart: codes 4 GiB and scales 256 MiB apart."""
    rng = np.random.default_rng(5)
    m, k, sizes, stride = 24, 256, [5, 40], 1 << 33
    off, n = R.boundaries(sizes), sum(sizes)
    ca, sa = random_packed(rng, 2 * m, k)
    cb, sb = random_packed(rng, n, k)
    dA, dSA = ctx.empty(stride // 2 + m * k // 2, np.uint8), ctx.empty(stride // 32 + m * k // 32, np.uint8)
    for g in range(2):
        ctx.h2d(dA.offset(g * stride // 2), pack(ca[g * m:(g + 1) * m]))
        ctx.h2d(dSA.offset(g * stride // 32), sa[g * m:(g + 1) * m])
    dB, dSB = to_device(ctx, cb, sb, k)
    dC = ctx.upload(np.zeros((n, m), np.float32))
    ctx.mxfp4_gemm_grouped(2, m, n, k, 1.0, dA, dSA, k, stride, dB, dSB, k, ctx.upload(off), 0.0, dC, m, R.TYPES["f32"])
    got = dC.to_host().astype(np.float64)
    dA.free()
    dSA.free()
    A, B = values(ca, sa).reshape(2, m, k), values(cb, sb)
    for g in range(2):
        x = B[off[g]:off[g + 1]]
        R.assert_product(got[off[g]:off[g + 1]], x @ A[g].T, np.abs(x) @ np.abs(A[g]).T, k, "f32")


def test_results_are_the_same_every_time(ctx):
    for sizes in ("tiny", "skewed", "long"):
        first = run_product(ctx, "f32", 300, 520, GROUPS[sizes], seed=2)
        assert np.array_equal(first, run_product(ctx, "f32", 300, 520, GROUPS[sizes], seed=2))


def test_refusals(ctx):
    d = ctx.upload(np.zeros(1 << 14, np.uint8))
    o = ctx.upload(np.array([0, 4], np.int64))

    def quant(type=0, trans=0, k=64, n=4, X=d, ldx=64, codes=d, scales=d, ld=128):
        ctx.mxfp4_quantize(type, trans, k, n, X, ldx, codes, scales, ld)

    def dequant(type=0, k=64, n=4, codes=d, scales=d, ld=128, X=d, ldx=64):
        ctx.mxfp4_dequantize(type, k, n, codes, scales, ld, X, ldx)

    def gemm(m=4, n=4, k=64, A=d, sA=d, lda=128, B=d, sB=d, ldb=128, C=d, ldc=4, ctype=0):
        ctx.mxfp4_gemm(m, n, k, 1.0, A, sA, lda, B, sB, ldb, 0.0, C, ldc, ctype)

    def grouped(groups=1, m=4, n=4, k=64, A=d, sA=d, lda=128, strideA=512, B=d, sB=d, ldb=128, off=o, C=d, ldc=4, ctype=0):
        ctx.mxfp4_gemm_grouped(groups, m, n, k, 1.0, A, sA, lda, strideA, B, sB, ldb, off, 0.0, C, ldc, ctype)

    convert = [dict(type=3), dict(k=-1), dict(n=-1), dict(X=None), dict(ldx=63), dict(codes=None), dict(scales=None),
               dict(ld=64), dict(ld=160), dict(k=129, ldx=129), dict(codes=d.offset(8)), dict(scales=d.offset(2)),
               dict(ld=(1 << 23) + 128), dict(n=1 << 31)]
    both = [dict(m=-1), dict(n=-1), dict(k=-1), dict(k=129), dict(lda=64), dict(ldb=192), dict(ldc=3), dict(ctype=3),
            dict(A=None), dict(sA=None), dict(B=None), dict(sB=None), dict(C=None), dict(A=d.offset(4)),
            dict(sB=d.offset(1)), dict(m=1 << 31, ldc=1 << 31)]
    cases = [(quant, a) for a in convert + [dict(trans=2), dict(trans=1, n=65)]] + [(dequant, a) for a in convert]
    cases += [(gemm, a) for a in both] + [(grouped, a) for a in both + [
        dict(groups=-1), dict(groups=2, strideA=384), dict(strideA=100), dict(strideA=-128), dict(off=None),
        dict(groups=(1 << 20) + 1)]]
    for fn, args in cases:
        with pytest.raises(WgblasError, match="status -1"):
            fn(**args)
    quant(n=0, X=None, codes=None, scales=None)
    dequant(k=0, X=None, codes=None, scales=None)
    gemm(m=0, A=None, sA=None, B=None, sB=None, C=None)
    grouped(groups=0, A=None, sA=None, B=None, sB=None, C=None, off=None)
    ctx.synchronize()


@pytest.mark.parametrize("k", [(1 << 23) + 1, 1 << 31, (1 << 63) - 100, (1 << 63) - 1])
def test_refuses_k_too_large_to_round_up(ctx, k):
    d = ctx.upload(np.zeros(1 << 10, np.uint8))
    o = ctx.upload(np.array([0, 1], np.int64))
    ld = 1 << 23
    for call in (lambda: ctx.mxfp4_quantize(R.TYPES["f32"], TRANS, k, 1, d, 1, d, d, ld),
                 lambda: ctx.mxfp4_quantize(R.TYPES["f32"], NO_TRANS, k, 1, d, k, d, d, ld),
                 lambda: ctx.mxfp4_dequantize(R.TYPES["f32"], k, 1, d, d, ld, d, k),
                 lambda: ctx.mxfp4_gemm(1, 1, k, 1.0, d, d, ld, d, d, ld, 0.0, d, 1, R.TYPES["f32"]),
                 lambda: ctx.mxfp4_gemm_grouped(1, 1, 1, k, 1.0, d, d, ld, ld, d, d, ld, o, 0.0, d, 1, R.TYPES["f32"])):
        with pytest.raises(WgblasError, match="status -1"):
            call()
