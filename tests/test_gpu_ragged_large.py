"""Grouped and 4-bit products at sizes that the small-tile kernels leave to the
256 x 256 tiles: whole rounds of tiles on a persistent launch, the rest as 128
x 128 tiles, more tiles than a block can list, more groups than lanes. All
columns of a sample of rows against float64 products."""
import numpy as np
import pytest

from tests import ragged as R
from tests.test_gpu_mxfp4 import pack, runs, values
from wgblas_amd import NO_TRANS, TRANS

pytestmark = pytest.mark.gpu


def sample(rng, rows, count=160):
    """Rows of every part of a tile, the first and the last among them."""
    edges = [r for b in range(0, rows, 128) for r in (b, b + 127) if r < rows][:80]
    return np.unique(np.concatenate([edges, [rows - 1], rng.integers(0, rows, count)])).astype(np.int64)


def values16(rng, shape, t):
    """Storage of small normals, quickly (float16 / float32 of one rounding)."""
    x = rng.standard_normal(shape, dtype=np.float32)
    if t == "bf16":
        return (x.view(np.uint32) >> 16).astype(np.uint16)
    return x.astype(R.STORE[t])


# m, k, sizes: 16 x 18 tiles of 256 (one round and a few), 33 x 18 (two rounds and a few), 8 x 40 (just over a round)
COLUMNS = [(4000, 778, [1300, 0, 1, 2047, 300, 77]), (8200, 520, [1300, 0, 1, 2047, 300, 77]),
           (2048, 1026, [256] * 20 + [1000, 3000, 1200]), (4096, 1024, [4096])]


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t,ct,beta", [("bf16", "bf16", 0.0), ("f16", "f32", 0.0), ("bf16", "f32", 0.5), ("f16", "f16", -0.5)])
@pytest.mark.parametrize("m,k,sizes", COLUMNS)
def test_columns(ctx, t, ct, beta, trans, m, k, sizes):
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups = int(off[-1]), len(sizes)
    A = values16(rng, (groups, m, k) if trans == TRANS else (groups, k, m), t)
    B = values16(rng, (n, k), t)
    C0 = R.encode(np.full((n, m), np.nan, np.float32), ct) if beta == 0.0 else values16(rng, (n, m), ct)
    dA, dB, dC, dO = ctx.upload(A), ctx.upload(B), ctx.upload(C0), ctx.upload(off)
    lda = A.shape[2]
    ctx.gemm_grouped(R.TYPES[t], trans, groups, m, n, k, 0.5, dA, lda, m * k, dB, k, dO, beta, dC, m, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    rows = sample(rng, m)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        W = R.decode(A[g, rows].T if trans == TRANS else A[g][:, rows], t)
        x = R.decode(B[lo:hi], t)
        R.assert_product(R.decode(got[lo:hi, rows], ct), x @ W, np.abs(x) @ np.abs(W), k, ct, 0.5, beta,
                         R.decode(C0[lo:hi, rows], ct))


@pytest.mark.parametrize("t,ct,beta", [("bf16", "f32", 0.0), ("f16", "f16", 0.0), ("bf16", "f32", 1.0)])
@pytest.mark.parametrize("m,n,sizes", [(2000, 1500, [1700, 0, 1, 900, 1313, 129]), (4096, 2048, [700, 64, 900, 0, 513, 1111]),
                                       (2056, 4104, [900, 1100, 3])])
def test_k(ctx, t, ct, beta, m, n, sizes):
    rng = np.random.default_rng(m + n)
    off = R.boundaries(sizes)
    k, groups = int(off[-1]), len(sizes)
    A, B = values16(rng, (k, m), t), values16(rng, (k, n), t)
    C0 = R.encode(np.full((groups, n, m), np.nan, np.float32), ct) if beta == 0.0 else values16(rng, (groups, n, m), ct)
    dA, dB, dC, dO = ctx.upload(A), ctx.upload(B), ctx.upload(C0), ctx.upload(off)
    ctx.gemm_grouped_k(R.TYPES[t], groups, m, n, k, 0.5, dA, m, dB, n, dO, beta, dC, m, n * m, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    rows = sample(rng, m)
    for g in range(groups):
        a, b = R.decode(A[off[g]:off[g + 1]][:, rows], t), R.decode(B[off[g]:off[g + 1]], t)
        R.assert_product(R.decode(got[g][:, rows], ct), b.T @ a, np.abs(b).T @ np.abs(a), sizes[g], ct, 0.5, beta,
                         R.decode(C0[g][:, rows], ct))


@pytest.mark.parametrize("ct", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("m,k,sizes", [(8200, 1504, [1300, 0, 1, 2047, 300, 77]), (4096, 1536, [4096]), (4100, 1408, [850] * 4),
                                       (8192, 640, [4000, 300]), (4100, 384, [10] * 20), (4100, 448, [25] * 20)])
def test_mxfp4(ctx, ct, m, k, sizes):
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups, ld = int(off[-1]), len(sizes), runs(k)

    def packed(rows):
        code, byte = np.zeros((rows, ld), np.uint8), np.zeros((rows, ld // 32), np.uint8)
        code[:, :k] = rng.integers(0, 16, (rows, k), dtype=np.uint8)
        byte[:, :(k + 31) // 32] = rng.integers(118, 124, (rows, (k + 31) // 32), dtype=np.uint8)
        return code, byte

    ca, sa = packed(groups * m)
    cb, sb = packed(n)
    dA, dSA, dB, dSB = ctx.upload(pack(ca)), ctx.upload(sa), ctx.upload(pack(cb)), ctx.upload(sb)
    dC, dO = ctx.upload(R.encode(np.full((n, m), np.nan, np.float32), ct)), ctx.upload(off)
    ctx.mxfp4_gemm_grouped(groups, m, n, k, 1.0, dA, dSA, ld, m * ld, dB, dSB, ld, dO, 0.0, dC, m, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dSA, dB, dSB, dC, dO):
        d.free()
    rows = sample(rng, m)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if lo < hi:
            W, x = values(ca[g * m + rows], sa[g * m + rows]).T, values(cb[lo:hi], sb[lo:hi])
            R.assert_product(R.decode(got[lo:hi, rows], ct), x @ W, np.abs(x) @ np.abs(W), k, ct)


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,sizes,pad,shift", [
    (4096, 1024, [4096], 0, 0), (2049, 513, [2049], 0, 0), (2049, 513, [2049], 0, 1), (4100, 384, [10] * 20, 0, 0),
    (4100, 383, [10] * 20, 0, 0), (1500, 400, [3000, 2000, 500], 1, 0), (1500, 401, [3000, 2000, 500], 1, 1),
    (600, 90, [20, 30, 700, 3], 1 << 20, 0)])
def test_columns_other_tiles_and_alignments(ctx, t, trans, m, k, sizes, pad, shift):
    """128 x 128 and 128 x 32 tiles, operands moved to an aligned workspace, leading dimensions past the copies' offsets."""
    rng = np.random.default_rng(m + k + shift)
    off = R.boundaries(sizes)
    n, groups = int(off[-1]), len(sizes)
    rows, cols = (k, m) if trans == TRANS else (m, k)
    wide = pad >= 1 << 20
    lda, ldb = (rows, k + pad) if wide else (rows + pad, k + pad)
    A, B = values16(rng, (groups, cols, lda), t), values16(rng, (n, k if wide else ldb), t)
    dA, dO, dC = ctx.upload(np.concatenate([A.reshape(-1)[:shift], A.reshape(-1)])), ctx.upload(off), ctx.empty((n, m), np.float32)
    if wide:
        dB = ctx.empty(n * ldb, R.STORE[t])
        for j in range(n):
            ctx.h2d(dB.offset(j * ldb), B[j])
    else:
        dB = ctx.upload(np.concatenate([B.reshape(-1)[:shift], B.reshape(-1)]))
    ctx.gemm_grouped(R.TYPES[t], trans, groups, m, n, k, 1.0, dA.offset(shift), lda, cols * lda, dB.offset(shift), ldb, dO, 0.0,
                     dC, m, R.TYPES["f32"])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    pick = sample(rng, m, 60)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        W = R.decode(A[g, pick, :k].T if trans == TRANS else A[g][:, pick], t)
        x = R.decode(B[lo:hi, :k], t)
        R.assert_product(got[lo:hi, pick].astype(np.float64), x @ W, np.abs(x) @ np.abs(W), k, "f32")


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,sizes,pad,shift", [(4096, 4096, [1024], 0, 0), (2049, 2051, [600], 0, 0), (2049, 2051, [600], 0, 1),
                                                 (1500, 3001, [900, 300, 0, 40], 1, 1)])
def test_k_other_tiles_and_alignments(ctx, t, m, n, sizes, pad, shift):
    rng = np.random.default_rng(m + n + shift)
    off = R.boundaries(sizes)
    k, groups = int(off[-1]), len(sizes)
    A, B = values16(rng, (k, m + pad), t), values16(rng, (k, n + pad), t)
    dA = ctx.upload(np.concatenate([A.reshape(-1)[:shift], A.reshape(-1)]))
    dB = ctx.upload(np.concatenate([B.reshape(-1)[:shift], B.reshape(-1)]))
    dO, dC = ctx.upload(off), ctx.empty((groups, n, m), np.float32)
    ctx.gemm_grouped_k(R.TYPES[t], groups, m, n, k, 1.0, dA.offset(shift), m + pad, dB.offset(shift), n + pad, dO, 0.0, dC, m,
                       n * m, R.TYPES["f32"])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    pick = sample(rng, m, 60)
    for g in range(groups):
        a, b = R.decode(A[off[g]:off[g + 1]][:, pick], t), R.decode(B[off[g]:off[g + 1], :n], t)
        R.assert_product(got[g][:, pick].astype(np.float64), b.T @ a, np.abs(b).T @ np.abs(a), sizes[g], "f32")


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("m,k,sizes", [(100, 200, [70, 90, 65]), (100, 203, [70, 90, 65]), (700, 150, [300, 200, 129]),
                                       (700, 157, [300, 200, 129]), (2304, 1003, [1100, 1300, 520]), (2304, 1000, [1100, 1300, 520]),
                                       (300, 5, [90, 70, 64]), (4100, 203, [9] * 20)])
def test_what_is_past_k_is_never_used(ctx, t, trans, m, k, sizes):
    """NaN and Inf in the padding behind every column and in the middle group's tokens: the other groups' results are
    finite and right, the middle group's are NaN."""
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups, bad = int(off[-1]), len(sizes), 1
    rows, cols = (k, m) if trans == TRANS else (m, k)
    lda, ldb = rows + 2 + rows % 2, k + 2 + k % 2
    nan, inf = R.encode(np.array([np.nan, np.inf], np.float32), t)
    A, B = values16(rng, (groups, cols, lda), t), values16(rng, (n, ldb), t)
    A[:, :, rows:], B[:, k:] = nan, inf
    B[off[bad]:off[bad + 1], :k] = nan
    dA, dB, dO, dC = ctx.upload(A), ctx.upload(B), ctx.upload(off), ctx.empty((n, m), np.float32)
    ctx.gemm_grouped(R.TYPES[t], trans, groups, m, n, k, 1.0, dA, lda, cols * lda, dB, ldb, dO, 0.0, dC, m, R.TYPES["f32"])
    got = dC.to_host()
    pick = sample(rng, m, 40)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if g == bad:
            assert np.isnan(got[lo:hi]).all()
            continue
        W = R.decode(A[g, pick, :k].T if trans == TRANS else A[g][:, pick], t)
        x = R.decode(B[lo:hi, :k], t)
        R.assert_product(got[lo:hi, pick].astype(np.float64), x @ W, np.abs(x) @ np.abs(W), k, "f32")
    # the weight gradient: k is the tokens, whose ends are the next group's tokens
    Y = values16(rng, (n, m + 2 + m % 2), t)
    Y[:, m:] = nan
    dY, dW = ctx.upload(Y), ctx.empty((groups, m, k), np.float32)
    ctx.gemm_grouped_k(R.TYPES[t], groups, k, m, n, 1.0, dB, ldb, dY, Y.shape[1], dO, 0.0, dW, k, m * k, R.TYPES["f32"])
    grad = dW.to_host()
    for d in (dA, dB, dO, dC, dY, dW):
        d.free()
    for g in range(groups):
        if g == bad:
            assert np.isnan(grad[g]).all()
            continue
        x, y = R.decode(B[off[g]:off[g + 1], :k], t), R.decode(Y[off[g]:off[g + 1]][:, pick], t)
        R.assert_product(grad[g][pick].astype(np.float64), y.T @ x, np.abs(y).T @ np.abs(x), sizes[g], "f32")


def test_calls_in_turn_on_two_contexts(ctx):
    """Each context has its own stream and workspace; products of odd leading dimensions (moved to the workspace) of two
    contexts, started before either is waited for, do not disturb one another."""
    from wgblas_amd import Context

    rng = np.random.default_rng(2)
    m, k, n = 1501, 801, 1700
    with Context(0) as other:
        work = []
        for c in (ctx, other):
            A, B = values16(rng, (m, k), "bf16"), values16(rng, (n, k), "bf16")
            work.append((c, A, B, c.upload(A), c.upload(B), c.upload(np.array([0, n], np.int64)), c.empty((n, m), np.float32)))
        for _ in range(3):
            for c, A, B, dA, dB, dO, dC in work:
                c.gemm_grouped(R.TYPES["bf16"], TRANS, 1, m, n, k, 1.0, dA, k, m * k, dB, k, dO, 0.0, dC, m, R.TYPES["f32"])
        for c, A, B, dA, dB, dO, dC in work:
            W, x = R.decode(A, "bf16").T, R.decode(B, "bf16")
            R.assert_product(dC.to_host().astype(np.float64), x @ W, np.abs(x) @ np.abs(W), k, "f32")


def test_more_tiles_than_a_block_lists(ctx):
    """64 tiles a block are listed: 132 x 129 tiles of 256 need more blocks than CUs."""
    rng = np.random.default_rng(1)
    m, n, k = 33700, 33000, 64
    A, B = values16(rng, (m, k), "bf16"), values16(rng, (n, k), "bf16")
    dA, dB, dC = ctx.upload(A), ctx.upload(B), ctx.empty((n, m), np.uint16)
    ctx.gemm_grouped(R.TYPES["bf16"], TRANS, 2, m, n, k, 1.0, dA, k, m * k, dB, k,
                     ctx.upload(np.array([0, n, n], np.int64)), 0.0, dC, m)
    rows = sample(rng, m, 60)
    got = dC.to_host()[:, rows]
    dC.free()
    W, x = R.decode(A[rows], "bf16").T, R.decode(B, "bf16")
    R.assert_product(R.decode(got, "bf16"), x @ W, np.abs(x) @ np.abs(W), k, "bf16")


@pytest.mark.parametrize("groups,most", [(65, 40), (200, 9), (700, 3)])
def test_more_groups_than_lanes(ctx, groups, most):
    rng = np.random.default_rng(groups)
    m, k = 300, 136
    sizes = rng.integers(0, most, groups)
    sizes[5] = 700  # a group of whole tiles among the short ones
    off = R.boundaries(sizes)
    n = int(off[-1])
    A, B = values16(rng, (groups, m, k), "bf16"), values16(rng, (n, k), "bf16")
    dA, dB, dO, dC = ctx.upload(A), ctx.upload(B), ctx.upload(off), ctx.empty((n, m), np.float32)
    ctx.gemm_grouped(R.TYPES["bf16"], TRANS, groups, m, n, k, 1.0, dA, k, m * k, dB, k, dO, 0.0, dC, m, R.TYPES["f32"])
    Y = ctx.upload(values16(rng, (n, m), "bf16"))
    dW = ctx.empty((groups, m, k), np.float32)
    ctx.gemm_grouped_k(R.TYPES["bf16"], groups, k, m, n, 1.0, dB, k, Y, m, dO, 0.0, dW, k, m * k, R.TYPES["f32"])
    got, grad, y64 = dC.to_host(), dW.to_host(), R.decode(Y.to_host(), "bf16")
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        x, W, y = R.decode(B[lo:hi], "bf16"), R.decode(A[g], "bf16").T, y64[lo:hi]
        R.assert_product(got[lo:hi].astype(np.float64), x @ W, np.abs(x) @ np.abs(W), k, "f32")
        R.assert_product(grad[g].astype(np.float64), y.T @ x, np.abs(y).T @ np.abs(x), int(sizes[g]), "f32")
