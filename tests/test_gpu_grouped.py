"""Grouped products (wgb_gemm_grouped, wgb_gemm_grouped_k) against products in
float64, group by group: types, layouts, raggedness, strides, alignment,
alpha / beta rules, values in places that must not be read, gradients."""
import numpy as np
import pytest

from tests import ragged as R
from wgblas_amd import NO_TRANS, TRANS, WgblasError

pytestmark = pytest.mark.gpu

SIZES = {
    "one": [1],
    "even": [40, 40, 40],
    "empty_ends": [0, 7, 0, 0, 130, 1, 0],
    "skewed": [3, 0, 300, 1, 17],
    "many": [1, 2, 0, 5] * 20,
    "long": [700, 515],
    "tiny": [1, 1, 2, 1, 0, 1, 3, 1],
}


def run_columns(ctx, t, ct, trans, m, k, sizes, pads=(0, 0, 0), alpha=1.0, beta=0.0, shift=0, spare=0, seed=0):
    """One wgb_gemm_grouped call on host-made operands; returns C as (columns, ldc) storage and what it should hold.

    `pads`: of A, B, C's leading dimensions; `shift`: elements that A and B start past their allocation's start;
    `spare`: columns of B and C after the last group's."""
    rng = np.random.default_rng(seed)
    off = R.boundaries(sizes)
    n, groups = int(off[-1]) + spare, len(sizes)
    a_rows, a_cols = (k, m) if trans == TRANS else (m, k)
    lda, ldb, ldc = max(1, a_rows + pads[0]), max(1, k + pads[1]), m + pads[2]
    A = R.columns(rng, a_rows, groups * a_cols, lda, t)
    B = R.columns(rng, k, n, ldb, t)
    if spare:
        B[n - spare:] = R.encode(np.full((spare, ldb), np.nan), t)
    C0 = R.encode(np.full((n, ldc), np.nan) if beta == 0.0 else rng.standard_normal((n, ldc)), ct)
    pad = np.zeros(shift, R.STORE[t])
    dA = ctx.upload(np.concatenate([pad, A.reshape(-1)]) if A.size + shift else np.zeros(1, R.STORE[t]))
    dB = ctx.upload(np.concatenate([pad, B.reshape(-1)]) if B.size + shift else np.zeros(1, R.STORE[t]))
    dC, dO = ctx.upload(C0), ctx.upload(off)
    ctx.gemm_grouped(R.TYPES[t], trans, groups, m, n, k, alpha, dA.offset(shift), lda, a_cols * lda, dB.offset(shift),
                     ldb, dO, beta, dC, ldc, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    A64 = R.decode(A, t).reshape(groups, a_cols, lda)[:, :, :a_rows]
    B64, C64 = R.decode(B, t)[:, :k], R.decode(C0, ct)[:, :m]
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        W = A64[g].T if trans == TRANS else A64[g]  # k x m
        exact, absdot = B64[lo:hi] @ W, np.abs(B64[lo:hi]) @ np.abs(W)
        R.assert_product(R.decode(got[lo:hi, :m], ct), exact, absdot, k, ct, alpha, beta, C64[lo:hi])
    # padding and columns of no group keep their bits
    raw, raw0 = got.view(np.uint8).reshape(n, -1), C0.view(np.uint8).reshape(n, -1)
    es = got.dtype.itemsize
    assert np.array_equal(raw[:, m * es:], raw0[:, m * es:])
    assert np.array_equal(raw[int(off[-1]):], raw0[int(off[-1]):])
    return got


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t,ct", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("sizes", sorted(SIZES))
def test_columns_types_and_raggedness(ctx, t, ct, trans, sizes):
    run_columns(ctx, t, ct, trans, 136, 200, SIZES[sizes], seed=len(sizes))


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 64), (3, 1000), (257, 7), (128, 64), (129, 65), (520, 513), (256, 1024)])
@pytest.mark.parametrize("sizes", ["skewed", "tiny"])
def test_columns_odd_sizes(ctx, t, trans, m, k, sizes):
    run_columns(ctx, t, t, trans, m, k, SIZES[sizes], seed=m + k)


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pads,shift", [((0, 0, 5), 0), ((8, 8, 8), 0), ((1, 1, 1), 0), ((2, 6, 3), 2), ((1, 0, 0), 1),
                                        ((0, 0, 0), 1), ((0, 3, 0), 3)])
@pytest.mark.parametrize("sizes", ["skewed", "tiny", "long"])
def test_columns_strides_and_alignment(ctx, t, trans, pads, shift, sizes):
    run_columns(ctx, t, t, trans, 264, 192, SIZES[sizes], pads, shift=shift, spare=4, seed=shift)


@pytest.mark.parametrize("t,ct", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("alpha,beta", [(1.5, 0.5), (-0.25, 1.0), (0.0, 0.5), (0.0, 0.0), (2.0, 0.0)])
@pytest.mark.parametrize("sizes", ["skewed", "tiny", "long"])
def test_columns_alpha_beta(ctx, t, ct, alpha, beta, sizes):
    run_columns(ctx, t, ct, TRANS, 200, 96, SIZES[sizes], (0, 0, 2), alpha, beta, seed=3)
    run_columns(ctx, t, ct, NO_TRANS, 200, 96, SIZES[sizes], (0, 0, 2), alpha, beta, seed=4)


@pytest.mark.parametrize("sizes", ["skewed", "tiny"])
def test_columns_without_k_scale_c(ctx, sizes):
    run_columns(ctx, "bf16", "bf16", TRANS, 70, 0, SIZES[sizes], beta=0.5)
    run_columns(ctx, "f32", "f32", NO_TRANS, 70, 0, SIZES[sizes], beta=0.0)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_columns_larger(ctx, t):
    run_columns(ctx, t, t, TRANS, 1000, 1100, [300, 0, 411, 90, 257], seed=9)
    run_columns(ctx, t, t, NO_TRANS, 1000, 1100, [300, 0, 411, 90, 257], seed=10)


def test_columns_special_values_stay_in_their_group(ctx):
    """An Inf or NaN in one token or one expert reaches only that token's or that expert's results."""
    rng = np.random.default_rng(5)
    m, k, sizes = 96, 160, [5, 40, 3]
    off, n = R.boundaries(sizes), sum(sizes)
    A, B = R.columns(rng, k, 3 * m, k, "bf16"), R.columns(rng, k, n, k, "bf16")
    A[2 * m + 7, 3] = 0x7F80  # +Inf in row 7 of the last group's op(A)
    B[10, 100] = 0x7FC0  # NaN in token 10
    dC = ctx.upload(np.zeros((n, m), np.float32))
    ctx.gemm_grouped(R.TYPES["bf16"], TRANS, 3, m, n, k, 1.0, ctx.upload(A), k, m * k, ctx.upload(B), k, ctx.upload(off),
                     0.0, dC, m, R.TYPES["f32"])
    finite = np.isfinite(dC.to_host())
    want = np.ones((n, m), bool)
    want[10] = False
    want[45:, 7] = False
    assert np.array_equal(finite, want)


def test_columns_boundaries_outside_the_columns_are_clamped(ctx):
    rng = np.random.default_rng(6)
    m, k, n = 40, 64, 30
    A, B = R.columns(rng, k, 2 * m, k, "bf16"), R.columns(rng, k, n, k, "bf16")
    dC = ctx.upload(np.zeros((n, m), np.float32))
    ctx.gemm_grouped(R.TYPES["bf16"], TRANS, 2, m, n, k, 1.0, ctx.upload(A), k, m * k, ctx.upload(B), k,
                     ctx.upload(np.array([-5, 11, 1000], np.int64)), 0.0, dC, m, R.TYPES["f32"])
    A64, B64 = R.decode(A, "bf16"), R.decode(B, "bf16")
    got = dC.to_host().astype(np.float64)
    for lo, hi, g in ((0, 11, 0), (11, 30, 1)):
        W = A64[g * m:(g + 1) * m].T
        R.assert_product(got[lo:hi], B64[lo:hi] @ W, np.abs(B64[lo:hi]) @ np.abs(W), k, "f32")


def test_columns_offsets_past_32_bits(ctx):
    """Expert weights 2^31 elements apart (4 GiB): addresses need 64 bits."""
    rng = np.random.default_rng(7)
    m, k, sizes, stride = 48, 72, [9, 33], (1 << 31) + 8
    off, n = R.boundaries(sizes), sum(sizes)
    A, B = R.columns(rng, k, 2 * m, k, "bf16"), R.columns(rng, k, n, k, "bf16")
    dA = ctx.empty(stride + m * k, np.uint16)
    for g in range(2):
        ctx.h2d(dA.offset(g * stride), A[g * m:(g + 1) * m])
    dC = ctx.upload(np.zeros((n, m), np.float32))
    ctx.gemm_grouped(R.TYPES["bf16"], TRANS, 2, m, n, k, 1.0, dA, k, stride, ctx.upload(B), k, ctx.upload(off), 0.0, dC,
                     m, R.TYPES["f32"])
    got = dC.to_host().astype(np.float64)
    dA.free()
    A64, B64 = R.decode(A, "bf16"), R.decode(B, "bf16")
    for g in range(2):
        W, x = A64[g * m:(g + 1) * m].T, B64[off[g]:off[g + 1]]
        R.assert_product(got[off[g]:off[g + 1]], x @ W, np.abs(x) @ np.abs(W), k, "f32")


def run_k(ctx, t, ct, m, n, sizes, pads=(0, 0, 0), alpha=1.0, beta=0.0, shift=0, spare=0, seed=0):
    rng = np.random.default_rng(seed)
    off = R.boundaries(sizes)
    k, groups = int(off[-1]) + spare, len(sizes)
    lda, ldb, ldc = m + pads[0], n + pads[1], m + pads[2]
    A, B = R.columns(rng, m, k, lda, t), R.columns(rng, n, k, ldb, t)
    if spare:
        A[k - spare:] = R.encode(np.full((spare, lda), np.nan), t)
        B[k - spare:] = R.encode(np.full((spare, ldb), np.inf), t)
    C0 = R.encode(np.full((groups * n, ldc), np.nan) if beta == 0.0 else rng.standard_normal((groups * n, ldc)), ct)
    pad = np.zeros(shift, R.STORE[t])
    dA, dB = ctx.upload(np.concatenate([pad, A.reshape(-1)])), ctx.upload(np.concatenate([pad, B.reshape(-1)]))
    dC, dO = ctx.upload(C0), ctx.upload(off)
    ctx.gemm_grouped_k(R.TYPES[t], groups, m, n, k, alpha, dA.offset(shift), lda, dB.offset(shift), ldb, dO, beta, dC,
                       ldc, n * ldc, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    A64, B64 = R.decode(A, t)[:, :m], R.decode(B, t)[:, :n]
    C64 = R.decode(C0, ct)[:, :m]
    for g in range(groups):
        a, b = A64[off[g]:off[g + 1]], B64[off[g]:off[g + 1]]
        R.assert_product(R.decode(got[g * n:(g + 1) * n, :m], ct), b.T @ a, np.abs(b).T @ np.abs(a), sizes[g], ct, alpha,
                         beta, C64[g * n:(g + 1) * n])
    es = got.dtype.itemsize
    raw, raw0 = got.view(np.uint8).reshape(groups * n, -1), C0.view(np.uint8).reshape(groups * n, -1)
    assert np.array_equal(raw[:, m * es:], raw0[:, m * es:])
    return got


@pytest.mark.parametrize("t,ct", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("sizes", sorted(SIZES))
def test_k_types_and_raggedness(ctx, t, ct, sizes):
    run_k(ctx, t, ct, 136, 72, SIZES[sizes], seed=len(sizes))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 200), (200, 1), (3, 5), (129, 257), (128, 128), (264, 520)])
@pytest.mark.parametrize("sizes", ["skewed", "tiny"])
def test_k_odd_sizes(ctx, t, m, n, sizes):
    run_k(ctx, t, t, m, n, SIZES[sizes], seed=m + n)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pads,shift", [((0, 0, 5), 0), ((8, 8, 8), 0), ((1, 1, 1), 0), ((2, 6, 3), 1), ((0, 0, 0), 2),
                                        ((0, 3, 0), 3)])
@pytest.mark.parametrize("sizes", ["skewed", "long"])
def test_k_strides_and_alignment(ctx, t, pads, shift, sizes):
    run_k(ctx, t, t, 264, 136, SIZES[sizes], pads, shift=shift, spare=4, seed=shift)


@pytest.mark.parametrize("t,ct", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("alpha,beta", [(1.5, 0.5), (-0.25, 1.0), (0.0, 0.5), (0.0, 0.0)])
def test_k_alpha_beta(ctx, t, ct, alpha, beta):
    """Also the accumulation of gradients (beta = 1), where an empty group's gradient stays."""
    run_k(ctx, t, ct, 200, 96, SIZES["empty_ends"], (0, 0, 2), alpha, beta, seed=3)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_k_larger(ctx, t):
    run_k(ctx, t, "f32", 1032, 1300, [300, 0, 411, 90, 257, 1, 64, 128, 30, 2, 63, 65], seed=9)


def test_results_are_the_same_every_time(ctx):
    first = run_columns(ctx, "bf16", "f32", TRANS, 300, 520, SIZES["skewed"], seed=2)
    assert np.array_equal(first, run_columns(ctx, "bf16", "f32", TRANS, 300, 520, SIZES["skewed"], seed=2))
    first = run_k(ctx, "bf16", "f32", 300, 120, SIZES["skewed"], seed=2)
    assert np.array_equal(first, run_k(ctx, "bf16", "f32", 300, 120, SIZES["skewed"], seed=2))


def test_gradients_against_differences(ctx):
    """For L = sum(R * Y), Y the forward product in f32: <dW, E> and <dX, E> against central differences of L along
    random directions E. L is linear in W and in X, so a difference of step 1 is exact but for the rounding of the two
    Y, each within (k + 2) 2^-23 sum |w x|."""
    rng = np.random.default_rng(11)
    m, k, sizes = 60, 44, [0, 13, 1, 30]
    off, n, groups = R.boundaries(sizes), sum(sizes), len(sizes)
    f32 = R.TYPES["f32"]
    W, X, Rm = (rng.standard_normal(s).astype(np.float32) for s in ((groups * m, k), (n, k), (n, m)))
    dO, dR = ctx.upload(off), ctx.upload(Rm)

    def loss(w, x):
        y = ctx.empty((n, m), np.float32)
        ctx.gemm_grouped(f32, TRANS, groups, m, n, k, 1.0, ctx.upload(w), k, m * k, ctx.upload(x), k, dO, 0.0, y, m)
        return float((y.to_host().astype(np.float64) * Rm).sum())

    dX, dW = ctx.empty((n, k), np.float32), ctx.empty((groups * m, k), np.float32)
    ctx.gemm_grouped(f32, NO_TRANS, groups, k, n, m, 1.0, ctx.upload(W), k, m * k, dR, m, dO, 0.0, dX, k)
    ctx.gemm_grouped_k(f32, groups, k, m, n, 1.0, ctx.upload(X), k, dR, m, dO, 0.0, dW, k, m * k)
    group = np.repeat(np.arange(groups), sizes)
    for which, grad, base in (("w", dW, W), ("x", dX, X)):
        E = rng.standard_normal(base.shape).astype(np.float32)
        up, down = base + E, base - E
        diff = (loss(up, X) - loss(down, X)) / 2 if which == "w" else (loss(W, up) - loss(W, down)) / 2
        g = grad.to_host().astype(np.float64)
        # the directions actually taken, as the sums were rounded
        step = (up.astype(np.float64) - down.astype(np.float64)) / 2
        Wa = np.abs(W).reshape(groups, m, k)[group] + np.abs(E if which == "w" else 0 * W).reshape(groups, m, k)[group]
        Xa = np.abs(X) + (np.abs(E) if which == "x" else 0)
        size = (np.abs(Rm)[:, :, None] * Wa * Xa[:, None, :]).sum()
        assert abs((g * step).sum() - diff) <= 3 * (max(m, k, n) + 2) * 2.0 ** -23 * size


def test_refusals(ctx):
    f = np.zeros(64, np.float32)
    d, o = ctx.upload(f), ctx.upload(np.array([0, 4], np.int64))

    def columns(type=0, transA=0, groups=1, m=4, n=4, k=4, A=d, lda=4, strideA=16, B=d, ldb=4, off=o, C=d, ldc=4, ctype=0):
        ctx.gemm_grouped(type, transA, groups, m, n, k, 1.0, A, lda, strideA, B, ldb, off, 0.0, C, ldc, ctype)

    def ragged_k(type=0, groups=1, m=4, n=4, k=4, A=d, lda=4, B=d, ldb=4, off=o, C=d, ldc=4, strideC=16, ctype=0):
        ctx.gemm_grouped_k(type, groups, m, n, k, 1.0, A, lda, B, ldb, off, 0.0, C, ldc, strideC, ctype)

    both = [dict(type=3), dict(type=-1), dict(type=0, ctype=2), dict(type=1, ctype=2), dict(groups=-1), dict(m=-1), dict(n=-1),
            dict(k=-1), dict(m=1 << 31, lda=1 << 31, ldc=1 << 31), dict(groups=(1 << 20) + 1, strideA=16), dict(lda=3),
            dict(ldb=3), dict(ldc=3), dict(A=None), dict(B=None), dict(C=None), dict(off=None)]
    cases = [(columns, a) for a in both + [dict(transA=2), dict(strideA=-1), dict(groups=2, strideA=15),
                                           dict(transA=1, m=8, groups=2, strideA=31, ldc=8)]]
    cases += [(ragged_k, a) for a in both[:9] + both[10:] + [dict(strideC=-1), dict(groups=2, strideC=15)]]
    for fn, args in cases:
        with pytest.raises(WgblasError, match="status -1"):
            fn(**args)
    # nothing to do: no operand is needed
    columns(m=0, A=None, B=None, C=None, off=None)
    columns(n=0, A=None, B=None, C=None, off=None)
    columns(groups=0, A=None, B=None, C=None, off=None)
    ragged_k(n=0, A=None, B=None, C=None, off=None)
    ragged_k(groups=0, A=None, B=None, C=None, off=None)
    ctx.synchronize()
