"""The 256 x 256 kernel where its turns are least regular: MXFP4 operands of several ragged groups, k an odd multiple of
128 (half of the last k-tile) before a block's next tile, rests that are cut along k in the middle of such a one, and more
groups than a wave has lanes. All columns of a sample of rows against float64 products, and the same bits from call to
call. That the cases take this kernel is checked on the CPU (tests/test_ragged_host_side.py)."""
import numpy as np
import pytest

from tests import ragged as R
from tests.test_gpu_mxfp4 import runs, values
from tests.test_gpu_ragged_large import sample, values16
from wgblas_amd import NO_TRANS, TRANS

pytestmark = pytest.mark.gpu


def share(total, groups, seed):
    """Uneven sizes of `groups` groups, one in five of them empty."""
    rng = np.random.default_rng(seed)
    chance = rng.random(groups) + 0.2
    chance[rng.permutation(groups)[: groups // 5]] = 0.0
    return rng.multinomial(total, chance / chance.sum()).tolist()


# m, k, sizes, whether the rest is cut along k
MXFP4 = [(8190, 1152, [3000, 0, 1, 2555, 2444], False),  # 32 x 33 tiles: four rounds and 32 tiles
         (8190, 1100, [3000, 0, 1, 2555, 2444], False),  # k inside a block of 32
         (8192, 1152, [255, 6001, 256, 0, 5488], False),
         (2048, 1152, share(40000, 70, 1), False),
         (2040, 6272, [5000, 700, 3300], True),
         (4100, 6272, [4150, 100], True)]


def packed(rng, rows, k):
    """Random codes, two a byte, and scales of a matrix of k x rows, zeros past k."""
    codes, scales = rng.integers(0, 256, (rows, runs(k) // 2), dtype=np.uint8), rng.integers(118, 124, (rows, runs(k) // 32), dtype=np.uint8)
    codes[:, (k + 1) // 2:] = 0
    if k % 2:
        codes[:, k // 2] &= 15
    scales[:, (k + 31) // 32:] = 0
    return codes, scales


def decoded(codes, scales):
    return values(np.stack([codes & 15, codes >> 4], 2).reshape(len(codes), -1), scales)


@pytest.mark.parametrize("ct", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,sizes,cut", MXFP4)
def test_mxfp4(ctx, ct, m, k, sizes, cut):
    """One token's last block is NaN: its results are, no other's."""
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups, ld = int(off[-1]), len(sizes), runs(k)
    ca, sa = packed(rng, groups * m, k)
    cb, sb = packed(rng, n, k)
    bad = n // 2
    sb[bad, (k - 1) // 32] = 255
    dA, dSA, dB, dSB, dO = (ctx.upload(x) for x in (ca, sa, cb, sb, off))
    out = []
    for _ in range(2):
        dC = ctx.upload(R.encode(np.full((n, m), 7.0, np.float32), ct))
        ctx.mxfp4_gemm_grouped(groups, m, n, k, 1.0, dA, dSA, ld, m * ld, dB, dSB, ld, dO, 0.0, dC, m, R.TYPES[ct])
        out.append(dC.to_host())
        dC.free()
    for d in (dA, dSA, dB, dSB, dO):
        d.free()
    got = out[0]
    assert (got.view(np.uint8) == out[1].view(np.uint8)).all()
    rows = sample(rng, m, 40)[:: 1 if groups < 10 else 4]
    assert np.isnan(R.decode(got[bad], ct)).all()
    for g in range(groups):
        at = np.arange(off[g], off[g + 1])
        at = at[at != bad]
        if not len(at):
            continue
        W, x = decoded(ca[g * m + rows], sa[g * m + rows]).T, decoded(cb[at], sb[at])
        R.assert_product(R.decode(got[np.ix_(at, rows)], ct), x @ W, np.abs(x) @ np.abs(W), k, ct)


# m, k, sizes, whether the rest is cut along k
COLUMNS = [(1024, 520, share(20000, 66, 2), False), (768, 264, share(30000, 90, 3), False), (1022, 516, share(45000, 130, 4), False)]


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t,ct,beta", [("bf16", "f32", 0.0), ("f16", "f16", 0.5)])
@pytest.mark.parametrize("m,k,sizes,cut", COLUMNS)
def test_columns_of_more_groups_than_lanes(ctx, t, ct, beta, trans, m, k, sizes, cut):
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups = int(off[-1]), len(sizes)
    A = values16(rng, (groups, m, k) if trans == TRANS else (groups, k, m), t)
    B = values16(rng, (n, k), t)
    C0 = R.encode(np.full((n, m), np.nan, np.float32), ct) if beta == 0.0 else values16(rng, (n, m), ct)
    dA, dB, dC, dO = ctx.upload(A), ctx.upload(B), ctx.upload(C0), ctx.upload(off)
    ctx.gemm_grouped(R.TYPES[t], trans, groups, m, n, k, 0.5, dA, A.shape[2], m * k, dB, k, dO, beta, dC, m, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dB, dC, dO):
        d.free()
    rows = sample(rng, m, 40)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        W = R.decode(A[g, rows].T if trans == TRANS else A[g][:, rows], t)
        x = R.decode(B[lo:hi], t)
        R.assert_product(R.decode(got[lo:hi, rows], ct), x @ W, np.abs(x) @ np.abs(W), k, ct, 0.5, beta,
                         R.decode(C0[lo:hi, rows], ct))


# m, n, sizes, whether the rest is cut along k
K = [(512, 512, share(33000, 128, 5), False), (1000, 500, share(40000, 128, 6), False), (500, 512, share(106000, 66, 7), True)]


@pytest.mark.parametrize("t,ct,beta", [("bf16", "f32", 0.0), ("f16", "f16", 0.5)])
@pytest.mark.parametrize("m,n,sizes,cut", K)
def test_k_of_more_groups_than_lanes(ctx, t, ct, beta, m, n, sizes, cut):
    rng = np.random.default_rng(m + n)
    off = R.boundaries(sizes)
    k, groups = int(off[-1]), len(sizes)
    A, B = values16(rng, (k, m), t), values16(rng, (k, n), t)
    C0 = R.encode(np.full((groups, n, m), np.nan, np.float32), ct) if beta == 0.0 else values16(rng, (groups, n, m), ct)
    dA, dB, dO = ctx.upload(A), ctx.upload(B), ctx.upload(off)
    out = []
    for _ in range(2):
        dC = ctx.upload(C0)
        ctx.gemm_grouped_k(R.TYPES[t], groups, m, n, k, 0.5, dA, m, dB, n, dO, beta, dC, m, n * m, R.TYPES[ct])
        out.append(dC.to_host())
        dC.free()
    for d in (dA, dB, dO):
        d.free()
    got = out[0]
    assert (got.view(np.uint8) == out[1].view(np.uint8)).all()
    rows = sample(rng, m, 40)
    for g in range(groups):
        a, b = R.decode(A[off[g]:off[g + 1]][:, rows], t), R.decode(B[off[g]:off[g + 1]], t)
        R.assert_product(R.decode(got[g][:, rows], ct), b.T @ a, np.abs(b).T @ np.abs(a), sizes[g], ct, 0.5, beta,
                         R.decode(C0[g][:, rows], ct))
