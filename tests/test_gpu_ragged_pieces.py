"""Products whose 256 x 256 tiles are a little more than whole rounds, at long k: the rest's tiles are cut into pieces of k
and added up. Against float64 products, and the same bits from call to call."""
import numpy as np
import pytest

from tests import ragged as R
from tests.test_gpu_mxfp4 import pack, runs, values
from tests.test_gpu_ragged_large import sample, values16
from wgblas_amd import NO_TRANS, TRANS

pytestmark = pytest.mark.gpu

# tiles past a round of 256 (pieces of a tile): 40 (3), 8 (4), 8 (8, the last ones shorter), 16 (8), 96 (1)
COLUMNS = [(2048, 2104, [1300, 0, 1, 2047, 300, 5000]), (2048, 2104, [8192, 40]), (2048, 4744, [8000, 300]),
           (4096, 4104, [4096, 0, 90]), (2048, 2104, [8192, 2900])]


@pytest.mark.parametrize("trans", [NO_TRANS, TRANS])
@pytest.mark.parametrize("t,ct,beta,cut", [("bf16", "bf16", 0.0, 0), ("f16", "f32", 0.5, 0), ("bf16", "f32", 0.0, 3)])
@pytest.mark.parametrize("m,k,sizes", COLUMNS)
def test_columns(ctx, t, ct, beta, cut, trans, m, k, sizes):
    """cut: k and m off multiples of a copy, with odd leading dimensions (moved to the workspace before the sums' part)."""
    m, k = m - cut, k - cut
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups = int(off[-1]), len(sizes)
    A = values16(rng, (groups, m, k) if trans == TRANS else (groups, k, m), t)
    B = values16(rng, (n, k), t)
    C0 = R.encode(np.full((n, m), np.nan, np.float32), ct) if beta == 0.0 else values16(rng, (n, m), ct)
    dA, dB, dO = ctx.upload(A), ctx.upload(B), ctx.upload(off)
    out = []
    for _ in range(2):
        dC = ctx.upload(C0)
        ctx.gemm_grouped(R.TYPES[t], trans, groups, m, n, k, 0.5, dA, A.shape[2], m * k, dB, k, dO, beta, dC, m, R.TYPES[ct])
        out.append(dC.to_host())
        dC.free()
    for d in (dA, dB, dO):
        d.free()
    got = out[0]
    assert (got.view(np.uint8) == out[1].view(np.uint8)).all()
    rows = sample(rng, m, 60)
    for g in range(groups):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        W = R.decode(A[g, rows].T if trans == TRANS else A[g][:, rows], t)
        x = R.decode(B[lo:hi], t)
        R.assert_product(R.decode(got[lo:hi, rows], ct), x @ W, np.abs(x) @ np.abs(W), k, ct, 0.5, beta,
                         R.decode(C0[lo:hi, rows], ct))


# 9 x 10 tiles a group, 14 past a round; the rest's groups are the shortest ones. The last: 16 x 17 tiles, 16 past a round
@pytest.mark.parametrize("t,ct,beta", [("bf16", "f32", 0.0), ("f16", "f16", 0.5)])
@pytest.mark.parametrize("m,n,sizes", [(2304, 2304 + 8, [2200, 2300, 2100]), (2200, 2400, [2600, 0, 4500]),
                                       (2200, 2400, [3000, 3000, 700]), (4096, 4100, [4200])])
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
    rows = sample(rng, m, 60)
    for g in range(groups):
        a, b = R.decode(A[off[g]:off[g + 1]][:, rows], t), R.decode(B[off[g]:off[g + 1]], t)
        R.assert_product(R.decode(got[g][:, rows], ct), b.T @ a, np.abs(b).T @ np.abs(a), sizes[g], ct, 0.5, beta,
                         R.decode(C0[g][:, rows], ct))


@pytest.mark.parametrize("ct,m,k,sizes", [("bf16", 2048, 6272, [8000, 300]), ("f32", 4090, 8192, [4300])])
def test_mxfp4(ctx, ct, m, k, sizes):
    rng = np.random.default_rng(m + k)
    off = R.boundaries(sizes)
    n, groups, ld = int(off[-1]), len(sizes), runs(k)

    def packed(rows):
        code = rng.integers(0, 16, (rows, ld), dtype=np.uint8)
        return code, rng.integers(118, 124, (rows, ld // 32), dtype=np.uint8)

    ca, sa = packed(groups * m)
    cb, sb = packed(n)
    dA, dSA, dB, dSB = ctx.upload(pack(ca)), ctx.upload(sa), ctx.upload(pack(cb)), ctx.upload(sb)
    dC, dO = ctx.upload(R.encode(np.full((n, m), np.nan, np.float32), ct)), ctx.upload(off)
    if groups == 1:
        ctx.mxfp4_gemm(m, n, k, 1.0, dA, dSA, ld, dB, dSB, ld, 0.0, dC, m, R.TYPES[ct])
    else:
        ctx.mxfp4_gemm_grouped(groups, m, n, k, 1.0, dA, dSA, ld, m * ld, dB, dSB, ld, dO, 0.0, dC, m, R.TYPES[ct])
    got = dC.to_host()
    for d in (dA, dSA, dB, dSB, dC, dO):
        d.free()
    rows = sample(rng, m, 40)
    for g in range(groups):
        W, x = values(ca[g * m + rows], sa[g * m + rows]).T, values(cb[off[g]:off[g + 1]], sb[off[g]:off[g + 1]])
        R.assert_product(R.decode(got[off[g]:off[g + 1], rows], ct), x @ W, np.abs(x) @ np.abs(W), k, ct)
