"""f16 rows are rounded from their fp32 values wherever they lie: in a whole 16-byte chunk of a row or in its cut end. The
inputs are products whose rounding to f16 in one step differs from that through fp32."""
import numpy as np
import pytest

from tests import ragged as R

pytestmark = pytest.mark.gpu

F16 = R.TYPES["f16"]


def twice(a, b):
    """(products a b through fp32 to f16, in one step): a fp32, b f16, so that they are exact in float64."""
    p = a.astype(np.float64) * b.astype(np.float64)
    with np.errstate(over="ignore"):
        return p.astype(np.float32).astype(np.float16), p.astype(np.float16)


def pairs(rng, count):
    """fp32 and f16 numbers whose product the two ways of rounding differ in."""
    a, b = [], []
    while sum(map(len, a)) < count:
        x = rng.uniform(0.5, 2.0, 1 << 20).astype(np.float32)
        y = rng.uniform(0.5, 2.0, 1 << 20).astype(np.float16)
        through, once = twice(x, y)
        a.append(x[through != once])
        b.append(y[through != once])
    return np.concatenate(a)[:count], np.concatenate(b)[:count]


@pytest.mark.parametrize("d", [13, 8, 3, 2053])
def test_sums(ctx, d):
    """One slot: the sum is w y."""
    w, y = pairs(np.random.default_rng(d), 60)
    n = len(w)
    places = np.arange(n, dtype=np.int32).reshape(n, 1)
    dY, dP, dW, dC = ctx.upload(np.repeat(y[:, None], d, 1)), ctx.upload(places), ctx.upload(w), ctx.empty((n, d), np.float16)
    ctx.route_combine(F16, d, n, 1, dY, d, dP, dW, 0.0, dC, d, F16)
    assert np.array_equal(dC.to_host(), np.repeat(twice(w, y)[0][:, None], d, 1))
    out = ctx.upload(np.zeros((n, d), np.float16))
    ctx.route_gather(F16, d, n, 1, dY, d, dP, dW, out, d)
    assert np.array_equal(out.to_host(), np.repeat(twice(w, y)[0][:, None], d, 1))
    for b in (dY, dP, dW, dC, out):
        b.free()


@pytest.mark.parametrize("d", [13, 8, 3, 2053])
def test_the_rows_own_term(ctx, d):
    """No slot has a place: the result is beta c."""
    rng = np.random.default_rng(d)
    c = np.arange(0x3C00, 0x4000, dtype=np.uint16).view(np.float16)  # 1 to 2
    n, found = len(c), 0
    dY, dP, dW = ctx.empty((n, d), np.float16), ctx.upload(np.full((n, 1), -1, np.int32)), ctx.upload(np.ones((n, 1), np.float32))
    while found < 12:
        beta = rng.uniform(0.5, 2.0, 1).astype(np.float32)
        through, once = twice(np.repeat(beta, n), c)
        if (through == once).all():
            continue
        found += 1
        dC = ctx.upload(np.repeat(c[:, None], d, 1))
        ctx.route_combine(F16, d, n, 1, dY, d, dP, dW, float(beta[0]), dC, d, F16)
        assert np.array_equal(dC.to_host(), np.repeat(through[:, None], d, 1)), beta
        dC.free()
    for b in (dY, dP, dW):
        b.free()
