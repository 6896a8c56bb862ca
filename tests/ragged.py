"""Host-side helpers of the grouped and 4-bit operators' tests: 16-bit types in
numpy, ragged boundaries, and error bounds.

Bounds. Products of 16-bit values are exact in fp32 and fp32 products round
once, sums are held in fp32, so a result before its last rounding is within
(k + 2) 2^-23 sum |a b| of the exact one, whatever the order of the sum (2^-23
a step leaves room for a matrix instruction that truncates). The last rounding
adds half a unit of the type C is held in: 2^-8 (bf16), 2^-11 (f16, and half
its smallest subnormal, 2^-25), 2^-24 (f32) of the value; past the type's range
the result is an Inf.
"""
import numpy as np

from wgblas_amd import BF16, F16, F32

TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
STORE = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
HALF_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
OVERFLOW = {"f32": 2.0 ** 128 * (1 - 2.0 ** -25), "f16": 65520.0, "bf16": 2.0 ** 128 * (1 - 2.0 ** -9)}
SMALLEST = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}


def encode(x, t):
    """float64 -> the type's storage, to nearest even (bf16 as its 16 bits)."""
    if t != "bf16":
        return np.asarray(x, np.float64).astype(STORE[t])
    # through float32, whose own rounding the tests' inputs (few bits) do not meet
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7FC0), r).astype(np.uint16)


def decode(x, t):
    """Storage -> float64."""
    if t != "bf16":
        return x.astype(np.float64)
    return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def boundaries(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)


def columns(rng, rows, cols, ld, t, fill=np.nan):
    """A column-major matrix of normals in storage form, its padding set to `fill`: shape (cols, ld)."""
    x = np.full((cols, ld), fill)
    x[:, :rows] = rng.standard_normal((cols, rows))
    return encode(x, t)


def assert_product(got, exact, absdot, k, ct, alpha=1.0, beta=0.0, c0=None):
    """Every element of got (float64) within the bound above of alpha exact + beta c0."""
    want = alpha * exact
    sums = (k + 2) * 2.0 ** -23 * abs(alpha) * absdot
    if beta != 0.0:
        want = want + beta * c0
        sums = sums + 2.0 ** -23 * (np.abs(alpha * exact) + np.abs(beta * c0))
    bound = sums + (np.abs(want) + sums) * HALF_UNIT[ct] + SMALLEST[ct]
    # a result past the largest number of C's type is an Inf of its sign (halfway to the next power of two rounds up)
    top = OVERFLOW[ct]
    over = np.abs(want) - bound >= top
    assert np.array_equal(got[over], np.sign(want[over]) * np.inf)
    near = ~over & (np.abs(want) + bound >= top)
    err = np.where(over | (near & np.isinf(got)), 0.0, np.abs(got - want))
    bad = ~(err <= bound)
    assert not bad.any(), (f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: got {got[bad][0]}, "
                           f"want {want[bad][0]}, bound {bound[bad][0]}")
