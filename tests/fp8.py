"""FP8 matrices in numpy, by the definition: E4M3 codes and a scale for each 128 x block values."""
import numpy as np

RUN = 128


def runs(k):
    return (k + RUN - 1) // RUN * RUN


def code_values():
    """The value of each of the 256 codes, from its sign, exponent and mantissa bits."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (1.0 + f / 8.0) * np.exp2(e - 7.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


VALUES = code_values()


def quantize(x, block):
    """x (n, k) float64 -> codes (n, runs(k)) and scales (runs(k) / 128, ceil(n / block)), both by the definition."""
    n, k = x.shape
    cols = (n + block - 1) // block
    full = np.zeros((cols * block, runs(k)))
    full[:n, :k] = x
    tiles = full.reshape(cols, block, -1, RUN)
    bad = ~np.isfinite(tiles).all(axis=(1, 3))
    top = np.where(bad, 1.0, np.abs(np.where(np.isfinite(tiles), tiles, 0.0)).max(axis=(1, 3)))
    f, e = np.frexp(top)  # top = f 2^e, f in [0.5, 1): 448 = 0.875 2^9
    e = np.where(top == 0, -126, np.maximum(e - 9 + (f > 0.875), -126))
    v = np.where(bad[:, None, :, None], 0.0, tiles) / np.exp2(e.astype(np.float64))[:, None, :, None]
    magnitudes = VALUES[:127]
    low = np.searchsorted(magnitudes, np.abs(v), side="right") - 1
    high = np.minimum(low + 1, 126)
    down, up = np.abs(v) - magnitudes[low], magnitudes[high] - np.abs(v)
    code = np.where((up < down) | ((up == down) & (low % 2 == 1)), high, low)
    code = np.where(bad[:, None, :, None], 0, code + 128 * np.signbit(v))
    scales = np.where(bad, np.nan, np.exp2(e.astype(np.float64))).T
    return code.reshape(cols * block, -1)[:n].astype(np.uint8), np.ascontiguousarray(scales.astype(np.float32))


def values(codes, scales, block):
    """What codes (n, runs(k)) and scales stand for, float64."""
    n, length = codes.shape
    s = scales.astype(np.float64).T.repeat(block, axis=0)[:n].repeat(RUN, axis=1)[:, :length]
    return VALUES[codes] * s


def random_matrix(rng, columns, length, block):
    """Codes as quantising gives them for normal values, and scales of any kind: (codes, scales, values (columns, length))."""
    codes, scales = quantize(rng.standard_normal((columns, length)), block)
    scales = (scales * rng.uniform(0.5, 2.0, scales.shape)).astype(np.float32)
    return codes, scales, values(codes, scales, block)[:, :length]


def to_device(ctx, codes, scales, ld, lds):
    """With leading dimensions ld and lds; what is past the last run of 128 and the last column block is NaN."""
    c = np.full((codes.shape[0], ld), 0x7F, np.uint8)
    c[:, :codes.shape[1]] = codes
    s = np.full((scales.shape[0], lds), np.nan, np.float32)
    s[:, :scales.shape[1]] = scales
    return ctx.upload(c), ctx.upload(s)
