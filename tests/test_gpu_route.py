"""Routing to experts: choices and order exactly, weights, gradients and moved rows against float64.

Bounds. A score is an exponential of a rounded difference, a sum of up to 1024 of them and a division: the difference
|l - max| <= D is off by 2^-24 D, the exponential by 2 units, the sum (each addend off alike) by 10 roundings (4 lanes'
worth of 16 in a row, then a tree: at most 16 + 6), so a relative 2^-24 (2 D + 2 * 2 + 22 + 2); renormalising adds a sum of
at most 64 of them (4 in a row and a tree of 6) and a division, scale a product."""
import numpy as np
import pytest

from tests import ragged as R
from tests import routing as Q
from wgblas_amd import SIGMOID, SOFTMAX

pytestmark = pytest.mark.gpu

SCORING = {"softmax": SOFTMAX, "sigmoid": SIGMOID}
STEP = 2.0 ** -24


def padded(x, pad, t, fill=np.nan):
    full = np.full((x.shape[0], x.shape[1] + pad), fill)
    full[:, :x.shape[1]] = x
    return R.encode(full, t)


def run_route(ctx, stored, t, experts, scoring, topk, bias=None, groups=1, top_groups=1, best=1, renorm=0, scale=1.0):
    n = stored.shape[0]
    d, b = ctx.upload(stored), None if bias is None else ctx.upload(bias.astype(np.float32))
    ids, w = ctx.upload(np.full((n, topk), 99, np.int32)), ctx.upload(np.full((n, topk), np.nan, np.float32))
    ctx.route(R.TYPES[t], SCORING[scoring], experts, n, topk, d, stored.shape[1], b, groups, top_groups, best, renorm, scale,
              ids, w)
    out = ids.to_host(), w.to_host()
    for x in (d, b, ids, w):
        if x is not None:
            x.free()
    return out


def weight_bound(logits, experts):
    finite = np.where(np.isfinite(logits), logits, 0.0)
    spread = finite.max(axis=1) - finite.min(axis=1)
    return STEP * (2 * np.maximum(spread, np.abs(finite).max(axis=1)) + 48)[:, None]


CASES = [  # experts, n, topk, scoring, bias, groups, top_groups, best
    (1, 3, 1, "softmax", False, 1, 1, 1), (2, 70, 2, "sigmoid", True, 1, 1, 1), (8, 33, 2, "softmax", False, 1, 1, 1),
    (16, 17, 16, "sigmoid", False, 1, 1, 1), (17, 100, 3, "softmax", True, 1, 1, 1), (60, 129, 6, "softmax", False, 1, 1, 1),
    (64, 300, 8, "softmax", False, 8, 3, 1), (64, 50, 8, "sigmoid", True, 8, 4, 2), (96, 40, 6, "softmax", False, 4, 1, 2),
    (160, 64, 6, "softmax", False, 8, 3, 1), (256, 200, 8, "sigmoid", True, 8, 4, 2), (256, 30, 64, "softmax", False, 1, 1, 1),
    (264, 31, 8, "sigmoid", True, 33, 5, 2), (384, 65, 8, "sigmoid", True, 1, 1, 1), (512, 9, 10, "softmax", False, 64, 7, 2),
    (1000, 5, 64, "sigmoid", True, 8, 2, 1), (1024, 6, 3, "softmax", False, 1, 1, 1), (63, 40, 2, "sigmoid", False, 63, 2, 2),
]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("renorm,scale,pad", [(0, 1.0, 0), (1, 2.5, 3)])
@pytest.mark.parametrize("experts,n,topk,scoring,bias,groups,top_groups,best", CASES)
def test_route(ctx, t, renorm, scale, pad, experts, n, topk, scoring, bias, groups, top_groups, best):
    """16-bit logits are equal often: the lowest expert goes first."""
    rng = np.random.default_rng(experts + n)
    stored = padded(rng.standard_normal((n, experts)) * 2.0, pad, t)
    logits = R.decode(stored, t)[:, :experts]
    b = (0.1 * rng.standard_normal(experts)).astype(np.float32) if bias else None
    ids, w = run_route(ctx, stored, t, experts, scoring, topk, b, groups, top_groups, best, renorm, scale)
    want, weights = Q.route(logits, scoring, topk, None if b is None else b.astype(np.float64), groups, top_groups, best,
                            renorm, scale)
    assert np.array_equal(ids, want)
    assert (np.abs(w - weights) <= weight_bound(logits, experts) * 2 * np.abs(weights)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,topk,groups,top_groups,best", [(8, 4, 1, 1, 1), (64, 6, 8, 2, 2), (300, 5, 1, 1, 1),
                                                                 (600, 5, 4, 2, 1)])
@pytest.mark.parametrize("bias", [False, True])
def test_masks_and_special_values(ctx, scoring, experts, topk, groups, top_groups, best, bias):
    """Rows that a mask leaves empty or nearly so, Infs and NaNs, all experts equal."""
    rng = np.random.default_rng(experts)
    x = rng.standard_normal((12, experts))
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, experts - 1] = 0.5
    x[2, ::2] = -np.inf
    x[3] = 0.0
    x[4, 3] = np.nan
    x[5] = np.nan
    x[6, 2] = np.inf
    x[7, [1, 4]] = np.inf
    x[8] = -3e38
    x[9] = 3e38
    x[10, topk // 2:] = -np.inf
    x[11, 1] = np.finfo(np.float32).min
    x = x.astype(np.float32)
    b = (0.1 * rng.standard_normal(experts)).astype(np.float32) if bias else None
    if bias:
        b[experts // 2] = -np.inf
    for renorm in (0, 1):
        ids, w = run_route(ctx, x, "f32", experts, scoring, topk, b, groups, top_groups, best, renorm)
        with np.errstate(invalid="ignore", over="ignore"):
            want, weights = Q.route(x.astype(np.float64), scoring, topk, None if b is None else b.astype(np.float64), groups,
                                    top_groups, best, renorm)
        assert np.array_equal(ids, want)
        assert np.array_equal(np.isnan(w), np.isnan(weights))
        fine = ~np.isnan(weights)
        assert (np.abs(w - weights)[fine] <= 2.0 ** -17 * np.abs(weights)[fine]).all()


def test_values_next_to_each_other(ctx):
    """Choice values that differ by less than fp32 holds: the order is that of 64 bits."""
    rng = np.random.default_rng(0)
    experts, n = 32, 200
    x = rng.standard_normal((n, experts)).astype(np.float32)
    p = Q.scores(x, "sigmoid")
    b = (0.5 - p[0]).astype(np.float32)  # token 0: all choice values within a few 2^-25 of each other
    for token in range(1, n):
        x[token] = np.nextafter(x[0], np.where(rng.random(experts) < 0.5, -np.inf, np.inf)).astype(np.float32)
    ids, _ = run_route(ctx, x, "f32", experts, "sigmoid", 8, b)
    choice = Q.scores(x, "sigmoid") + b.astype(np.float64)
    assert (np.ptp(choice, axis=1) < 2.0 ** -22).all()
    gaps = np.abs(np.diff(np.sort(choice, axis=1), axis=1))
    sure = gaps.min(axis=1) > 1e-13  # what two float64 evaluations may differ by is far less
    assert sure.sum() > 100
    want = Q.route(x.astype(np.float64), "sigmoid", 8, b.astype(np.float64))[0]
    assert np.array_equal(ids[sure], want[sure])


@pytest.mark.parametrize("experts,n,topk", [(1, 1, 1), (8, 1, 2), (64, 16, 8), (5, 300, 1), (256, 128, 8), (256, 129, 8),
                                            (1024, 700, 3), (3, 5000, 2), (384, 40000, 8), (60, 4097, 6), (16, 0, 2)])
@pytest.mark.parametrize("missing", [0.0, 0.3, 1.0])
def test_order(ctx, experts, n, topk, missing):
    rng = np.random.default_rng(n)
    ids = rng.integers(0, experts, (n, topk)).astype(np.int32)
    ids[rng.random((n, topk)) < missing] = -1
    if n > 4 and missing == 0.3:
        ids[0, 0], ids[1, 0], ids[2, 0] = experts, 2 ** 31 - 1, -2 ** 31  # outside: no place
    d = ctx.upload(ids)
    off = ctx.upload(np.full(experts + 1, -7, np.int64))
    places, pairs = (ctx.upload(np.full(n * topk + 4, 77, np.int32)) for _ in range(2))
    ctx.route_order(experts, n, topk, d, off, places, pairs)
    offsets, want_places, want_pairs = Q.order(ids, experts)
    assert np.array_equal(off.to_host(), offsets)
    assert np.array_equal(places.to_host()[:n * topk], want_places.reshape(-1)) and (places.to_host()[n * topk:] == 77).all()
    assert np.array_equal(pairs.to_host()[:n * topk], want_pairs) and (pairs.to_host()[n * topk:] == 77).all()
    for x in (d, off, places, pairs):
        x.free()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm,scale,pad", [(0, 1.0, 0), (1, 2.5, 3)])
@pytest.mark.parametrize("experts,n,topk", [(1, 2, 1), (8, 33, 2), (17, 40, 17), (64, 100, 8), (128, 9, 8), (250, 20, 6),
                                            (300, 5, 64), (1024, 3, 4)])
def test_route_grad(ctx, t, scoring, renorm, scale, pad, experts, n, topk):
    rng = np.random.default_rng(experts)
    stored = padded(rng.standard_normal((n, experts)), pad, t)
    logits = R.decode(stored, t)[:, :experts]
    if n > 4:  # masked experts and slots without one
        logits = logits.copy()
        logits[3] = -np.inf
        logits[4, 1:] = -np.inf
        stored[:, :experts] = R.encode(logits, t)
    ids, _ = Q.route(logits, scoring, topk, renorm=renorm)
    dw = rng.standard_normal((n, topk)).astype(np.float32)
    dL, dI, dW = ctx.upload(stored), ctx.upload(ids), ctx.upload(dw)
    out = ctx.upload(padded(np.full((n, experts), 5.0), pad, t, fill=5.0))
    ctx.route_grad(R.TYPES[t], SCORING[scoring], experts, n, topk, dL, experts + pad, dI, renorm, scale, dW, out, experts + pad)
    got = R.decode(out.to_host(), t)
    want = Q.grad(logits, scoring, ids, dw.astype(np.float64), renorm, scale)
    # every term of a logit's gradient is a product of scores (each off as a weight is), of dw and of 1 / S, S >= the
    # largest score; the terms are of the size of the sum of |dw| p / S
    p = Q.scores(logits, scoring)
    chosen = np.where(ids < 0, 0.0, np.take_along_axis(p, np.maximum(ids, 0), 1))
    total = chosen.sum(axis=1, keepdims=True) if renorm else np.ones((n, 1))
    total = np.where(total == 0, 1.0, total)
    size = scale * ((np.abs(dw) * chosen).sum(axis=1, keepdims=True) / total + np.abs(dw).max(axis=1, keepdims=True)) / total * p
    bound = 8 * weight_bound(logits, experts) * size
    assert (np.abs(got[:, :experts] - want) <= bound + np.abs(want) * R.HALF_UNIT[t] + (2.0 ** -25 if t == "f16" else 2.0 ** -149)).all()
    assert (got[:, experts:] == 5.0).all()
    for x in (dL, dI, dW, out):
        x.free()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
def test_route_grad_against_differences(ctx, scoring, renorm):
    """Central differences of the weights that the forward call itself gives, in float64 of its definition."""
    rng = np.random.default_rng(2)
    experts, n, topk = 12, 3, 4
    x = rng.standard_normal((n, experts)).astype(np.float32)
    ids, _ = run_route(ctx, x, "f32", experts, scoring, topk, renorm=renorm)
    dw = rng.standard_normal((n, topk)).astype(np.float32)
    out = ctx.empty((n, experts), np.float32)
    ctx.route_grad(R.TYPES["f32"], SCORING[scoring], experts, n, topk, ctx.upload(x), experts, ctx.upload(ids), renorm, 1.0,
                   ctx.upload(dw), out, experts)
    got, h = out.to_host(), 1e-4

    def value(z, token):
        p = Q.scores(z, scoring)[token, ids[token]]
        return float((dw[token] * (p / p.sum() if renorm else p)).sum())

    for token in range(n):
        for e in range(experts):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[token, e] += h
            down[token, e] -= h
            # the third derivative of these functions is below 1 here: h^2 / 6 and the gradient's own rounding
            assert abs((value(up, token) - value(down, token)) / (2 * h) - got[token, e]) < 4e-6


def test_the_same_expert_twice(ctx):
    """ids that a caller made: an expert's gradients add up, in the slots' order."""
    x = np.array([[0.3, -1.0, 2.0, 0.1]], np.float32)
    ids = np.array([[2, 2, 0, 2]], np.int32)
    dw = np.array([[1.0, 0.5, -2.0, 0.25]], np.float32)
    for scoring in ("softmax", "sigmoid"):
        out = ctx.empty((1, 4), np.float32)
        ctx.route_grad(R.TYPES["f32"], SCORING[scoring], 4, 1, 4, ctx.upload(x), 4, ctx.upload(ids), 0, 1.0, ctx.upload(dw), out, 4)
        want = Q.grad(x.astype(np.float64), scoring, ids, dw.astype(np.float64))
        assert (np.abs(out.to_host() - want) <= 2.0 ** -20 * np.abs(dw).sum()).all()


ROWS = [(1, 1, 1), (2, 3, 2), (8, 33, 3), (64, 100, 8), (257, 9, 6), (1000, 40, 1), (4096, 17, 9), (5000, 3, 64), (33, 700, 2)]


def move_inputs(rng, n, topk, missing):
    places = rng.permutation(n * topk).astype(np.int32).reshape(n, topk)
    places[rng.random((n, topk)) < missing] = -1
    if n > 2 and missing:
        places[0, 0], places[1, 0] = n * topk, 2 ** 31 - 1  # outside: skipped
    return places, rng.standard_normal((n, topk)).astype(np.float32)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,n,topk", ROWS)
@pytest.mark.parametrize("pad,missing", [(0, 0.0), (3, 0.3)])
def test_gather(ctx, t, d, n, topk, pad, missing):
    rng = np.random.default_rng(d)
    places, w = move_inputs(rng, n, topk, missing)
    x = padded(rng.standard_normal((n, d)), pad, t)
    dX, dP, dW = ctx.upload(x), ctx.upload(places), ctx.upload(w)
    there = (places >= 0) & (places < n * topk)
    for weighted in (False, True):
        host = R.encode(rng.standard_normal((n * topk, d + pad)), t)
        dY = ctx.upload(host)
        ctx.route_gather(R.TYPES[t], d, n, topk, dX, d + pad, dP, dW if weighted else None, dY, d + pad)
        want = host.copy()
        for token, slot in np.argwhere(there):
            row = R.decode(x[token, :d], t)
            # a product of two fp32 numbers rounds once to fp32, then to the type
            row = (row.astype(np.float32) * w[token, slot]).astype(np.float64) if weighted else row
            want[places[token, slot], :d] = R.encode(row, t)
        assert np.array_equal(dY.to_host().view(np.uint8), want.view(np.uint8))
        dY.free()
    for v in (dX, dP, dW):
        v.free()


@pytest.mark.parametrize("t,ct", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("d,n,topk", ROWS)
@pytest.mark.parametrize("pad,missing,beta", [(0, 0.0, 0.0), (3, 0.3, -0.5), (0, 1.0, 0.0)])
def test_combine(ctx, t, ct, d, n, topk, pad, missing, beta):
    rng = np.random.default_rng(d + 1)
    places, w = move_inputs(rng, n, topk, missing)
    y = padded(rng.standard_normal((n * topk, d)), pad, t)
    there = (places >= 0) & (places < n * topk)
    rows = np.where(there[:, :, None], R.decode(y, t)[np.where(there, places, 0)][:, :, :d], 0.0)
    dY, dP, dW = ctx.upload(y), ctx.upload(places), ctx.upload(w)
    for weighted in (False, True):
        host = R.encode(rng.standard_normal((n, d + pad)) if beta else np.full((n, d + pad), np.nan), ct)
        dC = ctx.upload(host)
        ctx.route_combine(R.TYPES[t], d, n, topk, dY, d + pad, dP, dW if weighted else None, beta, dC, d + pad, R.TYPES[ct])
        raw = dC.to_host()
        terms = rows * (w.astype(np.float64)[:, :, None] if weighted else 1.0)
        R.assert_product(R.decode(raw, ct)[:, :d], terms.sum(1), np.abs(terms).sum(1), topk, ct, 1.0, beta,
                         R.decode(host, ct)[:, :d])
        assert np.array_equal(raw[:, d:].tobytes(), host[:, d:].tobytes())
        dC.free()
    for v in (dY, dP, dW):
        v.free()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,n,topk", ROWS)
@pytest.mark.parametrize("pad,missing,in_place", [(0, 0.0, False), (3, 0.3, True)])
def test_combine_grad(ctx, t, d, n, topk, pad, missing, in_place):
    rng = np.random.default_rng(d + 2)
    places, w = move_inputs(rng, n, topk, missing)
    y, dc = padded(rng.standard_normal((n * topk, d)), pad, t), padded(rng.standard_normal((n, d)), pad, t)
    there = (places >= 0) & (places < n * topk)
    dY, dP, dW, dC = ctx.upload(y), ctx.upload(places), ctx.upload(w), ctx.upload(dc)
    out = dY if in_place else ctx.upload(y)
    dw = ctx.upload(np.full((n, topk), np.nan, np.float32))
    ctx.route_combine_grad(R.TYPES[t], d, n, topk, dC, d + pad, dY, d + pad, dP, dW, out, d + pad, dw)
    want = y.copy()
    for token, slot in np.argwhere(there):
        row = (R.decode(dc[token, :d], t).astype(np.float32) * w[token, slot]).astype(np.float64)
        want[places[token, slot], :d] = R.encode(row, t)
    assert np.array_equal(out.to_host().view(np.uint8), want.view(np.uint8))
    rows = np.where(there[:, :, None], R.decode(y, t)[np.where(there, places, 0)][:, :, :d], 0.0)
    terms = rows * R.decode(dc, t)[:, None, :d]
    R.assert_product(dw.to_host().astype(np.float64), terms.sum(2), np.abs(terms).sum(2), d, "f32")
    for v in {dY, dP, dW, dC, out, dw}:
        v.free()
