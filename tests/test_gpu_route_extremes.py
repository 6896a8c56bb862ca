"""Routing where fp32 numbers lose what the definition needs: groups whose two best values nearly cancel, scores far below
fp32's range that are divided by their sum, one expert that has nearly all of the softmax, ids that a bias chose. Against
float64 by the definition (tests/routing.py) and by sums that do not cancel (tests/routing_gradient.py).

Bounds. A weight is off by a relative W = 2 weight_bound (tests/test_gpu_route.py). A logit's gradient is a sum of products
of two scores or weights, the complement of one, and a difference of two of what came back: it is within (3 W + (slots + 8)
2^-24) of the sum of the terms' magnitudes (each term's difference, products and place in the sum round once)."""
import numpy as np
import pytest

from tests import ragged as R
from tests import routing as Q
from tests import routing_gradient as G
from tests.test_gpu_route import SCORING, STEP, run_route, weight_bound

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -149  # a step of fp32's subnormals
SMALLEST = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the type's


# ---- the choice ----------------------------------------------------------------------


def group_gaps(choice, groups, top_groups):
    """How far the last kept group's score (the sum of its two best) is from the next one's."""
    best = np.sort(np.sort(choice.reshape(len(choice), groups, -1), axis=2)[:, :, -2:].sum(2), axis=1)
    return best[:, groups - top_groups] - best[:, groups - top_groups - 1]


@pytest.mark.parametrize("experts,groups,top_groups", [(16, 8, 4), (24, 8, 3), (64, 4, 1), (256, 8, 4), (528, 33, 10), (1024, 64, 7)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [1e3, 1e4, 1e6])
def test_groups_whose_two_best_nearly_cancel(ctx, experts, groups, top_groups, scoring, size):
    """One expert of a group has a bias near `size`, the others one near -size: the sum is of the size of the scores, its
    terms' roundings are not."""
    rng = np.random.default_rng(experts)
    n, per = 64000 // experts, experts // groups
    x = rng.standard_normal((n, experts)).astype(np.float32)
    b = (-size + 0.1 * rng.standard_normal(experts)).astype(np.float32)
    first = np.arange(groups) * per + rng.integers(0, per, groups)
    b[first] = (size + 0.1 * rng.standard_normal(groups)).astype(np.float32)
    choice = Q.scores(x, scoring) + b.astype(np.float64)
    sure = group_gaps(choice, groups, top_groups) > 1e-9  # a float64 value of 1e6 is rounded at 1.2e-10
    assert sure.mean() > 0.99
    ids, _ = run_route(ctx, x, "f32", experts, scoring, top_groups, b, groups, top_groups, 2)
    # the top_groups largest values are the kept groups' first experts: their order is not the question here
    want, _ = Q.route(x[sure].astype(np.float64), scoring, top_groups, b.astype(np.float64), groups, top_groups, 2)
    assert np.array_equal(np.sort(ids[sure], axis=1), np.sort(want, axis=1))


def test_groups_whose_sums_leave_fp32(ctx):
    """The two best values' sum is past fp32's largest number, of either sign."""
    experts, groups = 12, 4
    b = np.zeros(experts, np.float32)
    b[[0, 1, 3, 4]] = 3.0e38
    b[1] = 2.9e38
    b[[6, 7, 8]] = -3.0e38
    b[[9, 10, 11]] = -3.1e38
    x = np.random.default_rng(0).standard_normal((40, experts)).astype(np.float32)
    for top_groups in (1, 2, 3):
        topk = 3 * top_groups
        ids, _ = run_route(ctx, x, "f32", experts, "sigmoid", topk, b, groups, top_groups, 2)
        want, _ = Q.route(x.astype(np.float64), "sigmoid", topk, b.astype(np.float64), groups, top_groups, 2)
        # values of 3e38 that differ by a score are one value in float64: the lowest goes first
        assert np.array_equal(ids, want), top_groups


@pytest.mark.parametrize("experts", [8, 12])
def test_groups_with_nan_come_after_numbers(ctx, experts):
    """Also after numbers far below zero, and the lowest group of those with a NaN first."""
    groups, per = 4, experts // 4
    b = np.full(experts, -1.0e35, np.float32)
    b[per:2 * per] = [0.0] + [np.nan] * (per - 1)  # its second best is NaN
    b[2 * per:3 * per] = [1.0] + [np.nan] * (per - 1)
    b[3 * per:] = -2.0e35
    x = np.random.default_rng(0).standard_normal((5, experts)).astype(np.float32)
    for top_groups in (1, 2, 3):
        ids, _ = run_route(ctx, x, "f32", experts, "sigmoid", per, b, groups, top_groups, 2)
        want, _ = Q.route(x.astype(np.float64), "sigmoid", per, b.astype(np.float64), groups, top_groups, 2)
        assert np.array_equal(ids, want), top_groups


# ---- weights and their gradients -------------------------------------------------------


def run_grad(ctx, x, t, scoring, ids, dw, renorm, scale=1.0):
    n, experts = x.shape
    dL, dI, dW = ctx.upload(R.encode(x, t)), ctx.upload(ids), ctx.upload(dw)
    out = ctx.empty((n, experts), R.STORE[t])
    ctx.route_grad(R.TYPES[t], SCORING[scoring], experts, n, ids.shape[1], dL, experts, dI, renorm, scale, dW, out, experts)
    got = R.decode(out.to_host(), t)
    for d in (dL, dI, dW, out):
        d.free()
    return got


def check_grad(ctx, x, t, scoring, ids, dw, renorm, scale=1.0):
    x = R.decode(R.encode(x, t), t)
    got = run_grad(ctx, x, t, scoring, ids, dw, renorm, scale)
    want, size = G.grad(x, scoring, ids, dw.astype(np.float64), renorm, scale)
    bound = (3 * 2 * weight_bound(x, x.shape[1]) + (ids.shape[1] + 8) * STEP) * size
    # the result's own rounding, and some of fp32's steps where it or a score is subnormal
    bound += np.abs(want) * R.HALF_UNIT[t] + SMALLEST[t] + 8 * LEAST * max(np.abs(dw).max(), 1.0) * max(scale, 1.0)
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= bound).all(), (np.argwhere(~(off <= bound))[0], np.nanmax(off / bound))


LEVELS = [-60.0, -80.0, -86.5, -88.5, -95.0, -104.0, -120.0, -300.0, -700.0]


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("experts,topk", [(8, 2), (60, 6), (384, 8), (64, 64)])
def test_weights_of_small_sigmoids(ctx, level, experts, topk):
    rng = np.random.default_rng(experts)
    x = (level + rng.standard_normal((30, experts))).astype(np.float32)
    x[:4, ::2] = -np.inf
    for renorm, scale in ((1, 2.5), (0, 1.0)):
        ids, w = run_route(ctx, x, "f32", experts, "sigmoid", topk, renorm=renorm, scale=scale)
        want, weights = Q.route(x.astype(np.float64), "sigmoid", topk, renorm=renorm, scale=scale)
        assert np.array_equal(ids, want)
        # without the sum's division the scores themselves may be subnormal: an exponential and a quotient of that size
        assert (np.abs(w - weights) <= weight_bound(x, experts) * 2 * np.abs(weights) + (0.0 if renorm else 4 * LEAST)).all()


@pytest.mark.parametrize("ahead", [20.0, 80.0, 87.5, 95.0, 104.0, 150.0, 700.0])
@pytest.mark.parametrize("experts,topk,groups", [(16, 4, 1), (64, 6, 8), (600, 5, 1)])
def test_weights_of_experts_far_below_the_largest(ctx, ahead, experts, topk, groups):
    """A bias keeps the largest logits from being chosen: the others' softmax scores are divided by their own sum."""
    rng = np.random.default_rng(experts)
    x = rng.standard_normal((30, experts)).astype(np.float32)
    b = np.zeros(experts, np.float32)
    x[:, 1] += ahead
    b[1] = -100.0
    b[3:] = rng.permutation(experts - 3) / np.float32(experts)  # so far apart that the small scores do not decide
    if groups > 1:
        b[:experts // groups] = -100.0
    ids, w = run_route(ctx, x, "f32", experts, "softmax", topk, b, groups, max(1, groups // 2), 1, renorm=1)
    want, weights = Q.route(x.astype(np.float64), "softmax", topk, b.astype(np.float64), groups, max(1, groups // 2), 1, renorm=1)
    assert np.array_equal(ids, want) and (ids != 1).all()
    # only differences of the logits and of the largest chosen one enter; the bound counts those from the largest of all
    assert (np.abs(w - weights) <= weight_bound(x, experts) * 2 * np.abs(weights)).all()
    dw = rng.standard_normal((30, topk)).astype(np.float32)
    check_grad(ctx, x, "f32", "softmax", ids, dw, 1, 2.5)


def test_scores_that_64_bits_hold_as_zero(ctx):
    """Masks of the type's lowest value: no weight, as -Inf, where others are left and where none is."""
    low = np.finfo(np.float32).min
    x = np.full((3, 8), low, np.float32)
    x[1, 2], x[2, [0, 5]] = -90.0, [-1.0, -700.0]
    for t in ("f32", "bf16"):
        stored = R.encode(np.maximum(x, -3.38e38), t)
        for renorm in (0, 1):
            ids, w = run_route(ctx, stored, t, 8, "sigmoid", 3, renorm=renorm)
            want, weights = Q.route(R.decode(stored, t), "sigmoid", 3, renorm=renorm)
            assert np.array_equal(ids, want)
            assert (np.abs(w - weights) <= 2.0 ** -17 * np.abs(weights) + 4 * LEAST).all()
            check_grad(ctx, R.decode(stored, t), t, "sigmoid", want, np.full((3, 3), 1.5, np.float32), renorm)
    b = np.zeros(8, np.float32)
    b[2] = -5.0
    x[1, 2] = 1.0
    ids, w = run_route(ctx, x, "f32", 8, "softmax", 3, b, renorm=1)
    assert np.array_equal(ids[1], [0, 1, 3]) and (w[1] == 0.0).all()  # expert 2 has all of the softmax
    assert (np.abs(w[0] - 1 / 3) <= 2.0 ** -22).all()  # all alike


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("experts,topk", [(8, 2), (60, 6), (300, 64)])
def test_gradient_of_small_sigmoids(ctx, t, level, experts, topk):
    rng = np.random.default_rng(experts)
    x = R.decode(R.encode(level + rng.standard_normal((30, experts)), t), t)
    x[:4, ::2] = -np.inf
    dw = (3.0 * rng.standard_normal((30, topk))).astype(np.float32)
    for renorm, scale in ((1, 1.0), (1, 2.5), (0, 1.0)):
        ids, _ = Q.route(x, "sigmoid", topk, renorm=renorm)
        check_grad(ctx, x, t, "sigmoid", ids, dw, renorm, scale)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm,scale", [(0, 1.0), (0, 2.5), (1, 2.5)])
@pytest.mark.parametrize("ahead", [0.0, 6.0, 12.0, 16.0, 20.0, 40.0, 100.0])
@pytest.mark.parametrize("experts,topk", [(8, 1), (8, 8), (60, 6), (128, 8), (600, 33)])
def test_gradient_of_a_dominating_expert(ctx, t, scoring, renorm, scale, ahead, experts, topk):
    """One logit far ahead: its score is nearly 1, its gradient what the others leave."""
    rng = np.random.default_rng(experts + topk)
    x = rng.standard_normal((20, experts))
    x[np.arange(20), rng.integers(0, experts, 20)] += ahead
    x = R.decode(R.encode(x, t), t)
    dw = rng.standard_normal((20, topk)).astype(np.float32)
    dw[5:10] = dw[5:10, :1] * (1 + 2.0 ** -12 * rng.standard_normal((5, topk)))  # nearly the same for all slots
    ids, _ = Q.route(x, scoring, topk)
    check_grad(ctx, x, t, scoring, ids, dw, renorm, scale)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("experts,topk,groups,top_groups", [(16, 4, 1, 1), (64, 6, 8, 2), (600, 5, 4, 1)])
@pytest.mark.parametrize("ahead", [0.0, 14.0, 60.0])
def test_gradient_of_what_a_bias_chose(ctx, scoring, renorm, experts, topk, groups, top_groups, ahead):
    """ids of the forward call with a bias and groups, of which the largest logit may not be one."""
    rng = np.random.default_rng(experts)
    x = rng.standard_normal((40, experts)).astype(np.float32)
    x[:, 3] += ahead
    b = rng.standard_normal(experts).astype(np.float32)
    b[3] = -3.0
    ids, _ = run_route(ctx, x, "f32", experts, scoring, topk, b, groups, top_groups, 2, renorm)
    want, _ = Q.route(x.astype(np.float64), scoring, topk, b.astype(np.float64), groups, top_groups, 2, renorm)
    assert np.array_equal(ids, want)
    dw = rng.standard_normal((40, topk)).astype(np.float32)
    check_grad(ctx, x, "f32", scoring, ids, dw, renorm, 2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
def test_gradient_of_an_expert_that_is_there_twice(ctx, scoring, renorm):
    """ids that a caller made, some of no expert: the slots' gradients add up, also where one expert has nearly all."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 20)).astype(np.float32)
    x[::2, 4] += 15.0
    ids = rng.integers(-1, 6, (50, 7)).astype(np.int32)
    ids[7, 2], ids[8, 0], ids[9] = 20, 2 ** 31 - 1, -5
    dw = rng.standard_normal((50, 7)).astype(np.float32)
    check_grad(ctx, x, "f32", scoring, ids, dw, renorm, 1.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
def test_nan_gradients_stay_in_their_row(ctx, scoring, renorm):
    """A softmax with a NaN or an Inf has no scores, its row's gradients are NaN; a NaN sigmoid that is not chosen changes
    no other's."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 8)).astype(np.float32)
    x[1, 5], x[2, 0] = np.nan, np.inf
    ids = np.array([[0, 1], [0, 1], [2, 1], [3, 4]], np.int32)
    dw = rng.standard_normal((4, 2)).astype(np.float32)
    got = run_grad(ctx, x, "f32", scoring, ids, dw, renorm)
    if scoring == "softmax":
        assert np.array_equal(np.isnan(got), np.isin(np.arange(4), [1, 2])[:, None].repeat(8, 1))
    else:
        got[1, 5] = 0.0  # of the NaN itself: 0 times its slope
        assert not np.isnan(got).any()
