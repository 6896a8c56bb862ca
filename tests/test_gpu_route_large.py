"""Routing of many tokens: scores too near to tell in fp32, and rows of more than the caches hold, at whole dwords and
between them; the bounds are tests/test_gpu_route.py's."""
import numpy as np
import pytest

from tests import ragged as R
from tests import routing as Q
from tests.test_gpu_route import run_route
from wgblas_amd import SIGMOID, SOFTMAX  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,topk,groups,top_groups,best", [(128, 8, 1, 1, 1), (256, 8, 8, 4, 2), (384, 6, 1, 1, 1)])
def test_many_tokens_near_each_other(ctx, t, scoring, experts, topk, groups, top_groups, best):
    """Logits within 1e-6 of one value and a bias of a few steps: fp32 scores tie, float64 ones decide."""
    rng = np.random.default_rng(experts)
    n = 700
    logits = 0.3 + 1e-6 * rng.integers(-3, 4, (n, experts))
    logits[n // 2:] = rng.standard_normal((n - n // 2, experts))
    stored = R.encode(logits, t)
    bias = (1e-7 * rng.integers(-2, 3, experts)).astype(np.float32)
    ids, _ = run_route(ctx, stored, t, experts, scoring, topk, bias, groups, top_groups, best)
    want, _ = Q.route(R.decode(stored, t), scoring, topk, bias.astype(np.float64), groups, top_groups, best)
    assert np.array_equal(ids, want)


BIG = [(2101, 1100, 8), (4096, 600, 7)]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,n,topk", BIG)
@pytest.mark.parametrize("pad", [0, 1])
def test_rows_past_the_caches(ctx, t, d, n, topk, pad):
    rng = np.random.default_rng(d + pad)
    places = rng.permutation(n * topk).astype(np.int32).reshape(n, topk)
    places[rng.random((n, topk)) < 0.1] = -1
    w = rng.standard_normal((n, topk)).astype(np.float32)
    there = places >= 0
    ld = d + pad
    x, dc = (R.encode(rng.standard_normal((n, ld)), t) for _ in range(2))
    old = R.encode(rng.standard_normal((n * topk, ld)), t)
    kind = R.TYPES[t]
    dX, dDC, dP, dW, dY = (ctx.upload(v) for v in (x, dc, places, w, old))
    # gather, weighted: fp32 products of the row and its weight, rounded to the type
    ctx.route_gather(kind, d, n, topk, dX, ld, dP, dW, dY, ld)
    token, slot = np.nonzero(there)
    want = old.copy()
    rows = R.decode(x[:, :d], t).astype(np.float32)[token] * w[token, slot][:, None]
    want[places[token, slot], :d] = R.encode(rows.astype(np.float64), t)
    assert np.array_equal(dY.to_host().view(np.uint8), want.view(np.uint8))
    # combine those rows again
    terms = np.where(there[:, :, None], R.decode(want, t)[np.where(there, places, 0)][:, :, :d], 0.0) * w[:, :, None].astype(np.float64)
    dC = ctx.upload(np.zeros((n, ld), R.STORE[t]))
    ctx.route_combine(kind, d, n, topk, dY, ld, dP, dW, 0.0, dC, ld, kind)
    raw = dC.to_host()
    R.assert_product(R.decode(raw, t)[:, :d], terms.sum(1), np.abs(terms).sum(1), topk, t)
    assert not raw[:, d:].any()
    # and its gradient, in place
    dw = ctx.empty((n, topk), np.float32)
    ctx.route_combine_grad(kind, d, n, topk, dDC, ld, dY, ld, dP, dW, dY, ld, dw)
    g = R.decode(dc, t)[:, None, :d]
    terms = np.where(there[:, :, None], R.decode(want, t)[np.where(there, places, 0)][:, :, :d], 0.0) * g
    R.assert_product(dw.to_host().astype(np.float64), terms.sum(2), np.abs(terms).sum(2), d, "f32")
    rows = R.decode(dc[:, :d], t).astype(np.float32)[token] * w[token, slot][:, None]
    want[places[token, slot], :d] = R.encode(rows.astype(np.float64), t)
    assert np.array_equal(dY.to_host().view(np.uint8), want.view(np.uint8))
    for v in (dX, dDC, dP, dW, dY, dC, dw):
        v.free()


@pytest.mark.parametrize("experts,n,topk,missing", [(256, 20000, 8, 0.2), (1024, 5001, 3, 0.0), (1, 70000, 1, 0.5)])
def test_order_of_many(ctx, experts, n, topk, missing):
    rng = np.random.default_rng(n)
    ids = (rng.zipf(1.3, (n, topk)) % experts).astype(np.int32)
    ids[rng.random((n, topk)) < missing] = -1
    offsets, places, pairs = ctx.empty(experts + 1, np.int64), ctx.empty((n, topk), np.int32), ctx.empty(n * topk, np.int32)
    dI = ctx.upload(ids)
    ctx.route_order(experts, n, topk, dI, offsets, places, pairs)
    for got, want in zip((offsets, places, pairs), Q.order(ids, experts)):
        assert np.array_equal(got.to_host(), want)
    for v in (offsets, places, pairs, dI):
        v.free()
