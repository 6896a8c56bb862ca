"""A layer of experts, run as it is used: route, order, gather, quantise, product, combine, and back to the gradients of
its input, its router and its weights. Every step is checked against float64 of what the step read; the whole against
float64 without any 8-bit rounding, within what those roundings allow. In a captured graph, and from two contexts at
once, it gives the same bits."""
import ctypes
import threading

import numpy as np
import pytest

from tests import fp8 as F
from tests import ragged as R
from tests import routing as Q
from tests.test_gpu_fp8 import DROPPED
from wgblas_amd import NO_TRANS, SIGMOID, TRANS

pytestmark = pytest.mark.gpu

BF16, F32 = R.TYPES["bf16"], R.TYPES["f32"]


class Layer:
    """Weights of `experts` matrices out x inner in fp8 (128 x 128 scales), and room for n tokens."""

    def __init__(self, c, rng, n, experts, topk, inner, out, groups):
        self.c, self.n, self.experts, self.topk, self.inner, self.out, self.groups = c, n, experts, topk, inner, out, groups
        self.weights = R.encode(rng.standard_normal((experts, out, inner)) / np.sqrt(inner), "bf16")
        self.bias_host = (0.1 * rng.standard_normal(experts)).astype(np.float32)
        self.W, self.bias = c.upload(self.weights), c.upload(self.bias_host)
        rows, li, lo = n * topk, F.runs(inner), F.runs(out)
        self.rows, self.li, self.lo = rows, li, lo
        per = (out + 127) // 128  # an expert's column blocks
        self.Wc, self.Ws, self.per = c.empty((experts, out, li), np.uint8), c.empty((experts, li // 128, per), np.float32), per
        for e in range(experts):
            c.fp8_quantize(BF16, NO_TRANS, 128, inner, out, self.W.ptr + 2 * e * out * inner, inner,
                           self.Wc.ptr + e * out * li, li, self.Ws.ptr + 4 * e * (li // 128) * per, per)
        self.logits, self.x, self.dc = c.empty((n, experts), np.float32), c.empty((n, inner), np.uint16), c.empty((n, out), np.uint16)
        self.ids, self.w = c.empty((n, topk), np.int32), c.empty((n, topk), np.float32)
        self.offsets, self.places, self.pairs = c.empty(experts + 1, np.int64), c.empty((n, topk), np.int32), c.empty(rows, np.int32)
        self.xs, self.xc, self.xsc = c.empty((rows, inner), np.uint16), c.empty((rows, li), np.uint8), c.empty((li // 128, rows), np.float32)
        self.ys, self.y = c.empty((rows, out), np.uint16), c.empty((n, out), np.float32)
        self.dys, self.dw = c.empty((rows, out), np.uint16), c.empty((n, topk), np.float32)
        self.dyc, self.dysc = c.empty((rows, lo), np.uint8), c.empty((lo // 128, rows), np.float32)
        self.dxs, self.dx = c.empty((rows, inner), np.uint16), c.empty((n, inner), np.float32)
        self.dlogits, self.dW = c.empty((n, experts), np.float32), c.empty((experts, out, inner), np.float32)
        self.results = ("ids", "w", "offsets", "places", "y", "dw", "dx", "dlogits", "dW")

    def set(self, rng):
        for a, host in ((self.logits, rng.standard_normal((self.n, self.experts)).astype(np.float32)),
                        (self.x, R.encode(rng.standard_normal((self.n, self.inner)), "bf16")),
                        (self.dc, R.encode(rng.standard_normal((self.n, self.out)), "bf16"))):
            self.c.h2d(a.ptr, host)

    def run(self):
        c, n, e, topk, inner, out, rows, li, lo = (self.c, self.n, self.experts, self.topk, self.inner, self.out, self.rows,
                                                   self.li, self.lo)
        c.route(F32, SIGMOID, e, n, topk, self.logits, e, self.bias, self.groups, max(1, self.groups // 2), 1, 1, 2.5, self.ids, self.w)
        c.route_order(e, n, topk, self.ids, self.offsets, self.places, self.pairs)
        c.route_gather(BF16, inner, n, topk, self.x, inner, self.places, None, self.xs, inner)
        c.fp8_quantize(BF16, NO_TRANS, 1, inner, rows, self.xs, inner, self.xc, li, self.xsc, rows)
        c.fp8_gemm_grouped(TRANS, e, out, rows, inner, 1.0, self.Wc, li, out * li, 128, self.Ws, self.per, li // 128 * self.per,
                           self.xc, li, self.xsc, rows, self.offsets, 0.0, self.ys, out, BF16)
        c.route_combine(BF16, out, n, topk, self.ys, out, self.places, self.w, 0.0, self.y, out, F32)
        # back
        c.route_combine_grad(BF16, out, n, topk, self.dc, out, self.ys, out, self.places, self.w, self.dys, out, self.dw)
        c.route_grad(F32, SIGMOID, e, n, topk, self.logits, e, self.ids, 1, 2.5, self.dw, self.dlogits, e)
        c.fp8_quantize(BF16, NO_TRANS, 1, out, rows, self.dys, out, self.dyc, lo, self.dysc, rows)
        c.fp8_gemm_grouped(NO_TRANS, e, inner, rows, out, 1.0, self.Wc, li, out * li, 128, self.Ws, self.per, li // 128 * self.per,
                           self.dyc, lo, self.dysc, rows, self.offsets, 0.0, self.dxs, inner, BF16)
        c.route_combine(BF16, inner, n, topk, self.dxs, inner, self.places, None, 0.0, self.dx, inner, F32)
        c.gemm_grouped_k(BF16, e, inner, out, rows, 1.0, self.xs, inner, self.dys, out, self.offsets, 0.0, self.dW, inner,
                         out * inner, F32)

    def host(self, names=None):
        self.c.synchronize()
        return {k: getattr(self, k).to_host().copy() for k in names or self.results}

    def buffers(self):
        return [v for v in vars(self).values() if hasattr(v, "nbytes") and hasattr(v, "ptr")]


def code_error(x, codes, scales, block):
    """(values of the codes, how far they may be from x: half a step of a normal code or of a subnormal one)."""
    s = scales.astype(np.float64).T.repeat(block, axis=0)[:len(x)].repeat(F.RUN, axis=1)[:, :x.shape[1]]
    v = F.values(codes, scales, block)[:, :x.shape[1]]
    allowed = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s)
    assert (np.abs(v - x) <= allowed).all()
    return v, allowed


def grouped(off, B, A):
    return np.concatenate([B[off[g]:off[g + 1]] @ A[g] for g in range(len(A))])


@pytest.mark.parametrize("n,experts,topk,inner,out,groups", [(1, 8, 2, 256, 128, 1), (3, 16, 4, 130, 257, 4), (500, 8, 2, 384, 300, 1),
                                                             (300, 64, 6, 200, 136, 8)])
def test_the_whole_layer(ctx, n, experts, topk, inner, out, groups):
    rng = np.random.default_rng(n)
    layer = Layer(ctx, rng, n, experts, topk, inner, out, groups)
    layer.set(rng)
    # rows behind the last pair are never written; here every pair has a place
    layer.run()
    h = layer.host([k for k in vars(layer) if hasattr(getattr(layer, k), "to_host")])
    logits, w = h["logits"].astype(np.float64), h["w"].astype(np.float64)
    ids, _ = Q.route(logits, "sigmoid", topk, layer.bias_host.astype(np.float64), groups, max(1, groups // 2), 1, 1, 2.5)
    assert np.array_equal(h["ids"], ids)
    off, places, _ = Q.order(ids, experts)
    assert np.array_equal(h["offsets"], off) and np.array_equal(h["places"], places)
    x, dc = R.decode(h["x"], "bf16"), R.decode(h["dc"], "bf16")
    xs = np.zeros((n * topk, inner))
    xs[places.reshape(-1)] = x.repeat(topk, axis=0)
    assert np.array_equal(R.decode(h["xs"], "bf16"), xs)
    # what the codes stand for
    W = R.decode(layer.weights, "bf16").reshape(experts, out, inner)
    per = [code_error(W[e], h["Wc"][e], h["Ws"][e], 128) for e in range(experts)]
    Wq, We = (np.stack([p[i] for p in per]) for i in (0, 1))
    xq, xe = code_error(xs, h["xc"], h["xsc"], 1)
    # products
    Wt = Wq.transpose(0, 2, 1)
    exact, absdot = grouped(off, xq, Wt), grouped(off, np.abs(xq), np.abs(Wt))
    ys = R.decode(h["ys"], "bf16")
    R.assert_product(ys, exact, absdot, inner + DROPPED["bf16"] * 2.0 ** 23, "bf16")
    terms = ys[places] * w[:, :, None]
    R.assert_product(h["y"].astype(np.float64), terms.sum(1), np.abs(terms).sum(1), topk, "f32")
    # the whole without 8-bit roundings: theirs, the product's and bf16's, through the weights; (1 + 2^-8) covers the rest of the sum
    full = grouped(off, xs, W.transpose(0, 2, 1))
    Wa = np.abs(W).transpose(0, 2, 1)
    off_by = grouped(off, np.abs(xs), We.transpose(0, 2, 1)) + grouped(off, xe, Wa) + grouped(off, xe, We.transpose(0, 2, 1))
    off_by += (2.0 ** -8 + 2.0 ** -9) * absdot
    bound = (off_by[places] * np.abs(w)[:, :, None]).sum(1) * (1 + 2.0 ** -8)
    assert (np.abs(h["y"] - (full[places] * w[:, :, None]).sum(1)) <= bound).all()
    # back: rows' gradients, the weights', the logits'
    dys = np.zeros((n * topk, out))
    dys[places.reshape(-1)] = R.decode(R.encode((dc.astype(np.float32)[:, None] * h["w"][:, :, None]).astype(np.float64), "bf16"),
                                       "bf16").reshape(-1, out)
    assert np.array_equal(R.decode(h["dys"], "bf16"), dys)
    terms = ys[places] * dc[:, None]
    R.assert_product(h["dw"].astype(np.float64), terms.sum(2), np.abs(terms).sum(2), out, "f32")
    want = Q.grad(logits, "sigmoid", ids, h["dw"].astype(np.float64), 1, 2.5)
    # dl = 2.5 (dw / S - dot / S^2) p (1 - p), p <= S, so each term is at most 2.5 sum |dw|. In units of 2^-24 of itself a
    # score is off by 4, S by 4 + topk <= 10, dot by 4 + 2 topk <= 16, a quotient by 1 more, p (1 - p) scale by 11: the first
    # term by 10 + 1 + 11 = 22, the second by 16 + 20 + 2 + 11 = 49, their difference's rounding 1 each: 2.5 * 73 <= 2^8 units
    assert (np.abs(h["dlogits"] - want) <= 2.0 ** -16 * np.abs(h["dw"]).sum(1, keepdims=True)).all()
    dyq, _ = code_error(dys, h["dyc"], h["dysc"], 1)
    R.assert_product(R.decode(h["dxs"], "bf16"), grouped(off, dyq, Wq), grouped(off, np.abs(dyq), np.abs(Wq)),
                     out + DROPPED["bf16"] * 2.0 ** 23, "bf16")
    terms = R.decode(h["dxs"], "bf16")[places]
    R.assert_product(h["dx"].astype(np.float64), terms.sum(1), np.abs(terms).sum(1), topk, "f32")
    for e in range(experts):
        a, b = dys[off[e]:off[e + 1]], xs[off[e]:off[e + 1]]
        R.assert_product(h["dW"][e].astype(np.float64), a.T @ b, np.abs(a).T @ np.abs(b), len(a) + 1, "f32")
    for b in layer.buffers():
        b.free()


def test_replays_of_a_captured_layer():
    """A graph keeps the workspace that it was captured with, also when later calls need a larger one."""
    from wgblas_amd import Context

    hip = ctypes.CDLL("libamdhip64.so")

    def check(status):
        assert status == 0, f"HIP status {status}"

    rng = np.random.default_rng(1)
    with Context(0) as c:
        layer = Layer(c, rng, 2500, 32, 4, 520, 300, 4)
        layer.set(rng)
        layer.run()
        c.synchronize()
        stream = ctypes.c_void_p(c.stream)
        graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
        check(hip.hipStreamBeginCapture(stream, 1))  # thread-local mode
        try:
            layer.run()
        finally:
            check(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        check(hip.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, ctypes.c_size_t(0)))
        for replay in range(4):
            if replay == 1:
                larger = Layer(c, rng, 9000, 64, 8, 256, 128, 1)
                larger.set(rng)
                larger.run()
            layer.set(rng)
            layer.run()
            eager = layer.host()
            for name in layer.results:
                a = getattr(layer, name)
                c.h2d(a.ptr, np.full(a.nbytes, 0xEE, np.uint8))
            check(hip.hipGraphLaunch(executable, stream))
            got = layer.host()
            for name in layer.results:
                assert got[name].tobytes() == eager[name].tobytes(), (replay, name)
        check(hip.hipGraphExecDestroy(executable))
        check(hip.hipGraphDestroy(graph))


def test_two_contexts_at_once():
    """Each from a thread of its own, both in flight: the bits of one alone."""
    from wgblas_amd import Context

    with Context(0) as a, Context(0) as b:
        layers = [Layer(c, np.random.default_rng(2), 1800, 16, 3, 384, 264, 1) for c in (a, b)]
        for layer in layers:
            layer.set(np.random.default_rng(4))
        layers[0].run()
        alone = layers[0].host()
        got = [None, None]

        def work(i):
            for _ in range(5):
                layers[i].run()
            got[i] = layers[i].host()

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for result in got:
            for name, want in alone.items():
                assert result[name].tobytes() == want.tobytes(), name


@pytest.mark.parametrize("d,n,topk", [(5, 3, 2), (257, 40, 6), (1000, 9, 11)])
def test_rows_gradients_against_differences(ctx, d, n, topk):
    """combine is linear in the weights and in the rows: a step of any size gives the difference <dC, dCombine> exactly,
    but for the sums' own roundings, (topk + 2 + d) 2^-23 of the terms' magnitudes. gather's gradient is combine: <gather X, G>
    = <X, combine G>."""
    rng = np.random.default_rng(d)
    places = rng.permutation(n * topk).astype(np.int32).reshape(n, topk)
    places[rng.random((n, topk)) < 0.2] = -1
    there = places >= 0
    w, y, dc = (rng.standard_normal(s).astype(np.float32) for s in ((n, topk), (n * topk, d), (n, d)))
    dP, dDC = ctx.upload(places), ctx.upload(dc)
    dC, dw, dy = ctx.empty((n, d), np.float32), ctx.empty((n, topk), np.float32), ctx.upload(np.zeros_like(y))

    def combine(w, y):
        a, b = ctx.upload(w), ctx.upload(y)
        ctx.route_combine(F32, d, n, topk, b, d, dP, a, 0.0, dC, d, F32)
        out = dC.to_host().astype(np.float64)
        a.free(), b.free()
        return out

    a, b = ctx.upload(w), ctx.upload(y)
    ctx.route_combine_grad(F32, d, n, topk, dDC, d, b, d, dP, a, dy, d, dw)
    got_w, got_y = dw.to_host(), dy.to_host()
    assert (got_w[~there] == 0).all()
    base = combine(w, y)
    for slot in range(topk):  # every token's weight of a slot at once: tokens are apart
        step = np.zeros_like(w)
        step[:, slot] = 0.5
        change = ((combine(w + step, y) - base) * dc).sum(1) / 0.5
        rows = np.where(there[:, :, None], y[np.where(there, places, 0)], 0.0).astype(np.float64)
        # two sums, over the step of 0.5, and that step's own rounding: four times the terms
        size = ((np.abs(rows) * (np.abs(w) + 0.5)[:, :, None]).sum(1) * np.abs(dc)).sum(1) * 4
        assert (np.abs(change - got_w[:, slot]) <= (topk + 2 + d) * 2.0 ** -23 * size).all()
    v = rng.standard_normal(y.shape).astype(np.float32)  # a direction of the rows
    change = ((combine(w, y + v) - base) * dc).sum()
    moved = (y + v).astype(np.float64) - y
    rows = lambda x: np.abs(np.where(there[:, :, None], x[np.where(there, places, 0)], 0.0)) * np.abs(w)[:, :, None]  # noqa: E731
    size = ((rows(y) + rows(y + v)) * np.abs(dc)[:, None]).sum()
    assert abs(change - (got_y.astype(np.float64) * moved).sum()) <= (topk + 3) * 2.0 ** -23 * size
    x, g = rng.standard_normal((n, d)).astype(np.float32), rng.standard_normal(y.shape).astype(np.float32)
    dX, out = ctx.upload(x), ctx.upload(np.zeros_like(y))
    ctx.route_gather(F32, d, n, topk, dX, d, dP, a, out, d)
    back = combine(w, g)
    left, right = (out.to_host().astype(np.float64) * g).sum(), (back * x).sum()
    size = (rows(g) * np.abs(x)[:, None]).sum()
    assert abs(left - right) <= (topk + 2) * 2.0 ** -23 * size
