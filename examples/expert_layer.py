"""A layer of experts, trained in bf16 and served from 4-bit weights.

    python examples/expert_layer.py [--steps N]

Tokens go to the expert whose direction they are nearest to (the router), are
sorted by expert, and every product of a training step is one call for all
experts, whatever their shares of the tokens:

    forward          Y(:, j)  = W_g x_j        wgb_gemm_grouped, WGB_TRANS
    input gradient   dX(:, j) = W_g^T dy_j     wgb_gemm_grouped, WGB_NO_TRANS
    weight gradient  dW_g     = dY_g X_g^T     wgb_gemm_grouped_k, in fp32

Afterwards the weights are quantised to MXFP4 once, and single tokens are
quantised and multiplied with them (wgb_mxfp4_quantize, wgb_mxfp4_gemm_grouped).

Arrays are row-major here (tokens by features, weights out by in), which is the
library's column-major frame read the other way.
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from wgblas_amd import BF16, F32, NO_TRANS, TRANS, Context  # noqa: E402


def to_bf16(x):
    """float32 -> bfloat16 bits, to nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def route(x, directions):
    """Tokens sorted by expert, and the experts' boundaries."""
    expert = (x @ directions.T).argmax(1)
    order = np.argsort(expert, kind="stable")
    sizes = np.bincount(expert, minlength=len(directions))
    return order, np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)


class ExpertLayer:
    """Device buffers of `experts` matrices out x inner and of up to `tokens` tokens."""

    def __init__(self, ctx, weights, tokens):
        self.ctx, self.tokens = ctx, tokens
        self.experts, self.out, self.inner = weights.shape
        self.weights = ctx.upload(to_bf16(weights))
        self.x, self.y = ctx.empty((tokens, self.inner), np.uint16), ctx.empty((tokens, self.out), np.float32)
        self.dy, self.dx = ctx.empty((tokens, self.out), np.uint16), ctx.empty((tokens, self.inner), np.float32)
        self.dw = ctx.empty(weights.shape, np.float32)
        self.offsets = ctx.empty(self.experts + 1, np.int64)

    def count(self, x):
        """Tokens of x, which the buffers have to hold."""
        if len(x) > self.tokens:
            raise ValueError(f"{len(x)} tokens, there is room for {self.tokens}")
        return len(x)

    def forward(self, x, offsets):
        n, ctx = self.count(x), self.ctx
        ctx.h2d(self.x.ptr, to_bf16(x))
        ctx.h2d(self.offsets.ptr, offsets)
        ctx.gemm_grouped(BF16, TRANS, self.experts, self.out, n, self.inner, 1.0, self.weights, self.inner,
                         self.out * self.inner, self.x, self.inner, self.offsets, 0.0, self.y, self.out, F32)
        return self.y.to_host()[:n]

    def backward(self, dy):
        """(gradient of the weights, gradient of the input) of the last forward's tokens."""
        n, ctx = self.count(dy), self.ctx
        ctx.h2d(self.dy.ptr, to_bf16(dy))
        ctx.gemm_grouped(BF16, NO_TRANS, self.experts, self.inner, n, self.out, 1.0, self.weights, self.inner,
                         self.out * self.inner, self.dy, self.out, self.offsets, 0.0, self.dx, self.inner, F32)
        ctx.gemm_grouped_k(BF16, self.experts, self.inner, self.out, n, 1.0, self.x, self.inner, self.dy, self.out,
                           self.offsets, 0.0, self.dw, self.inner, self.out * self.inner, F32)
        return self.dw.to_host(), self.dx.to_host()[:n]

    def update(self, weights):
        self.ctx.h2d(self.weights.ptr, to_bf16(weights))


class ServedLayer:
    """The same layer with its weights in MXFP4."""

    def __init__(self, layer):
        ctx, self.layer = layer.ctx, layer
        self.ld = (layer.inner + 127) // 128 * 128
        columns = layer.experts * layer.out  # all experts' weights in one call
        self.codes, self.scales = self._room(columns)
        ctx.mxfp4_quantize(BF16, NO_TRANS, layer.inner, columns, layer.weights, layer.inner, self.codes, self.scales, self.ld)
        self.x_codes, self.x_scales = self._room(layer.tokens)

    def _room(self, columns):
        ctx = self.layer.ctx
        return ctx.empty((columns, self.ld // 2), np.uint8), ctx.empty((columns, self.ld // 32), np.uint8)

    def forward(self, x, offsets):
        n, s, ctx = self.layer.count(x), self.layer, self.layer.ctx
        ctx.h2d(s.x.ptr, to_bf16(x))
        ctx.h2d(s.offsets.ptr, offsets)
        ctx.mxfp4_quantize(BF16, NO_TRANS, s.inner, n, s.x, s.inner, self.x_codes, self.x_scales, self.ld)
        ctx.mxfp4_gemm_grouped(s.experts, s.out, n, s.inner, 1.0, self.codes, self.scales, self.ld, s.out * self.ld,
                               self.x_codes, self.x_scales, self.ld, s.offsets, 0.0, s.y, s.out, F32)
        return s.y.to_host()[:n]


def main(steps=60, experts=6, inner=192, out=160, tokens=1500, seed=0, log=print):
    """Trains the layer on a teacher's outputs; returns (first loss, last loss, largest relative difference of the 4-bit layer)."""
    rng = np.random.default_rng(seed)
    directions = rng.standard_normal((experts, inner)) + 0.1 * rng.standard_normal(inner)
    teacher = rng.standard_normal((experts, out, inner)).astype(np.float32) / np.sqrt(inner)
    weights = np.zeros_like(teacher)
    losses = []
    with Context(0) as ctx:
        layer = ExpertLayer(ctx, weights, tokens)
        for step in range(steps):
            x = rng.standard_normal((tokens, inner)).astype(np.float32)
            order, offsets = route(x, directions)
            x = x[order]
            expert = np.repeat(np.arange(experts), np.diff(offsets))
            target = np.einsum("toi,ti->to", teacher[expert], x)
            error = layer.forward(x, offsets) - target
            losses.append(float((error ** 2).mean()))
            dw, _ = layer.backward(error)
            share = np.maximum(np.diff(offsets), 1)[:, None, None]
            weights -= 0.7 * dw / share
            layer.update(weights)
            if step % 10 == 0 or step == steps - 1:
                log(f"step {step:3d}  loss {losses[-1]:.5f}  tokens per expert {np.diff(offsets).tolist()}")
        served = ServedLayer(layer)
        worst = 0.0
        for count in (1, 3, 200):  # single tokens and a short prompt
            x = rng.standard_normal((count, inner)).astype(np.float32)
            order, offsets = route(x, directions)
            x = x[order]
            exact, got = layer.forward(x, offsets).copy(), served.forward(x, offsets)
            difference = float(np.linalg.norm(got - exact) / np.linalg.norm(exact))
            worst = max(worst, difference)
            log(f"{count:3d} tokens from 4-bit weights: relative difference {difference:.3f}")
    return losses[0], losses[-1], worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    main(ap.parse_args().steps)
