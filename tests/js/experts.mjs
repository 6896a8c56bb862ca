// Routing and the 8-bit products of the JS layer. With the argument "refusals"
// only what the checks in front of the addon say (no GPU); else also results,
// against float64 by the definitions, on the real addon.
import { test, run, assert, assertEqual, assertRejects } from "./harness.mjs";
import {
  init, cleanup, GpuVector, Fp8Matrix, randomFloat32Array, fp8Gemm, fp8GemmGrouped, route, routeGrad, routeOrder, routeGather,
  routeCombine, routeCombineGrad,
} from "../../wgblas_amd/js/index.mjs";

const rnd = (n, seed) => randomFloat32Array(n, -1, 1, seed);
const close = (got, want, what, bound = 1e-5) => {
  assertEqual(got.length, want.length, `${what}: length`);
  for (let i = 0; i < want.length; ++i)
    assert(Math.abs(got[i] - want[i]) <= bound * (1 + Math.abs(want[i])), `${what}[${i}]: ${got[i]} against ${want[i]}`);
};
const same = (got, want, what) => {
  assertEqual(got.length, want.length, `${what}: length`);
  for (let i = 0; i < want.length; ++i) assert(Number(got[i]) === Number(want[i]), `${what}[${i}]: ${got[i]} against ${want[i]}`);
};

if (process.argv[2] !== "refusals") {
  test("Fp8Matrix: values within half a code, transposes, residency, several matrices", async () => {
    const device = await init();
    const k = 130, n = 5, x = rnd(2 * k * n, 1);
    for (const block of [1, 128]) {
      const got = await Fp8Matrix.quantize(device, x, k, n, block, 2).read();
      // half a step of 3 bits of mantissa; a scale of the largest, at most 1 / 224, times half the least code 2^-9
      for (let i = 0; i < x.length; ++i) assert(Math.abs(got[i] - x[i]) <= Math.max(Math.abs(x[i]) / 16, 2 ** -10 / 224), `value ${i}`);
      const xt = new Float32Array(x.length);
      for (let g = 0; g < 2; ++g)
        for (let j = 0; j < n; ++j) for (let p = 0; p < k; ++p) xt[g * k * n + p * n + j] = x[g * k * n + j * k + p];
      same(await Fp8Matrix.quantize(device, GpuVector.from(device, xt), k, n, block, 2, n, "transpose").read(), got, "transposed");
    }
  });

  test("fp8Gemm and fp8GemmGrouped: products of the values the codes stand for", async () => {
    const device = await init();
    const m = 9, k = 140, n = 11, groups = 3, offsets = [0, 4, 4, 10];
    for (const t of [true, false]) {
      const rows = t ? k : m, cols = t ? m : k;
      const A = Fp8Matrix.quantize(device, rnd(groups * rows * cols, 2), rows, cols, 128, groups);
      const B = Fp8Matrix.quantize(device, rnd(k * n, 3), k, n), C = rnd(n * (m + 1), 4);
      const a = await A.read(), b = await B.read(), want = Float32Array.from(C);
      for (let g = 0; g < groups; ++g)
        for (let j = offsets[g]; j < offsets[g + 1]; ++j)
          for (let i = 0; i < m; ++i) {
            let s = 0;
            for (let p = 0; p < k; ++p) s += a[g * rows * cols + (t ? i * k + p : p * m + i)] * b[j * k + p];
            want[j * (m + 1) + i] = 1.5 * s - 0.5 * C[j * (m + 1) + i];
          }
      const trans = t ? "transpose" : "no-transpose";
      close((await fp8GemmGrouped(device, trans, 1.5, A, B, offsets, -0.5, C, m + 1)).C, want, `grouped ${trans}`, 1e-4);
      const one = Fp8Matrix.quantize(device, rnd(groups * rows * cols, 2).subarray(0, rows * cols), rows, cols, 128);
      const gC = GpuVector.from(device, C);
      assertEqual(Object.keys(await fp8Gemm(device, trans, 1.5, one, B, -0.5, gC, m + 1)).length, 0, "nothing for a resident C");
      const dense = await gC.read();
      close(dense.subarray(0, 4 * (m + 1)), want.subarray(0, 4 * (m + 1)), `dense ${trans}`, 1e-4);
    }
  });

  test("a routed layer: choice, order, rows there and back, gradients", async () => {
    const device = await init();
    const n = 7, experts = 6, topk = 2, d = 5;
    const logits = rnd(n * experts, 5), bias = rnd(experts, 6);
    for (const scoring of ["softmax", "sigmoid"]) {
      const { ids, weights } = await route(device, scoring, experts, n, topk, logits, experts, { bias, renorm: true, scale: 2 });
      const p = [];
      for (let t = 0; t < n; ++t) {
        const l = Array.from(logits.subarray(t * experts, (t + 1) * experts)), total = l.reduce((s, v) => s + Math.exp(v), 0);
        p.push(l.map((v) => (scoring === "softmax" ? Math.exp(v) / total : 1 / (1 + Math.exp(-v)))));
        const order = p[t].map((v, e) => [v + bias[e], e]).sort((a, b) => b[0] - a[0]).slice(0, topk).map((v) => v[1]);
        same(ids.subarray(t * topk, (t + 1) * topk), order, `experts of token ${t}`);
        const sum = order.reduce((s, e) => s + p[t][e], 0);
        close(weights.subarray(t * topk, (t + 1) * topk), order.map((e) => (2 * p[t][e]) / sum), "weights");
      }
      const { offsets, places, pairs } = await routeOrder(device, experts, n, topk, ids);
      const sorted = Array.from(ids.keys()).sort((a, b) => ids[a] - ids[b] || a - b);
      same(pairs, sorted, "pairs");
      sorted.forEach((pair, column) => assertEqual(places[pair], column, "place"));
      for (let e = 0; e <= experts; ++e) assertEqual(Number(offsets[e]), ids.filter((v) => v < e).length, "offset");
      const X = rnd(n * d, 7), Y = new Float32Array(n * topk * d);
      const moved = (await routeGather(device, d, n, topk, X, d, places, null, Y, d)).Y;
      places.forEach((at, pair) => {
        const token = Math.floor(pair / topk);
        same(moved.subarray(at * d, at * d + d), X.subarray(token * d, token * d + d), "row");
      });
      const C = rnd(n * d, 8);
      const back = (await routeCombine(device, d, n, topk, moved, d, places, weights, 1, C, d)).C;
      close(back, C.map((c, i) => c + 2 * X[i]), "weights sum to the scale");
      const dC = rnd(n * d, 9), gY = GpuVector.from(device, moved);
      const { dweights } = await routeCombineGrad(device, d, n, topk, GpuVector.from(device, dC), d, gY, d, places, weights, gY, d);
      const dY = await gY.read();
      places.forEach((at, pair) => {
        const token = Math.floor(pair / topk), g = dC.subarray(token * d, token * d + d);
        close(dY.subarray(at * d, at * d + d), g.map((v) => weights[pair] * v), "row's gradient");
        close([dweights[pair]], [g.reduce((s, v, i) => s + v * X[token * d + i], 0)], "weight's gradient");
      });
      const dl = (await routeGrad(device, scoring, experts, n, topk, logits, experts, ids, dweights, { renorm: true, scale: 2 })).dlogits;
      for (let t = 0; t < n; ++t) {
        const own = Array.from(ids.subarray(t * topk, (t + 1) * topk)), sum = own.reduce((s, e) => s + p[t][e], 0);
        const dot = own.reduce((s, e, i) => s + dweights[t * topk + i] * p[t][e], 0);
        const ds = new Array(experts).fill(0);
        own.forEach((e, i) => (ds[e] = 2 * (dweights[t * topk + i] / sum - dot / sum ** 2)));
        const inner = ds.reduce((s, v, e) => s + v * p[t][e], 0);
        const want = ds.map((v, e) => (scoring === "softmax" ? p[t][e] * (v - inner) : v * p[t][e] * (1 - p[t][e])));
        close(dl.subarray(t * experts, (t + 1) * experts), want, "logits' gradient");
      }
    }
  });

  test("refusals that need a matrix", async () => {
    const device = await init();
    const A = Fp8Matrix.quantize(device, rnd(40, 1), 10, 4), W = Fp8Matrix.quantize(device, rnd(40, 1), 10, 4, 128);
    const two = Fp8Matrix.quantize(device, rnd(80, 1), 10, 4, 1, 2), C = new Float32Array(16);
    await assertRejects(() => fp8Gemm(device, "transpose", 1, [1], A, 0, C, 4), "A must be an Fp8Matrix");
    await assertRejects(() => fp8Gemm(device, "t", 1, A, A, 0, C, 4), "transA");
    await assertRejects(() => fp8Gemm(device, "transpose", 1, A, W, 0, C, 4), "blocks of one column");
    await assertRejects(() => fp8Gemm(device, "no-transpose", 1, A, A, 0, C, 10), "blocks of 128");
    await assertRejects(() => fp8Gemm(device, "no-transpose", 1, W, A, 0, new Float32Array(40), 10), "same k");
    await assertRejects(() => fp8Gemm(device, "transpose", 1, two, A, 0, C, 4), "one matrix");
    await assertRejects(() => fp8Gemm(device, "transpose", 1, A, A, 0, C, 3), "ldc");
    await assertRejects(() => fp8Gemm(device, "transpose", 1, A, A, 0, new Float32Array(15), 4), "C does not have enough");
    await assertRejects(() => fp8GemmGrouped(device, "transpose", 1, two, A, [0, 4], 0, C, 4), "groups + 1");
    A.destroy();
    await assertRejects(() => fp8Gemm(device, "transpose", 1, A, A, 0, C, 4), "destroyed");
    await assertRejects(() => A.read(), "destroyed");
  });
}

test("refusals", async () => {
  const device = await init();
  const f = (n) => new Float32Array(n), i = (n) => new Int32Array(n);
  await assertRejects(async () => Fp8Matrix.quantize(device, f(41), 42, 1), "X does not have enough");
  await assertRejects(async () => Fp8Matrix.quantize(device, f(41), 10, 4, 1, 2), "X does not have enough");
  await assertRejects(async () => Fp8Matrix.quantize(device, f(40), 10, 4, 64), "block");
  await assertRejects(async () => Fp8Matrix.quantize(device, f(40), 10, 4, 1, 1, 9), "ldx");
  await assertRejects(async () => Fp8Matrix.quantize(device, f(40), 10, 4, 1, 1, 10, "t"), "trans");
  await assertRejects(async () => Fp8Matrix.quantize(device, [1], 1, 1), "X must be");
  await assertRejects(() => route(device, "linear", 4, 2, 1, f(8), 4), "scoring");
  await assertRejects(() => route(device, "softmax", 4, 2, 5, f(8), 4), "topk must be at most experts");
  await assertRejects(() => route(device, "softmax", 4, 2, 0, f(8), 4), "topk");
  await assertRejects(() => route(device, "softmax", 4, 2, 1, f(7), 4), "logits does not have enough");
  await assertRejects(() => route(device, "softmax", 4, 2, 1, f(8), 3), "ld of logits");
  await assertRejects(() => route(device, "softmax", 4, 2, 1, f(8), 4, { bias: f(3) }), "bias does not have enough");
  await assertRejects(() => route(device, "softmax", 4, 2, 1, f(8), 4, { groups: 3 }), "groups must divide");
  await assertRejects(() => route(device, "softmax", 4, 2, 1, f(8), 4, { groups: 2, topGroups: 3 }), "topGroups");
  await assertRejects(() => route(device, "softmax", 4, 2, 1, f(8), 4, { best: 3 }), "best");
  await assertRejects(() => routeOrder(device, 1025, 2, 1, i(2)), "experts");
  await assertRejects(() => routeOrder(device, 4, 2, 2, i(3)), "ids does not have enough");
  await assertRejects(() => routeOrder(device, 4, 2, 2, f(4)), "ids must be an Int32Array");
  await assertRejects(() => routeGather(device, 3, 2, 2, f(6), 3, i(4), null, f(11), 3), "Y does not have enough");
  await assertRejects(() => routeGather(device, 3, 2, 2, f(6), 3, i(4), f(3), f(12), 3), "weights does not have enough");
  await assertRejects(() => routeCombine(device, 3, 2, 2, f(12), 2, i(4), null, 0, f(6), 3), "ld of Y");
  await assertRejects(() => routeCombineGrad(device, 3, 2, 2, f(6), 3, f(12), 3, i(4), null, f(12), 3), "weights");
  await assertRejects(() => routeGrad(device, "softmax", 4, 2, 1, f(8), 4, i(2), f(1)), "dweights does not have enough");
  const { offsets, places } = await routeOrder(device, 3, 0, 2, i(0));
  assertEqual(offsets.length, 4, "boundaries of no tokens");
  assertEqual(places.length, 0, "places of no tokens");
  cleanup();
});

run();
