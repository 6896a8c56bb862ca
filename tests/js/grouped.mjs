// The grouped and 4-bit routines of the JS layer through grouped_addon.cjs:
// results, residency, shapes and refusals.
import { test, run, assert, assertEqual, assertRejects } from "./harness.mjs";
import {
  init, cleanup, GpuVector, Mxfp4Matrix, randomFloat32Array, sgemmGrouped, sgemmGroupedK, mxfp4Gemm, mxfp4GemmGrouped,
} from "../../wgblas_amd/js/index.mjs";

const rnd = (n, seed) => randomFloat32Array(n, -1, 1, seed);
const close = (got, want, what) => {
  assertEqual(got.length, want.length, `${what}: length`);
  for (let i = 0; i < want.length; ++i)
    assert(Math.abs(got[i] - want[i]) <= 1e-5 * (1 + Math.abs(want[i])), `${what}[${i}]: ${got[i]} against ${want[i]}`);
};

// groups of 3, 0, 5 and 1 of 10 columns
const offsets = [0, 3, 3, 8, 9], groups = 4, m = 5, n = 10, k = 7;

function forward(A, t, B, C, alpha, beta, lda, strideA, ldb, ldc) {
  const out = Float32Array.from(C);
  for (let g = 0; g < groups; ++g)
    for (let j = offsets[g]; j < offsets[g + 1]; ++j)
      for (let i = 0; i < m; ++i) {
        let s = 0;
        for (let p = 0; p < k; ++p) s += A[g * strideA + (t ? i * lda + p : p * lda + i)] * B[j * ldb + p];
        out[j * ldc + i] = alpha * s + beta * C[j * ldc + i];
      }
  return out;
}

for (const t of [false, true])
  test(`sgemmGrouped, ${t ? "transpose" : "no-transpose"}: host arrays and GpuVector`, async () => {
    const device = await init();
    const lda = (t ? k : m) + 2, strideA = (t ? m : k) * lda, ldb = k + 1, ldc = m + 3;
    const A = rnd(groups * strideA, 1), B = rnd(n * ldb, 2), C = rnd(n * ldc, 3);
    const want = forward(A, t, B, C, 1.5, 0.5, lda, strideA, ldb, ldc);
    const before = Float32Array.from(C);
    const trans = t ? "transpose" : "no-transpose";
    const r = await sgemmGrouped(device, trans, groups, m, n, k, 1.5, A, lda, strideA, B, ldb, offsets, 0.5, C, ldc);
    close(r.C, want, "C");
    close(C, before, "the input C");
    const [gA, gB, gC] = [A, B, C].map((x) => GpuVector.from(device, x));
    const e = await sgemmGrouped(device, trans, groups, m, n, k, 1.5, gA, lda, strideA, gB, ldb, Int32Array.from(offsets), 0.5,
                                 gC, ldc);
    assertEqual(Object.keys(e).length, 0, "nothing returned for a resident C");
    close(await gC.read(), want, "resident C");
    [gA, gB, gC].forEach((x) => x.destroy());
  });

test("sgemmGroupedK: gradients of the groups, an empty one scaled", async () => {
  const device = await init();
  const A = rnd(n * m, 4), B = rnd(n * k, 5), C = rnd(groups * m * k, 6);
  const want = Float32Array.from(C);
  for (let g = 0; g < groups; ++g)
    for (let j = 0; j < k; ++j)
      for (let i = 0; i < m; ++i) {
        let s = 0;
        for (let p = offsets[g]; p < offsets[g + 1]; ++p) s += A[p * m + i] * B[p * k + j];
        want[g * m * k + j * m + i] = 2 * s - C[g * m * k + j * m + i];
      }
  const big = BigInt64Array.from(offsets.map(BigInt));
  close((await sgemmGroupedK(device, groups, m, k, n, 2, A, m, B, k, big, -1, C, m, m * k)).C, want, "C");
});

test("Mxfp4Matrix: the format's rounding, transposes, residency", async () => {
  const device = await init();
  // one block whose scale is 1: largest magnitude in [4, 8)
  const x = Float32Array.from([0, 0.25, 0.26, 0.75, 1.25, 1.26, 1.75, 2.5, 3.5, 5, 5.1, 7.9, -0.3, -6]);
  const q = Mxfp4Matrix.quantize(device, x, x.length, 1);
  close(await q.read(), Float32Array.from([0, 0, 0.5, 1, 1, 1.5, 2, 2, 4, 4, 6, 6, -0.5, -6]), "codes");
  assertEqual(q.ld, 128, "ld");
  const X = rnd(50 * 9, 7);
  const Xt = new Float32Array(X.length);
  for (let j = 0; j < 9; ++j) for (let p = 0; p < 50; ++p) Xt[p * 9 + j] = X[j * 50 + p];
  const a = await Mxfp4Matrix.quantize(device, X, 50, 9).read();
  const b = await Mxfp4Matrix.quantize(device, GpuVector.from(device, Xt), 50, 9, 9, "transpose").read();
  close(a, b, "transpose");
  q.destroy();
  q.destroy();
});

test("mxfp4Gemm and mxfp4GemmGrouped: products of the values the codes stand for", async () => {
  const device = await init();
  const kk = 70;
  const A = Mxfp4Matrix.quantize(device, rnd(kk * groups * m, 8), kk, groups * m), B = Mxfp4Matrix.quantize(device, rnd(kk * n, 9), kk, n);
  const a = await A.read(), b = await B.read(), C = rnd(n * m, 10);
  const dot = (i, j) => {
    let s = 0;
    for (let p = 0; p < kk; ++p) s += a[i * kk + p] * b[j * kk + p];
    return s;
  };
  const want = Float32Array.from(C);
  for (let g = 0; g < groups; ++g)
    for (let j = offsets[g]; j < offsets[g + 1]; ++j) for (let i = 0; i < m; ++i) want[j * m + i] = dot(g * m + i, j) + 0.5 * C[j * m + i];
  close((await mxfp4GemmGrouped(device, groups, m, 1, A, B, offsets, 0.5, C, m)).C, want, "grouped");
  const all = new Float32Array(n * groups * m);
  for (let j = 0; j < n; ++j) for (let i = 0; i < groups * m; ++i) all[j * groups * m + i] = dot(i, j);
  const gC = GpuVector.from(device, all);
  await mxfp4Gemm(device, 1, A, B, -1, gC, groups * m);
  close(await gC.read(), new Float32Array(all.length), "dense, minus itself");
});

test("nothing to do returns the arrays that came in", async () => {
  const device = await init();
  const z = new Float32Array(0), C = rnd(4, 1);
  assert((await sgemmGrouped(device, "transpose", 0, 2, 2, 2, 1, z, 2, 0, rnd(4, 2), 2, [0], 0, C, 2)).C === C, "no groups");
  assert((await sgemmGroupedK(device, 1, 0, 2, 0, 1, z, 1, z, 2, [0, 0], 0, C, 1, 0)).C === C, "no rows");
});

test("refusals", async () => {
  const device = await init();
  const A = rnd(40, 1), B = rnd(20, 2), C = rnd(20, 3), off = [0, 2, 4];
  const call = (o) => {
    const a = { device, trans: "transpose", groups: 2, m: 4, n: 4, k: 5, alpha: 1, A, lda: 5, strideA: 20, B, ldb: 5, off, beta: 0, C, ldc: 4, ...o };
    return () => sgemmGrouped(a.device, a.trans, a.groups, a.m, a.n, a.k, a.alpha, a.A, a.lda, a.strideA, a.B, a.ldb, a.off, a.beta, a.C, a.ldc);
  };
  await call({})();
  for (const [o, text] of [
    [{ device: {} }, "device must be"], [{ trans: "T" }, "must be 'no-transpose' or 'transpose'"], [{ alpha: NaN }, "alpha"],
    [{ beta: "1" }, "beta must be a number"], [{ m: 1.5 }, "must be integers"], [{ k: -1 }, "must be non-negative"],
    [{ A: new Float64Array(40) }, "A must be"], [{ C: GpuVector.from(device, C) }, "all host arrays or all GpuVector"],
    [{ off: [0, 2] }, "groups + 1"], [{ off: [0, 3, 2] }, "not decrease"], [{ off: [0, 2, 5] }, "within the columns"],
    [{ off: [1, 2, 4] }, "start at 0"], [{ off: "x" }, "offsets must be"], [{ off: [0, 0.5, 4] }, "not decrease"], [{ lda: 4 }, "lda"],
    [{ strideA: 19 }, "strideA"], [{ ldb: 4 }, "ldb"], [{ ldc: 3 }, "ldc"], [{ A: rnd(39, 1) }, "A does not have enough"],
    [{ B: rnd(19, 1) }, "B does not have enough"], [{ C: rnd(15, 1) }, "C does not have enough"],
  ]) await assertRejects(call(o), text, JSON.stringify(Object.keys(o)));
  await assertRejects(async () => Mxfp4Matrix.quantize(device, A, 41, 1), "X does not have enough");
  await assertRejects(async () => Mxfp4Matrix.quantize(device, A, 10, 4, 9), "ldx");
  await assertRejects(async () => Mxfp4Matrix.quantize(device, A, 10, 4, 10, "t"), "trans");
  await assertRejects(async () => Mxfp4Matrix.quantize(device, [1], 1, 1), "X must be");
  const q = Mxfp4Matrix.quantize(device, A, 10, 4), other = Mxfp4Matrix.quantize(device, A, 8, 4);
  await assertRejects(() => mxfp4Gemm(device, 1, A, q, 0, rnd(16, 1), 4), "A must be an Mxfp4Matrix");
  await assertRejects(() => mxfp4Gemm(device, 1, q, other, 0, rnd(16, 1), 4), "same k");
  await assertRejects(() => mxfp4Gemm(device, 1, q, q, 0, rnd(15, 1), 4), "C does not have enough");
  await assertRejects(() => mxfp4Gemm(device, 1, q, q, 0, rnd(16, 1), 3), "ldc");
  await assertRejects(() => mxfp4GemmGrouped(device, 2, 4, 1, q, q, [0, 1, 4], 0, rnd(16, 1), 4), "groups * m columns");
  const second = await init({ powerPreference: "low-power" });
  if (second !== device) await assertRejects(() => mxfp4Gemm(second, 1, q, q, 0, rnd(16, 1), 4), "different GPUDevice");
  q.destroy();
  await assertRejects(() => mxfp4Gemm(device, 1, q, q, 0, rnd(16, 1), 4), "destroyed");
  cleanup();
});

run();
