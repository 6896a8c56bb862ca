// The grouped and 4-bit routines through the real addon and library, with a
// stand-in for the HIP runtime in place of a GPU (tests/test_js_addon.py): what
// they compute is nothing, which calls they make is the test. Every operand has
// a size of its own, so that its allocation names it.
import {
  init, cleanup, GpuVector, Mxfp4Matrix, sgemmGrouped, sgemmGroupedK, mxfp4Gemm, mxfp4GemmGrouped,
} from "../../wgblas_amd/js/index.mjs";

const f = (n) => new Float32Array(n);
async function main() {
  const device = await init();

  // 3 groups, m 5, n 10, k 7; A 9 x 5 a group at stride 50, B 8 x 10, C 6 x 10
  await sgemmGrouped(device, "transpose", 3, 5, 10, 7, 1.5, f(150), 9, 50, f(80), 8, [0, 3, 3, 9], 0.5, f(60), 6);
  await sgemmGrouped(device, "no-transpose", 3, 5, 10, 7, -2, f(151), 6, 51, f(81), 8, [0, 3, 3, 9], 0, f(61), 6);
  const [A, B, C] = [152, 82, 62].map((n) => GpuVector.from(device, f(n)));
  await sgemmGrouped(device, "transpose", 3, 5, 10, 7, 1, A, 9, 50, B, 8, Int32Array.from([0, 3, 3, 9]), 1, C, 6);
  // 2 groups of 11 columns; A 4 x 11 at 5, B 6 x 11 at 7, C 4 x 6 a group at 8, stride 49
  await sgemmGroupedK(device, 2, 4, 6, 11, 0.25, f(55), 5, f(77), 7, BigInt64Array.from([0n, 2n, 11n]), -1, f(98), 8, 49);
  // MXFP4: k 130 (ld 256); 3 x 4 columns of weights, 9 of tokens
  const W = Mxfp4Matrix.quantize(device, f(12 * 131), 130, 12, 131);
  const X = Mxfp4Matrix.quantize(device, f(130 * 10), 130, 9, 10, "transpose");
  await W.read();
  await mxfp4Gemm(device, 2, W, X, 0.75, f(9 * 13), 13);
  await mxfp4GemmGrouped(device, 3, 4, 3, W, X, [0, 1, 1, 9], 0.125, f(9 * 5), 5);
  cleanup();
}

main().catch((e) => {
  console.error(e);
  process.exitCode = 1;
});
