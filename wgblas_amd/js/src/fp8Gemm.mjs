// fp8Gemm: C <- alpha*op(A)*B + beta*C for 8-bit A and B (Fp8Matrix; B k x n in
// blocks of one column), C m x n float32, column-major (wgb_fp8_gemm). 'transpose':
// A is k x m in blocks of 1 or 128 columns; 'no-transpose': m x k in blocks of
// 128. fp8GemmGrouped: the same for ragged groups of B's columns, group g with
// A's matrix g (wgb_fp8_gemm_grouped). wgblas has no counterpart.
// Return { C } (a new Float32Array) when C is a host array, {} when it is a
// GpuVector (updated in place); plus gpuTimeMs when init({benchmark:true}).
import { checkScalar, checkTrans, execute, NO_TRANS, TRANS } from "./gemm_common.mjs";
import { checkFlat, checkLength, checkOffsets, checkSizes, F32, span } from "./grouped_common.mjs";
import { Fp8Matrix } from "./classes/Fp8Matrix.mjs";
import { requireGpuDevice, requireSameDevice } from "./device.mjs";
import { native } from "./native.mjs";

function checkCall(routine, device, transA, alpha, A, B, beta, C, ldc) {
  requireGpuDevice(device);
  requireSameDevice(device, routine, { C });
  checkTrans("transA", transA);
  for (const [name, X] of [["A", A], ["B", B]]) {
    if (!(X instanceof Fp8Matrix)) throw new Error(`${name} must be an Fp8Matrix.`);
    if (X._codes === null) throw new Error(`${name} was destroyed.`);
    if (X.device !== device) throw new Error(`${routine}: ${name} belongs to a different GPUDevice than the one passed in.`);
  }
  checkScalar("alpha", alpha);
  checkScalar("beta", beta);
  checkSizes("ldc", [ldc]);
  const t = transA === "transpose";
  const m = t ? A.n : A.k;
  if (B.block !== 1 || B.matrices !== 1) throw new Error("B must be one matrix in blocks of one column.");
  if (!t && A.block !== 128) throw new Error("A must be in blocks of 128 columns for 'no-transpose'.");
  if ((t ? A.k : A.n) !== B.k) throw new Error("op(A) and B must have the same k.");
  const resident = checkFlat({ C });
  if (ldc < Math.max(1, m)) throw new Error("ldc must be >= max(1, m).");
  checkLength("C", C, span(m, B.n, ldc));
  return { resident, m, trans: t ? TRANS : NO_TRANS };
}

function run(device, groups, call, alpha, A, B, bounds, beta, C, ldc) {
  const { resident, m, trans } = call;
  if (m === 0 || B.n === 0 || groups === 0) return resident ? {} : { C };
  return execute(device, bounds ? [bounds] : [], C, resident, Float32Array, (ctx, p, pC) =>
    native().fp8Gemm(ctx, trans, groups, m, B.n, B.k, alpha, A._codes, A.ld, A.n * A.ld, A.block, A._scales, A.lds, B._codes,
                     B.ld, B._scales, B.lds, bounds ? p[0] : null, beta, pC, ldc, F32),
  );
}

export async function fp8Gemm(device, transA, alpha, A, B, beta, C, ldc) {
  const call = checkCall("fp8Gemm", device, transA, alpha, A, B, beta, C, ldc);
  if (A.matrices !== 1) throw new Error("A must be one matrix.");
  return run(device, -1, call, alpha, A, B, null, beta, C, ldc);
}

export async function fp8GemmGrouped(device, transA, alpha, A, B, offsets, beta, C, ldc) {
  const call = checkCall("fp8GemmGrouped", device, transA, alpha, A, B, beta, C, ldc);
  return run(device, A.matrices, call, alpha, A, B, checkOffsets(offsets, A.matrices, B.n), beta, C, ldc);
}
