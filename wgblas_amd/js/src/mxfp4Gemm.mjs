// mxfp4Gemm: C <- alpha*A^T*B + beta*C for A (k x m) and B (k x n) in MXFP4,
// C m x n float32, column-major (wgb_mxfp4_gemm). mxfp4GemmGrouped: the same
// for ragged groups of B's columns, group g with columns g*m .. g*m + m - 1 of
// A (wgb_mxfp4_gemm_grouped). wgblas has no counterpart.
// Return { C } (a new Float32Array) when C is a host array, {} when it is a
// GpuVector (updated in place); plus gpuTimeMs when init({benchmark:true}).
import { checkScalar, execute } from "./gemm_common.mjs";
import { checkFlat, checkLength, checkOffsets, checkSizes, F32, span } from "./grouped_common.mjs";
import { Mxfp4Matrix } from "./classes/Mxfp4Matrix.mjs";
import { requireGpuDevice, requireSameDevice } from "./device.mjs";
import { native } from "./native.mjs";

function checkCall(routine, device, alpha, A, B, beta, C, ldc, m) {
  requireGpuDevice(device);
  requireSameDevice(device, routine, { C });
  for (const [name, X] of [["A", A], ["B", B]]) {
    if (!(X instanceof Mxfp4Matrix)) throw new Error(`${name} must be an Mxfp4Matrix.`);
    if (X._codes === null) throw new Error(`${name} was destroyed.`);
    if (X.device !== device) throw new Error(`${routine}: ${name} belongs to a different GPUDevice than the one passed in.`);
  }
  checkScalar("alpha", alpha);
  checkScalar("beta", beta);
  checkSizes("ldc", [ldc]);
  if (A.k !== B.k) throw new Error("A and B must have the same k.");
  const resident = checkFlat({ C });
  if (ldc < Math.max(1, m)) throw new Error("ldc must be >= max(1, m).");
  checkLength("C", C, span(m, B.n, ldc));
  return resident;
}

export async function mxfp4Gemm(device, alpha, A, B, beta, C, ldc) {
  const m = A instanceof Mxfp4Matrix ? A.n : 0;
  const resident = checkCall("mxfp4Gemm", device, alpha, A, B, beta, C, ldc, m);
  if (m === 0 || B.n === 0) return resident ? {} : { C };
  return execute(device, [], C, resident, Float32Array, (ctx, p, pC) =>
    native().mxfp4Gemm(ctx, -1, m, B.n, A.k, alpha, A._codes, A._scales, A.ld, 0, B._codes, B._scales, B.ld, null, beta, pC, ldc,
                       F32),
  );
}

export async function mxfp4GemmGrouped(device, groups, m, alpha, A, B, offsets, beta, C, ldc) {
  checkSizes("groups and m", [groups, m]);
  const resident = checkCall("mxfp4GemmGrouped", device, alpha, A, B, beta, C, ldc, m);
  if (A.n < groups * m) throw new Error("A must have groups * m columns.");
  const bounds = checkOffsets(offsets, groups, B.n);
  if (groups === 0 || m === 0 || B.n === 0) return resident ? {} : { C };
  return execute(device, [bounds], C, resident, Float32Array, (ctx, p, pC) =>
    native().mxfp4Gemm(ctx, groups, m, B.n, A.k, alpha, A._codes, A._scales, A.ld, m * A.ld, B._codes, B._scales, B.ld, p[0],
                       beta, pC, ldc, F32),
  );
}
