// sgemmGrouped: the products of ragged groups of columns, each group with a
// matrix of its own (wgb_gemm_grouped in float32): C(:, j) <- alpha*op(A_g)*
// B(:, j) + beta*C(:, j) for offsets[g] <= j < offsets[g + 1]. sgemmGroupedK:
// C_g <- alpha*A(:, g)*B(:, g)^T + beta*C_g, the gradient of the groups'
// matrices (wgb_gemm_grouped_k). Column-major throughout (tokens by features
// in row-major storage); wgblas has no counterpart.
// Return { C } (a new Float32Array) for host arrays, {} when the operands are
// GpuVector (C updated in place); plus gpuTimeMs when init({benchmark:true}).
import { checkScalar, checkTrans, execute, NO_TRANS, TRANS } from "./gemm_common.mjs";
import { checkFlat, checkLength, checkOffsets, checkSizes, F32, span } from "./grouped_common.mjs";
import { requireGpuDevice, requireSameDevice } from "./device.mjs";
import { native } from "./native.mjs";

export async function sgemmGrouped(device, transA, groups, m, n, k, alpha, A, lda, strideA, B, ldb, offsets, beta, C,
                                   ldc) {
  requireGpuDevice(device);
  requireSameDevice(device, "sgemmGrouped", { A, B, C });
  checkTrans("transA", transA);
  checkScalar("alpha", alpha);
  checkScalar("beta", beta);
  checkSizes("groups, m, n, k, lda, strideA, ldb, and ldc", [groups, m, n, k, lda, strideA, ldb, ldc]);
  const resident = checkFlat({ A, B, C });
  const bounds = checkOffsets(offsets, groups, n);
  const t = transA === "transpose";
  const rows = t ? k : m, cols = t ? m : k;
  if (lda < Math.max(1, rows)) throw new Error("lda must be >= max(1, rows of A).");
  if (groups > 1 && strideA < span(rows, cols, lda)) throw new Error("strideA must cover a group's A.");
  if (ldb < Math.max(1, k)) throw new Error("ldb must be >= max(1, k).");
  if (ldc < Math.max(1, m)) throw new Error("ldc must be >= max(1, m).");
  if (m === 0 || n === 0 || groups === 0) return resident ? {} : { C };
  checkLength("A", A, (groups - 1) * strideA + span(rows, cols, lda));
  checkLength("B", B, span(k, n, ldb));
  checkLength("C", C, span(m, n, ldc));
  return execute(device, [A, B, bounds], C, resident, Float32Array, (ctx, p, pC) =>
    native().gemmGrouped(ctx, F32, t ? TRANS : NO_TRANS, groups, m, n, k, alpha, p[0], lda, strideA, p[1], ldb, p[2], beta, pC,
                         ldc, F32),
  );
}

export async function sgemmGroupedK(device, groups, m, n, k, alpha, A, lda, B, ldb, offsets, beta, C, ldc, strideC) {
  requireGpuDevice(device);
  requireSameDevice(device, "sgemmGroupedK", { A, B, C });
  checkScalar("alpha", alpha);
  checkScalar("beta", beta);
  checkSizes("groups, m, n, k, lda, ldb, ldc, and strideC", [groups, m, n, k, lda, ldb, ldc, strideC]);
  const resident = checkFlat({ A, B, C });
  const bounds = checkOffsets(offsets, groups, k);
  if (lda < Math.max(1, m)) throw new Error("lda must be >= max(1, m).");
  if (ldb < Math.max(1, n)) throw new Error("ldb must be >= max(1, n).");
  if (ldc < Math.max(1, m)) throw new Error("ldc must be >= max(1, m).");
  if (groups > 1 && strideC < span(m, n, ldc)) throw new Error("strideC must cover a group's C.");
  if (m === 0 || n === 0 || groups === 0) return resident ? {} : { C };
  checkLength("A", A, span(m, k, lda));
  checkLength("B", B, span(n, k, ldb));
  checkLength("C", C, (groups - 1) * strideC + span(m, n, ldc));
  return execute(device, [A, B, bounds], C, resident, Float32Array, (ctx, p, pC) =>
    native().gemmGroupedK(ctx, F32, groups, m, n, k, alpha, p[0], lda, p[1], ldb, p[2], beta, pC, ldc, strideC, F32),
  );
}
