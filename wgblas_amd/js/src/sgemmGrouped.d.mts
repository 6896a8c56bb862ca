// TypeScript declarations for sgemmGrouped and sgemmGroupedK (src/sgemmGrouped.mjs).
import { HipDevice } from "./init.mjs";
import { GpuVector } from "./classes/GpuVector.mjs";
import type { Timed, Trans } from "./types.mjs";

/** Boundaries of the groups: groups + 1 integers from 0, never decreasing. */
export type Offsets = Int32Array | BigInt64Array | number[];

/**
 * C(:, j) = alpha op(A_g) B(:, j) + beta C(:, j) for offsets[g] <= j < offsets[g + 1].
 * Column-major: A_g (at g * strideA elements) is m x k, or k x m for "transpose"; B is k x n, C m x n.
 * Columns of no group keep their values. Host arrays: the result comes back as a new Float32Array.
 */
export declare function sgemmGrouped(
  device: HipDevice, transA: Trans, groups: number, m: number, n: number, k: number, alpha: number,
  A: Float32Array, lda: number, strideA: number, B: Float32Array, ldb: number, offsets: Offsets,
  beta: number, C: Float32Array, ldc: number,
): Promise<{ C: Float32Array } & Timed>;

/** Resident operands: C is updated in place on the device. */
export declare function sgemmGrouped(
  device: HipDevice, transA: Trans, groups: number, m: number, n: number, k: number, alpha: number,
  A: GpuVector, lda: number, strideA: number, B: GpuVector, ldb: number, offsets: Offsets,
  beta: number, C: GpuVector, ldc: number,
): Promise<Timed>;

/**
 * C_g = alpha A(:, g) B(:, g)^T + beta C_g over the columns of each group: A is m x k, B n x k,
 * C_g (at g * strideC elements) m x n, column-major. An empty group gives beta C_g.
 */
export declare function sgemmGroupedK(
  device: HipDevice, groups: number, m: number, n: number, k: number, alpha: number,
  A: Float32Array, lda: number, B: Float32Array, ldb: number, offsets: Offsets,
  beta: number, C: Float32Array, ldc: number, strideC: number,
): Promise<{ C: Float32Array } & Timed>;

/** Resident operands: C is updated in place on the device. */
export declare function sgemmGroupedK(
  device: HipDevice, groups: number, m: number, n: number, k: number, alpha: number,
  A: GpuVector, lda: number, B: GpuVector, ldb: number, offsets: Offsets,
  beta: number, C: GpuVector, ldc: number, strideC: number,
): Promise<Timed>;
