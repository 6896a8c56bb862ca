// TypeScript declarations for mxfp4Gemm and mxfp4GemmGrouped (src/mxfp4Gemm.mjs).
import { HipDevice } from "./init.mjs";
import { GpuVector } from "./classes/GpuVector.mjs";
import { Mxfp4Matrix } from "./classes/Mxfp4Matrix.mjs";
import type { Offsets } from "./sgemmGrouped.mjs";
import type { Timed } from "./types.mjs";

/** C = alpha A^T B + beta C: A k x m, B k x n, C m x n, column-major; a new Float32Array. */
export declare function mxfp4Gemm(
  device: HipDevice, alpha: number, A: Mxfp4Matrix, B: Mxfp4Matrix, beta: number, C: Float32Array, ldc: number,
): Promise<{ C: Float32Array } & Timed>;

/** Resident C: updated in place on the device. */
export declare function mxfp4Gemm(
  device: HipDevice, alpha: number, A: Mxfp4Matrix, B: Mxfp4Matrix, beta: number, C: GpuVector, ldc: number,
): Promise<Timed>;

/**
 * C(:, j) = alpha A_g^T B(:, j) + beta C(:, j) for offsets[g] <= j < offsets[g + 1], A_g the m columns of A from
 * column g * m on.
 */
export declare function mxfp4GemmGrouped(
  device: HipDevice, groups: number, m: number, alpha: number, A: Mxfp4Matrix, B: Mxfp4Matrix, offsets: Offsets,
  beta: number, C: Float32Array, ldc: number,
): Promise<{ C: Float32Array } & Timed>;

/** Resident C: updated in place on the device. */
export declare function mxfp4GemmGrouped(
  device: HipDevice, groups: number, m: number, alpha: number, A: Mxfp4Matrix, B: Mxfp4Matrix, offsets: Offsets,
  beta: number, C: GpuVector, ldc: number,
): Promise<Timed>;
