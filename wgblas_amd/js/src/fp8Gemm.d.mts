// TypeScript declarations for fp8Gemm and fp8GemmGrouped (src/fp8Gemm.mjs).
import { HipDevice } from "./init.mjs";
import { GpuVector } from "./classes/GpuVector.mjs";
import { Fp8Matrix } from "./classes/Fp8Matrix.mjs";
import type { Offsets } from "./sgemmGrouped.mjs";
import type { Timed, Trans } from "./types.mjs";

/** C = alpha op(A) B + beta C: B k x n, C m x n, column-major; a new Float32Array. */
export declare function fp8Gemm(
  device: HipDevice, transA: Trans, alpha: number, A: Fp8Matrix, B: Fp8Matrix, beta: number, C: Float32Array, ldc: number,
): Promise<{ C: Float32Array } & Timed>;

/** Resident C: updated in place on the device. */
export declare function fp8Gemm(
  device: HipDevice, transA: Trans, alpha: number, A: Fp8Matrix, B: Fp8Matrix, beta: number, C: GpuVector, ldc: number,
): Promise<Timed>;

/** C(:, j) = alpha op(A_g) B(:, j) + beta C(:, j) for offsets[g] <= j < offsets[g + 1], A_g the matrix g of A. */
export declare function fp8GemmGrouped(
  device: HipDevice, transA: Trans, alpha: number, A: Fp8Matrix, B: Fp8Matrix, offsets: Offsets, beta: number,
  C: Float32Array, ldc: number,
): Promise<{ C: Float32Array } & Timed>;

/** Resident C: updated in place on the device. */
export declare function fp8GemmGrouped(
  device: HipDevice, transA: Trans, alpha: number, A: Fp8Matrix, B: Fp8Matrix, offsets: Offsets, beta: number,
  C: GpuVector, ldc: number,
): Promise<Timed>;
