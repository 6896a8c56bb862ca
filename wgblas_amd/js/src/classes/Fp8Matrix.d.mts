// TypeScript declarations for Fp8Matrix (src/classes/Fp8Matrix.mjs).
import { HipDevice } from "../init.mjs";
import { GpuVector } from "./GpuVector.mjs";
import type { Trans } from "../types.mjs";

/** Matrices k x n of 8-bit floats (E4M3) on the device, a scale for each block of 128 along k by `block` columns. */
export declare class Fp8Matrix {
  readonly k: number;
  readonly n: number;
  /** Columns of a block: 1 (activations) or 128 (weights). */
  readonly block: 1 | 128;
  readonly matrices: number;
  /** Codes between columns, a multiple of 128. */
  readonly ld: number;
  /** Scales between blocks along k. */
  readonly lds: number;
  readonly device: HipDevice;
  /** Quantises X: the matrices one behind another, k x n column-major, or n x k for "transpose". */
  static quantize(
    device: HipDevice, X: Float32Array | GpuVector, k: number, n: number, block?: 1 | 128, matrices?: number, ldx?: number,
    trans?: Trans,
  ): Fp8Matrix;
  static quantize(
    X: Float32Array | GpuVector, k: number, n: number, block?: 1 | 128, matrices?: number, ldx?: number, trans?: Trans,
  ): Fp8Matrix;
  /** The values they stand for, k x n, column-major and dense. */
  read(): Promise<Float32Array>;
  /** Frees the device allocations (safe to call twice). */
  destroy(): void;
}
