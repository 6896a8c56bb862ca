// TypeScript declarations for Mxfp4Matrix (src/classes/Mxfp4Matrix.mjs).
import { HipDevice } from "../init.mjs";
import { GpuVector } from "./GpuVector.mjs";
import type { Trans } from "../types.mjs";

/** A k x n matrix of 4-bit floats on the device, in blocks of 32 along k with a power of two each. */
export declare class Mxfp4Matrix {
  readonly k: number;
  readonly n: number;
  /** Elements between columns, a multiple of 128. */
  readonly ld: number;
  readonly device: HipDevice;
  /** Quantises X: k x n column-major, or n x k for "transpose". */
  static quantize(device: HipDevice, X: Float32Array | GpuVector, k: number, n: number, ldx?: number, trans?: Trans): Mxfp4Matrix;
  static quantize(X: Float32Array | GpuVector, k: number, n: number, ldx?: number, trans?: Trans): Mxfp4Matrix;
  /** The values it stands for, k x n, column-major and dense. */
  read(): Promise<Float32Array>;
  /** Frees the device allocations (safe to call twice). */
  destroy(): void;
}
