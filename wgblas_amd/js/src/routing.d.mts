// TypeScript declarations for the routing calls (src/routing.mjs).
import { HipDevice } from "./init.mjs";
import { GpuVector } from "./classes/GpuVector.mjs";
import type { Timed } from "./types.mjs";

export type Scoring = "softmax" | "sigmoid";
export type RouteOptions = {
  /** Added to the scores for the choice alone. */
  bias?: Float32Array | null;
  /** Groups of experts, of which topGroups stay, by their `best` largest choice values. */
  groups?: number;
  topGroups?: number;
  best?: 1 | 2;
  /** Whether the weights are divided by their sum. */
  renorm?: boolean;
  scale?: number;
};

/** The topk experts of each token and their weights; ids are -1 where no expert is left. */
export declare function route(
  device: HipDevice, scoring: Scoring, experts: number, n: number, topk: number, logits: Float32Array | GpuVector, ldl: number,
  options?: RouteOptions,
): Promise<{ ids: Int32Array; weights: Float32Array } & Timed>;

/** The logits' gradient, dense, from the weights'. */
export declare function routeGrad(
  device: HipDevice, scoring: Scoring, experts: number, n: number, topk: number, logits: Float32Array | GpuVector, ldl: number,
  ids: Int32Array, dweights: Float32Array, options?: { renorm?: boolean; scale?: number },
): Promise<{ dlogits: Float32Array } & Timed>;

/** The pairs (token, expert) in the order of their expert. */
export declare function routeOrder(
  device: HipDevice, experts: number, n: number, topk: number, ids: Int32Array,
): Promise<{ offsets: BigInt64Array; places: Int32Array; pairs: Int32Array } & Timed>;

/** Tokens' columns to their places, times their weights (null: 1). */
export declare function routeGather(
  device: HipDevice, d: number, n: number, topk: number, X: Float32Array, ldx: number, places: Int32Array,
  weights: Float32Array | null, Y: Float32Array, ldy: number,
): Promise<{ Y: Float32Array } & Timed>;
export declare function routeGather(
  device: HipDevice, d: number, n: number, topk: number, X: GpuVector, ldx: number, places: Int32Array,
  weights: Float32Array | null, Y: GpuVector, ldy: number,
): Promise<Timed>;

/** The weighted sums of the columns at tokens' places, plus beta C. */
export declare function routeCombine(
  device: HipDevice, d: number, n: number, topk: number, Y: Float32Array, ldy: number, places: Int32Array,
  weights: Float32Array | null, beta: number, C: Float32Array, ldc: number,
): Promise<{ C: Float32Array } & Timed>;
export declare function routeCombine(
  device: HipDevice, d: number, n: number, topk: number, Y: GpuVector, ldy: number, places: Int32Array,
  weights: Float32Array | null, beta: number, C: GpuVector, ldc: number,
): Promise<Timed>;

/** routeCombine's gradients; dY may be the GpuVector Y. */
export declare function routeCombineGrad(
  device: HipDevice, d: number, n: number, topk: number, dC: Float32Array, lddc: number, Y: Float32Array, ldy: number,
  places: Int32Array, weights: Float32Array, dY: Float32Array, lddy: number,
): Promise<{ dY: Float32Array; dweights: Float32Array } & Timed>;
export declare function routeCombineGrad(
  device: HipDevice, d: number, n: number, topk: number, dC: GpuVector, lddc: number, Y: GpuVector, ldy: number,
  places: Int32Array, weights: Float32Array, dY: GpuVector, lddy: number,
): Promise<{ dweights: Float32Array } & Timed>;
