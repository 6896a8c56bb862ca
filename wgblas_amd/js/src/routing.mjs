// Routing of tokens to experts: the experts of each token and their weights
// (route), the pairs (token, expert) in the order of their expert (routeOrder),
// the tokens' columns copied there (routeGather) and added up again
// (routeCombine), and the gradients (routeGrad, routeCombineGrad; the gradient
// of routeGather's X is routeCombine without weights). Matrices are column-major,
// Float32Array or GpuVector; ids, places and weights (topk x n) are host arrays.
// wgblas has no counterpart.
// Return their host results by name (those in a GpuVector are left there), plus
// gpuTimeMs when init({benchmark:true}).
import { checkScalar } from "./gemm_common.mjs";
import { checkFlat, checkLength, checkSizes, F32, span } from "./grouped_common.mjs";
import { GpuVector } from "./classes/GpuVector.mjs";
import { requireGpuDevice, requireSameDevice } from "./device.mjs";
import { lastGpuTimeMs } from "./init.mjs";
import { native } from "./native.mjs";

const SCORING = { softmax: 0, sigmoid: 1 };

/** launch(ctx, pointers of the inputs, of the outputs); outputs are uploaded first, since calls leave parts as they were. */
function call(device, inputs, outputs, launch) {
  const nat = native();
  const ctx = device.ctx();
  const temps = [];
  const pointer = (X) => {
    if (X === null) return null;
    if (X instanceof GpuVector) return X._buf;
    const p = nat.malloc(ctx, X.byteLength);
    temps.push(p);
    if (X.length > 0) nat.upload(ctx, p, X);
    return p;
  };
  try {
    const pIn = inputs.map(pointer), entries = Object.entries(outputs), pOut = entries.map(([, X]) => pointer(X));
    launch(nat, ctx, pIn, pOut);
    const t = lastGpuTimeMs(device);
    const result = t === undefined ? {} : { gpuTimeMs: t };
    entries.forEach(([name, X], i) => {
      if (X instanceof GpuVector) return;
      result[name] = new X.constructor(X.length);
      if (X.length > 0) nat.download(ctx, pOut[i], result[name]);
    });
    return result;
  } finally {
    for (const p of temps) nat.free(ctx, p);
  }
}

function checkTopk(n, topk) {
  checkSizes("n and topk", [n, topk]);
  if (topk < 1 || topk > 64) throw new Error("topk must be from 1 to 64.");
  if (n * topk >= 2 ** 31) throw new Error("n * topk must be below 2^31.");
}

function checkExperts(experts) {
  checkSizes("experts", [experts]);
  if (experts < 1 || experts > 1024) throw new Error("experts must be from 1 to 1024.");
}

function checkList(name, type, X, need) {
  if (!(X instanceof type)) throw new Error(`${name} must be ${type === Int32Array ? "an Int32Array" : "a Float32Array"}.`);
  checkLength(name, X, need);
}

function checkScoring(scoring) {
  if (!Object.prototype.hasOwnProperty.call(SCORING, scoring)) throw new Error("scoring must be 'softmax' or 'sigmoid'.");
  return SCORING[scoring];
}

function checkMatrix(name, X, rows, cols, ld) {
  checkSizes(`ld of ${name}`, [ld]);
  if (ld < Math.max(1, rows)) throw new Error(`ld of ${name} must be >= max(1, its rows).`);
  checkLength(name, X, span(rows, cols, ld));
}

/** { ids: Int32Array, weights: Float32Array }; options: bias, groups, topGroups, best, renorm, scale. */
export async function route(device, scoring, experts, n, topk, logits, ldl, options = {}) {
  requireGpuDevice(device);
  requireSameDevice(device, "route", { logits });
  const { bias = null, groups = 1, topGroups = groups, best = 1, renorm = false, scale = 1 } = options;
  const kind = checkScoring(scoring);
  checkExperts(experts);
  checkTopk(n, topk);
  if (topk > experts) throw new Error("topk must be at most experts.");
  checkFlat({ logits });
  checkMatrix("logits", logits, experts, n, ldl);
  if (bias !== null) checkList("bias", Float32Array, bias, experts);
  checkSizes("groups, topGroups, and best", [groups, topGroups, best]);
  if (groups < 1 || experts % groups !== 0) throw new Error("groups must divide experts.");
  if (topGroups < 1 || topGroups > groups) throw new Error("topGroups must be from 1 to groups.");
  if (best !== 1 && best !== 2) throw new Error("best must be 1 or 2.");
  checkScalar("scale", scale);
  const out = { ids: new Int32Array(n * topk), weights: new Float32Array(n * topk) };
  if (n === 0) return out;
  return call(device, [logits, bias], out, (nat, ctx, i, o) =>
    nat.route(ctx, F32, kind, experts, n, topk, i[0], ldl, i[1], groups, topGroups, best, renorm ? 1 : 0, scale, o[0], o[1]),
  );
}

/** { dlogits }: dense, experts x n, from the weights' gradient and route's ids; options: renorm and scale as there. */
export async function routeGrad(device, scoring, experts, n, topk, logits, ldl, ids, dweights, options = {}) {
  requireGpuDevice(device);
  requireSameDevice(device, "routeGrad", { logits });
  const { renorm = false, scale = 1 } = options;
  const kind = checkScoring(scoring);
  checkExperts(experts);
  checkTopk(n, topk);
  if (topk > experts) throw new Error("topk must be at most experts.");
  checkFlat({ logits });
  checkMatrix("logits", logits, experts, n, ldl);
  checkList("ids", Int32Array, ids, n * topk);
  checkList("dweights", Float32Array, dweights, n * topk);
  checkScalar("scale", scale);
  const out = { dlogits: new Float32Array(n * experts) };
  if (n === 0) return out;
  return call(device, [logits, ids, dweights], out, (nat, ctx, i, o) =>
    nat.routeGrad(ctx, F32, kind, experts, n, topk, i[0], ldl, i[1], renorm ? 1 : 0, scale, i[2], o[0], experts),
  );
}

/** { offsets: BigInt64Array, places: Int32Array, pairs: Int32Array } */
export async function routeOrder(device, experts, n, topk, ids) {
  requireGpuDevice(device);
  checkExperts(experts);
  checkTopk(n, topk);
  checkList("ids", Int32Array, ids, n * topk);
  const out = { offsets: new BigInt64Array(experts + 1), places: new Int32Array(n * topk), pairs: new Int32Array(n * topk) };
  if (n === 0) return out;
  return call(device, [ids], out, (nat, ctx, i, o) => nat.routeOrder(ctx, experts, n, topk, i[0], o[0], o[1], o[2]));
}

function checkRows(routine, device, d, n, topk, places, weights, matrices) {
  requireGpuDevice(device);
  requireSameDevice(device, routine, matrices);
  checkSizes("d", [d]);
  checkTopk(n, topk);
  checkFlat(matrices);
  checkList("places", Int32Array, places, n * topk);
  if (weights !== null) checkList("weights", Float32Array, weights, n * topk);
}

/** { Y }: column places[t*topk + s] is weights' (null: 1) times X's column t; the others are as they were. */
export async function routeGather(device, d, n, topk, X, ldx, places, weights, Y, ldy) {
  checkRows("routeGather", device, d, n, topk, places, weights, { X, Y });
  checkMatrix("X", X, d, n, ldx);
  checkMatrix("Y", Y, d, n * topk, ldy);
  if (d === 0 || n === 0) return Y instanceof GpuVector ? {} : { Y };
  return call(device, [X, places, weights], { Y }, (nat, ctx, i, o) =>
    nat.routeGather(ctx, F32, d, n, topk, i[0], ldx, i[1], i[2], o[0], ldy),
  );
}

/** { C }: column t is the sum of weights' (null: 1) times Y's columns places[t*topk + s], plus beta times itself. */
export async function routeCombine(device, d, n, topk, Y, ldy, places, weights, beta, C, ldc) {
  checkRows("routeCombine", device, d, n, topk, places, weights, { Y, C });
  checkScalar("beta", beta);
  checkMatrix("Y", Y, d, n * topk, ldy);
  checkMatrix("C", C, d, n, ldc);
  if (d === 0 || n === 0) return C instanceof GpuVector ? {} : { C };
  return call(device, [Y, places, weights], { C }, (nat, ctx, i, o) =>
    nat.routeCombine(ctx, F32, d, n, topk, i[0], ldy, i[1], i[2], beta, o[0], ldc, F32),
  );
}

/** { dY, dweights }: routeCombine's gradients from C's; dY may be the GpuVector Y. */
export async function routeCombineGrad(device, d, n, topk, dC, lddc, Y, ldy, places, weights, dY, lddy) {
  checkRows("routeCombineGrad", device, d, n, topk, places, weights, { dC, Y, dY });
  if (weights === null) throw new Error("weights must be a Float32Array.");
  checkMatrix("dC", dC, d, n, lddc);
  checkMatrix("Y", Y, d, n * topk, ldy);
  checkMatrix("dY", dY, d, n * topk, lddy);
  if (dY === Y && lddy !== ldy) throw new Error("lddy must be ldy where dY is Y.");
  const dweights = new Float32Array(n * topk);
  if (d === 0 || n === 0) return dY instanceof GpuVector ? { dweights } : { dY, dweights };
  return call(device, [dC, Y, places, weights], { dY, dweights }, (nat, ctx, i, o) =>
    nat.routeCombineGrad(ctx, F32, d, n, topk, i[0], lddc, i[1], ldy, i[2], i[3], o[0], lddy, o[1]),
  );
}
