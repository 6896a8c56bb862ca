// One or more k x n matrices of 8-bit floats on the device (E4M3), with an fp32
// scale for each block of 128 values along k, of `block` columns (1:
// activations and gradients, 128: weights). `_codes` holds a byte a value, each
// column in whole runs of 128 (`ld`), `_scales` a row of `lds` column blocks for
// each run. wgblas has no counterpart.
import { HipDevice, getDevice } from "../init.mjs";
import { native } from "../native.mjs";
import { checkFlat, checkLength, checkSizes, F32, span } from "../grouped_common.mjs";
import { requireSameDevice } from "../device.mjs";

export class Fp8Matrix {
  constructor(codes, scales, k, n, block, matrices, device) {
    this._codes = codes;
    this._scales = scales;
    this.k = k;
    this.n = n;
    this.block = block;
    this.matrices = matrices;
    this.ld = Math.max(128, Math.ceil(k / 128) * 128);
    this.lds = Math.max(1, Math.ceil(n / block));
    this.device = device;
  }

  /**
   * Fp8Matrix.quantize([device,] X, k, n, block = 1, matrices = 1, ldx?, trans = 'no-transpose'):
   * X holds the matrices one behind another, each k x n column-major, or n x k
   * for 'transpose' (its transpose is quantised); ldx defaults to its rows. A
   * Float32Array is uploaded for the call, a GpuVector read in place.
   */
  static quantize(deviceOrData, ...rest) {
    const explicit = deviceOrData instanceof HipDevice;
    const device = explicit ? deviceOrData : getDevice();
    const X = explicit ? rest.shift() : deviceOrData;
    const [k, n] = rest;
    const block = rest[2] === undefined ? 1 : rest[2], matrices = rest[3] === undefined ? 1 : rest[3];
    const trans = rest[5] === undefined ? "no-transpose" : rest[5];
    if (trans !== "no-transpose" && trans !== "transpose") throw new Error("trans must be 'no-transpose' or 'transpose'.");
    if (block !== 1 && block !== 128) throw new Error("block must be 1 or 128.");
    checkSizes("k, n, and matrices", [k, n, matrices]);
    if (k > 2 ** 23) throw new Error("k must be at most 2^23.");
    const resident = checkFlat({ X });
    requireSameDevice(device, "Fp8Matrix.quantize", { X });
    const t = trans === "transpose";
    const rows = t ? n : k, cols = t ? k : n;
    const ldx = rest[4] === undefined ? Math.max(1, rows) : rest[4];
    checkSizes("ldx", [ldx]);
    if (ldx < Math.max(1, rows)) throw new Error("ldx must be >= max(1, rows of X).");
    if (matrices > 0) checkLength("X", X, span(rows, cols, ldx) > 0 ? (matrices - 1) * ldx * cols + span(rows, cols, ldx) : 0);
    const made = new Fp8Matrix(null, null, k, n, block, matrices, device);
    const nat = native();
    const ctx = device.ctx();
    const buffers = [];
    const room = (bytes) => {
      buffers.push(nat.malloc(ctx, bytes));
      return buffers[buffers.length - 1];
    };
    let temp = null;
    try {
      made._codes = room(matrices * n * made.ld);
      made._scales = room((matrices * made.ld * made.lds) / 32);
      if (!resident) {
        temp = nat.malloc(ctx, X.byteLength);
        nat.upload(ctx, temp, X);
      }
      nat.fp8Quantize(ctx, F32, t ? 1 : 0, block, matrices, k, n, resident ? X._buf : temp, ldx, made._codes, made.ld,
                      made._scales, made.lds);
      return made;
    } catch (e) {
      for (const b of buffers) nat.free(ctx, b);
      throw e;
    } finally {
      if (temp !== null) nat.free(ctx, temp);
    }
  }

  /** The values it stands for: a Float32Array of the matrices, k x n, column-major and dense. */
  async read() {
    if (this._codes === null) throw new Error("Fp8Matrix.read: the matrix was destroyed.");
    const nat = native();
    const ctx = this.device.ctx();
    const out = new Float32Array(this.matrices * this.k * this.n);
    if (out.length === 0) return out;
    const temp = nat.malloc(ctx, out.byteLength);
    try {
      nat.fp8Dequantize(ctx, F32, this.block, this.matrices, this.k, this.n, this._codes, this.ld, this._scales, this.lds, temp,
                        this.k);
      nat.download(ctx, temp, out);
    } finally {
      nat.free(ctx, temp);
    }
    return out;
  }

  /** Frees the device allocations (safe to call twice). */
  destroy() {
    for (const b of [this._codes, this._scales])
      if (b !== null && this.device._ctx !== null) native().free(this.device._ctx, b);
    this._codes = this._scales = null;
  }
}
