// A k x n matrix of 4-bit floats on the device (MXFP4: blocks of 32 along k
// with a power of two each): `_codes` holds two codes a byte, `_scales` a byte
// a block, each column in whole runs of 128 elements (`ld`). wgblas has no
// counterpart.
import { HipDevice, getDevice } from "../init.mjs";
import { native } from "../native.mjs";
import { checkFlat, checkLength, checkSizes, F32, span } from "../grouped_common.mjs";
import { requireSameDevice } from "../device.mjs";

export class Mxfp4Matrix {
  constructor(codes, scales, k, n, ld, device) {
    this._codes = codes;
    this._scales = scales;
    this.k = k;
    this.n = n;
    this.ld = ld;
    this.device = device;
  }

  /**
   * Mxfp4Matrix.quantize([device,] X, k, n, ldx?, trans = 'no-transpose'):
   * X is k x n column-major, or n x k for 'transpose' (its transpose is
   * quantised); ldx defaults to its rows. A Float32Array is uploaded for the
   * call, a GpuVector read in place.
   */
  static quantize(deviceOrData, ...rest) {
    const explicit = deviceOrData instanceof HipDevice;
    const device = explicit ? deviceOrData : getDevice();
    const X = explicit ? rest.shift() : deviceOrData;
    const [k, n] = rest;
    const trans = rest[3] === undefined ? "no-transpose" : rest[3];
    if (trans !== "no-transpose" && trans !== "transpose") throw new Error("trans must be 'no-transpose' or 'transpose'.");
    checkSizes("k and n", [k, n]);
    const resident = checkFlat({ X });
    requireSameDevice(device, "Mxfp4Matrix.quantize", { X });
    const t = trans === "transpose";
    const rows = t ? n : k, cols = t ? k : n;
    const ldx = rest[2] === undefined ? Math.max(1, rows) : rest[2];
    checkSizes("ldx", [ldx]);
    if (ldx < Math.max(1, rows)) throw new Error("ldx must be >= max(1, rows of X).");
    checkLength("X", X, span(rows, cols, ldx));
    const ld = Math.max(128, Math.ceil(k / 128) * 128);
    const nat = native();
    const ctx = device.ctx();
    const buffers = [];
    const room = (bytes) => {
      buffers.push(nat.malloc(ctx, bytes));
      return buffers[buffers.length - 1];
    };
    let temp = null;
    try {
      const codes = room((n * ld) / 2), scales = room((n * ld) / 32);
      if (!resident) {
        temp = nat.malloc(ctx, X.byteLength);
        nat.upload(ctx, temp, X);
      }
      nat.mxfp4Quantize(ctx, F32, t ? 1 : 0, k, n, resident ? X._buf : temp, ldx, codes, scales, ld);
      return new Mxfp4Matrix(codes, scales, k, n, ld, device);
    } catch (e) {
      for (const b of buffers) nat.free(ctx, b);
      throw e;
    } finally {
      if (temp !== null) nat.free(ctx, temp);
    }
  }

  /** The values it stands for: a Float32Array of k x n, column-major and dense. */
  async read() {
    const nat = native();
    const ctx = this.device.ctx();
    const out = new Float32Array(this.k * this.n);
    if (out.length === 0) return out;
    const temp = nat.malloc(ctx, out.byteLength);
    try {
      nat.mxfp4Dequantize(ctx, F32, this.k, this.n, this._codes, this._scales, this.ld, temp, this.k);
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

