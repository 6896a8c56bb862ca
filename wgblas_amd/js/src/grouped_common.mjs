// Checks and execution shared by the grouped and 4-bit routines. wgblas has no
// counterpart of them; names, order and wording of the checks follow its
// other routines.
import { GpuVector } from "./classes/GpuVector.mjs";

export const F32 = 0;  // WGB_F32

/** Throws unless every value is a non-negative integer. */
export function checkSizes(names, values) {
  for (const v of values) if (!Number.isInteger(v)) throw new Error(`${names} must be integers.`);
  for (const v of values) if (v < 0) throw new Error(`${names} must be non-negative.`);
}

/** Operands are Float32Array or Float32Array-backed GpuVector, all of one kind. */
export function checkFlat(operands) {
  const entries = Object.entries(operands);
  for (const [name, X] of entries)
    if (!(X instanceof Float32Array) && !(X instanceof GpuVector && X.dtype === Float32Array))
      throw new Error(`${name} must be a Float32Array or a Float32Array-backed GpuVector.`);
  const resident = entries.filter(([, X]) => X instanceof GpuVector).length;
  if (resident !== 0 && resident !== entries.length)
    throw new Error(`${entries.map(([n]) => n).join(", ")} must be all host arrays or all GpuVector.`);
  return resident !== 0;
}

/** Throws unless X holds `need` elements. */
export function checkLength(name, X, need) {
  if (X.length < need) throw new Error(`${name} does not have enough elements for the given dimensions.`);
}

/**
 * groups + 1 boundaries (Int32Array, BigInt64Array or an array of integers),
 * never decreasing, from 0 to at most `columns`; returned as BigInt64Array.
 */
export function checkOffsets(offsets, groups, columns) {
  const ok = offsets instanceof Int32Array || offsets instanceof BigInt64Array || Array.isArray(offsets);
  if (!ok) throw new Error("offsets must be an Int32Array, a BigInt64Array or an array of integers.");
  if (offsets.length !== groups + 1) throw new Error("offsets must hold groups + 1 boundaries.");
  const out = new BigInt64Array(groups + 1);
  for (let g = 0; g <= groups; ++g) {
    const v = Number(offsets[g]);
    if (!Number.isInteger(v) || v < 0 || v > columns || (g > 0 && v < Number(out[g - 1])))
      throw new Error("offsets must not decrease and must stay within the columns.");
    out[g] = BigInt(v);
  }
  if (out[0] !== 0n) throw new Error("offsets must start at 0.");
  return out;
}

/** Elements of `cols` columns of `rows` at leading dimension ld. */
export const span = (rows, cols, ld) => (cols > 0 && rows > 0 ? (cols - 1) * ld + rows : 0);

