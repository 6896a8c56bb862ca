// cpu_addon.cjs with the grouped and 4-bit calls, in float64 under the C ABI's
// semantics: lets the JS layer's routines for them run without a GPU.
"use strict";

const base = require("./cpu_addon.cjs");
const stub = require("./stub_addon.cjs");

const raw = (c, b) => stub._stub.bytes(c, b);
const f32 = (c, b) => new Float32Array(raw(c, b).buffer, 0, raw(c, b).byteLength >> 2);
const bounds = (c, b) => Array.from(new BigInt64Array(raw(c, b).buffer), Number);
const LEVELS = [0, 0.5, 1, 1.5, 2, 3, 4, 6];

function store(C, at, alpha, sum, beta) {
  C[at] = alpha * sum + (beta !== 0 ? beta * C[at] : 0);
}

const value = (codes, scales, ld, p, j) => {
  const byte = codes[j * (ld / 2) + (p >> 1)], code = p & 1 ? byte >> 4 : byte & 15, s = scales[j * (ld / 32) + (p >> 5)];
  return (code & 8 ? -1 : 1) * LEVELS[code & 7] * (s === 255 ? NaN : 2 ** (s - 127));
};

module.exports = Object.assign({}, base, {
  gemmGrouped(c, type, ta, groups, m, n, k, alpha, A, lda, strideA, B, ldb, off, beta, C, ldc, ctype) {
    if (type !== 0 || ctype !== 0) throw new Error("the stand-in computes in float32 only");
    const a = f32(c, A), b = f32(c, B), out = f32(c, C), o = bounds(c, off);
    for (let g = 0; g < groups; ++g)
      for (let j = o[g]; j < o[g + 1]; ++j)
        for (let i = 0; i < m; ++i) {
          let s = 0;
          for (let p = 0; p < k; ++p) s += a[g * strideA + (ta ? i * lda + p : p * lda + i)] * b[j * ldb + p];
          store(out, j * ldc + i, alpha, s, beta);
        }
  },
  gemmGroupedK(c, type, groups, m, n, k, alpha, A, lda, B, ldb, off, beta, C, ldc, strideC, ctype) {
    if (type !== 0 || ctype !== 0) throw new Error("the stand-in computes in float32 only");
    const a = f32(c, A), b = f32(c, B), out = f32(c, C), o = bounds(c, off);
    for (let g = 0; g < groups; ++g)
      for (let j = 0; j < n; ++j)
        for (let i = 0; i < m; ++i) {
          let s = 0;
          for (let p = o[g]; p < o[g + 1]; ++p) s += a[p * lda + i] * b[p * ldb + j];
          store(out, g * strideC + j * ldc + i, alpha, s, beta);
        }
  },
  mxfp4Quantize(c, type, trans, k, n, X, ldx, codes, scales, ld) {
    const x = f32(c, X), q = raw(c, codes), e = raw(c, scales);
    for (let j = 0; j < n; ++j)
      for (let b = 0; b < Math.ceil(k / 128) * 4; ++b) {
        const v = [];
        for (let p = 32 * b; p < 32 * b + 32; ++p) v.push(p < k ? (trans ? x[p * ldx + j] : x[j * ldx + p]) : 0);
        const top = Math.max(...v.map(Math.abs));
        const s = !v.every(Number.isFinite) ? 255 : top === 0 ? 0 : Math.max(0, Math.floor(Math.log2(top)) - 2 + 127);
        e[j * (ld / 32) + b] = s;
        v.forEach((y, i) => {
          let best = 0;
          if (s !== 255) {
            const z = Math.abs(y) / 2 ** (s - 127);
            for (let l = 1; l < 8; ++l) {
              const d = Math.abs(z - LEVELS[l]), was = Math.abs(z - LEVELS[best]);
              if (d < was || (d === was && l % 2 === 0)) best = l;
            }
            if (y < 0) best += 8;
          }
          const at = j * (ld / 2) + 16 * b + (i >> 1);
          q[at] = i & 1 ? (q[at] & 15) | (best << 4) : best;
        });
      }
  },
  mxfp4Dequantize(c, type, k, n, codes, scales, ld, X, ldx) {
    const x = f32(c, X);
    for (let j = 0; j < n; ++j) for (let p = 0; p < k; ++p) x[j * ldx + p] = value(raw(c, codes), raw(c, scales), ld, p, j);
  },
  mxfp4Gemm(c, groups, m, n, k, alpha, A, sA, lda, strideA, B, sB, ldb, off, beta, C, ldc, ctype) {
    if (ctype !== 0) throw new Error("the stand-in computes in float32 only");
    const out = f32(c, C), o = groups < 0 ? [0, n] : bounds(c, off);
    for (let g = 0; g < Math.abs(groups); ++g)
      for (let j = o[g]; j < o[g + 1]; ++j)
        for (let i = 0; i < m; ++i) {
          let s = 0;
          for (let p = 0; p < k; ++p)
            s += value(raw(c, A), raw(c, sA), lda, p, (g * strideA) / lda + i) * value(raw(c, B), raw(c, sB), ldb, p, j);
          store(out, j * ldc + i, alpha, s, beta);
        }
  },
});
