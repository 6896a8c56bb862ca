// FP8: matrices of 8-bit floats (E4M3) with an fp32 scale for each block of
// 128 values along k, of one column (activations, gradients) or of 128
// (weights): their conversion from and to f32 / f16 / bf16, and their
// products (fp8_tile.h).
//
// Quantisation: a block's scale is the least power of two s >= 2^-126 with
// max |x| / s <= 448, the largest code. So x / s is exact, its rounding to a
// code depends on nothing but x, and of a code's 16 binades at most one is
// given away; with s = max |x| / 448 itself every value would be divided and
// rounded twice. Scales that come with weights may be any numbers.
#include "fp8_tile.h"

namespace {

using namespace wgb_ragged;
using wgb::fail;

typedef float f2v __attribute__((ext_vector_type(2)));

// From the fp32 bits of a block's largest magnitude: its scale's bits, and
// those of the scale's reciprocal. 448 = 1.75 2^8.
__device__ __forceinline__ uint32_t scale_bits(uint32_t top) {
  const uint32_t e = top >> 23;
  if (e == 255) return 0x7fc00000u;
  const int s = (int)e - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(s < 1 ? 1 : s) << 23;
}
// Four codes of four values and the scale's bits (Inf and NaN: codes 0).
__device__ __forceinline__ uint32_t codes4(const float *x, uint32_t scale) {
  if (scale == 0x7fc00000u) return 0;
  const float inverse = __uint_as_float((254u << 23) - scale);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, r, true);
}
__device__ __forceinline__ uint32_t top_of(uint32_t t, float x) {
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;  // NaN above Inf above the rest
  return t > a ? t : a;
}

template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
  T v[8];
};
template <class T>
__device__ __forceinline__ void load8(const T *x, int64_t left, float (&f)[8]) {
  if (left >= 8) {
    const Eight<T> v = *reinterpret_cast<const Eight<T> *>(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)v.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? (float)x[i] : 0.0f;
  }
}

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
// Past the caches, if STREAM.
template <bool STREAM, class V>
__device__ __forceinline__ void put(uint8_t *to, V codes) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(codes, reinterpret_cast<V *>(to));
  else
    *reinterpret_cast<V *>(to) = codes;
}

template <int ROR>
__device__ __forceinline__ uint32_t max_ror(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x120 + ROR, 0xf, 0xf, true);
  return x > y ? x : y;
}
// The largest of a row of 16 lanes, in all of them.
__device__ __forceinline__ uint32_t row_max(uint32_t x) { return max_ror<1>(max_ror<2>(max_ror<4>(max_ror<8>(x)))); }

// Blocks of one column, along the contiguous axis: 16 lanes have a block, 8
// values each. Bound by memory. STREAM, here and below: the values are more than
// the caches hold, and codes are stored past them (bf16 8192 x 4096: 17.8 us,
// 5.6 TB/s, and 22.4 us through them).
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void quantize_kernel(const T *X, int64_t ldx, int64_t k, int64_t n, uint8_t *codes,
                                                       int64_t ld, float *scales, int64_t lds) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), k0 = (int64_t)blockIdx.y * 512 + lane * 8;
  if (j >= n || k0 >= (k + 127) / 128 * 128) return;  // whole blocks of lanes
  float f[8];
  load8(X + j * ldx + k0, k - k0, f);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = top_of(top, f[i]);
  const uint32_t scale = scale_bits(row_max(top));
  put<STREAM>(codes + j * ld + k0, u2{codes4(f, scale), codes4(f + 4, scale)});
  if ((lane & 15) == 0) scales[k0 / 128 * lds + j] = __uint_as_float(scale);
}

// 128 x 128 values a block: 32 columns at a time, 16 lanes a column (f32
// 8192 x 4096: 29.4 us, 5.7 TB/s).
template <class T, bool STREAM>
__global__ __launch_bounds__(512) void quantize_square_kernel(const T *X, int64_t ldx, int64_t k, int64_t n, uint8_t *codes,
                                                              int64_t ld, float *scales, int64_t lds, int blocks_k) {
  __shared__ uint32_t tops[8];
  const int t = threadIdx.x, kb = (int)(blockIdx.x % blocks_k);
  const int64_t jb = blockIdx.x / blocks_k, k0 = (int64_t)kb * 128 + (t & 15) * 8;
  float f[4][8];
  uint32_t top = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t j = jb * 128 + q * 32 + (t >> 4);
    if (j < n) {
      load8(X + j * ldx + k0, k - k0, f[q]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[q][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = top_of(top, f[q][i]);
  }
  top = row_max(top);
  uint32_t other = (uint32_t)__shfl_xor((int)top, 16);
  top = top > other ? top : other;
  other = (uint32_t)__shfl_xor((int)top, 32);
  top = top > other ? top : other;
  if ((t & 63) == 0) tops[t >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = top > tops[w] ? top : tops[w];
  const uint32_t scale = scale_bits(top);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t j = jb * 128 + q * 32 + (t >> 4);
    if (j < n) put<STREAM>(codes + j * ld + k0, u2{codes4(f[q], scale), codes4(f[q] + 4, scale)});
  }
  if (t == 0) scales[kb * lds + jb] = __uint_as_float(scale);
}

// Blocks along the strided axis, 128 x 128 values a block of threads: a wave has
// 16 rows of k, a lane 16 bytes of neighbouring columns in some of them, so that
// loads are as wide as those along the contiguous axis (two columns a lane and
// 16 rows: 2.9 TB/s). A lane's codes of a column, RG rows of k, go through LDS
// (four dwords more after every lane's columns: two lanes in a bank) and out as
// 128-byte lines. STREAM loads past the caches (bf16 16384 x 4096: 43 us,
// 4.7 TB/s, and 50 us through them; stores past them too: 45 us), at whole dwords
// only: at halves that is slower (bf16 16384 x 4096 at 4097: 46.8 us, 43.9 through
// the caches; 4099 x 8191 at 8191: 32.7 and 28.1).
template <class T, bool SQUARE, bool STREAM>
__global__ __launch_bounds__(512) void quantize_strided_kernel(const T *X, int64_t ldx, int64_t k, int64_t n,
                                                               uint8_t *codes, int64_t ld, float *scales, int64_t lds,
                                                               int blocks_k) {
  constexpr int V = 16 / sizeof(T), LR = 128 / V, G = 64 / LR, RG = 16 / G;  // columns, lanes a row, rows at once, a lane's rows
  __shared__ __attribute__((aligned(16))) uint32_t lines[128 * 32 + 4 * LR];
  __shared__ uint32_t tops[8][128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, g = lane / LR, c0 = lane % LR * V;
  const int kb = (int)(blockIdx.x % blocks_k);
  const int64_t j0 = blockIdx.x / blocks_k * 128, j = j0 + c0, k0 = (int64_t)kb * 128 + wave * 16 + g * RG;
  typedef int Any __attribute__((ext_vector_type(4), aligned(2)));
  struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[V];
  };
  const T *x = X + k0 * ldx + j;
  Any raw[RG];
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    raw[r] = Any{0, 0, 0, 0};
    if (k0 + r >= k) continue;
    if (j + V <= n) {
      const Any *from = reinterpret_cast<const Any *>(x + r * ldx);
      if constexpr (STREAM)
        raw[r] = __builtin_nontemporal_load(from);
      else
        raw[r] = *from;
    } else if (j < n) {
      Vec v;
#pragma unroll
      for (int c = 0; c < V; ++c) v.v[c] = j + c < n ? x[r * ldx + c] : (T)0.0f;
      raw[r] = __builtin_bit_cast(Any, v);
    }
  }
  float f[V][RG];
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const Vec v = __builtin_bit_cast(Vec, raw[r]);
#pragma unroll
    for (int c = 0; c < V; ++c) f[c][r] = (float)v.v[c];
  }
  // the columns' largest: of the lane, of the wave's lanes with the same columns, of the waves
#pragma unroll
  for (int c = 0; c < V; ++c) {
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < RG; ++r) top = top_of(top, f[c][r]);
#pragma unroll
    for (int d = LR; d < 64; d <<= 1) {
      const uint32_t other = (uint32_t)__shfl_xor((int)top, d);
      top = top > other ? top : other;
    }
    if (g == 0) tops[wave][c0 + c] = top;
  }
  __syncthreads();
  uint32_t scale[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    scale[c] = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) scale[c] = scale[c] > tops[w][c0 + c] ? scale[c] : tops[w][c0 + c];
  }
  if constexpr (SQUARE) {
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < V; ++c) top = top > scale[c] ? top : scale[c];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t other = (uint32_t)__shfl_xor((int)top, d);
      top = top > other ? top : other;
    }
#pragma unroll
    for (int c = 0; c < V; ++c) scale[c] = top;
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    scale[c] = scale_bits(scale[c]);
    uint32_t *line = lines + (c0 + c) * 32 + lane % LR * 4 + wave * 4 + g * (RG / 4);
#pragma unroll
    for (int q = 0; q < RG / 4; ++q) line[q] = codes4(f[c] + 4 * q, scale[c]);
  }
  if (wave == 0 && g == 0) {
    if constexpr (SQUARE) {
      if (lane == 0) scales[kb * lds + j0 / 128] = __uint_as_float(scale[0]);
    } else {
#pragma unroll
      for (int c = 0; c < V; ++c)
        if (j + c < n) scales[kb * lds + j + c] = __uint_as_float(scale[c]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int col = (t >> 3) + 64 * q, chunk = t & 7;
    if (j0 + col < n)
      put<false>(codes + (j0 + col) * ld + kb * 128 + chunk * 16, *reinterpret_cast<const v4i *>(lines + col * 32 + (col / V + chunk) * 4));
  }
}

// A lane has 16 bytes of output: code * scale in fp32, rounded to the output's
// type. Bound by memory. STREAM: the output is more than the caches hold, and
// stored past them (bf16 8192 x 4096: 17.0 us, 5.9 TB/s, and 29.7 us through
// them); at whole dwords only.
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t *codes, int64_t ld, const float *scales, int64_t lds,
                                                         int shift, int64_t k, int64_t n, T *X, int64_t ldx) {
  constexpr int V = 16 / sizeof(T);
  const int64_t j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), k0 = ((int64_t)blockIdx.y * 64 + (threadIdx.x & 63)) * V;
  if (j >= n || k0 >= k) return;
  struct __attribute__((aligned(V))) Dwords {
    uint32_t d[V / 4];
  };
  const Dwords q = *reinterpret_cast<const Dwords *>(codes + j * ld + k0);
  const float scale = scales[k0 / 128 * lds + (j >> shift)];
  struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[V];
  } v;
#pragma unroll
  for (int h = 0; h < V / 4; ++h) {
    const f2v lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.d[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.d[h], true);
    v.v[4 * h] = (T)wgb::in_fp32(lo[0] * scale);
    v.v[4 * h + 1] = (T)wgb::in_fp32(lo[1] * scale);
    v.v[4 * h + 2] = (T)wgb::in_fp32(hi[0] * scale);
    v.v[4 * h + 3] = (T)wgb::in_fp32(hi[1] * scale);
  }
  T *x = X + j * ldx + k0;
  if (k - k0 >= V) {
    typedef int Any __attribute__((ext_vector_type(4), aligned(4)));
    if constexpr (STREAM)
      __builtin_nontemporal_store(__builtin_bit_cast(Any, v), reinterpret_cast<Any *>(x));
    else
      *reinterpret_cast<Vec *>(x) = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < k - k0) x[i] = v.v[i];
  }
}

int64_t blocks128(int64_t k) { return (k + 127) / 128; }
// More than the caches hold: 8 L2 caches of 4 MB.
template <class T>
bool streams(int64_t k, int64_t n) {
  return k * n * (int64_t)sizeof(T) > (int64_t)32 << 20;
}

template <class T, bool STREAM>
int quantize(wgb_ctx *ctx, int trans, int block, int64_t k, int64_t n, const void *X, int64_t ldx, uint8_t *codes,
             int64_t ld, float *scales, int64_t lds) {
  const int blocks_k = (int)blocks128(k);
  const int64_t tiles = blocks_k * blocks128(n);
  // as few threads as check_convert allows, 512 of a tile
  if ((trans == WGB_TRANS || block == 128) && tiles >= (int64_t)1 << 23)
    return fail(WGB_ERR_INVALID_VALUE, "wgb_fp8_quantize: too many blocks");
  const T *x = (const T *)X;
  if (trans == WGB_TRANS) {
    if (block == 128)
      quantize_strided_kernel<T, true, STREAM><<<(unsigned)tiles, 512, 0, ctx->stream>>>(x, ldx, k, n, codes, ld, scales, lds, blocks_k);
    else
      quantize_strided_kernel<T, false, STREAM><<<(unsigned)tiles, 512, 0, ctx->stream>>>(x, ldx, k, n, codes, ld, scales, lds, blocks_k);
  } else if (block == 128) {
    quantize_square_kernel<T, STREAM><<<(unsigned)tiles, 512, 0, ctx->stream>>>(x, ldx, k, n, codes, ld, scales, lds, blocks_k);
  } else {
    const dim3 grid((unsigned)((n + 3) / 4), (unsigned)((k + 511) / 512));
    quantize_kernel<T, STREAM><<<grid, 256, 0, ctx->stream>>>(x, ldx, k, n, codes, ld, scales, lds);
  }
  WGB_CHECK_LAUNCH("wgb_fp8_quantize");
  return WGB_OK;
}

template <class T>
int quantize_as(wgb_ctx *ctx, int trans, int block, int64_t k, int64_t n, const void *X, int64_t ldx, uint8_t *codes,
                int64_t ld, float *scales, int64_t lds) {
  const bool stream = streams<T>(k, n) && (trans == WGB_NO_TRANS || (((uintptr_t)X | ldx * sizeof(T)) & 3) == 0);
  return (stream ? quantize<T, true> : quantize<T, false>)(ctx, trans, block, k, n, X, ldx, codes, ld, scales, lds);
}

template <class T>
int dequantize(wgb_ctx *ctx, int block, int64_t k, int64_t n, const uint8_t *codes, int64_t ld, const float *scales,
               int64_t lds, void *X, int64_t ldx) {
  const int shift = block == 128 ? 7 : 0, along = (int)((k * sizeof(T) + 1023) / 1024);
  const bool stream = streams<T>(k, n) && (((uintptr_t)X | ldx * sizeof(T)) & 3) == 0;
  const dim3 grid((unsigned)((n + 3) / 4), (unsigned)along);
  if (stream)
    dequantize_kernel<T, true><<<grid, 256, 0, ctx->stream>>>(codes, ld, scales, lds, shift, k, n, (T *)X, ldx);
  else
    dequantize_kernel<T, false><<<grid, 256, 0, ctx->stream>>>(codes, ld, scales, lds, shift, k, n, (T *)X, ldx);
  WGB_CHECK_LAUNCH("wgb_fp8_dequantize");
  return WGB_OK;
}

// Codes and scales of a matrix whose contiguous axis is `length` long, of `columns` columns.
int check_codes(const char *what, int64_t length, int64_t columns, int block, const void *codes, int64_t ld,
                const void *scales, int64_t lds, bool needed) {
  if (ld <= 0 || ld < length || ld % 128 != 0 || ld > ((int64_t)1 << 23))
    return fail(WGB_ERR_INVALID_VALUE, std::string("the leading dimension of ") + what +
                                           " must be a multiple of 128, at least its columns' length, at most 2^23");
  if (lds < 1 || lds < (columns + block - 1) / block || lds > ((int64_t)1 << 28))
    return fail(WGB_ERR_INVALID_VALUE,
                std::string("the scales' leading dimension of ") + what + " must be at least its column blocks, at most 2^28");
  if (!needed) return WGB_OK;
  if (!codes || !scales) return fail(WGB_ERR_INVALID_VALUE, std::string("the codes or scales of ") + what + " are null");
  if (!wgb::aligned16(codes) || ((uintptr_t)scales & 3))
    return fail(WGB_ERR_INVALID_VALUE,
                std::string("the codes of ") + what + " must be 16-byte aligned, its scales 4-byte aligned");
  return WGB_OK;
}

int check_convert(int type, int block, int64_t k, int64_t n) {
  if (type != WGB_F32 && type != WGB_F16 && type != WGB_BF16)
    return fail(WGB_ERR_INVALID_VALUE, "type must be WGB_F32, WGB_F16 or WGB_BF16");
  if (block != 1 && block != 128) return fail(WGB_ERR_INVALID_VALUE, "block must be 1 or 128");
  if (k < 0 || n < 0) return fail(WGB_ERR_INVALID_VALUE, "k and n must be non-negative");
  // a launch has fewer than 2^32 threads along an axis, of which a column has 64, in blocks of four columns
  if (n > ((int64_t)1 << 26) - 4) return fail(WGB_ERR_INVALID_VALUE, "n must be at most 2^26 - 4");
  return WGB_OK;
}

// Estimated times of tiles (ragged_tile.h) at k = 1024: first and each further
// one on a CU. Measured from 1024 x 1024 x 4096 (64 x 64 tiles: 15.5 us into
// bf16, 19.5 into fp32), 2048 x 2048 x 8192 (128 x 128: 57 and 86) and 8192 x
// 4096 x 4096 (128 x 128: 147 and 245, 256 x 256: 122 and 218).
template <bool ROWS, bool EXACT>
constexpr TileCost cost(int T) {
  if (!EXACT) {
    return T == 64 ? TileCost{3.0, 1.5}
           : ROWS  ? (T == 128 ? TileCost{6.6, 4.3} : TileCost{14.5, 14.5})
                   : (T == 128 ? TileCost{6.4, 3.7} : TileCost{12.0, 12.0});
  }
  return T == 64  ? (ROWS ? TileCost{4.2, 2.3} : TileCost{3.7, 2.1})
         : T == 128 ? (ROWS ? TileCost{10.3, 7.4} : TileCost{9.4, 6.8})
                    : TileCost{22.0, 22.0};
}

template <bool AMC, bool ROWS, bool EXACT>
int product(wgb_ctx *ctx, Args &p) {
  typedef Fp8Kernel<128, 128, 2, 2, AMC, ROWS, EXACT, 2> K128;
  const int64_t mean = p.n / p.groups;
  if (mean <= 32) {
    // Few columns: reading A counts, streamed through LDS, or with too few
    // blocks for the CUs straight into registers, the waves sharing k.
    const int64_t blocks = (p.m + 127) / 128 * (p.n < p.groups ? p.n : p.groups);
    if constexpr (!AMC) {
      if (blocks < ctx->num_cus)
        return mean <= 16 ? launch_columns<Fp8Skinny<2, 1, ROWS, EXACT>>(ctx, p) : launch_columns<Fp8Skinny<2, 2, ROWS, EXACT>>(ctx, p);
    }
    return launch_columns<Fp8Kernel<128, 32, 4, 1, AMC, ROWS, EXACT, 4>>(ctx, p);
  }
  const double k = (double)p.k, size = p.c_f32 ? 4 : 2;
  const TileCost c64 = cost<ROWS, EXACT>(64), c128 = cost<ROWS, EXACT>(128), c256 = cost<ROWS, EXACT>(256);
  const double t64 = small_time(64, c64, per_cu(ctx, p, 64, expected_columns(p, 64)), k, size);
  const double t128 = small_time(128, c128, per_cu(ctx, p, 128, expected_columns(p, 128)), k, size);
  // with a scale for each row and exact sums v_fma and the conversions bound
  // it, and 256 x 256 tiles win nothing (8192 x 4096 x 4096: 261 us on 128 x 128 tiles, 256)
  if constexpr (!ROWS || !EXACT) {
    const double t256 = rounds_time(c256, c128, per_cu(ctx, p, 256, expected_columns(p, 256)), k, size, most_pieces(p.k, 128));
    if (t256 <= t128 && t256 <= t64) return launch_columns_rounds<Fp8Large<AMC, ROWS, EXACT>, K128>(ctx, p);
  }
  if (t128 <= t64) return launch_columns<K128>(ctx, p);
  return launch_columns<Fp8Kernel<64, 64, 2, 2, AMC, ROWS, EXACT, 2>>(ctx, p);
}

int run_product(wgb_ctx *ctx, int transA, int64_t groups, int64_t m, int64_t n, int64_t k, float alpha, const uint8_t *A,
                int64_t lda, int64_t strideA, int blockA, const float *scaleA, int64_t ldsa, int64_t strideScaleA,
                const uint8_t *B, int64_t ldb, const float *scaleB, int64_t ldsb, const int64_t *d_offsets, bool grouped,
                float beta, void *C, int64_t ldc, int ctype) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if (ctype != WGB_F32 && ctype != WGB_F16 && ctype != WGB_BF16)
    return fail(WGB_ERR_INVALID_VALUE, "the type of C must be WGB_F32, WGB_F16 or WGB_BF16");
  if (transA != WGB_NO_TRANS && transA != WGB_TRANS)
    return fail(WGB_ERR_INVALID_VALUE, "transA must be WGB_NO_TRANS or WGB_TRANS");
  if (blockA != 128 && (blockA != 1 || transA == WGB_NO_TRANS))
    return fail(WGB_ERR_INVALID_VALUE, "blockA must be 128, or with WGB_TRANS 1 or 128");
  if (groups < 0 || m < 0 || n < 0 || k < 0)
    return fail(WGB_ERR_INVALID_VALUE, "groups, m, n, and k must be non-negative");
  if (groups > (1 << 20)) return fail(WGB_ERR_INVALID_VALUE, "groups must be at most 2^20");
  if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX)
    return fail(WGB_ERR_INVALID_VALUE, "m, n, and k must be below 2^31");
  const bool amc = transA == WGB_NO_TRANS;
  const bool none = m == 0 || n == 0 || groups == 0, reads = !none && k > 0 && alpha != 0.0f;
  const int64_t length = amc ? m : k, columns = amc ? k : m;
  if ((st = check_codes("A", length, columns, blockA, A, lda, scaleA, ldsa, reads))) return st;
  if ((st = check_codes("B", k, n, 1, B, ldb, scaleB, ldsb, reads))) return st;
  if (strideA < 0 || strideA % 16 != 0 || (groups > 1 && strideA < columns * lda))
    return fail(WGB_ERR_INVALID_VALUE, "strideA must be a multiple of 16 and cover a group's columns");
  const int64_t rows_s = blocks128(length), cols_s = (columns + blockA - 1) / blockA;
  if (strideScaleA < 0 || (groups > 1 && rows_s > 0 && strideScaleA < (rows_s - 1) * ldsa + cols_s))
    return fail(WGB_ERR_INVALID_VALUE, "strideScaleA must cover a group's scales");
  if (ldc < (m > 1 ? m : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldc must be >= max(1, m)");
  if (none) return WGB_OK;
  if (grouped && !d_offsets) return fail(WGB_ERR_INVALID_VALUE, "d_offsets is null");
  if (!C) return fail(WGB_ERR_INVALID_VALUE, "C is null");
  Args p = {};
  p.m = m;
  p.n = n;
  p.k = blocks128(k) * 128;
  p.a_depth = k;
  p.A = (const char *)A;
  p.B = (const char *)B;
  p.lda = lda;
  p.ldb = ldb;
  p.stride_a = strideA;
  p.a_rows = blocks128(m) * 128;
  p.block_scale_a = scaleA;
  p.block_scale_b = scaleB;
  p.a_row = amc ? ldsa : 1;
  p.a_k = amc ? 1 : ldsa;
  p.a_group = strideScaleA;
  p.b_k = ldsb;
  p.a_shift = blockA == 128 ? 7 : 0;
  p.off = grouped ? d_offsets : nullptr;
  p.groups = (int)groups;
  p.C = C;
  p.ldc = ldc;
  p.alpha = alpha;
  p.beta = beta;
  p.c_f32 = ctype == WGB_F32;
  p.c_f16 = ctype == WGB_F16;
  wgb::timing_begin(ctx);
  if (amc)
    st = p.c_f32 ? product<true, false, true>(ctx, p) : product<true, false, false>(ctx, p);
  else if (blockA == 1)
    st = p.c_f32 ? product<false, true, true>(ctx, p) : product<false, true, false>(ctx, p);
  else
    st = p.c_f32 ? product<false, false, true>(ctx, p) : product<false, false, false>(ctx, p);
  wgb::timing_end(ctx);
  return st;
}

}  // namespace

extern "C" int wgb_fp8_quantize(wgb_ctx *ctx, int type, int trans, int block, int64_t k, int64_t n, const void *X,
                                int64_t ldx, uint8_t *codes, int64_t ld, float *scales, int64_t lds) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_convert(type, block, k, n))) return st;
  if (trans != WGB_NO_TRANS && trans != WGB_TRANS)
    return fail(WGB_ERR_INVALID_VALUE, "trans must be WGB_NO_TRANS or WGB_TRANS");
  const int64_t rows = trans == WGB_TRANS ? n : k;
  if (ldx < (rows > 1 ? rows : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldx must be >= max(1, rows of X)");
  if ((st = check_codes("the result", k, n, block, codes, ld, scales, lds, k > 0 && n > 0))) return st;
  if (k == 0 || n == 0) return WGB_OK;
  if (!X) return fail(WGB_ERR_INVALID_VALUE, "X is null");
  wgb::timing_begin(ctx);
  st = type == WGB_F32   ? quantize_as<float>(ctx, trans, block, k, n, X, ldx, codes, ld, scales, lds)
       : type == WGB_F16 ? quantize_as<_Float16>(ctx, trans, block, k, n, X, ldx, codes, ld, scales, lds)
                         : quantize_as<__bf16>(ctx, trans, block, k, n, X, ldx, codes, ld, scales, lds);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_fp8_dequantize(wgb_ctx *ctx, int type, int block, int64_t k, int64_t n, const uint8_t *codes,
                                  int64_t ld, const float *scales, int64_t lds, void *X, int64_t ldx) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_convert(type, block, k, n))) return st;
  if (ldx < (k > 1 ? k : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldx must be >= max(1, k)");
  if ((st = check_codes("the matrix", k, n, block, codes, ld, scales, lds, k > 0 && n > 0))) return st;
  if (k == 0 || n == 0) return WGB_OK;
  if (!X) return fail(WGB_ERR_INVALID_VALUE, "X is null");
  wgb::timing_begin(ctx);
  st = type == WGB_F32   ? dequantize<float>(ctx, block, k, n, codes, ld, scales, lds, X, ldx)
       : type == WGB_F16 ? dequantize<_Float16>(ctx, block, k, n, codes, ld, scales, lds, X, ldx)
                         : dequantize<__bf16>(ctx, block, k, n, codes, ld, scales, lds, X, ldx);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_fp8_gemm(wgb_ctx *ctx, int transA, int64_t m, int64_t n, int64_t k, float alpha, const uint8_t *A,
                            int64_t lda, int blockA, const float *scaleA, int64_t ldsa, const uint8_t *B, int64_t ldb,
                            const float *scaleB, int64_t ldsb, float beta, void *C, int64_t ldc, int ctype) {
  return run_product(ctx, transA, 1, m, n, k, alpha, A, lda, 0, blockA, scaleA, ldsa, 0, B, ldb, scaleB, ldsb, nullptr,
                     false, beta, C, ldc, ctype);
}

extern "C" int wgb_fp8_gemm_grouped(wgb_ctx *ctx, int transA, int64_t groups, int64_t m, int64_t n, int64_t k, float alpha,
                                    const uint8_t *A, int64_t lda, int64_t strideA, int blockA, const float *scaleA,
                                    int64_t ldsa, int64_t strideScaleA, const uint8_t *B, int64_t ldb, const float *scaleB,
                                    int64_t ldsb, const int64_t *d_offsets, float beta, void *C, int64_t ldc, int ctype) {
  return run_product(ctx, transA, groups, m, n, k, alpha, A, lda, strideA, blockA, scaleA, ldsa, strideScaleA, B, ldb,
                     scaleB, ldsb, d_offsets, true, beta, C, ldc, ctype);
}
