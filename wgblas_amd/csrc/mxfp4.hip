// MXFP4: matrices of 4-bit floats in blocks of 32 along k with a power of two
// each (the OCP microscaling format: E2M1 codes, E8M0 scales), their
// conversion from and to f32 / f16 / bf16, and their products.
//
// Storage of a k x n matrix at leading dimension ld (a multiple of 128
// elements): column j has its codes at codes + j ld / 2, two a byte, the
// first in the low half, and its scales at scales + j ld / 32, 2^(s - 127)
// for byte s, 0xff for NaN. The elements from k to the next multiple of 128
// are zeros with scale 0, so products read whole runs of 128.
//
// Quantisation: with e = floor(log2 max |x|) over a block the scale is
// 2^(e - 2) (the largest code is 6 = 1.5 2^2), at least 2^-127, and each
// x / scale goes to the nearest code, ties to the even one, magnitudes above
// 6 to 6. A block that holds an Inf or NaN gets scale 0xff: all of it reads
// as NaN, so that what is not finite stays visible in any product.
#include "ragged_tile.h"

namespace {

using namespace wgb_ragged;
using wgb::fail;

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint16_t u2 __attribute__((ext_vector_type(2)));

// Two neighbours of a block as they are loaded: one dword of 16-bit values,
// two of fp32.
template <class E>
struct Pair;

template <>
struct Pair<F32> {
  typedef f2 V;
  static __device__ __forceinline__ V zero() { return V{0.0f, 0.0f}; }
  static __device__ __forceinline__ V make(float a, float b) { return V{a, b}; }
  // magnitudes as whole numbers (NaN above Inf above the rest)
  static __device__ __forceinline__ uint32_t top(uint32_t t, V v) {
    const uint32_t a = __float_as_uint(v[0]) & 0x7fffffffu, b = __float_as_uint(v[1]) & 0x7fffffffu;
    t = t > a ? t : a;
    return t > b ? t : b;
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t t) { return t; }
  template <int SEL>
  static __device__ __forceinline__ uint32_t code(uint32_t old, V v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, v[0], v[1], scale, SEL);
  }
  static __device__ __forceinline__ f2 widen(V v) { return v; }
};

// 16-bit: both magnitudes of a dword at once
__device__ __forceinline__ uint32_t top16(uint32_t t, uint32_t v) {
  const u2 a = __builtin_bit_cast(u2, v & 0x7fff7fffu), b = __builtin_bit_cast(u2, t);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
}

template <>
struct Pair<Bf16> {
  typedef uint32_t V;
  static __device__ __forceinline__ V zero() { return 0; }
  static __device__ __forceinline__ V make(uint16_t a, uint16_t b) { return (uint32_t)a | ((uint32_t)b << 16); }
  static __device__ __forceinline__ uint32_t top(uint32_t t, V v) { return top16(t, v); }
  // of the running pair of maxima: the larger as fp32 bits
  static __device__ __forceinline__ uint32_t bits(uint32_t t) {
    const uint32_t lo = t & 0xffffu, hi = t >> 16;
    return (lo > hi ? lo : hi) << 16;
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t code(uint32_t old, V v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(b2, v), scale, SEL);
  }
  static __device__ __forceinline__ f2 widen(V v) {
    return f2{__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)};
  }
};

template <>
struct Pair<F16> {
  typedef uint32_t V;
  static __device__ __forceinline__ V zero() { return 0; }
  static __device__ __forceinline__ V make(uint16_t a, uint16_t b) { return (uint32_t)a | ((uint32_t)b << 16); }
  static __device__ __forceinline__ uint32_t top(uint32_t t, V v) { return top16(t, v); }
  static __device__ __forceinline__ uint32_t bits(uint32_t t) {
    const uint32_t lo = t & 0xffffu, hi = t >> 16;
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)(lo > hi ? lo : hi)));
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t code(uint32_t old, V v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(h2, v), scale, SEL);
  }
  static __device__ __forceinline__ f2 widen(V v) {
    const h2 h = __builtin_bit_cast(h2, v);
    return f2{(float)h[0], (float)h[1]};
  }
};

// The scale byte of a block from the fp32 bits of its largest magnitude:
// exponent field less 2 and at least 0 (subnormals and zero end there), 0xff
// for Inf and NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
  const uint32_t e = bits >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}

// Eight codes of four pairs. The conversion instruction divides by a scale
// given as fp32; 2^-127 is no normal number there, so blocks of that scale
// (magnitudes below 2^-124) go through fp32 times 2^64.
template <class E>
__device__ __forceinline__ uint32_t codes8(const typename Pair<E>::V (&v)[4], uint32_t byte) {
  typedef Pair<E> P;
  uint32_t r = 0;
  if (byte == 255) return 0;
  if (byte == 0) {
    const float up = 0x1p64f, scale = 0x1p-63f;
    f2 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = P::widen(v[i]);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, w[0][0] * up, w[0][1] * up, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, w[1][0] * up, w[1][1] * up, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, w[2][0] * up, w[2][1] * up, scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, w[3][0] * up, w[3][1] * up, scale, 3);
    return r;
  }
  const float scale = __uint_as_float(byte << 23);
  r = P::template code<0>(r, v[0], scale);
  r = P::template code<1>(r, v[1], scale);
  r = P::template code<2>(r, v[2], scale);
  r = P::template code<3>(r, v[3], scale);
  return r;
}

// Largest of a quad's values (lanes 4 i .. 4 i + 3).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true);  // lane ^ 1
  x = x > y ? x : y;
  y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true);  // lane ^ 2
  return x > y ? x : y;
}

// Blocks along the contiguous axis: a lane has 8 elements of a column, a quad
// a block. Bound by memory: one pass, loads of 16 bytes a lane. 16384 columns of
// 4096 bf16 values: 30 us, 5.6 TB/s; 17 columns: 2.5 us, a launch.
template <class E>
__global__ __launch_bounds__(256) void quantize_kernel(const typename E::store *X, int64_t ldx, int64_t k, int64_t n,
                                                       uint8_t *codes, uint8_t *scales, int64_t ld, int segs) {
  typedef Pair<E> P;
  typedef typename E::store T;
  const int64_t total = n * segs, stride = (int64_t)gridDim.x * 256;
  // whole quads: segs is a multiple of 16
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
    const int64_t j = i / segs;
    const int s = (int)(i - j * segs);
    const T *x = X + j * ldx + s * 8;
    const int64_t left = k - (int64_t)s * 8;
    typename P::V v[4];
    if (left >= 8) {
      struct __attribute__((packed, aligned(sizeof(T)))) V8 {
        typename P::V p[4];
      };
      const V8 w = *reinterpret_cast<const V8 *>(x);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = w.p[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[c] = P::zero();
        if constexpr (E::kBits == 32) {
          if (2 * c < left) v[c] = P::make(x[2 * c], 2 * c + 1 < left ? x[2 * c + 1] : 0.0f);
        } else {
          const uint16_t *u = reinterpret_cast<const uint16_t *>(x);
          if (2 * c < left) v[c] = P::make(u[2 * c], 2 * c + 1 < left ? u[2 * c + 1] : (uint16_t)0);
        }
      }
    }
    uint32_t t = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) t = P::top(t, v[c]);
    const uint32_t byte = scale_byte(quad_max(P::bits(t)));
    *reinterpret_cast<uint32_t *>(codes + j * (ld / 2) + s * 4) = codes8<E>(v, byte);
    if ((threadIdx.x & 3) == 0) scales[j * (ld / 32) + s / 4] = (uint8_t)byte;
  }
}

// Blocks along the strided axis. A lane has two neighbouring columns of one
// block: 32 loads of two elements (256 contiguous bytes a wave for 16-bit
// types). The eight waves have eight blocks in a row of the same 128 columns;
// their codes go through LDS (16-byte chunks at chunk ^ column, no two lanes
// of a quarter wave in the same banks) and out as 128-byte lines. Bound by
// memory: 8192 x 16384 in bf16 93 us, 3.8 TB/s (the two-element loads keep
// fewer bytes in flight than the 16-byte ones above).
template <class E>
__global__ __launch_bounds__(512) void quantize_strided_kernel(const typename E::store *X, int64_t ldx, int64_t k,
                                                               int64_t n, uint8_t *codes, uint8_t *scales, int64_t ld,
                                                               int blocks, int groups_k) {
  typedef Pair<E> P;
  typedef typename E::store T;
  __shared__ v4i lines[128][8];
  __shared__ __align__(8) uint8_t bytes[128][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kb0 = (int)(blockIdx.x % groups_k) * 8, kb = kb0 + wave;
  const int64_t j0 = (int64_t)(blockIdx.x / groups_k) * 128, j = j0 + 2 * lane;
  if (kb < blocks && j < n) {
    const bool two = j + 1 < n;
    const int64_t k0 = (int64_t)kb * 32, left = k - k0;
    const T *x = X + k0 * ldx + j;
    typename P::V v[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      v[r] = P::zero();
      if (r < left) {
        struct __attribute__((packed, aligned(sizeof(T)))) V2 {
          typename P::V p;
        };
        if (two) {
          v[r] = reinterpret_cast<const V2 *>(x + r * ldx)->p;
        } else if constexpr (E::kBits == 32) {
          v[r] = P::make(x[r * ldx], 0.0f);
        } else {
          v[r] = P::make(reinterpret_cast<const uint16_t *>(x)[r * ldx], 0);
        }
      }
    }
    uint32_t bits[2];
    if constexpr (E::kBits == 32) {
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int r = 0; r < 32; ++r) {
        const uint32_t p = __float_as_uint(v[r][0]) & 0x7fffffffu, q = __float_as_uint(v[r][1]) & 0x7fffffffu;
        a = a > p ? a : p;
        b = b > q ? b : q;
      }
      bits[0] = a;
      bits[1] = b;
    } else {
      uint32_t t = 0;
#pragma unroll
      for (int r = 0; r < 32; ++r) t = P::top(t, v[r]);
      bits[0] = P::bits(t & 0xffffu);
      bits[1] = P::bits(t >> 16);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t byte = scale_byte(bits[c]);
      v4i out;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        typename P::V w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * q + 2 * i;
          if constexpr (E::kBits == 32)
            w[i] = P::make(v[r][c], v[r + 1][c]);
          else  // the two rows' halves c side by side
            w[i] = __builtin_amdgcn_perm(v[r + 1], v[r], c == 0 ? 0x05040100u : 0x07060302u);
        }
        out[q] = (int)codes8<E>(w, byte);
      }
      lines[2 * lane + c][wave ^ (lane & 7)] = out;
      bytes[2 * lane + c][wave] = (uint8_t)byte;
    }
  }
  __syncthreads();
  const int here = blocks - kb0 < 8 ? blocks - kb0 : 8;  // a multiple of 4
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int col = (threadIdx.x >> 3) + 64 * q, chunk = threadIdx.x & 7;
    if (j0 + col < n && chunk < here)
      *reinterpret_cast<v4i *>(codes + (j0 + col) * (ld / 2) + (kb0 + chunk) * 16) = lines[col][chunk ^ ((col >> 1) & 7)];
  }
  const int col = threadIdx.x >> 1, half = threadIdx.x & 1;
  if (col < 128 && j0 + col < n && 4 * half < here)
    *reinterpret_cast<int *>(scales + (j0 + col) * (ld / 32) + kb0 + 4 * half) =
        *reinterpret_cast<const int *>(&bytes[col][4 * half]);
}

// A lane has 8 codes of a column: value * scale in fp32 (both exact), rounded
// once to the output's type. Bound by memory: 8192 x 16384 to bf16 64 us, 5.2
// TB/s.
template <class E>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t *codes, const uint8_t *scales, int64_t ld,
                                                         int64_t k, int64_t n, typename E::store *X, int64_t ldx,
                                                         int segs) {
  typedef typename E::store T;
  const int64_t total = n * segs, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
    const int64_t j = i / segs;
    const int s = (int)(i - j * segs);
    const uint32_t q = *reinterpret_cast<const uint32_t *>(codes + j * (ld / 2) + s * 4);
    const uint32_t byte = scales[j * (ld / 32) + s / 4];
    const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
    f2 w[4];
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
    w[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    w[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2);
    w[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
    typedef T V8 __attribute__((ext_vector_type(8)));
    V8 v;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[2 * c] = (T)(w[c][0] * scale);
      v[2 * c + 1] = (T)(w[c][1] * scale);
    }
    T *x = X + j * ldx + s * 8;
    const int64_t left = k - (int64_t)s * 8;
    if (left >= 8) {
      struct __attribute__((packed, aligned(sizeof(T)))) U {
        V8 p;
      };
      reinterpret_cast<U *>(x)->p = v;
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < left) x[c] = v[c];
    }
  }
}

int64_t runs128(int64_t k) { return (k + 127) / 128 * 128; }

unsigned lane_grid(wgb_ctx *ctx, int64_t lanes) {
  const int64_t want = (lanes + 255) / 256, most = (int64_t)ctx->num_cus * 32;
  return (unsigned)(want < most ? want : most);
}

template <class E>
int quantize(wgb_ctx *ctx, int trans, int64_t k, int64_t n, const void *X, int64_t ldx, uint8_t *codes, uint8_t *scales,
             int64_t ld) {
  typedef typename E::store T;
  if (trans == WGB_NO_TRANS) {
    const int segs = (int)(runs128(k) / 8);
    quantize_kernel<E><<<lane_grid(ctx, n * segs), 256, 0, ctx->stream>>>((const T *)X, ldx, k, n, codes, scales, ld, segs);
    WGB_CHECK_LAUNCH("quantize_kernel");
  } else {
    const int blocks = (int)(runs128(k) / 32), groups_k = (blocks + 7) / 8;
    const int64_t grid = (n + 127) / 128 * groups_k;
    if (grid > INT32_MAX) return fail(WGB_ERR_INVALID_VALUE, "wgb_mxfp4_quantize: too many blocks");
    quantize_strided_kernel<E><<<(unsigned)grid, 512, 0, ctx->stream>>>((const T *)X, ldx, k, n, codes, scales, ld, blocks,
                                                                        groups_k);
    WGB_CHECK_LAUNCH("quantize_strided_kernel");
  }
  return WGB_OK;
}

template <class E>
int dequantize(wgb_ctx *ctx, int64_t k, int64_t n, const uint8_t *codes, const uint8_t *scales, int64_t ld, void *X,
               int64_t ldx) {
  const int segs = (int)((k + 7) / 8);
  dequantize_kernel<E><<<lane_grid(ctx, n * segs), 256, 0, ctx->stream>>>(codes, scales, ld, k, n,
                                                                         (typename E::store *)X, ldx, segs);
  WGB_CHECK_LAUNCH("dequantize_kernel");
  return WGB_OK;
}

int check_packed(const char *what, int64_t k, const void *codes, const void *scales, int64_t ld, bool needed) {
  // against k itself, which may be too large to be rounded up
  if (ld <= 0 || ld < k || ld % 128 != 0 || ld > ((int64_t)1 << 23))
    return fail(WGB_ERR_INVALID_VALUE,
                std::string("the leading dimension of ") + what + " must be a multiple of 128, at least k, at most 2^23");
  if (!needed) return WGB_OK;
  if (!codes || !scales) return fail(WGB_ERR_INVALID_VALUE, std::string("the codes or scales of ") + what + " are null");
  if (!wgb::aligned16(codes) || ((uintptr_t)scales & 3))
    return fail(WGB_ERR_INVALID_VALUE,
                std::string("the codes of ") + what + " must be 16-byte aligned, its scales 4-byte aligned");
  return WGB_OK;
}

int check_convert(int type, int64_t k, int64_t n) {
  if (type != WGB_F32 && type != WGB_F16 && type != WGB_BF16)
    return fail(WGB_ERR_INVALID_VALUE, "type must be WGB_F32, WGB_F16 or WGB_BF16");
  if (k < 0 || n < 0) return fail(WGB_ERR_INVALID_VALUE, "k and n must be non-negative");
  if (n > INT32_MAX) return fail(WGB_ERR_INVALID_VALUE, "n must be below 2^31");
  return WGB_OK;
}

int product(wgb_ctx *ctx, Args &p) {
  const int64_t mean = p.n / p.groups;
  if (mean <= 32) {
    // Few columns, as in the 16-bit products: 64 experts of 4096 x 2048 take
    // 44 us streamed with two stages (66 with four, which leave one block a
    // CU), 82 us with the waves sharing k.
    const int64_t blocks = (p.m + 127) / 128 * (p.n < p.groups ? p.n : p.groups);
    if (blocks < ctx->num_cus)
      return mean <= 16 ? launch_columns<SkinnyKernel<Fp4, 2, 1>>(ctx, p) : launch_columns<SkinnyKernel<Fp4, 2, 2>>(ctx, p);
    return launch_columns<Kernel<Fp4, 128, 32, 4, 1, false, false, true, false, 2>>(ctx, p);
  }
  const double k = (double)p.k, size = p.c_f32 ? 4 : 2;
  const TileCost c64 = {4.0, 1.5}, c128 = {5.6, 3.3}, c256 = {10.5, 10.5};
  const double t64 = small_time(64, c64, per_cu(ctx, p, 64, expected_columns(p, 64)), k, size);
  const double t128 = small_time(128, c128, per_cu(ctx, p, 128, expected_columns(p, 128)), k, size);
  const double t256 = rounds_time(c256, c128, per_cu(ctx, p, 256, expected_columns(p, 256)), k, size, most_pieces(p.k, 256));
  if (t256 <= t128 && t256 <= t64)
    return launch_columns_rounds<TurnKernel<Fp4, false, false, false>, Kernel<Fp4, 128, 128, 2, 2, false, false, true, false, 2>>(ctx, p);
  if (t128 <= t64) return launch_columns<Kernel<Fp4, 128, 128, 2, 2, false, false, true, false, 2>>(ctx, p);
  return launch_columns<Kernel<Fp4, 64, 64, 2, 2, false, false, true, false, 2>>(ctx, p);
}

int run_product(wgb_ctx *ctx, int64_t groups, int64_t m, int64_t n, int64_t k, float alpha, const uint8_t *A,
                const uint8_t *scaleA, int64_t lda, int64_t strideA, const uint8_t *B, const uint8_t *scaleB, int64_t ldb,
                const int64_t *d_offsets, bool grouped, float beta, void *C, int64_t ldc, int ctype) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if (ctype != WGB_F32 && ctype != WGB_F16 && ctype != WGB_BF16)
    return fail(WGB_ERR_INVALID_VALUE, "the type of C must be WGB_F32, WGB_F16 or WGB_BF16");
  if (groups < 0 || m < 0 || n < 0 || k < 0)
    return fail(WGB_ERR_INVALID_VALUE, "groups, m, n, and k must be non-negative");
  if (groups > (1 << 20)) return fail(WGB_ERR_INVALID_VALUE, "groups must be at most 2^20");
  if (m > INT32_MAX || n > INT32_MAX) return fail(WGB_ERR_INVALID_VALUE, "m and n must be below 2^31");
  const bool none = m == 0 || n == 0 || groups == 0, reads = !none && k > 0 && alpha != 0.0f;
  if ((st = check_packed("A", k, A, scaleA, lda, reads))) return st;
  if ((st = check_packed("B", k, B, scaleB, ldb, reads))) return st;
  if (strideA < 0 || strideA % 128 != 0 || (groups > 1 && strideA < m * lda))
    return fail(WGB_ERR_INVALID_VALUE, "strideA must be a multiple of 128 and cover a group's m columns");
  if (ldc < (m > 1 ? m : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldc must be >= max(1, m)");
  if (none) return WGB_OK;
  if (grouped && !d_offsets) return fail(WGB_ERR_INVALID_VALUE, "d_offsets is null");
  if (!C) return fail(WGB_ERR_INVALID_VALUE, "C is null");
  Args p = {};
  p.m = m;
  p.n = n;
  p.k = runs128(k);
  p.A = (const char *)A;
  p.B = (const char *)B;
  p.lda = lda / 2;
  p.ldb = ldb / 2;
  p.stride_a = strideA / 2;
  p.scale_a = scaleA;
  p.scale_b = scaleB;
  p.off = grouped ? d_offsets : nullptr;
  p.groups = (int)groups;
  p.C = C;
  p.ldc = ldc;
  p.alpha = alpha;
  p.beta = beta;
  p.c_f32 = ctype == WGB_F32;
  p.c_f16 = ctype == WGB_F16;
  wgb::timing_begin(ctx);
  st = product(ctx, p);
  wgb::timing_end(ctx);
  return st;
}

}  // namespace

extern "C" int wgb_mxfp4_quantize(wgb_ctx *ctx, int type, int trans, int64_t k, int64_t n, const void *X, int64_t ldx,
                                  uint8_t *codes, uint8_t *scales, int64_t ld) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_convert(type, k, n))) return st;
  if (trans != WGB_NO_TRANS && trans != WGB_TRANS)
    return fail(WGB_ERR_INVALID_VALUE, "trans must be WGB_NO_TRANS or WGB_TRANS");
  const int64_t rows = trans == WGB_TRANS ? n : k;
  if (ldx < (rows > 1 ? rows : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldx must be >= max(1, rows of X)");
  if ((st = check_packed("the result", k, codes, scales, ld, k > 0 && n > 0))) return st;
  if (k == 0 || n == 0) return WGB_OK;
  if (!X) return fail(WGB_ERR_INVALID_VALUE, "X is null");
  wgb::timing_begin(ctx);
  st = type == WGB_F32   ? quantize<F32>(ctx, trans, k, n, X, ldx, codes, scales, ld)
       : type == WGB_F16 ? quantize<F16>(ctx, trans, k, n, X, ldx, codes, scales, ld)
                         : quantize<Bf16>(ctx, trans, k, n, X, ldx, codes, scales, ld);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_mxfp4_dequantize(wgb_ctx *ctx, int type, int64_t k, int64_t n, const uint8_t *codes,
                                    const uint8_t *scales, int64_t ld, void *X, int64_t ldx) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_convert(type, k, n))) return st;
  if (ldx < (k > 1 ? k : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldx must be >= max(1, k)");
  if ((st = check_packed("the matrix", k, codes, scales, ld, k > 0 && n > 0))) return st;
  if (k == 0 || n == 0) return WGB_OK;
  if (!X) return fail(WGB_ERR_INVALID_VALUE, "X is null");
  wgb::timing_begin(ctx);
  st = type == WGB_F32   ? dequantize<F32>(ctx, k, n, codes, scales, ld, X, ldx)
       : type == WGB_F16 ? dequantize<F16>(ctx, k, n, codes, scales, ld, X, ldx)
                         : dequantize<Bf16>(ctx, k, n, codes, scales, ld, X, ldx);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_mxfp4_gemm(wgb_ctx *ctx, int64_t m, int64_t n, int64_t k, float alpha, const uint8_t *A,
                              const uint8_t *scaleA, int64_t lda, const uint8_t *B, const uint8_t *scaleB, int64_t ldb,
                              float beta, void *C, int64_t ldc, int ctype) {
  return run_product(ctx, 1, m, n, k, alpha, A, scaleA, lda, 0, B, scaleB, ldb, nullptr, false, beta, C, ldc, ctype);
}

extern "C" int wgb_mxfp4_gemm_grouped(wgb_ctx *ctx, int64_t groups, int64_t m, int64_t n, int64_t k, float alpha,
                                      const uint8_t *A, const uint8_t *scaleA, int64_t lda, int64_t strideA,
                                      const uint8_t *B, const uint8_t *scaleB, int64_t ldb, const int64_t *d_offsets,
                                      float beta, void *C, int64_t ldc, int ctype) {
  return run_product(ctx, groups, m, n, k, alpha, A, scaleA, lda, strideA, B, scaleB, ldb, d_offsets, true, beta, C, ldc,
                     ctype);
}
