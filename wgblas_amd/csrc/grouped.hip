// Grouped products with ragged groups: wgb_gemm_grouped (ragged columns) and
// wgb_gemm_grouped_k (ragged k), for f32, f16 and bf16 operands.
//
// wgblas has no grouped product; an expert layer's products would be one
// sgemm per expert, with the groups' sizes copied to the host first. Here one
// launch covers all groups and reads their boundaries on the GPU
// (ragged_tile.h).
#include "ragged_tile.h"

namespace {

using namespace wgb_ragged;
using wgb::fail;

int64_t type_size(int type) { return type == WGB_F32 ? 4 : 2; }

bool known_type(int type) { return type == WGB_F32 || type == WGB_F16 || type == WGB_BF16; }

// Whether 16-byte copies can read a matrix: dword-aligned addresses, and the
// lane offsets of a 256-column tile inside 32 bits.
bool copyable(const void *p, int64_t ld_bytes, int64_t stride_bytes) {
  return ((uintptr_t)p & 3) == 0 && ld_bytes % 4 == 0 && stride_bytes % 4 == 0 && ld_bytes < ((int64_t)1 << 22);
}

template <class E>
constexpr TileCost cost(int T) {
  return E::kBits == 32 ? (T == 64 ? TileCost{20, 15.2} : TileCost{64, 59.3})
                        : (T == 64 ? TileCost{5.4, 4.1} : T == 128 ? TileCost{12.5, 9.5} : TileCost{23.5, 23.5});
}

// The tile (64, 128 or 256 square) whose estimated time is least; 256 needs
// 16-bit operands that can be copied.
template <class E, bool VEC>
int choose(wgb_ctx *ctx, const Args &p, double k, double n64, double n128, double n256) {
  const double size = p.c_f32 ? 4 : 2;
  const double t64 = small_time(64, cost<E>(64), per_cu(ctx, p, 64, n64), k, size);
  const double t128 = small_time(128, cost<E>(128), per_cu(ctx, p, 128, n128), k, size);
  if (VEC && E::kBits == 16) {
    const double t256 = rounds_time(cost<E>(256), cost<E>(128), per_cu(ctx, p, 256, n256), k, size);
    if (t256 <= t128 && t256 <= t64) return 256;
  }
  return t128 <= t64 ? 128 : 64;
}

template <class E, bool AMC, bool VEC>
int run_columns(wgb_ctx *ctx, Args &p) {
  const int64_t mean = p.n / p.groups;
  if (mean <= 32) {
    // Few columns: reading A counts. Whole rows of blocks stream it through
    // LDS (64 experts of 2048 x 1024 in bf16: 27 us, the waves-share-k kernel
    // 37); with too few blocks for the CUs the waves share k instead (8192 x
    // 4096, one column: 5.8 against 10 us in fp4).
    const int64_t blocks = (p.m + 127) / 128 * (p.n < p.groups ? p.n : p.groups);
    if constexpr (!AMC) {
      if (blocks < ctx->num_cus)
        return mean <= 16 ? launch_columns<SkinnyKernel<E, 2, 1>>(ctx, p) : launch_columns<SkinnyKernel<E, 2, 2>>(ctx, p);
    }
    return launch_columns<Kernel<E, 128, 32, 4, 1, AMC, false, VEC, false, 4>>(ctx, p);
  }
  const int T = choose<E, VEC>(ctx, p, (double)p.k, expected_columns(p, 64), expected_columns(p, 128), expected_columns(p, 256));
  if constexpr (VEC && E::kBits == 16) {
    if (T == 256)
      return launch_columns_rounds<TurnKernel<E, AMC, false, false>, Kernel<E, 128, 128, 2, 2, AMC, false, VEC, false, 2>>(ctx, p);
  }
  if (T == 128) return launch_columns<Kernel<E, 128, 128, 2, 2, AMC, false, VEC, false, 2>>(ctx, p);
  return launch_columns<Kernel<E, 64, 64, 2, 2, AMC, false, VEC, false, 2>>(ctx, p);
}

template <class E, bool VEC>
int run_k(wgb_ctx *ctx, Args &p) {
  auto across = [&](int64_t T) { return (double)((p.n + T - 1) / T * p.groups); };
  const int T = choose<E, VEC>(ctx, p, (double)p.k / p.groups, across(64), across(128), across(256));
  if constexpr (VEC && E::kBits == 16) {
    if (T == 256)
      return launch_k_rounds<TurnKernel<E, true, true, true>, Kernel<E, 128, 128, 2, 2, true, true, VEC, true, 2>>(ctx, p);
  }
  if (T == 128) return launch_k<Kernel<E, 128, 128, 2, 2, true, true, VEC, true, 2>>(ctx, p);
  return launch_k<Kernel<E, 64, 64, 2, 2, true, true, VEC, true, 2>>(ctx, p);
}

template <class E>
int dispatch_columns(wgb_ctx *ctx, Args &p, bool amc, bool vec) {
  if (amc) return vec ? run_columns<E, true, true>(ctx, p) : run_columns<E, true, false>(ctx, p);
  return vec ? run_columns<E, false, true>(ctx, p) : run_columns<E, false, false>(ctx, p);
}

// Checks shared by both forms. `k` is null-free of meaning where a dimension is zero.
int check_sizes(int type, int ctype, int64_t groups, int64_t m, int64_t n, int64_t k) {
  if (!known_type(type)) return fail(WGB_ERR_INVALID_VALUE, "type must be WGB_F32, WGB_F16 or WGB_BF16");
  if (ctype != type && ctype != WGB_F32)
    return fail(WGB_ERR_INVALID_VALUE, "the type of C must be the operands' type or WGB_F32");
  if (groups < 0 || m < 0 || n < 0 || k < 0)
    return fail(WGB_ERR_INVALID_VALUE, "groups, m, n, and k must be non-negative");
  if (groups > (1 << 20)) return fail(WGB_ERR_INVALID_VALUE, "groups must be at most 2^20");
  if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX)
    return fail(WGB_ERR_INVALID_VALUE, "m, n, and k must be below 2^31");
  return WGB_OK;
}

}  // namespace

extern "C" int wgb_gemm_grouped(wgb_ctx *ctx, int type, int transA, int64_t groups, int64_t m, int64_t n, int64_t k,
                                float alpha, const void *A, int64_t lda, int64_t strideA, const void *B, int64_t ldb,
                                const int64_t *d_offsets, float beta, void *C, int64_t ldc, int ctype) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_sizes(type, ctype, groups, m, n, k))) return st;
  if (transA != WGB_NO_TRANS && transA != WGB_TRANS)
    return fail(WGB_ERR_INVALID_VALUE, "transA must be WGB_NO_TRANS or WGB_TRANS");
  const int64_t a_rows = transA == WGB_TRANS ? k : m, a_cols = transA == WGB_TRANS ? m : k;
  if (lda < (a_rows > 1 ? a_rows : 1)) return fail(WGB_ERR_INVALID_VALUE, "lda must be >= max(1, rows of A)");
  if (strideA < 0 || (groups > 1 && strideA < (a_cols > 0 ? (a_cols - 1) * lda + a_rows : 0)))
    return fail(WGB_ERR_INVALID_VALUE, "strideA must cover a group's A");
  if (ldb < (k > 1 ? k : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldb must be >= max(1, k)");
  if (ldc < (m > 1 ? m : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldc must be >= max(1, m)");
  if (m == 0 || n == 0 || groups == 0) return WGB_OK;
  if (!d_offsets) return fail(WGB_ERR_INVALID_VALUE, "d_offsets is null");
  if (!C) return fail(WGB_ERR_INVALID_VALUE, "C is null");
  if (k > 0 && alpha != 0.0f && (!A || !B)) return fail(WGB_ERR_INVALID_VALUE, "A or B is null");
  const int64_t es = type_size(type);
  Args p = {};
  p.m = m;
  p.n = n;
  p.k = k;
  p.A = (const char *)A;
  p.B = (const char *)B;
  p.lda = lda * es;
  p.ldb = ldb * es;
  p.stride_a = strideA * es;
  p.off = d_offsets;
  p.groups = (int)groups;
  p.C = C;
  p.ldc = ldc;
  p.alpha = alpha;
  p.beta = beta;
  p.c_f32 = ctype == WGB_F32;
  const bool vec = copyable(A, p.lda, p.stride_a) && copyable(B, p.ldb, 0);
  wgb::timing_begin(ctx);
  const bool amc = transA == WGB_NO_TRANS;
  st = type == WGB_F32   ? dispatch_columns<F32>(ctx, p, amc, vec)
       : type == WGB_F16 ? dispatch_columns<F16>(ctx, p, amc, vec)
                         : dispatch_columns<Bf16>(ctx, p, amc, vec);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_gemm_grouped_k(wgb_ctx *ctx, int type, int64_t groups, int64_t m, int64_t n, int64_t k, float alpha,
                                  const void *A, int64_t lda, const void *B, int64_t ldb, const int64_t *d_offsets,
                                  float beta, void *C, int64_t ldc, int64_t strideC, int ctype) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_sizes(type, ctype, groups, m, n, k))) return st;
  if (lda < (m > 1 ? m : 1)) return fail(WGB_ERR_INVALID_VALUE, "lda must be >= max(1, m)");
  if (ldb < (n > 1 ? n : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldb must be >= max(1, n)");
  if (ldc < (m > 1 ? m : 1)) return fail(WGB_ERR_INVALID_VALUE, "ldc must be >= max(1, m)");
  if (strideC < 0 || (groups > 1 && strideC < (n > 0 ? (n - 1) * ldc + m : 0)))
    return fail(WGB_ERR_INVALID_VALUE, "strideC must cover a group's C");
  if (m == 0 || n == 0 || groups == 0) return WGB_OK;
  if (!d_offsets) return fail(WGB_ERR_INVALID_VALUE, "d_offsets is null");
  if (!C) return fail(WGB_ERR_INVALID_VALUE, "C is null");
  if (k > 0 && alpha != 0.0f && (!A || !B)) return fail(WGB_ERR_INVALID_VALUE, "A or B is null");
  const int64_t es = type_size(type);
  Args p = {};
  p.m = m;
  p.n = n;
  p.k = k;
  p.A = (const char *)A;
  p.B = (const char *)B;
  p.lda = lda * es;
  p.ldb = ldb * es;
  p.off = d_offsets;
  p.groups = (int)groups;
  p.C = C;
  p.ldc = ldc;
  p.stride_c = strideC;
  p.alpha = alpha;
  p.beta = beta;
  p.c_f32 = ctype == WGB_F32;
  const bool vec = copyable(A, p.lda, 0) && copyable(B, p.ldb, 0);
  wgb::timing_begin(ctx);
  st = type == WGB_F32   ? (vec ? run_k<F32, true>(ctx, p) : run_k<F32, false>(ctx, p))
       : type == WGB_F16 ? (vec ? run_k<F16, true>(ctx, p) : run_k<F16, false>(ctx, p))
                         : (vec ? run_k<Bf16, true>(ctx, p) : run_k<Bf16, false>(ctx, p));
  wgb::timing_end(ctx);
  return st;
}
