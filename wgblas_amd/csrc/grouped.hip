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

// The tile (64, 128 or 256 square) whose estimated time is least, and that
// time; 256 needs 16-bit operands that can be copied. Operands that cannot
// cost about three times as much (bf16 4096^3 at an odd leading dimension:
// 347 TFLOP/s on 128 x 128 tiles).
template <class E>
int choose(wgb_ctx *ctx, const Args &p, bool vec, double k, double n64, double n128, double n256, double &time) {
  const double size = p.c_f32 ? 4 : 2;
  auto cost_of = [&](int T) {
    TileCost c = cost<E>(T);
    return vec ? c : TileCost{3 * c.first, 3 * c.next};
  };
  const double t64 = small_time(64, cost_of(64), per_cu(ctx, p, 64, n64), k, size);
  const double t128 = small_time(128, cost_of(128), per_cu(ctx, p, 128, n128), k, size);
  time = t128 <= t64 ? t128 : t64;
  if (vec && E::kBits == 16) {
    const double t256 = rounds_time(cost_of(256), cost_of(128), per_cu(ctx, p, 256, n256), k, size,
                                    most_pieces((int64_t)k, 64));
    if (t256 <= time) {
      time = t256;
      return 256;
    }
  }
  return t128 <= t64 ? 128 : 64;
}

template <class E>
int choose_columns(wgb_ctx *ctx, const Args &p, bool vec, double &time) {
  return choose<E>(ctx, p, vec, (double)p.k, expected_columns(p, 64), expected_columns(p, 128), expected_columns(p, 256),
                   time);
}

template <class E>
int choose_k(wgb_ctx *ctx, const Args &p, bool vec, double &time) {
  auto across = [&](int64_t T) { return (double)((p.n + T - 1) / T * p.groups); };
  return choose<E>(ctx, p, vec, (double)p.k / p.groups, across(64), across(128), across(256), time);
}

// Columns of `rows` 16-bit values moved to a leading dimension that 16-byte
// copies can read (whole chunks, the rest of the last one zeros).
__global__ __launch_bounds__(256) void align_kernel(const uint16_t *X, int64_t ld, int64_t stride, int64_t cols,
                                                    int64_t total, int rows, int chunks, v4i *Y) {
  struct __attribute__((packed, aligned(2))) Chunk {
    v4i v;
  };
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total * chunks; i += step) {
    const int64_t col = i / chunks;
    const int at = (int)(i - col * chunks) * 8;
    const uint16_t *x = X + col / cols * stride + col % cols * ld + at;
    v4i v;
    if (at + 8 <= rows) {
      v = reinterpret_cast<const Chunk *>(x)->v;
    } else {
      typedef uint16_t u8 __attribute__((ext_vector_type(8)));
      u8 u = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (at + c < rows) u[c] = x[c];
      v = __builtin_bit_cast(v4i, u);
    }
    Y[i] = v;
  }
}

// Operands that cannot be copied (16-bit values at odd leading dimensions or
// addresses) are first moved into the context's workspace where that and the
// faster product take less time than the slower product: `now` and `then` are
// the products' estimates, the move is a read and a write at 4.5 TB/s. Where
// there is no memory for the copies the slower product runs, which needs none.
// a_cols: columns of a group's A. Sets vec where it did.
int align_operands(wgb_ctx *ctx, Args &p, double now, double then, int64_t a_rows, int64_t a_cols, int64_t a_groups,
                   int64_t b_rows, int64_t b_cols, bool &vec) {
  const bool move_a = !copyable(p.A, p.lda, p.stride_a), move_b = !copyable(p.B, p.ldb, 0);
  const int64_t a_chunks = (a_rows + 7) / 8, b_chunks = (b_rows + 7) / 8;
  const int64_t a_total = a_cols * a_groups, bytes_a = move_a ? a_total * a_chunks * 16 : 0,
                bytes_b = move_b ? b_cols * b_chunks * 16 : 0;
  if (a_chunks * 16 >= (int64_t)1 << 22 || b_chunks * 16 >= (int64_t)1 << 22) return WGB_OK;
  if (then + 2.0 * (double)(bytes_a + bytes_b) / 4.5e6 + 3.0 >= now) return WGB_OK;
  const int st = wgb::ensure_op_workspace(ctx, (size_t)(bytes_a + bytes_b) + parts_bytes(ctx));
  if (st) return st == WGB_ERR_ALLOC ? WGB_OK : st;
  p.parts = (float *)((char *)ctx->op_ws + bytes_a + bytes_b);
  auto move = [&](const char *X, int64_t ld, int64_t stride, int64_t cols, int64_t total, int64_t rows, int64_t chunks,
                  char *Y) {
    const int64_t want = (total * chunks + 255) / 256, most = (int64_t)ctx->num_cus * 32;
    align_kernel<<<(unsigned)(want < most ? want : most), 256, 0, ctx->stream>>>(
        (const uint16_t *)X, ld / 2, stride / 2, cols, total, (int)rows, (int)chunks, (v4i *)Y);
  };
  char *ws = (char *)ctx->op_ws;
  if (move_a) {
    move(p.A, p.lda, p.stride_a, a_cols, a_total, a_rows, a_chunks, ws);
    p.A = ws;
    p.lda = a_chunks * 16;
    p.stride_a = a_cols * p.lda;
    ws += bytes_a;
  }
  if (move_b) {
    move(p.B, p.ldb, 0, b_cols, b_cols, b_rows, b_chunks, ws);
    p.B = ws;
    p.ldb = b_chunks * 16;
  }
  WGB_CHECK_LAUNCH("align_kernel");
  vec = true;
  return WGB_OK;
}

template <class E, bool AMC, bool VEC>
int run_columns(wgb_ctx *ctx, Args &p) {
  const int64_t mean = p.n / p.groups;
  if (mean <= 32) {
    // Few columns: reading A counts. Whole rows of blocks stream it through
    // LDS (64 experts of 2048 x 1024 in bf16: 27 us, the waves-share-k kernel
    // 37); with too few blocks for the CUs the waves share k instead (8192 x
    // 4096, one column: 5.8 against 10 us in fp4), as they do where the
    // operands cannot be copied.
    const int64_t blocks = (p.m + 127) / 128 * (p.n < p.groups ? p.n : p.groups);
    if constexpr (!AMC) {
      if (!VEC || blocks < ctx->num_cus)
        return mean <= 16 ? launch_columns<SkinnyKernel<E, 2, 1>>(ctx, p) : launch_columns<SkinnyKernel<E, 2, 2>>(ctx, p);
    }
    if constexpr (VEC || AMC) return launch_columns<Kernel<E, 128, 32, 4, 1, AMC, false, VEC, false, 4>>(ctx, p);
  }
  double time;
  const int T = choose_columns<E>(ctx, p, VEC, time);
  if constexpr (VEC && E::kBits == 16) {
    if (T == 256)
      return launch_columns_rounds<TurnKernel<E, AMC, false, false>, Kernel<E, 128, 128, 2, 2, AMC, false, VEC, false, 2>>(ctx, p);
  }
  if (T == 128) return launch_columns<Kernel<E, 128, 128, 2, 2, AMC, false, VEC, false, 2>>(ctx, p);
  return launch_columns<Kernel<E, 64, 64, 2, 2, AMC, false, VEC, false, 2>>(ctx, p);
}

template <class E, bool VEC>
int run_k(wgb_ctx *ctx, Args &p) {
  double time;
  const int T = choose_k<E>(ctx, p, VEC, time);
  if constexpr (VEC && E::kBits == 16) {
    if (T == 256)
      return launch_k_rounds<TurnKernel<E, true, true, true>, Kernel<E, 128, 128, 2, 2, true, true, VEC, true, 2>>(ctx, p);
  }
  if (T == 128) return launch_k<Kernel<E, 128, 128, 2, 2, true, true, VEC, true, 2>>(ctx, p);
  return launch_k<Kernel<E, 64, 64, 2, 2, true, true, VEC, true, 2>>(ctx, p);
}

template <class E>
int dispatch_k(wgb_ctx *ctx, Args &p) {
  bool vec = copyable(p.A, p.lda, 0) && copyable(p.B, p.ldb, 0);
  if (!vec && E::kBits == 16 && p.alpha != 0.0f) {
    double now, then;
    choose_k<E>(ctx, p, false, now);
    choose_k<E>(ctx, p, true, then);
    const int st = align_operands(ctx, p, now, then, p.m, p.k, 1, p.n, p.k, vec);
    if (st) return st;
  }
  return vec ? run_k<E, true>(ctx, p) : run_k<E, false>(ctx, p);
}

template <class E>
int dispatch_columns(wgb_ctx *ctx, Args &p, bool amc) {
  bool vec = copyable(p.A, p.lda, p.stride_a) && copyable(p.B, p.ldb, 0);
  if (!vec && E::kBits == 16 && p.n / p.groups > 32 && p.k > 0 && p.alpha != 0.0f) {
    double now, then;
    choose_columns<E>(ctx, p, false, now);
    choose_columns<E>(ctx, p, true, then);
    const int st = align_operands(ctx, p, now, then, amc ? p.m : p.k, amc ? p.k : p.m, p.groups, p.k, p.n, vec);
    if (st) return st;
  }
  if (amc) return vec ? run_columns<E, true, true>(ctx, p) : run_columns<E, true, false>(ctx, p);
  return vec ? run_columns<E, false, true>(ctx, p) : run_columns<E, false, false>(ctx, p);
}

// Checks shared by both forms.
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
  wgb::timing_begin(ctx);
  const bool amc = transA == WGB_NO_TRANS;
  st = type == WGB_F32   ? dispatch_columns<F32>(ctx, p, amc)
       : type == WGB_F16 ? dispatch_columns<F16>(ctx, p, amc)
                         : dispatch_columns<Bf16>(ctx, p, amc);
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
  wgb::timing_begin(ctx);
  st = type == WGB_F32   ? dispatch_k<F32>(ctx, p)
       : type == WGB_F16 ? dispatch_k<F16>(ctx, p)
                         : dispatch_k<Bf16>(ctx, p);
  wgb::timing_end(ctx);
  return st;
}
