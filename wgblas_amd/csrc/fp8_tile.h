// Tiles of products of 8-bit floats (E4M3) with a scale for each block of 128
// along k, on the staging, tile order and epilogue of ragged_tile.h.
//
// C = sum over blocks b of k of sA(b) sB(b) sum over the block of a b: a k-tile
// of 128 bytes is one such block, and one v_mfma_f32_16x16x128_f8f6f4 its sum
// for 16 x 16 elements of C. Its result, from a zero accumulator, is multiplied
// with the two scales on its way into the fp32 sums: four v_fma a lane for the
// 32 cycles that the matrix core takes.
//
// That instruction adds up products in eights (k 8 i .. 8 i + 7 of a lane's
// bytes), aligned to the largest of the eight: what is below 2^-13 of it is
// lost (measured: 2^16 + 4 gives 2^16, the sums of eights among each other are
// fp32's). On normal values that is 1.3e-5 of the result (2-norm), without
// bias, a hundredth of a bf16 result's own rounding; an fp32 result would show
// it, so there the codes are widened to bf16, which holds them exactly, and
// multiplied by v_mfma_f32_16x16x32_bf16, whose sums are fp32's throughout, at
// half the rate.
//
// Operand layout: lane group g = lane / 16 has the bytes 16 g .. 16 g + 15 and
// 64 + 16 g .. of its row's k-tile, in A and in B alike (any order of k that
// both share gives the same sum). From row-contiguous tiles ("MC") they come
// by ds_read_b64_tr_b8: 16 lanes read 8 k-rows of 16 rows, each gets its row's
// 8 values.
#pragma once

#include "ragged_tile.h"

namespace wgb_ragged {

struct Fp8 {
  typedef uint8_t store;  // never stored: products come out in a wider type
  typedef v4i chunk;
  static constexpr int kBits = 8;
};

// What a lane multiplies: 32 codes, or those as bf16.
template <bool EXACT>
struct Codes;

template <>
struct Codes<false> {
  typedef v8i wide;
  static __device__ __forceinline__ wide widen(const v8i &x) { return x; }
  static __device__ __forceinline__ f4 dot(const wide &a, const wide &b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
  }
};

template <>
struct Codes<true> {
  struct wide {
    v4i part[4];
  };
  static __device__ __forceinline__ wide widen(const v8i &x) {
    wide w;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      w.part[c / 2][2 * (c & 1)] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[c], 1.0f, false));
      w.part[c / 2][2 * (c & 1) + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[c], 1.0f, true));
    }
    return w;
  }
  static __device__ __forceinline__ f4 dot(const wide &a, const wide &b) {
    f4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s) Bf16::mma(a.part[s], b.part[s], c, 0, 0, 0, 0, 0);
    return c;
  }
};

// The MFMA operands of a k-tile for MB blocks of 16 rows, `STEP` rows apart,
// from row `wrow`; only the first `used` blocks.
template <int BT, bool MC, int MB, int STEP = 16>
__device__ __forceinline__ void fetch_codes(const char *stage, int wrow, int lane, v8i (&out)[MB], int used = MB) {
  const int i16 = lane & 15, g = lane >> 4;
  if constexpr (!MC) {
    const int lo = (g ^ (i16 & 7)) * 16, hi = ((4 + g) ^ (i16 & 7)) * 16;
#pragma unroll
    for (int b = 0; b < MB; ++b)
      if (b == 0 || __builtin_expect(b < used, 1)) {
        const char *row = stage + (wrow + STEP * b + i16) * TB;
        const v4i x = *reinterpret_cast<const v4i *>(row + lo), y = *reinterpret_cast<const v4i *>(row + hi);
        out[b] = v8i{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      }
  } else {
    typedef int v2i __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) v2i *LdsV2;
    const int kr = 16 * g + (i16 >> 1);
    int at = kr * BT + ((wrow ^ (mc_key<8, BT / 16>(kr) << 4)) + (i16 & 1) * 8);
    asm volatile("" : "+v"(at));  // one register, not one for every block
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      if (b > 0 && __builtin_expect(b >= used, 0)) break;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v2i x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsV2)(stage + (at ^ (STEP * b)) + (64 * (q >> 1) + 8 * (q & 1)) * BT));
        out[b][2 * q] = x[0];
        out[b][2 * q + 1] = x[1];
      }
    }
  }
}

// The scales of a k-tile's rows of A, then of B's columns, a dword each,
// copied 64 at a time; the waves share the copies evenly (a wave past the last
// one copies the last again).
template <int BM, int BN, int NW>
struct BlockScaleStager {
  static constexpr int COPIES = (BM + BN + 63) / 64;
  static constexpr int LOADS = (COPIES + NW - 1) / NW;
  static constexpr int BYTES = COPIES * 256;
  static_assert(BM % 64 == 0, "A's copies are whole");

  const float *src[LOADS];  // scalar
  int64_t step[LOADS];      // from one k-tile to the next
  uint32_t voff[LOADS];     // this lane's dword, in bytes
  int at[LOADS];

  // tile's rows from m0, columns from lo + n0 on, of which n_left exist
  __device__ __forceinline__ void init(const Args &p, int g, int64_t m0, int64_t col0, int64_t n_left, int first, int wave,
                                       int lane) {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      int c = wave + r * NW;
      if (c >= COPIES) c = COPIES - 1;
      at[r] = c * 256;
      if (c * 64 < BM) {
        int64_t row = m0 + c * 64 + lane;
        if (row >= p.m) row = p.m - 1;
        src[r] = p.block_scale_a + g * p.a_group;
        step[r] = p.a_k;
        const int64_t first_row = m0 / p.block_a;
        src[r] += first_row * p.a_row;
        voff[r] = (uint32_t)((row / p.block_a - first_row) * p.a_row * 4);
      } else {
        int64_t col = c * 64 - BM + lane;
        if (col >= n_left) col = n_left - 1;
        src[r] = p.block_scale_b + col0;
        step[r] = p.b_k;
        voff[r] = (uint32_t)(col * 4);
      }
      src[r] += first * step[r];
    }
  }
  __device__ __forceinline__ void copy(char *stage, int kt) const {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) copy4_to_lds(scalar_at((const char *)(src[r] + kt * step[r]), voff[r]), stage + at[r]);
  }
};

// Products of a lane's blocks added to the sums. ROWS: A has a scale for each
// row (sa[i]: of the lane's four rows of block i), else one for all (sa[0][0]).
template <bool EXACT, bool ROWS, int MB, int NB>
__device__ __forceinline__ void multiply_codes(const v8i (&a)[MB], const v8i (&b)[NB], f4 (&acc)[MB][NB], const f4 (&sa)[ROWS ? MB : 1],
                                               const float (&sb)[NB]) {
  typedef Codes<EXACT> X;
  typename X::wide wa[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) wa[i] = X::widen(a[i]);
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const typename X::wide wb = X::widen(b[j]);
    const float s = sa[0][0] * sb[j];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const f4 x = X::dot(wa[i], wb);
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(x[q], ROWS ? sa[i][q] * sb[j] : s, acc[i][j][q]);
    }
  }
}

// One BM x BN tile of C a block, WM x WN waves, S stages of LDS.
template <int BM, int BN, int WM, int WN, bool AMC, bool ROWS, bool EXACT, int S>
struct Fp8Kernel {
  typedef Fp8 Element;
  typedef ColumnOrder Order;
  static constexpr int kBM = BM, kBN = BN, kWM = WM, kWN = WN;
  static constexpr bool kRK = false;
  static constexpr bool REST = BM == 128 && BN == 128;  // computes what a launch of 256 x 256 tiles leaves, too
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
  typedef Stager<Fp8, BM, AMC, NT> SA;
  typedef Stager<Fp8, BN, false, NT> SB;
  typedef BlockScaleStager<BM, BN, NW> SS;
  static constexpr int STAGE = SA::BYTES + SB::BYTES + SS::BYTES;
  static constexpr int LDS = S * STAGE;
  static constexpr int PER_TILE = SA::LOADS + SB::LOADS + SS::LOADS;  // copies of a k-tile, of one wave

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    Tile tile;
    Order order;
    Quarter quarter = {0, 0, 1};
    if (REST && p.round) {
      if (!quarter.find(p, order, blockIdx.x, false, tile)) return;
    } else {
      order.init(p, BN);
      if (!order.find(p, blockIdx.x, tile)) return;
    }
    const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
    const int64_t cols = tile.hi - tile.lo;
    if (m0 >= p.m || n0 >= cols) return;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);

    f4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    // alpha == 0 reads neither operand
    int nt = p.alpha == 0.0f ? 0 : (int)((p.k + TB - 1) / TB), first = 0;
    if (REST && quarter.pieces > 1) {
      const int most = (nt + quarter.pieces - 1) / quarter.pieces;
      first = quarter.piece * most;
      nt = nt - first < most ? nt - first : most;
    }
    if (nt > 0) {
      SA sa;
      SB sb;
      SS ss;
      // columns of 8-bit matrices are whole runs of 128; only A's k-rows (MC) end at k itself
      const int64_t depth = p.k - (int64_t)first * TB;
      sa.init(p.A + (int64_t)tile.g * p.stride_a, p.lda, m0, AMC ? p.a_rows : p.m, AMC ? depth : (int64_t)TB * nt, t);
      sb.init(p.B + tile.lo * p.ldb, p.ldb, n0, cols, (int64_t)TB * nt, t);
      sa.origin += first * sa.step();
      sb.origin += first * sb.step();
      ss.init(p, tile.g, m0, tile.lo + n0, cols - n0, first, wave, lane);
      const int whole = AMC && depth < (int64_t)nt * TB ? nt - 1 : nt;

      auto copy = [&](int kt) {
        char *st = smem + (kt % S) * STAGE;
        sa.copy(st, kt, wave);
        sb.copy(st + SA::BYTES, kt, wave);
        ss.copy(st + SA::BYTES + SB::BYTES, kt);
      };
      // k-rows past k read the k-tile's first one again: B's codes there are zeros
      auto fill = [&](int kt) {
        if (kt < whole) {
          copy(kt);
          return;
        }
        char *st = smem + (kt % S) * STAGE;
#pragma unroll
        for (int r = 0; r < SA::LOADS; ++r)
          copy_chunks(sa.origin + (int64_t)kt * sa.step(), sa.tail_voff(r), st + wave * 1024 + r * NT * 16);
        sb.copy(st + SA::BYTES, kt, wave);
        ss.copy(st + SA::BYTES + SB::BYTES, kt);
      };
      struct Operands {
        v8i a[MB], b[NB];
        f4 sa[ROWS ? MB : 1];
        float sb[NB];
      };
      auto fetch = [&](int kt, Operands &o) {
        const char *st = smem + (kt % S) * STAGE;
        fetch_codes<BM, AMC, MB>(st, wm, lane, o.a);
        fetch_codes<BN, false, NB>(st + SA::BYTES, wn, lane, o.b);
        const float *scales = reinterpret_cast<const float *>(st + SA::BYTES + SB::BYTES);
        if constexpr (ROWS) {
#pragma unroll
          for (int i = 0; i < MB; ++i) o.sa[i] = *reinterpret_cast<const f4 *>(scales + wm + 16 * i + 4 * (lane >> 4));
        } else {
          o.sa[0][0] = scales[wm];
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) o.sb[j] = scales[BM + wn + 16 * j + (lane & 15)];
      };
      auto multiply = [&](const Operands &o) { multiply_codes<EXACT, ROWS>(o.a, o.b, acc, o.sa, o.sb); };

      // Tile kt is read from stage kt % S while the copies of the next S - 1
      // are in flight or landed; its stage takes tile kt + S after the barrier
      // that ends its reads, and its products run behind that barrier.
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < nt) fill(i);
      wait_barrier<0>();
      Operands x, y;
      fetch(0, x);
      int kt = 0;
      // steady: two tiles a turn while tiles kt + S and kt + 1 + S are whole
      const int steady = whole - S - 1;
      for (; kt < steady; kt += 2) {
        wait_barrier<(S - 2) * PER_TILE>();
        copy(kt + S);
        fetch(kt + 1, y);
        multiply(x);
        wait_barrier<(S - 2) * PER_TILE>();
        copy(kt + 1 + S);
        fetch(kt + 2, x);
        multiply(y);
      }
      for (; kt < nt; ++kt) {
        wait_barrier<0>();
        if (kt + S < nt) fill(kt + S);
        if (kt + 1 < nt) fetch(kt + 1, y);
        multiply(x);
        if (kt + 1 < nt) x = y;
      }
    }

    if (REST && quarter.pieces > 1) {
      f4 *part = reinterpret_cast<f4 *>(p.parts) + ((int64_t)blockIdx.x * NW + wave) * (MB * NB * 64) + lane;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i) part[(j * MB + i) * 64] = acc[i][j];
      return;
    }
    store_tile<Fp8, 16>(p, tile.lo * p.ldc, acc, m0 + wm, n0 + wn, cols, lane);
  }
};

}  // namespace wgb_ragged
