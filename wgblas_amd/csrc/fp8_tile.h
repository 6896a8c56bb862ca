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
// fp32's), so at most 7 2^-13 of the largest, less than 2^-10 of the eight's
// magnitudes. Taken for 16-bit results, for twice the rate. On normal values it
// is 1.3e-5 of the result (2-norm, no bias found), where rounding a bf16 result is
// 1.7e-3 and an f16 one 2.07e-4 (2.08e-4 with it, 512 x 512 x 2048; about two of
// a thousand bf16 elements are the neighbouring number). One channel of every eight
// 1000 times as large: f16 2.27e-4, 2.08e-4 of it its rounding; two of eight whose
// products cancel: 2.1e-3 of an f16 result and 2.7e-3 of a bf16 one, more than
// their rounding. An fp32 result would show it everywhere: there the codes are
// widened to bf16, which holds them exactly, and multiplied by
// v_mfma_f32_16x16x32_bf16, whose sums are fp32's throughout, at half the rate.
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

// 8 bytes of k of this lane's row. A pointer of its own, as far as the compiler
// is told: it would wait for all copies to LDS that are under way otherwise,
// and those are waited for where their k-tiles are due.
typedef int v2i __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2i read_transposed(const char *__restrict__ at) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i *)at);
}

// The MFMA operands of a k-tile for MB blocks of 16 rows, `STEP` rows apart,
// from row `wrow`.
template <int BT, bool MC, int MB, int STEP = 16>
__device__ __forceinline__ void fetch_codes(const char *stage, int wrow, int lane, v8i (&out)[MB]) {
  const int i16 = lane & 15, g = lane >> 4;
  if constexpr (!MC) {
    const int lo = (g ^ (i16 & 7)) * 16, hi = ((4 + g) ^ (i16 & 7)) * 16;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const char *row = stage + (wrow + STEP * b + i16) * TB;
      const v4i x = *reinterpret_cast<const v4i *>(row + lo), y = *reinterpret_cast<const v4i *>(row + hi);
      out[b] = v8i{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
  } else {
    const int kr = 16 * g + (i16 >> 1);
    int at = kr * BT + ((wrow ^ (mc_key<8, BT / 16>(kr) << 4)) + (i16 & 1) * 8);
    asm volatile("" : "+v"(at));  // one register, not one for every block
#pragma unroll
    for (int b = 0; b < MB; ++b) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v2i x = read_transposed(stage + (at ^ (STEP * b)) + (64 * (q >> 1) + 8 * (q & 1)) * BT);
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
        const int64_t first_row = m0 >> p.a_shift;
        src[r] += first_row * p.a_row;
        voff[r] = (uint32_t)(((row >> p.a_shift) - first_row) * p.a_row * 4);
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

// The products of some row blocks with all column blocks, added to the sums.
// sb: the columns' scales; ROWS: A has a scale for each row (sa[i]: of the
// lane's four rows of block i), else the one for all is in sb. A block's
// products are scaled while the next ones are multiplied: the scheduler, left
// to itself, puts the v_fma right behind its MFMA and waits for it.
template <bool EXACT, bool ROWS, int MB, int NB, int FIRST, int COUNT>
__device__ __forceinline__ void multiply_codes(const v8i (&a)[COUNT], const typename Codes<EXACT>::wide (&b)[NB],
                                               f4 (&acc)[MB][NB], const f4 (&sa)[ROWS ? COUNT : 1], const float (&sb)[NB]) {
  typedef Codes<EXACT> X;
  constexpr int LAG = EXACT ? 1 : 2;
  typename X::wide w;
  f4 late[LAG + 1];
#pragma unroll
  for (int n = 0; n < COUNT * NB + LAG; ++n) {
    if (n < COUNT * NB) {
      if (n % NB == 0) w = X::widen(a[n / NB]);
      late[n % (LAG + 1)] = X::dot(w, b[n % NB]);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int m = n - LAG;
    if (m >= 0) {
      const int i = m / NB, j = m % NB;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        acc[FIRST + i][j][q] = fmaf(late[m % (LAG + 1)][q], ROWS ? sa[i][q] * sb[j] : sb[j], acc[FIRST + i][j][q]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// One BM x BN tile of C a block, WM x WN waves, S stages of LDS. 128 x 128 with
// exact sums and rows' own scales is bound by the conversions and v_fma (4096 x
// 2048 x 16384: 259 us, 1.06 PFLOP/s), 128 x 32 by reading A (49 experts of 4096
// x 2048 with 96 columns: 80 us, 5.1 TB/s).
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
    int nt = p.alpha == 0.0f ? 0 : (int)(p.k / TB), first = 0;
    if (REST && quarter.pieces > 1) {
      const int most = (nt + quarter.pieces - 1) / quarter.pieces;
      first = quarter.piece * most;
      nt = nt - first < most ? nt - first : most;
    }
    if (nt > 0) {
      SA sa;
      SB sb;
      SS ss;
      const int64_t depth = (AMC ? p.a_depth : p.k) - (int64_t)first * TB;
      sa.init(p.A + (int64_t)tile.g * p.stride_a, p.lda, m0, AMC ? p.a_rows : p.m, depth, t);
      sb.init(p.B + tile.lo * p.ldb, p.ldb, n0, cols, p.k - (int64_t)first * TB, t);
      sa.origin += first * sa.step();
      sb.origin += first * sb.step();
      ss.init(p, tile.g, m0, tile.lo + n0, cols - n0, first, wave, lane);
      const int whole = sa.soft_tail() && sa.whole_tiles() < nt ? sa.whole_tiles() : nt;

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
      // the row blocks in PARTS, each read while the one before is multiplied
      constexpr int PARTS = MB % 2 == 0 ? 2 : 1, PB = MB / PARTS;
      v8i a[PARTS][PB], b[NB];
      f4 scale_a[PARTS][ROWS ? PB : 1];
      float scale_b[NB];
      auto fetch_a = [&](const char *st, int part) {
        fetch_codes<BM, AMC, PB>(st, wm + 16 * PB * part, lane, a[part]);
        const float *scales = reinterpret_cast<const float *>(st + SA::BYTES + SB::BYTES);
        if constexpr (ROWS) {
#pragma unroll
          for (int i = 0; i < PB; ++i)
            scale_a[part][i] = *reinterpret_cast<const f4 *>(scales + wm + 16 * (PB * part + i) + 4 * (lane >> 4));
        }
      };
      auto fetch_b = [&](const char *st) {
        fetch_codes<BN, false, NB>(st + SA::BYTES, wn, lane, b);
        const float *scales = reinterpret_cast<const float *>(st + SA::BYTES + SB::BYTES);
#pragma unroll
        for (int j = 0; j < NB; ++j) scale_b[j] = scales[BM + wn + 16 * j + (lane & 15)];
        if constexpr (!ROWS) {
          const float rows = scales[wm];
#pragma unroll
          for (int j = 0; j < NB; ++j) scale_b[j] *= rows;
        }
      };

      // Tile kt is read from stage kt % S while the copies of the next S - 1
      // are in flight or landed; its stage takes tile kt + S after the barrier
      // that ends its reads.
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < nt) fill(i);
      wait_barrier<0>();
      const int steady = whole - S;  // tile kt + S exists and is whole
      for (int kt = 0; kt < nt; ++kt) {
        const char *st = smem + (kt % S) * STAGE;
        fetch_b(st);
        fetch_a(st, 0);
        typename Codes<EXACT>::wide wb[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) wb[j] = Codes<EXACT>::widen(b[j]);
        if constexpr (PARTS == 2) fetch_a(st, 1);
        multiply_codes<EXACT, ROWS, MB, NB, 0, PB>(a[0], wb, acc, scale_a[0], scale_b);
        if (kt < steady) {
          wait_barrier<(S - 2) * PER_TILE>();
          copy(kt + S);
        } else {
          wait_barrier<0>();
          if (kt + S < nt) fill(kt + S);
        }
        if constexpr (PARTS == 2) multiply_codes<EXACT, ROWS, MB, NB, PB, PB>(a[1], wb, acc, scale_a[1], scale_b);
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

// The 256 x 256 tile of the large products: 8 waves of 128 x 64 each, two on
// every SIMD. Their v_fma and LDS reads fill the time of each other's MFMAs, so
// nothing orders them but one barrier a k-tile (taking turns, as the 16-bit
// TurnKernel does, leaves a wave alone with its v_fma: 50 cycles an MFMA, not
// 32). A k-tile's row blocks are multiplied in PARTS; a part is read while the
// one before is multiplied. When the last part has been read, the barrier, which
// also ends the wait for the next k-tile's copies, frees the stage: the next
// k-tile's columns are read block by block into the registers that the last
// part's products leave, and the copies of the k-tile after that start. They
// are issued one by one between MFMAs, A's in the last part, B's in the next
// k-tile's first one: issued together, 64 KB took all waves 1000 to 1500
// cycles, at 64 bytes a cycle and CU, with no MFMA running.
// A block runs through tiles (w, w + blocks, ...). The next tile's first copies
// are issued before a tile is stored, when its operands' registers are free: in
// the midst of a tile they would have to be spilled, and each return of one
// waits for all copies and stores under way.
// 8192 x 4096 x 8192 into bf16: 224 us (2.45 PFLOP/s) and 226 with A
// row-contiguous, one call at a time; from call to call 255 and 231, bound by
// power; at k = 2048 2.0 to 2.1 PFLOP/s, for a tile's start and end.
template <bool AMC, bool ROWS, bool EXACT>
struct Fp8Large {
  static constexpr int BM = 256, BN = 256, WM = 2, WN = 4;
  static constexpr int kBM = BM, kBN = BN;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16, STEP = 16 * WN;
  static constexpr int PB = EXACT ? 1 : 2, PARTS = MB / PB;
  typedef Codes<EXACT> X;
  typedef Stager<Fp8, BM, AMC, NT> SA;
  typedef Stager<Fp8, BN, false, NT> SB;
  typedef BlockScaleStager<BM, BN, NW> SS;
  typedef TileTable<ColumnOrder> Table;
  static constexpr int STAGE = SA::BYTES + SB::BYTES + SS::BYTES;
  static constexpr int LDS = 2 * STAGE;
  static constexpr int COPIES_B = SB::LOADS + SS::LOADS;
  static_assert(SB::RPS == STEP, "a load is STEP columns");

  // The copies of a tile's k-tiles: of A, and of B with the scales.
  struct Copies {
    SA sa;
    SB sb;
    SS ss;

    __device__ __forceinline__ void init(const Args &p, const Tile &tile, int t) {
      const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN, cols = tile.hi - tile.lo;
      sa.init(p.A + (int64_t)tile.g * p.stride_a, p.lda, m0, AMC ? p.a_rows : p.m, AMC ? p.a_depth : p.k, t);
      sb.init(p.B + tile.lo * p.ldb, p.ldb, n0, cols, p.k, t);
      ss.init(p, tile.g, m0, tile.lo + n0, cols - n0, 0, __builtin_amdgcn_readfirstlane(t >> 6), t & 63);
    }
    __device__ __forceinline__ char *stage_of(char *smem, int kt) const { return smem + (kt & 1) * STAGE; }
    __device__ __forceinline__ void a(char *smem, int wave, int kt, int r) const {
      copy_chunks(sa.origin + kt * sa.step(), sa.voff[r], stage_of(smem, kt) + wave * 1024 + r * NT * 16);
    }
    __device__ __forceinline__ void b(char *smem, int wave, int kt, int r) const {
      char *st = stage_of(smem, kt) + SA::BYTES;
      if (r < SB::LOADS)
        copy_chunks(sb.origin + (int64_t)kt * TB, sb.voff[r], st + wave * 1024 + r * NT * 16);
      else
        ss.copy(st + SB::BYTES, kt);
    }
    // All of A of any k-tile: k-rows past k read the k-tile's first one again, B's codes there are zeros.
    __device__ __forceinline__ void all_a(char *smem, int wave, int kt) const {
      const bool cut = sa.soft_tail() && kt >= sa.whole_tiles();
#pragma unroll
      for (int r = 0; r < SA::LOADS; ++r)
        copy_chunks(sa.origin + kt * sa.step(), cut ? sa.tail_voff(r) : sa.voff[r],
                    stage_of(smem, kt) + wave * 1024 + r * NT * 16);
    }
    __device__ __forceinline__ void all_b(char *smem, int wave, int kt) const {
#pragma unroll
      for (int r = 0; r < COPIES_B; ++r) b(smem, wave, kt, r);
    }
  };

  // What a wave multiplies.
  struct Operands {
    v8i a[2][PB];  // the part that is multiplied and the next one
    f4 rows[2][ROWS ? PB : 1];
    v8i raw[NB];   // the next k-tile's columns and scales
    float next_a, next_b[NB];

    template <int P>
    __device__ __forceinline__ void fetch_a(const char *st, int wm, int lane) {
      fetch_codes<BM, AMC, PB>(st, wm + 16 * PB * P, lane, a[P & 1]);
      if constexpr (ROWS) {
        const float *s = reinterpret_cast<const float *>(st + SA::BYTES + SB::BYTES);
#pragma unroll
        for (int i = 0; i < PB; ++i) rows[P & 1][i] = *reinterpret_cast<const f4 *>(s + wm + 16 * (PB * P + i) + 4 * (lane >> 4));
      }
    }
    __device__ __forceinline__ void fetch_b(const char *st, int wn, int lane, int j) {
      v8i one[1];
      fetch_codes<BN, false, 1>(st + SA::BYTES, wn + STEP * j, lane, one);
      raw[j] = one[0];
    }
    __device__ __forceinline__ void fetch_scales(const char *st, int wm, int wn, int lane) {
      const float *s = reinterpret_cast<const float *>(st + SA::BYTES + SB::BYTES);
      if constexpr (!ROWS) next_a = s[wm];
#pragma unroll
      for (int j = 0; j < NB; ++j) next_b[j] = s[BM + wn + STEP * j + (lane & 15)];
    }
  };

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * 16;
    const int depth = p.alpha == 0.0f ? 0 : (int)(p.k / TB);  // k-tiles of every tile; alpha == 0 reads neither operand
    Table table;
    table.init(p, BN);
    Copies c;
    Operands o;
    f4 acc[MB][NB];

    // k-tile kt, of which the first USED column blocks of the tile exist.
    // STEADY: k-tiles kt + 1 and kt + 2 exist and are whole.
    auto k_tile = [&](auto used, auto steady, int kt) {
      constexpr int USED = decltype(used)::value;
      constexpr bool STEADY = decltype(steady)::value;
      const char *st = smem + (kt & 1) * STAGE, *next = smem + (~kt & 1) * STAGE;
      typename X::wide b[USED];
      float scale[USED];
#pragma unroll
      for (int j = 0; j < USED; ++j) {
        b[j] = X::widen(o.raw[j]);
        scale[j] = ROWS ? o.next_b[j] : o.next_a * o.next_b[j];
      }
      // part's products; behind(n) is run behind the n-th of PB USED
      auto multiply = [&](auto part, auto behind) {
        constexpr int P = decltype(part)::value;
        typename X::wide w[PB];
#pragma unroll
        for (int i = 0; i < PB; ++i) w[i] = X::widen(o.a[P & 1][i]);
        // a product is scaled behind the LAG next ones: left to itself the
        // scheduler puts the v_fma right behind its MFMA and waits for it
        constexpr int LAG = EXACT ? 1 : 2;
        f4 late[LAG + 1];
#pragma unroll
        for (int n = 0; n < PB * USED + LAG; ++n) {
          if (n < PB * USED) {
            late[n % (LAG + 1)] = X::dot(w[n % PB], b[n / PB]);
            __builtin_amdgcn_sched_barrier(0);
            behind(n);
          }
          const int m = n - LAG, i = m % PB, j = m / PB;
          if (m >= 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[PB * P + i][j][q] =
                  fmaf(late[m % (LAG + 1)][q], ROWS ? o.rows[P & 1][i][q] * scale[j] : scale[j], acc[PB * P + i][j][q]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        // the sums are made here: past a branch the v_fma would be far from their MFMAs, whose results all wait for them
#pragma unroll
        for (int i = 0; i < PB; ++i)
#pragma unroll
          for (int j = 0; j < USED; ++j) asm volatile("" : "+v"(acc[PB * P + i][j]));
      };
      // of the first part, or of the first two where a part has fewer products than B's k-tile has copies
      constexpr int AT_ONCE = PB * USED >= COPIES_B ? 1 : (COPIES_B + 2 * PB * USED - 1) / (2 * PB * USED);
      auto part = [&](auto at) {
        constexpr int P = decltype(at)::value;
        o.template fetch_a<P + 1>(st, wm, lane);
        if constexpr (P == 0 && !STEADY) {
          if (kt + 1 < depth) c.all_b(smem, wave, kt + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        multiply(at, [&](int n) {
          if (!STEADY || P > 1) return;
#pragma unroll
          for (int r = (P * PB * USED + n) * AT_ONCE; r < (P * PB * USED + n + 1) * AT_ONCE; ++r)
            if (r < COPIES_B) c.b(smem, wave, kt + 1, r);
        });
      };
      part(std::integral_constant<int, 0>());
      part(std::integral_constant<int, 1>());
      part(std::integral_constant<int, 2>());
      if constexpr (PARTS == 8) {
        part(std::integral_constant<int, 3>());
        part(std::integral_constant<int, 4>());
        part(std::integral_constant<int, 5>());
        part(std::integral_constant<int, 6>());
      }
      wait_barrier<0>();
      if constexpr (!STEADY) {
        if (kt + 2 < depth) c.all_a(smem, wave, kt + 2);
      }
      // (behind the last k-tile: what is read is not used)
      o.template fetch_a<0>(next, wm, lane);  // PARTS is even: the other registers
      o.fetch_scales(next, wm, wn, lane);
      __builtin_amdgcn_sched_barrier(0);
      constexpr int A_AT_ONCE = (SA::LOADS + PB * USED - 1) / (PB * USED);
      multiply(std::integral_constant<int, PARTS - 1>(), [&](int n) {
        if (n % PB == PB - 1) o.fetch_b(next, wn, lane, n / PB);
        if (!STEADY) return;
#pragma unroll
        for (int r = n * A_AT_ONCE; r < (n + 1) * A_AT_ONCE; ++r)
          if (r < SA::LOADS) c.a(smem, wave, kt + 2, r);
      });
    };
    auto k_tiles = [&](auto used) {
      const int whole = c.sa.soft_tail() ? c.sa.whole_tiles() : depth, steady = (whole < depth ? whole : depth) - 2;
      int kt = 0;
      for (; kt < steady; ++kt) k_tile(used, std::true_type(), kt);
      for (; kt < depth; ++kt) k_tile(used, std::false_type(), kt);
    };
    // The first copies of tile i (its k-tile 0, and A of k-tile 1): false if there is none.
    Tile tile;
    auto begin = [&](int i) {
      if (!table.get(i, tile)) return false;
      if (depth > 0) {
        c.init(p, tile, t);
        c.all_a(smem, wave, 0);
        c.all_b(smem, wave, 0);
        if (depth > 1) c.all_a(smem, wave, 1);
      }
      return true;
    };

    bool more = begin(0);
    for (int i = 1; more; ++i) {
      const int64_t row0 = (int64_t)tile.tm * BM + wm, n0 = (int64_t)tile.tn * BN, cols = tile.hi - tile.lo, at = tile.lo * p.ldc;
#pragma unroll
      for (int x = 0; x < MB; ++x)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[x][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
      if (depth > 0) {
        wait_barrier<0>();
#pragma unroll
        for (int j = 0; j < NB; ++j) o.fetch_b(smem, wn, lane, j);
        o.fetch_scales(smem, wm, wn, lane);
        o.template fetch_a<0>(smem, wm, lane);
        // column blocks in use: a group's last tile costs what its columns need
        if (cols - n0 > STEP * 3)
          k_tiles(std::integral_constant<int, 4>());
        else if (cols - n0 > STEP * 2)
          k_tiles(std::integral_constant<int, 3>());
        else if (cols - n0 > STEP)
          k_tiles(std::integral_constant<int, 2>());
        else
          k_tiles(std::integral_constant<int, 1>());
        // all waves have read the last k-tile's operands before its barrier; what they read behind it is not used
      }
      more = begin(i);
      store(p, at, acc, row0, n0 + wn, cols, lane);
    }
  }

  // Without guards for rows where there is nothing to guard.
  static __device__ __forceinline__ void store(const Args &p, int64_t at, const f4 (&acc)[MB][NB], int64_t row0, int64_t col0,
                                               int64_t cols, int lane) {
    const bool inside = p.beta == 0.0f && row0 + 16 * MB <= p.m;
    if (inside && p.stream)
      store_tile<Fp8, STEP, true, true>(p, at, acc, row0, col0, cols, lane);
    else if (inside)
      store_tile<Fp8, STEP, false, true>(p, at, acc, row0, col0, cols, lane);
    else
      store_tile<Fp8, STEP, false>(p, at, acc, row0, col0, cols, lane);
  }
};

// Few columns a group (single tokens): bound by reading A once. A block has R
// row blocks and CB column blocks of 16; its eight waves share k in k-tiles,
// load both operands straight into MFMA operand registers, the next k-tile ahead
// of the present one's MFMAs, and add their sums in LDS in the waves' order. A
// k-contiguous only. One column, repeated: 8192 x 8192 12.4 us (5.4 TB/s), 4096 x
// 4096 6.9; 16 columns, 8192 x 4096 9.0.
template <int R, int CB, bool ROWS, bool EXACT>
struct Fp8Skinny {
  static constexpr int kBM = 16 * R, kBN = 16 * CB;
  static constexpr int NW = 8, NT = 64 * NW;
  static constexpr int LDS = NW * R * CB * 1024;
  typedef Codes<EXACT> X;

  struct Operands {
    v8i a[R], b[CB];
    f4 sa[R];  // of the lane's four rows, or [0][0] for all
    float sb[CB];
  };

  static __device__ __forceinline__ v8i load(const char *row) {
    const v4i x = *reinterpret_cast<const v4i *>(row), y = *reinterpret_cast<const v4i *>(row + 64);
    return v8i{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  }

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    Tile tile;
    ColumnOrder order;
    order.init(p, kBN);
    if (!order.find(p, blockIdx.x, tile)) return;
    const int64_t m0 = (int64_t)tile.tm * kBM, n0 = tile.lo + (int64_t)tile.tn * kBN;
    const int nt = p.alpha == 0.0f ? 0 : (int)(p.k / TB);  // alpha == 0 reads neither operand

    // this lane's chunks and scales; past the end the last row or column is
    // read again (what it gives is never stored)
    const char *pa[R], *pb[CB];
    const float *sa[R][ROWS ? 4 : 1], *sb[CB];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = m0 + 16 * r + i16, last = p.m - 1;
      pa[r] = p.A + (int64_t)tile.g * p.stride_a + (row < last ? row : last) * p.lda + 16 * g;
#pragma unroll
      for (int q = 0; q < (ROWS ? 4 : 1); ++q) {
        const int64_t of = ROWS ? m0 + 16 * r + 4 * g + q : m0;  // a block's rows share a scale
        sa[r][q] = p.block_scale_a + tile.g * p.a_group + ((of < last ? of : last) >> p.a_shift) * p.a_row;
      }
    }
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      int64_t col = n0 + 16 * c + i16;
      if (col >= tile.hi) col = tile.hi - 1;
      pb[c] = p.B + col * p.ldb + 16 * g;
      sb[c] = p.block_scale_b + col;
    }
    auto fetch = [&](int kt, Operands &o) {
      const int64_t at = (int64_t)kt * TB;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        o.a[r] = load(pa[r] + at);
        if (ROWS || r == 0)
#pragma unroll
          for (int q = 0; q < (ROWS ? 4 : 1); ++q) o.sa[r][q] = sa[r][q][kt * p.a_k];
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        o.b[c] = load(pb[c] + at);
        o.sb[c] = sb[c][kt * p.b_k];
      }
    };
    f4 acc[R][CB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < CB; ++c) acc[r][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const Operands &o) {
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const typename X::wide b = X::widen(o.b[c]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const f4 x = X::dot(X::widen(o.a[r]), b);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[r][c][q] = fmaf(x[q], (ROWS ? o.sa[r][q] : o.sa[0][0]) * o.sb[c], acc[r][c][q]);
        }
      }
    };
    Operands x, y;
    int kt = wave;
    if (kt < nt) fetch(kt, x);
    while (kt < nt) {
      if (kt + NW < nt) fetch(kt + NW, y);
      multiply(x);
      kt += NW;
      if (kt >= nt) break;
      if (kt + NW < nt) fetch(kt + NW, x);
      multiply(y);
      kt += NW;
    }

    // the waves' sums, one block (r, c) after the other: lane's f4 as it is
    f4 *sums = reinterpret_cast<f4 *>(smem);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < CB; ++c) sums[(wave * R * CB + r * CB + c) * 64 + lane] = acc[r][c];
    __syncthreads();
    const int64_t cols = tile.hi - n0;
    if (wave >= R * CB) return;
    static_assert(R * CB <= NW, "a wave a block");
    f4 total[1][1] = {{sums[wave * 64 + lane]}};
#pragma unroll
    for (int v = 1; v < NW; ++v) total[0][0] += sums[(v * R * CB + wave) * 64 + lane];
    store_tile<Fp8, 16>(p, n0 * p.ldc, total, m0 + 16 * (wave / CB), 16 * (wave % CB), cols, lane);
  }
};

}  // namespace wgb_ragged
