// Tiles of ragged, grouped products on CDNA4's matrix cores, for 16-bit, fp32
// and MXFP4 operands with fp32 sums.
//
// Two shapes of raggedness, both with the group boundaries in device memory
// (a router's result; the host never waits for it):
//   * ragged columns: C(:, j) = alpha op(A_g) B(:, j) + beta C(:, j) for the
//     columns off[g] <= j < off[g + 1] of group g (forward products and input
//     gradients of expert layers). A block finds its tile itself: the groups'
//     numbers of column tiles are summed over the lanes of a wave, and the
//     launch has as many blocks as the worst split of the columns needs;
//   * ragged k: C_g = alpha A(:, off[g]:off[g+1]) B(:, off[g]:off[g+1])^T +
//     beta C_g (weight gradients).
//
// Everything is counted in bytes: a k-tile is 128 bytes of k (64 16-bit, 32
// fp32, 256 fp4 elements), an MFMA operand is 16 bytes a lane. One k-tile is
// two steps of 64 bytes, in which lane group g = lane / 16 supplies one
// 16-byte chunk of its row:
//   * 16-bit: one v_mfma_f32_16x16x32 on 8 elements a lane;
//   * fp32: four v_mfma_f32_16x16x4, element i of every lane's chunk in the
//     i-th (k permuted alike in both operands);
//   * fp4: one v_mfma_scale_f32_16x16x128 on a whole block of 32 codes a lane
//     with that block's scale, applied inside the instruction.
// Operands are staged in LDS as they lie in memory, by global_load_lds:
//   * k-contiguous: [row][128 bytes], the eight chunks of a row at chunk ^
//     (row & 7);
//   * row-contiguous ("MC"): [k][row], read back k-first: 16-bit by the
//     transposing read ds_read_b64_tr_b16 (16 lanes read 4 k-rows of 16 rows,
//     each gets its row's 4 values), fp32 by four 4-byte reads. Chunks are
//     XORed by k so that the rows one read touches start in different banks.
#pragma once

#include "common.h"
#include "tile_order.h"

namespace wgb_ragged {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

// ---- element kinds -----------------------------------------------------------

struct F32 {
  typedef float store;
  typedef int chunk __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr int kBits = 32;
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int, int, int) {
    const f4 fa = __builtin_bit_cast(f4, a), fb = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
  }
};

struct F16 {
  typedef _Float16 store;
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef int chunk __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr int kBits = 16;
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int, int, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

struct Bf16 {
  typedef __bf16 store;
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef int chunk __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr int kBits = 16;
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int, int, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

// MXFP4: two codes a byte, a scale byte for 32 of them. sa / sb hold the
// scales of the lane's chunks of both steps, step s in byte s.
struct Fp4 {
  typedef uint8_t store;  // never stored: products come out in a wider type
  typedef v4i chunk;
  static constexpr int kBits = 4;
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int step, int sa, int sb) {
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    if (step == 0)
      c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
    else
      c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 1, sa, 1, sb);
  }
};

// ---- arguments -----------------------------------------------------------------

struct Args {
  int64_t m, n, k;  // ragged columns: n = all columns; ragged k: k = all of k
  const char *A, *B;
  int64_t lda, ldb;   // bytes between columns
  int64_t stride_a;   // bytes between the groups' A (ragged columns)
  const uint8_t *scale_a, *scale_b;  // fp4: one byte per chunk of codes, at ld / 16 bytes
  const int64_t *off;  // groups + 1 boundaries in device memory; null: one group of all columns
  int groups;
  int tiles_m, tiles_n;  // tiles_n: ragged k only
  void *C;
  int64_t ldc, stride_c;  // elements; stride_c: ragged k only
  float alpha, beta;
  int c_f32;  // C holds fp32 (else the operands' type; fp4: bf16, or f16 with c_f16)
  int c_f16;
};

constexpr int kTileBytes = 128;  // bytes of k in a k-tile

// ---- finding a tile --------------------------------------------------------------

struct Tile {
  int64_t lo, hi;  // the group's columns (ragged columns) or its part of k (ragged k)
  int g, tm, tn;
};

// Boundaries as the kernels use them: inside [0, n] and never decreasing
// within a group, whatever the array holds.
__device__ __forceinline__ void group_range(const int64_t *off, int g, int64_t n, int64_t &lo, int64_t &hi) {
  lo = off[g];
  hi = off[g + 1];
  lo = lo < 0 ? 0 : lo > n ? n : lo;
  hi = hi < lo ? lo : hi > n ? n : hi;
}

// Tile of block w of a ragged-columns launch: false if there is none.
// Column tiles are counted per group over the lanes of each wave.
__device__ __forceinline__ bool find_columns(const Args &p, int bn, int w, Tile &t) {
  const int lane = threadIdx.x & 63;
  if (!p.off) {
    const int tn = (int)((p.n + bn - 1) / bn);
    const int total = p.tiles_m * tn;
    if (w >= total) return false;
    t.g = 0;
    t.lo = 0;
    t.hi = p.n;
    wgb_tiles::logical_tile(wgb_tiles::xcd_remap(w, total), p.tiles_m, tn, 0, t.tm, t.tn);
    return true;
  }
  // column tiles of groups lane, lane + 64, ...: all of them, then this block's group
  int all = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 64) {
    int64_t lo = 0, hi = 0;
    if (g0 + lane < p.groups) group_range(p.off, g0 + lane, p.n, lo, hi);
    int c = (int)((hi - lo + bn - 1) / bn);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) c += __shfl_xor(c, d);
    all += c;
  }
  const int64_t total = (int64_t)all * p.tiles_m;
  if (w >= total) return false;
  const int L = wgb_tiles::xcd_remap(w, (int)total);
  const int q = L / p.tiles_m;  // the column tile, over all groups
  int before = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 64) {
    int64_t lo = 0, hi = 0;
    if (g0 + lane < p.groups) group_range(p.off, g0 + lane, p.n, lo, hi);
    const int c = (int)((hi - lo + bn - 1) / bn);
    int sum = c;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    const uint64_t past = __ballot(before + sum > q);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int first = before + __shfl(sum - c, at);
      const int tn = __shfl(c, at);
      t.g = __builtin_amdgcn_readfirstlane(g0 + at);
      group_range(p.off, t.g, p.n, t.lo, t.hi);
      wgb_tiles::logical_tile(L - first * p.tiles_m, p.tiles_m, tn, 0, t.tm, t.tn);
      t.tm = __builtin_amdgcn_readfirstlane(t.tm);
      t.tn = __builtin_amdgcn_readfirstlane(t.tn);
      return true;
    }
    before += __shfl(sum, 63);
  }
  return false;
}

__device__ __forceinline__ void find_k(const Args &p, int w, Tile &t) {
  const int per = p.tiles_m * p.tiles_n;
  const int L = wgb_tiles::xcd_remap(w, per * p.groups);
  t.g = L / per;
  wgb_tiles::logical_tile(L - t.g * per, p.tiles_m, p.tiles_n, 0, t.tm, t.tn);
  group_range(p.off, t.g, p.k, t.lo, t.hi);
}

// ---- staging ---------------------------------------------------------------------

// A wave's 64 x 16 bytes from its lanes' addresses to LDS at `lds` + 16 lane
// (4-byte form: + 4 lane).
typedef __attribute__((address_space(3))) void *LdsPtr;
__device__ __forceinline__ void copy16_to_lds(const void *g, void *lds) {
  __builtin_amdgcn_global_load_lds(g, (LdsPtr)lds, 16, 0, 0);
}
__device__ __forceinline__ void copy4_to_lds(const void *g, void *lds) {
  __builtin_amdgcn_global_load_lds(g, (LdsPtr)lds, 4, 0, 0);
}

// Chunk keys of the row-contiguous layout, for k-row r of a tile whose rows
// have `chunks` chunks: 16-bit transposing reads touch k-rows 8 g .. 8 g + 3
// (32 bytes of each), fp32 reads k-rows 4 g (64 bytes of each).
template <int BITS, int CHUNKS>
__device__ __forceinline__ int mc_key(int r) {
  const int key = BITS == 16 ? ((r & 3) << 1) | (((r >> 3) & 1) << 3) : ((r >> 2) & 3) << 2;
  return key & (CHUNKS - 1);
}

template <class E, int BT, bool MC, int NT>
struct Stager {
  static constexpr int EPC = 128 / E::kBits;             // elements in a 16-byte chunk
  static constexpr int BK = kTileBytes * 8 / E::kBits;   // elements of k in a k-tile
  static constexpr int BYTES = BT * kTileBytes;          // of a staged tile
  static constexpr int LOADS = BYTES / 16 / NT;          // chunks a thread stages
  static constexpr int CPR = MC ? BT / EPC : 8;          // chunks in a staged row
  static constexpr int RPS = NT / CPR;                   // staged rows in one step of all threads
  static_assert(BYTES % (16 * NT) == 0 && NT % CPR == 0, "whole steps");

  const char *origin;    // element (row0, k = 0)
  int64_t ld;            // bytes
  int64_t rows_left;     // rows from row0 to the end of the matrix
  int64_t K;             // elements
  uint32_t voff[LOADS];  // this lane's chunks of k-tile 0, in bytes from origin
  int t;

  __device__ __forceinline__ int slot_row(int r) const { return t / CPR + r * RPS; }
  __device__ __forceinline__ int slot_chunk(int r) const {
    const int row = slot_row(r);
    return (t % CPR) ^ (MC ? mc_key<E::kBits, CPR>(row) : (row & 7));
  }

  __device__ __forceinline__ void init(const char *P, int64_t ld_, int64_t row0, int64_t rows, int64_t K_, int t_) {
    t = t_;
    ld = ld_;
    rows_left = rows - row0;
    K = K_;
    origin = MC ? P + row0 * E::kBits / 8 : P + row0 * ld;
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      int row = slot_row(r), chunk = slot_chunk(r);
      // lanes past the matrix read its last row (last chunk of rows): what
      // they read only reaches elements of C that are never written
      if (MC) {
        const int64_t last = (rows_left - 1) / EPC;
        if (chunk > last) chunk = (int)last;
      } else if (row >= rows_left) {
        row = (int)(rows_left - 1);
      }
      voff[r] = (uint32_t)(row * ld + chunk * 16);
    }
  }

  // k-tiles whose copies stay inside the matrix: in the row-contiguous layout
  // a last chunk that the end of the rows cuts reads on into the next k-row,
  // which the last one does not have.
  __device__ __forceinline__ int whole_tiles() const {
    const bool cut = MC && rows_left < BT;
    return (int)((cut ? (K > 0 ? K - 1 : 0) : K) / BK);
  }

  // k-tile kt straight to LDS: the scalar origin and 32-bit lane offsets.
  __device__ __forceinline__ void copy(char *stage, int kt, int wave) const {
    const uint64_t o64 = (uint64_t)(origin + (MC ? (int64_t)kt * BK * ld : (int64_t)kt * kTileBytes));
    uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)o64);
    uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(o64 >> 32));
    asm volatile("" : "+s"(lo), "+s"(hi));
    const char *o = (const char *)(((uint64_t)hi << 32) | lo);
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      uint32_t v = voff[r];
      asm volatile("" : "+v"(v));
      copy16_to_lds(o + v, stage + wave * 1024 + r * NT * 16);
    }
  }

  // Chunk r of k-tile kt through registers: rows past the matrix and k past
  // K read as zeros, at any alignment of the elements.
  __device__ __forceinline__ v4i load_guarded(int kt, int r) const {
    typedef typename E::chunk v4u;  // 16 bytes at the elements' alignment
    const int row = slot_row(r), chunk = slot_chunk(r);
    int64_t left, at;
    bool in;
    if (MC) {
      const int64_t kk = (int64_t)kt * BK + row;
      in = kk < K;
      left = rows_left - (int64_t)chunk * EPC;
      at = kk * ld + chunk * 16;
    } else {
      const int64_t kk = (int64_t)kt * BK + (int64_t)chunk * EPC;
      in = row < rows_left;
      left = K - kk;
      at = row * ld + (int64_t)kt * kTileBytes + chunk * 16;
    }
    v4i v = {0, 0, 0, 0};
    if (in && left >= EPC) {
      v = *reinterpret_cast<const v4u *>(origin + at);
    } else if (in && left > 0) {
      // fp4 has no cut chunks: K is whole runs of 128 elements
      if constexpr (E::kBits == 16) {
        typedef short s8 __attribute__((ext_vector_type(8)));
        s8 s = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) s[i] = reinterpret_cast<const short *>(origin + at)[i];
        v = __builtin_bit_cast(v4i, s);
      } else if constexpr (E::kBits == 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < left) v[i] = reinterpret_cast<const int *>(origin + at)[i];
      }
    }
    return v;
  }

  __device__ __forceinline__ void put(char *stage, int r, const v4i &v) const {
    *reinterpret_cast<v4i *>(stage + t * 16 + r * NT * 16) = v;
  }

  // The MFMA operands of step s for MB blocks of 16 rows from row `wrow`.
  template <int MB>
  static __device__ __forceinline__ void fetch(const char *stage, int wrow, int s, int lane, v4i (&out)[MB]) {
    const int i16 = lane & 15, g = lane >> 4;
    if constexpr (!MC) {
      // fp4: a lane group's two chunks are neighbours, so that one 2-byte
      // read has both scales
      const int chunk = (E::kBits == 4 ? 2 * g + s : 4 * s + g) ^ (i16 & 7);
#pragma unroll
      for (int b = 0; b < MB; ++b)
        out[b] = *reinterpret_cast<const v4i *>(stage + (wrow + 16 * b + i16) * kTileBytes + chunk * 16);
    } else if constexpr (E::kBits == 16) {
      typedef __attribute__((address_space(3))) s4 *LdsS4;
      constexpr int RB = BT * 2;
      // the 16 lanes of a group read k-rows kr .. kr + 3, four lanes a row
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        s4 h[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int kr = 32 * s + 8 * g + 4 * q + (i16 >> 2);
          const int at = (wrow + 16 * b) * 2 + (i16 & 3) * 8;
          h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LdsS4)(stage + kr * RB + (((at >> 4) ^ mc_key<16, CPR>(kr)) << 4) + (at & 15)));
        }
        typedef short s8 __attribute__((ext_vector_type(8)));
        const s8 w = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
        out[b] = __builtin_bit_cast(v4i, w);
      }
    } else {
      constexpr int RB = BT * 4;
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kr = 16 * s + 4 * g + i;
          const int at = (wrow + 16 * b + i16) * 4;
          out[b][i] = *reinterpret_cast<const int *>(stage + kr * RB + (((at >> 4) ^ mc_key<32, CPR>(kr)) << 4) + (at & 15));
        }
    }
  }
};

// The scales of a k-tile: 8 bytes a row, A's rows then B's, copied 4 bytes a
// lane. The waves share the copies evenly (a wave past the last one copies
// the last again, the same bytes to the same place), so that every wave has
// as many copies in flight.
template <int BM, int BN, int NW>
struct ScaleStager {
  static constexpr int BYTES = (BM + BN) * 8;
  static constexpr int COPIES = BYTES / 256;
  static constexpr int LOADS = (COPIES + NW - 1) / NW;
  static_assert(BYTES % 256 == 0 && BM % 32 == 0, "whole copies");

  const uint8_t *src[LOADS];
  int at[LOADS];
  int half;
  int64_t blocks;  // of 32 elements, in a row

  __device__ __forceinline__ void init(const uint8_t *sa, int64_t lda, int64_t m_left, const uint8_t *sb, int64_t ldb,
                                       int64_t n_left, int64_t K, int wave, int lane) {
    blocks = K / 32;
    half = lane & 1;
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      int c = wave + r * NW;
      if (c >= COPIES) c = COPIES - 1;
      at[r] = c * 256;
      int row = c * 32 + (lane >> 1);
      const bool b = c * 32 >= BM;
      if (b) row -= BM;
      const int64_t left = b ? n_left : m_left;
      if (row >= left) row = (int)(left - 1);
      src[r] = (b ? sb + row * ldb : sa + row * lda) + 4 * half;
    }
  }
  __device__ __forceinline__ void copy(char *stage, int kt) const {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) copy4_to_lds(src[r] + (int64_t)kt * 8, stage + at[r]);
  }
  // The last k-tile when it is half a tile: its second half counts as zeros.
  __device__ __forceinline__ void put_guarded(char *stage, int kt, int lane) const {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      int v = 0;
      if ((int64_t)kt * 8 + 4 * half < blocks) v = *reinterpret_cast<const int *>(src[r] + (int64_t)kt * 8);
      *reinterpret_cast<int *>(stage + at[r] + 4 * lane) = v;
    }
  }
  // Both steps' scales of this lane's rows.
  template <int MB>
  static __device__ __forceinline__ void fetch(const char *stage, int row, int lane, int (&out)[MB]) {
#pragma unroll
    for (int b = 0; b < MB; ++b)
      out[b] = *reinterpret_cast<const uint16_t *>(stage + (row + 16 * b + (lane & 15)) * 8 + (lane >> 4) * 2);
  }
};

// ---- the tile ----------------------------------------------------------------------

// s_waitcnt: at most n vector-memory operations in flight, LDS done.
constexpr int waitcnt_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4); }

template <int VM>
__device__ __forceinline__ void wait_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(VM));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <typename T>
__device__ __forceinline__ T to(float x) {
  return (T)x;
}

// alpha acc + beta C for a lane's runs of four rows of one column.
template <typename T, int MB, int NB>
__device__ __forceinline__ void epilogue(const Args &p, T *C, const f4 (&acc)[MB][NB], int64_t row0, int64_t rows,
                                         int64_t col0, int64_t cols, int lane) {
  typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const int i16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t col = col0 + 16 * j + i16;
    if (col >= cols) continue;
    T *cp = C + col * p.ldc;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int64_t row = row0 + 16 * i + 4 * g;
      f4 x = acc[i][j];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] *= p.alpha;
      if (row + 4 <= rows) {
        if (p.beta != 0.0f) {
          const V4 c = *reinterpret_cast<const V4 *>(cp + row);
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = fmaf(p.beta, (float)c[q], x[q]);
        }
        V4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = to<T>(x[q]);
        *reinterpret_cast<V4 *>(cp + row) = v;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (row + q < rows) {
            if (p.beta != 0.0f) x[q] = fmaf(p.beta, (float)cp[row + q], x[q]);
            cp[row + q] = to<T>(x[q]);
          }
      }
    }
  }
}

// One BM x BN tile of C a block, WM x WN waves. AMC / BMC: the operand is
// row-contiguous in memory. VEC: both operands can be copied by 16-byte
// (4-byte aligned) loads at 32-bit offsets; otherwise every k-tile goes
// through registers. RK: ragged k. S: stages of LDS.
template <class E, int BM, int BN, int WM, int WN, bool AMC, bool BMC, bool VEC, bool RK, int S>
struct Kernel {
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
  static constexpr bool kScaled = E::kBits == 4;
  typedef Stager<E, BM, AMC, NT> SA;
  typedef Stager<E, BN, BMC, NT> SB;
  typedef ScaleStager<kScaled ? BM : 32, kScaled ? BN : 32, NW> SS;
  static constexpr int SCALES = kScaled ? SS::BYTES : 0;
  static constexpr int STAGE = SA::BYTES + SB::BYTES + SCALES;
  static constexpr int LDS = S * STAGE;
  // vector-memory operations of one k-tile's copies, of one wave
  static constexpr int PER_TILE = SA::LOADS + SB::LOADS + (kScaled ? SS::LOADS : 0);

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    Tile tile;
    if constexpr (RK)
      find_k(p, blockIdx.x, tile);
    else if (!find_columns(p, BN, blockIdx.x, tile))
      return;
    const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
    const int64_t cols = RK ? p.n : tile.hi - tile.lo;
    int64_t K = RK ? tile.hi - tile.lo : p.k;
    if (p.alpha == 0.0f) K = 0;  // reads neither operand
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);

    f4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    const int nt = (int)((K + SA::BK - 1) / SA::BK);
    if (nt > 0) {
      SA sa;
      SB sb;
      SS ss;
      const char *A = RK ? p.A + tile.lo * p.lda : p.A + (int64_t)tile.g * p.stride_a;
      const char *B = RK ? p.B + tile.lo * p.ldb : p.B + tile.lo * p.ldb;
      sa.init(A, p.lda, m0, p.m, K, t);
      sb.init(B, p.ldb, n0, cols, K, t);
      if constexpr (kScaled) {
        const int64_t lsa = p.lda / 16, lsb = p.ldb / 16;
        ss.init(p.scale_a + (int64_t)tile.g * (p.stride_a / 16) + m0 * lsa, lsa, p.m - m0,
                p.scale_b + (tile.lo + n0) * lsb, lsb, cols - n0, K, wave, lane);
      }
      int whole = 0;
      if constexpr (VEC) {
        whole = sa.whole_tiles();
        const int wb = sb.whole_tiles();
        whole = whole < wb ? whole : wb;
      }

      auto guarded = [&](int kt) {
        char *st = smem + (kt % S) * STAGE;
#pragma unroll
        for (int r = 0; r < SA::LOADS; ++r) sa.put(st, r, sa.load_guarded(kt, r));
#pragma unroll
        for (int r = 0; r < SB::LOADS; ++r) sb.put(st + SA::BYTES, r, sb.load_guarded(kt, r));
        if constexpr (kScaled) ss.put_guarded(st + SA::BYTES + SB::BYTES, kt, lane);
      };
      auto copy = [&](int kt) {
        char *st = smem + (kt % S) * STAGE;
        sa.copy(st, kt, wave);
        sb.copy(st + SA::BYTES, kt, wave);
        if constexpr (kScaled) ss.copy(st + SA::BYTES + SB::BYTES, kt);
      };
      auto fill = [&](int kt) {
        if (VEC && kt < whole)
          copy(kt);
        else
          guarded(kt);
      };
      auto fetch = [&](int kt, int s, v4i (&a)[MB], v4i (&b)[NB]) {
        const char *st = smem + (kt % S) * STAGE;
        SA::template fetch<MB>(st, wm, s, lane, a);
        SB::template fetch<NB>(st + SA::BYTES, wn, s, lane, b);
      };
      auto fetch_scales = [&](int kt, int (&a)[MB], int (&b)[NB]) {
        if constexpr (kScaled) {
          const char *st = smem + (kt % S) * STAGE + SA::BYTES + SB::BYTES;
          SS::template fetch<MB>(st, wm, lane, a);
          SS::template fetch<NB>(st, BM + wn, lane, b);
        }
      };
      auto mma = [&](int s, const v4i (&a)[MB], const v4i (&b)[NB], const int (&qa)[MB], const int (&qb)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < MB; ++i) E::mma(a[i], b[j], acc[i][j], s, qa[i], qb[j]);
      };

      // Tile kt is read from stage kt % S while the copies of the next S - 1
      // are in flight or landed; its stage takes tile kt + S after the
      // barrier that ends its reads.
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < nt) fill(i);
      wait_barrier<0>();
      v4i xa[MB], xb[NB], ya[MB], yb[NB];
      int qa[MB] = {}, qb[NB] = {};
      fetch(0, 0, xa, xb);
      fetch_scales(0, qa, qb);
      int kt = 0;
      // steady: tile kt + S exists and is whole, so are those before it
      const int steady = (whole < nt ? whole : nt) - S;
      for (; kt < steady; ++kt) {
        fetch(kt, 1, ya, yb);
        mma(0, xa, xb, qa, qb);
        wait_barrier<(S - 2) * PER_TILE>();
        copy(kt + S);
        fetch(kt + 1, 0, xa, xb);
        mma(1, ya, yb, qa, qb);
        fetch_scales(kt + 1, qa, qb);
      }
      for (; kt < nt; ++kt) {
        fetch(kt, 1, ya, yb);
        mma(0, xa, xb, qa, qb);
        wait_barrier<0>();
        if (kt + S < nt) fill(kt + S);
        if (kt + 1 < nt) fetch(kt + 1, 0, xa, xb);
        mma(1, ya, yb, qa, qb);
        if (kt + 1 < nt) fetch_scales(kt + 1, qa, qb);
      }
    }

    const int64_t at = RK ? (int64_t)tile.g * p.stride_c : tile.lo * p.ldc;
    if constexpr (E::kBits == 32) {
      epilogue<float, MB, NB>(p, (float *)p.C + at, acc, m0 + wm, p.m, n0 + wn, cols, lane);
    } else if (p.c_f32) {
      epilogue<float, MB, NB>(p, (float *)p.C + at, acc, m0 + wm, p.m, n0 + wn, cols, lane);
    } else if constexpr (E::kBits == 4) {
      if (p.c_f16)
        epilogue<_Float16, MB, NB>(p, (_Float16 *)p.C + at, acc, m0 + wm, p.m, n0 + wn, cols, lane);
      else
        epilogue<__bf16, MB, NB>(p, (__bf16 *)p.C + at, acc, m0 + wm, p.m, n0 + wn, cols, lane);
    } else {
      epilogue<typename E::store, MB, NB>(p, (typename E::store *)p.C + at, acc, m0 + wm, p.m, n0 + wn, cols, lane);
    }
  }
};

template <class K>
__global__ __launch_bounds__(K::NT, 2) void ragged_kernel(Args p) {
  extern __shared__ __align__(1024) char ragged_smem[];
  K::run(p, ragged_smem);
}

// Blocks that a ragged-columns launch needs at most: a group of c columns has
// ceil(c / bn) column tiles, at most one of them partly filled.
inline int64_t column_tiles(const Args &p, int bn) {
  if (!p.off) return (p.n + bn - 1) / bn;
  return p.n / bn + (p.n < p.groups ? p.n : p.groups);
}

template <class K>
int launch(wgb_ctx *ctx, const Args &p, int64_t blocks) {
  if (blocks == 0) return WGB_OK;
  if (blocks > INT32_MAX) return wgb::fail(WGB_ERR_INVALID_VALUE, "grouped product: too many tiles");
  static const hipError_t attr =
      hipFuncSetAttribute((const void *)ragged_kernel<K>, hipFuncAttributeMaxDynamicSharedMemorySize, K::LDS);
  if (attr != hipSuccess) return wgb::fail_hip(attr, "LDS size of a grouped product");
  ragged_kernel<K><<<(unsigned)blocks, K::NT, K::LDS, ctx->stream>>>(p);
  WGB_CHECK_LAUNCH("ragged_kernel");
  return WGB_OK;
}

}  // namespace wgb_ragged
