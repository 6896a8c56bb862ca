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

#include <type_traits>

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
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int, int, int, int, int) {
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
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int, int, int, int, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

struct Bf16 {
  typedef __bf16 store;
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef int chunk __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr int kBits = 16;
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int, int, int, int, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

// MXFP4: two codes a byte, a scale byte for 32 of them. sa / sb hold the
// scales of the lane's chunks of two row blocks and both steps: block parity
// p, step s in byte 2 p + s.
struct Fp4 {
  typedef uint8_t store;  // never stored: products come out in a wider type
  typedef v4i chunk;
  static constexpr int kBits = 4;
  template <int SA, int SB>
  static __device__ __forceinline__ void scaled(const v4i &a, const v4i &b, f4 &c, int sa, int sb) {
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, SA, sa, SB, sb);
  }
  template <int SA>
  static __device__ __forceinline__ void scaled_b(const v4i &a, const v4i &b, f4 &c, int sa, int sb, int at) {
    if (at == 0)
      scaled<SA, 0>(a, b, c, sa, sb);
    else if (at == 1)
      scaled<SA, 1>(a, b, c, sa, sb);
    else if (at == 2)
      scaled<SA, 2>(a, b, c, sa, sb);
    else
      scaled<SA, 3>(a, b, c, sa, sb);
  }
  // step, block_a, block_b: known when the caller's loops are unrolled
  static __device__ __forceinline__ void mma(const v4i &a, const v4i &b, f4 &c, int step, int block_a, int sa, int block_b,
                                             int sb) {
    const int at_a = 2 * (block_a & 1) + step, at_b = 2 * (block_b & 1) + step;
    if (at_a == 0)
      scaled_b<0>(a, b, c, sa, sb, at_b);
    else if (at_a == 1)
      scaled_b<1>(a, b, c, sa, sb, at_b);
    else if (at_a == 2)
      scaled_b<2>(a, b, c, sa, sb, at_b);
    else
      scaled_b<3>(a, b, c, sa, sb, at_b);
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

// ---- finding a tile --------------------------------------------------------------

struct Tile {
  int64_t lo, hi;  // the group's columns (ragged columns) or its part of k (ragged k)
  int g, tm, tn;
};

// Boundaries as the kernels use them: inside [0, n] and never decreasing
// within a group, whatever the array holds.
__device__ __forceinline__ void clamp_range(int64_t n, int64_t &lo, int64_t &hi) {
  lo = lo < 0 ? 0 : lo > n ? n : lo;
  hi = hi < lo ? lo : hi > n ? n : hi;
}
__device__ __forceinline__ void group_range(const int64_t *off, int g, int64_t n, int64_t &lo, int64_t &hi) {
  lo = off[g];
  hi = off[g + 1];
  clamp_range(n, lo, hi);
}

// The tiles of a ragged-columns launch in order: first the groups' whole
// column tiles, one group after the other, each in bands (tile_order.h), then
// the tiles of the columns that are left over in each group, which cost less
// and even out the end. Either part is dealt to the XCDs in runs. Column tiles
// are counted over the lanes of each wave; up to 64 groups, one a lane, stay
// in registers.
struct ColumnFinder {
  int whole, total;      // tiles: of whole columns, all
  int bn;
  int lo, hi;            // lane's group: its columns (below 2^31),
  int sum, rest;         // whole column tiles, and leftovers, up to and with it

  // Groups g0 .. g0 + 63 into the lanes; before, rest_before: counts of the groups before them.
  __device__ __forceinline__ void scan(const Args &p, int g0, int before, int rest_before) {
    const int lane = threadIdx.x & 63;
    int64_t l = 0, h = 0;
    if (g0 + lane < p.groups) group_range(p.off, g0 + lane, p.n, l, h);
    lo = (int)l;
    hi = (int)h;
    sum = (hi - lo) / bn;
    rest = (hi - lo) % bn != 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d), rup = __shfl_up(rest, d);
      if (lane >= d) {
        sum += up;
        rest += rup;
      }
    }
    sum += before;
    rest += rest_before;
  }

  __device__ __forceinline__ void init(const Args &p, int bn_) {
    bn = bn_;
    if (!p.off) {
      whole = p.tiles_m * (int)(p.n / bn);
      total = p.tiles_m * (int)((p.n + bn - 1) / bn);
      return;
    }
    int all = 0, left = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
      scan(p, g0, all, left);
      all = __builtin_amdgcn_readlane(sum, 63);
      left = __builtin_amdgcn_readlane(rest, 63);
    }
    whole = all * p.tiles_m;
    total = whole + left * p.tiles_m;
  }

  // Tile w: false if there is none.
  __device__ __forceinline__ bool find(const Args &p, int w, Tile &t) {
    if (w >= total) return false;
    const bool left = w >= whole;
    const int L = left ? wgb_tiles::xcd_remap(w - whole, total - whole) : wgb_tiles::xcd_remap(w, whole);
    const int q = L / p.tiles_m;  // the column tile of its kind, over all groups
    int g0 = 0;
    uint64_t past = 1;
    if (!p.off) {
      t.g = 0;
      t.lo = 0;
      t.hi = p.n;
    } else {
      int before = 0, rest_before = 0;
      for (;; g0 += 64) {
        if (p.groups > 64) scan(p, g0, before, rest_before);
        past = __ballot((left ? rest : sum) > q);
        if (past || g0 + 64 >= p.groups) break;
        before = __builtin_amdgcn_readlane(sum, 63);
        rest_before = __builtin_amdgcn_readlane(rest, 63);
      }
      if (!past) return false;
    }
    const int at = __builtin_ctzll(past);
    if (p.off) {
      t.g = g0 + at;
      t.lo = __builtin_amdgcn_readlane(lo, at);
      t.hi = __builtin_amdgcn_readlane(hi, at);
    }
    const int tn = (int)(t.hi - t.lo) / bn;
    if (left) {
      t.tm = L - q * p.tiles_m;
      t.tn = tn;
    } else {
      const int first = p.off ? __builtin_amdgcn_readlane(sum, at) - tn : 0;
      wgb_tiles::logical_tile(L - first * p.tiles_m, p.tiles_m, tn, 0, t.tm, t.tn);
    }
    return true;
  }
};

// The tiles of a ragged-k launch: the groups from the longest to the shortest
// (up to 64 of them, one a lane; more stay in their order), the rounds of a
// persistent launch to and fro, so that blocks come out even; each group's
// tiles are dealt to all XCDs.
struct KFinder {
  int total, per;
  int lo, hi, rank;  // lane's group: its part of k (below 2^31), its place

  __device__ __forceinline__ void init(const Args &p, int) {
    per = p.tiles_m * p.tiles_n;
    total = per * p.groups;
    if (p.groups > 64) return;
    const int lane = threadIdx.x & 63;
    int64_t l = 0, h = 0;
    if (lane < p.groups) group_range(p.off, lane, p.k, l, h);
    lo = (int)l;
    hi = (int)h;
    rank = 0;
    const int size = hi - lo;
    for (int g = 0; g < p.groups; ++g) {
      const int other = __builtin_amdgcn_readlane(size, g);
      rank += other > size || (other == size && g < lane);
    }
    if (lane >= p.groups) rank = -1;
  }
  __device__ __forceinline__ bool find(const Args &p, int w, Tile &t) {
    if (w >= total) return false;
    const int round = w / (int)gridDim.x, begin = round * (int)gridDim.x;
    const int end = begin + (int)gridDim.x < total ? begin + (int)gridDim.x : total;
    const int at = round & 1 ? begin + end - 1 - w : w;
    const int place = at / per;
    wgb_tiles::logical_tile(wgb_tiles::xcd_remap(at - place * per, per), p.tiles_m, p.tiles_n, 0, t.tm, t.tn);
    if (p.groups <= 64) {
      t.g = __builtin_ctzll(__ballot(rank == place));
      t.lo = __builtin_amdgcn_readlane(lo, t.g);
      t.hi = __builtin_amdgcn_readlane(hi, t.g);
      return true;
    }
    t.g = place;
    // scalar loads: they do not wait for the copies in flight
    typedef const __attribute__((address_space(4))) int64_t *Constant;
    const Constant off = (Constant)(uintptr_t)p.off;
    t.lo = off[t.g];
    t.hi = off[t.g + 1];
    clamp_range(p.k, t.lo, t.hi);
    return true;
  }
};

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

// A wave's chunks at `from` (scalar) + `at` (32 bits a lane): the empty asm
// statements keep the compiler from making them per-lane 64-bit pointers.
__device__ __forceinline__ const char *scalar_at(const char *from, uint32_t at) {
  const uint64_t o64 = (uint64_t)from;
  uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)o64);
  uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(o64 >> 32));
  asm volatile("" : "+s"(lo), "+s"(hi));
  asm volatile("" : "+v"(at));
  return (const char *)(((uint64_t)hi << 32) | lo) + at;
}
__device__ __forceinline__ void copy_chunks(const char *from, uint32_t at, char *lds) {
  copy16_to_lds(scalar_at(from, at), lds);
}

// Chunk keys of the row-contiguous layout, for k-row r of a tile whose rows
// have `chunks` chunks: 16-bit transposing reads touch k-rows 8 g .. 8 g + 3
// (32 bytes of each), fp32 reads k-rows 4 g (64 bytes of each).
template <int BITS, int CHUNKS>
__device__ __forceinline__ int mc_key(int r) {
  const int key = BITS == 16 ? ((r & 3) << 1) | (((r >> 3) & 1) << 3) : ((r >> 2) & 3) << 2;
  return key & (CHUNKS - 1);
}

// k-tiles are 128 bytes of k: a whole cache line of every row. (Of 64 bytes,
// each line came from L2 twice, once for either half: 8192 x 16384 x 4096 in
// bf16 886 us, of which 180 were the copies'.)
constexpr int TB = 128;

template <int LOADS>
struct StagerData {
  const char *origin;    // element (row0, k = 0)
  int64_t ld;            // bytes
  int64_t rows_left;     // rows from row0 to the end of the matrix
  int64_t K;             // elements
  uint32_t voff[LOADS];  // this lane's chunks of k-tile 0, in bytes from origin
  int t;
};

template <class E, int BT, bool MC, int NT>
struct Stager : StagerData<BT * TB / 16 / NT> {
  static constexpr int EPC = 128 / E::kBits;         // elements in a 16-byte chunk
  static constexpr int BK = TB * 8 / E::kBits;       // elements of k in a k-tile
  static constexpr int BYTES = BT * TB;              // of a staged tile
  static constexpr int LOADS = BYTES / 16 / NT;      // chunks a thread stages
  static constexpr int CPR = MC ? BT / EPC : TB / 16;  // chunks in a staged row
  static constexpr int RPS = NT / CPR;               // staged rows in one step of all threads
  static_assert(BYTES % (16 * NT) == 0 && NT % CPR == 0, "whole steps");

  typedef StagerData<LOADS> Data;
  using Data::origin;
  using Data::ld;
  using Data::rows_left;
  using Data::K;
  using Data::voff;
  using Data::t;

  __device__ __forceinline__ int slot_row(int r) const { return t / CPR + r * RPS; }
  __device__ __forceinline__ int slot_chunk(int r) const {
    const int row = slot_row(r);
    return (t % CPR) ^ (MC ? mc_key<E::kBits, CPR>(row) : row & 7);
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

  // Bytes from one k-tile to the next.
  __device__ __forceinline__ int64_t step() const { return MC ? BK * ld : TB; }

  // k-tile kt.
  __device__ __forceinline__ void copy(char *stage, int kt, int wave) const {
    const char *from = origin + (int64_t)kt * step();
#pragma unroll
    for (int r = 0; r < LOADS; ++r) copy_chunks(from, voff[r], stage + wave * 1024 + r * NT * 16);
  }

  // fp4, a last k-tile of which only the first 64 bytes exist: the other four
  // chunks of a row read those again. What they hold does not matter (a code
  // is never Inf or NaN), for their scales are staged as 2^-127 in both
  // operands, and 36 * 2^-254 is nothing in fp32.
  __device__ __forceinline__ uint32_t half_voff(int r) const {
    return voff[r] - (slot_chunk(r) >= 4 ? 64u : 0u);
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
      at = row * ld + (int64_t)kt * TB + chunk * 16;
    }
    v4i v = {0, 0, 0, 0};
    if (in && left >= EPC) {
      v = *reinterpret_cast<const v4u *>(origin + at);
    } else if (in && left > 0) {
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

  // The MFMA operands of step s for MB blocks of 16 rows, `STEP` rows apart,
  // from row `wrow`; only the first `used` blocks.
  template <int MB, int STEP = 16>
  static __device__ __forceinline__ void fetch(const char *stage, int wrow, int s, int lane, v4i (&out)[MB],
                                               int used = MB) {
    const int i16 = lane & 15, g = lane >> 4;
    if constexpr (!MC) {
      // fp4: a lane group's two chunks are neighbours, so that
      // one 2-byte read has both scales
      const int chunk = (E::kBits == 4 ? 2 * g + s : 4 * s + g) ^ (i16 & 7);
#pragma unroll
      for (int b = 0; b < MB; ++b)
        if (b == 0 || __builtin_expect(b < used, 1))
          out[b] = *reinterpret_cast<const v4i *>(stage + (wrow + STEP * b + i16) * TB + chunk * 16);
    } else if constexpr (E::kBits == 16) {
      typedef __attribute__((address_space(3))) s4 *LdsS4;
      constexpr int RB = BT * 2;
      // the 16 lanes of a group read k-rows kr .. kr + 3, four lanes a row;
      // the key is the lane's own in every read, so a block's address is the
      // first one's with its bits changed (blocks do not carry into the wave's
      // first row)
      const int kr = 8 * g + (i16 >> 2);
      int at = kr * RB + ((wrow * 2 + (i16 & 3) * 8) ^ (mc_key<16, CPR>(kr) << 4));
      asm volatile("" : "+v"(at));  // one register, not one for every block
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        if (b > 0 && __builtin_expect(b >= used, 0)) break;
        s4 h[2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
          h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LdsS4)(stage + (at ^ (STEP * b * 2)) + (32 * s + 4 * q) * RB));
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
          const int at = (wrow + STEP * b + i16) * 4;
          out[b][i] = *reinterpret_cast<const int *>(stage + kr * RB + (((at >> 4) ^ mc_key<32, CPR>(kr)) << 4) + (at & 15));
        }
    }
  }
};

// The scales of a k-tile: 8 bytes a row, A's rows then B's, copied 4
// bytes a lane. The waves share the copies evenly (a wave past the last one
// copies the last again, the same bytes to the same place), so that every
// wave has as many copies in flight.
template <int BM, int BN, int NW>
struct ScaleStager {
  static constexpr int RB = TB / 16;        // bytes of a row
  static constexpr int WORDS = RB / 4;     // lanes of a row
  static constexpr int ROWS = 64 / WORDS;   // rows of a copy
  static constexpr int BYTES = (BM + BN) * RB;
  static constexpr int COPIES = BYTES / 256;
  static constexpr int LOADS = (COPIES + NW - 1) / NW;
  static_assert(BM % ROWS == 0 && BN % ROWS == 0, "whole copies");

  const uint8_t *src[LOADS];  // scalar: the copy's first row
  uint32_t voff[LOADS];       // this lane's dword
  int at[LOADS];
  int word;
  int64_t blocks;  // of 32 elements, in a row

  __device__ __forceinline__ void init(const uint8_t *sa, int64_t lda, int64_t m_left, const uint8_t *sb, int64_t ldb,
                                       int64_t n_left, int64_t K, int wave, int lane) {
    blocks = K / 32;
    word = lane % WORDS;
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      int c = wave + r * NW;
      if (c >= COPIES) c = COPIES - 1;
      at[r] = c * 256;
      const bool b = c * ROWS >= BM;
      int row = c * ROWS - (b ? BM : 0) + lane / WORDS;
      const int64_t left = b ? n_left : m_left, ld = b ? ldb : lda;
      if (row >= left) row = (int)(left - 1);
      src[r] = b ? sb : sa;
      voff[r] = (uint32_t)(row * ld + 4 * word);
    }
  }
  __device__ __forceinline__ void copy_part(char *stage, int kt, int r) const {
    copy4_to_lds(scalar_at((const char *)src[r] + (int64_t)kt * RB, voff[r]), stage + at[r]);
  }
  __device__ __forceinline__ void copy(char *stage, int kt) const {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) copy_part(stage, kt, r);
  }
  // The last k-tile when it is half a tile: its second half counts as zeros.
  __device__ __forceinline__ void put_guarded(char *stage, int kt, int lane) const {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      int v = 0;
      if ((int64_t)kt * RB + 4 * word < blocks) v = *reinterpret_cast<const int *>(src[r] + (int64_t)kt * RB + voff[r]);
      *reinterpret_cast<int *>(stage + at[r] + 4 * lane) = v;
    }
  }
  // Both steps' scales of this lane's rows, two row blocks to a register (Fp4::mma).
  template <int MB, int STEP = 16>
  static __device__ __forceinline__ void fetch(const char *stage, int row, int lane, int (&out)[(MB + 1) / 2], int used = MB) {
    // lanes share dwords; a lane group's two bytes are the low or the high half
    const char *at = stage + (row + (lane & 15)) * RB + (lane >> 5) * 4;
    const uint32_t half = ((lane >> 4) & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int b = 0; b < MB; b += 2)
      if (b == 0 || __builtin_expect(b < used, 1)) {
        const uint32_t lo = *reinterpret_cast<const uint32_t *>(at + STEP * b * RB);
        const uint32_t hi = b + 1 < MB ? *reinterpret_cast<const uint32_t *>(at + STEP * (b + 1) * RB) : 0u;
        out[b / 2] = (int)__builtin_amdgcn_perm(hi, lo, half);
      }
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

// Two 16x16 blocks' values of a column in two dwords each (four rows a lane:
// rows 4 g .. 4 g + 3) exchanged between lane groups, so that a lane has eight
// rows of one block: block i + (g & 1), rows 8 (g >> 1) .. + 7.
__device__ __forceinline__ v4i eight_rows(uint32_t x0, uint32_t x1, uint32_t y0, uint32_t y1) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(x0, y0, false, false));
  const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(x1, y1, false, false));
  return v4i{(int)a[0], (int)b[0], (int)a[1], (int)b[1]};
}

// alpha acc + beta C for a lane's runs of four rows of one column; column
// blocks are STEP columns apart. fp32 is stored in those runs (16 bytes a
// lane), 16-bit values in runs of eight rows (also 16 bytes) where there are
// two row blocks: with 8 bytes a lane 8192 x 16384 x 4096 took 788 us.
template <typename T, int MB, int NB, int STEP>
__device__ __forceinline__ void epilogue(const Args &p, T *C, const f4 (&acc)[MB][NB], int64_t row0, int64_t rows,
                                         int64_t col0, int64_t cols, int lane) {
  typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  constexpr bool PAIRS = sizeof(T) == 2 && MB % 2 == 0;
  const int i16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t col = col0 + STEP * j + i16;
    if (col >= cols) continue;
    T *cp = C + col * p.ldc;
    // a lane's four rows of row block i
    auto value = [&](int i) {
      const int64_t row = row0 + 16 * i + 4 * g;
      f4 x = acc[i][j];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] *= p.alpha;
      if (p.beta != 0.0f) {
        if (row + 4 <= rows) {
          const V4 c = *reinterpret_cast<const V4 *>(cp + row);
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = fmaf(p.beta, (float)c[q], x[q]);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (row + q < rows) x[q] = fmaf(p.beta, (float)cp[row + q], x[q]);
        }
      }
      V4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = (T)x[q];
      return v;
    };
    if constexpr (PAIRS) {
      typedef T V8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < MB; i += 2) {
        const u2 x = __builtin_bit_cast(u2, value(i)), y = __builtin_bit_cast(u2, value(i + 1));
        const V8 v = __builtin_bit_cast(V8, eight_rows(x[0], x[1], y[0], y[1]));
        const int64_t row = row0 + 16 * (i + (g & 1)) + 8 * (g >> 1);
        if (row + 8 <= rows) {
          *reinterpret_cast<V8 *>(cp + row) = v;
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (row + q < rows) cp[row + q] = v[q];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const V4 v = value(i);
        const int64_t row = row0 + 16 * i + 4 * g;
        if (row + 4 <= rows) {
          *reinterpret_cast<V4 *>(cp + row) = v;
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (row + q < rows) cp[row + q] = v[q];
        }
      }
    }
  }
}

// The epilogue in C's type; `at`: element of C where the group's part starts.
template <class E, int STEP, int MB, int NB>
__device__ __forceinline__ void store_tile(const Args &p, int64_t at, const f4 (&acc)[MB][NB], int64_t row0, int64_t col0,
                                           int64_t cols, int lane) {
  if (E::kBits == 32 || p.c_f32) {
    epilogue<float, MB, NB, STEP>(p, (float *)p.C + at, acc, row0, p.m, col0, cols, lane);
  } else if constexpr (E::kBits == 4) {
    if (p.c_f16)
      epilogue<_Float16, MB, NB, STEP>(p, (_Float16 *)p.C + at, acc, row0, p.m, col0, cols, lane);
    else
      epilogue<__bf16, MB, NB, STEP>(p, (__bf16 *)p.C + at, acc, row0, p.m, col0, cols, lane);
  } else if constexpr (E::kBits == 16) {
    epilogue<typename E::store, MB, NB, STEP>(p, (typename E::store *)p.C + at, acc, row0, p.m, col0, cols, lane);
  }
}

// One BM x BN tile of C a block, WM x WN waves. AMC / BMC: the operand is
// row-contiguous in memory. VEC: both operands can be copied by 16-byte
// (4-byte aligned) loads at 32-bit offsets; otherwise every k-tile goes
// through registers. RK: ragged k. S: stages of LDS.
template <class E, int BM, int BN, int WM, int WN, bool AMC, bool BMC, bool VEC, bool RK, int S>
struct Kernel {
  static constexpr int kBM = BM, kBN = BN;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
  static constexpr bool kScaled = E::kBits == 4;
  static constexpr bool kPersistent = false;  // a block a tile
  typedef Stager<E, BM, AMC, NT> SA;
  typedef Stager<E, BN, BMC, NT> SB;
  typedef ScaleStager<kScaled ? BM : 64, kScaled ? BN : 64, NW> SS;
  static constexpr int SCALES = kScaled ? SS::BYTES : 0;
  static constexpr int STAGE = SA::BYTES + SB::BYTES + SCALES;
  static constexpr int LDS = S * STAGE;
  // vector-memory operations of one k-tile's copies, of one wave
  static constexpr int PER_TILE = SA::LOADS + SB::LOADS + (kScaled ? SS::LOADS : 0);

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    Tile tile;
    typename std::conditional<RK, KFinder, ColumnFinder>::type finder;
    finder.init(p, BN);
    if (!finder.find(p, blockIdx.x, tile)) return;
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
        if constexpr (kScaled) {
          const int64_t at = (int64_t)kt * TB;
#pragma unroll
          for (int r = 0; r < SA::LOADS; ++r)
            copy_chunks(sa.origin + at, sa.half_voff(r), st + wave * 1024 + r * NT * 16);
#pragma unroll
          for (int r = 0; r < SB::LOADS; ++r)
            copy_chunks(sb.origin + at, sb.half_voff(r), st + SA::BYTES + wave * 1024 + r * NT * 16);
        } else {
#pragma unroll
          for (int r = 0; r < SA::LOADS; ++r) sa.put(st, r, sa.load_guarded(kt, r));
#pragma unroll
          for (int r = 0; r < SB::LOADS; ++r) sb.put(st + SA::BYTES, r, sb.load_guarded(kt, r));
        }
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
      auto fetch_scales = [&](int kt, int (&a)[(MB + 1) / 2], int (&b)[(NB + 1) / 2]) {
        if constexpr (kScaled) {
          const char *st = smem + (kt % S) * STAGE + SA::BYTES + SB::BYTES;
          SS::template fetch<MB>(st, wm, lane, a);
          SS::template fetch<NB>(st, BM + wn, lane, b);
        }
      };
      auto mma = [&](int s, const v4i (&a)[MB], const v4i (&b)[NB], const int (&qa)[(MB + 1) / 2],
                     const int (&qb)[(NB + 1) / 2]) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < MB; ++i) E::mma(a[i], b[j], acc[i][j], s, i, qa[i / 2], j, qb[j / 2]);
      };

      // Tile kt is read from stage kt % S while the copies of the next S - 1
      // are in flight or landed; its stage takes tile kt + S after the
      // barrier that ends its reads.
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < nt) fill(i);
      wait_barrier<0>();
      v4i xa[MB], xb[NB], ya[MB], yb[NB];
      int qa[(MB + 1) / 2] = {}, qb[(NB + 1) / 2] = {};
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
    store_tile<E, 16>(p, at, acc, m0 + wm, n0 + wn, cols, lane);
  }
};

// The 256 x 256 tile of the large products: 8 waves of 128 x 64 each (the
// columns in blocks of 16, 64 apart), two on every SIMD, which take turns.
// Time runs in slots between barriers: while one wave of a SIMD runs the 32
// MFMAs of a step (512 cycles of the matrix core) with the copies spread among
// them, the other reads its operands of the next step from LDS. Waves 4 - 7
// run one slot behind waves 0 - 3 (k-tile k, steps 0 and 1):
//   slot           4 k             4 k + 1     4 k + 2     4 k + 3     4 k + 4
//   waves 0 - 3    read 0          multiply 0  read 1      multiply 1  read 0
//   waves 4 - 7    multiply 1 (-)  read 0      multiply 0  read 1      multiply 1
// One block a CU runs through tiles (w, w + blocks, ...), and its k-tiles are
// one stream: the copies of the next tile's first k-tiles are under way while
// a tile is finished, and one half of the waves stores its part of C while
// the other multiplies. 16-bit: A's and B's k-tiles rotate through five units
// of 32 KB, all of LDS (A 0, B 0, A 1, B 1, ...). Both units of k-tile k - 1
// are free from slot 4 k on: waves 0 - 3 copy B k + 1 in "multiply 0" of k and
// A k + 2 in "multiply 1", waves 4 - 7 B k + 1 in "multiply 1" of k - 1 and
// A k + 2 in "multiply 0" of k; three or four slots before they are read. fp4
// also keeps scales and has four units: waves 0 - 3 copy all of k + 1 in
// "multiply 0" of k, waves 4 - 7 in "multiply 1" of k - 1.
template <class E, bool AMC, bool BMC, bool RK>
struct TurnKernel {
  static constexpr int BM = 256, BN = 256, WM = 2, WN = 4;
  static constexpr int kBM = BM, kBN = BN;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16, STEP = 16 * WN;
  static constexpr bool kScaled = E::kBits == 4;
  static constexpr bool kPersistent = true;  // at most one block a CU
  typedef Stager<E, BM, AMC, NT> SA;
  typedef Stager<E, BN, BMC, NT> SB;
  typedef ScaleStager<kScaled ? BM : 64, kScaled ? BN : 64, NW> SS;
  typedef typename std::conditional<RK, KFinder, ColumnFinder>::type Finder;
  static_assert(SA::BYTES == SB::BYTES, "equal units");
  static constexpr int UNIT = SA::BYTES;
  static constexpr int UNITS = kScaled ? 4 : 5;
  static constexpr int LDS = UNITS * UNIT + (kScaled ? 2 * SS::BYTES : 0);

  // k of a tile, and its k-tiles
  static __device__ __forceinline__ int depth(const Args &p, const Tile &t) {
    return p.alpha == 0.0f ? 0 : (int)(RK ? t.hi - t.lo : p.k);  // alpha == 0 reads neither operand
  }
  static __device__ __forceinline__ int tiles_k(int K) { return (K + SA::BK - 1) / SA::BK; }
  static __device__ __forceinline__ int rotate(int at) {  // two units on, in bytes
    return at + 2 * UNIT >= UNITS * UNIT ? at + (2 - UNITS) * UNIT : at + 2 * UNIT;
  }

  // The copies of one operand (which one is a scalar, so that both halves of
  // the waves share the code), k-tile after k-tile and tile after tile.
  struct Stream {
    StagerData<SA::LOADS> d;
    const char *from;  // the next k-tile's first byte
    int64_t step;
    int w, kt, nt, whole, unit;
    int parts;  // of a k-tile that the tile's columns need
    bool is_a;

    template <class S>
    __device__ __forceinline__ void open(const char *P, int64_t ld, int64_t row0, int64_t rows, int K, int t) {
      S s;
      s.init(P, ld, row0, rows, K, t);
      d = s;
      step = s.step();
      whole = s.whole_tiles();
    }
    // The first tile from w on that has k-tiles; nt == 0: none.
    __device__ __forceinline__ void seek(const Args &p, Finder &f, int t) {
      Tile tile;
      nt = 0;
      for (; f.find(p, w, tile); w += gridDim.x) {
        const int K = depth(p, tile);
        nt = tiles_k(K);
        if (nt == 0) continue;
        parts = SA::LOADS;
        if (!is_a && !BMC) {
          // a part is STEP columns
          static_assert(BMC || SB::RPS == STEP, "parts");
          const int64_t cols = (RK ? p.n : tile.hi - tile.lo) - (int64_t)tile.tn * BN;
          if (cols < BN) parts = (int)((cols + STEP - 1) / STEP);
        }
        if (is_a)
          open<SA>(RK ? p.A + tile.lo * p.lda : p.A + (int64_t)tile.g * p.stride_a, p.lda, (int64_t)tile.tm * BM, p.m, K, t);
        else
          open<SB>(p.B + tile.lo * p.ldb, p.ldb, (int64_t)tile.tn * BN, RK ? p.n : tile.hi - tile.lo, K, t);
        kt = 0;
        from = d.origin;
        break;
      }
    }
    __device__ __forceinline__ void start(const Args &p, Finder &f, int t, bool a) {
      is_a = a;
      w = blockIdx.x;
      unit = a ? 0 : UNIT;
      seek(p, f, t);
    }
    // k-tiles that can be copied one after the other without a look at what
    // comes: whole, and not the tile's last
    __device__ __forceinline__ int run() const { return (whole < nt - 1 ? whole : nt - 1) - kt; }
    __device__ __forceinline__ void copy_part(char *smem, int wave, int r) const {
      copy_chunks(from, d.voff[r], smem + unit + wave * 1024 + r * NT * 16);
    }
    __device__ __forceinline__ void advance() {
      ++kt;
      from += step;
      unit = rotate(unit);
    }
    template <class S>
    __device__ __forceinline__ void cut(char *smem, int wave) const {
      S s;
      (StagerData<SA::LOADS> &)s = d;
#pragma unroll
      for (int r = 0; r < S::LOADS; ++r)
        if constexpr (E::kBits == 4)
          copy_chunks(from, s.half_voff(r), smem + unit + wave * 1024 + r * NT * 16);
        else
          s.put(smem + unit, r, s.load_guarded(kt, r));
    }
    // The next k-tile, whatever it is: a cut one of 16-bit values goes through
    // registers.
    __device__ __forceinline__ void issue(const Args &p, Finder &f, char *smem, int t, int wave) {
      if (nt == 0) return;
      if (kt < whole) {
#pragma unroll
        for (int r = 0; r < SA::LOADS; ++r) copy_part(smem, wave, r);
      } else if (is_a) {
        cut<SA>(smem, wave);
      } else {
        cut<SB>(smem, wave);
      }
      advance();
      if (kt == nt) {
        w += gridDim.x;
        seek(p, f, t);
      }
    }
  };

  // The scales of both operands (fp4), alike.
  struct ScaleStream {
    SS s;
    int w, kt, nt, at;

    __device__ __forceinline__ void seek(const Args &p, Finder &f, int wave, int lane) {
      Tile tile;
      nt = 0;
      for (; f.find(p, w, tile); w += gridDim.x) {
        const int K = depth(p, tile);
        nt = tiles_k(K);
        if (nt == 0) continue;
        const int64_t lsa = p.lda / 16, lsb = p.ldb / 16;
        const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
        s.init(p.scale_a + (int64_t)tile.g * (p.stride_a / 16) + m0 * lsa, lsa, p.m - m0,
               p.scale_b + (tile.lo + n0) * lsb, lsb, tile.hi - tile.lo - n0, K, wave, lane);
        kt = 0;
        break;
      }
    }
    __device__ __forceinline__ void start(const Args &p, Finder &f, int wave, int lane) {
      w = blockIdx.x;
      at = UNITS * UNIT;
      seek(p, f, wave, lane);
    }
    __device__ __forceinline__ int run() const { return nt - 1 - kt; }
    __device__ __forceinline__ void advance() {
      ++kt;
      at ^= (UNITS * UNIT) ^ (UNITS * UNIT + SS::BYTES);
    }
    __device__ __forceinline__ void issue(const Args &p, Finder &f, char *smem, int wave, int lane) {
      if (nt == 0) return;
      if (kt < nt - 1)
        s.copy(smem + at, kt);
      else
        s.put_guarded(smem + at, kt, lane);
      advance();
      if (kt == nt) {
        w += gridDim.x;
        seek(p, f, wave, lane);
      }
    }
  };

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    constexpr int PARTS = SA::LOADS;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * 16;
    const bool second = wave >= NW / 2;
    Finder finder;
    finder.init(p, BN);

    f4 acc[MB][NB];
    v4i a[MB], b[NB];
    int qa[(MB + 1) / 2] = {}, qb[(NB + 1) / 2] = {};
    auto clear = [&]() {
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();

    Stream ca, cb;
    ScaleStream cs;
    ca.start(p, finder, t, true);
    cb.start(p, finder, t, false);
    if constexpr (kScaled) cs.start(p, finder, wave, lane);
    // ahead of the first slot: A 0, B 0 and, with five units, A 1
#pragma nounroll
    for (int i = 0; i < (UNITS == 5 ? 2 : 1); ++i) {
      ca.issue(p, finder, smem, t, wave);
      if (i == 0) cb.issue(p, finder, smem, t, wave);
      if constexpr (kScaled) cs.issue(p, finder, smem, wave, lane);
    }
    wait_barrier<0>();
    if (second) __builtin_amdgcn_s_barrier();

    int ua = 0, ub = UNIT, scales = UNITS * UNIT;  // the units and scales being read
    auto read = [&](int s, int nb) {
      SA::template fetch<MB>(smem + ua, wm, s, lane, a);
      SB::template fetch<NB, STEP>(smem + ub, wn, s, lane, b, nb);
      if (kScaled && s == 0) {
        SS::template fetch<MB>(smem + scales, wm, lane, qa);
        SS::template fetch<NB, STEP>(smem + scales, BM + wn, lane, qb, nb);
      }
    };
    auto multiply = [&](int s, int nb) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (j == 0 || __builtin_expect(j < nb, 1))
#pragma unroll
          for (int i = 0; i < MB; ++i) E::mma(a[i], b[j], acc[i][j], s, i, qa[i / 2], j, qb[j / 2]);
    };
    auto next_k = [&]() {
      ua = rotate(ua);
      ub = rotate(ub);
      if (kScaled) scales ^= (UNITS * UNIT) ^ (UNITS * UNIT + SS::BYTES);
    };

    auto steady = [&](int used, int count) {
      for (; count > 0; --count) {
        read(0, used);
        if (UNITS == 4)
#pragma unroll
          for (int r = 0; r < PARTS; ++r) ca.copy_part(smem, wave, r);
#pragma unroll
        for (int r = 0; r < PARTS; ++r)
          if (r == 0 || __builtin_expect(r < cb.parts, 1)) cb.copy_part(smem, wave, r);
        if constexpr (kScaled) cs.s.copy(smem + cs.at, cs.kt);
        wait_barrier<63>();
        __builtin_amdgcn_s_setprio(1);
        multiply(0, used);
        __builtin_amdgcn_s_setprio(0);
        cb.advance();
        if (UNITS == 4) ca.advance();
        if constexpr (kScaled) cs.advance();
        wait_barrier<63>();
        read(1, used);
        if (UNITS == 5)
#pragma unroll
          for (int r = 0; r < PARTS; ++r) ca.copy_part(smem, wave, r);
        // the next k-tile is there; the copies of A just issued may go on
        wait_barrier<UNITS == 5 ? PARTS : 0>();
        __builtin_amdgcn_s_setprio(1);
        multiply(1, used);
        __builtin_amdgcn_s_setprio(0);
        if (UNITS == 5) ca.advance();
        next_k();
        wait_barrier<63>();
      }
    };

    Tile tile;
    for (int w = blockIdx.x; finder.find(p, w, tile); w += gridDim.x) {
      const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
      const int64_t cols = RK ? p.n : tile.hi - tile.lo;
      const int nt = tiles_k(depth(p, tile));
      // column blocks in use: a group's last tile costs what its columns need
      int nb = NB;
      if (cols - n0 < BN) nb = (int)((cols - n0 + STEP - 1) / STEP);
      int kt = 0;
      while (kt < nt) {
        // The steady state, without a branch: k-tiles of which every copy is
        // whole and none the last of its tile.
        int count = ca.run();
        const int rb = cb.run();
        count = count < rb ? count : rb;
        if (kScaled) count = count < cs.run() ? count : cs.run();
        count = count < nt - kt ? count : nt - kt;
        if (count > 0) {
          kt += count;
          steady(nb, count);
        }
        if (kt == nt) break;
        // one k-tile, whatever it and its copies are
        read(0, nb);
        if (UNITS == 4) ca.issue(p, finder, smem, t, wave);
        cb.issue(p, finder, smem, t, wave);
        if constexpr (kScaled) cs.issue(p, finder, smem, wave, lane);
        wait_barrier<63>();
        multiply(0, nb);
        wait_barrier<63>();
        read(1, nb);
        if (UNITS == 5) ca.issue(p, finder, smem, t, wave);
        wait_barrier<0>();
        multiply(1, nb);
        next_k();
        wait_barrier<63>();
        ++kt;
      }
      const int64_t at = RK ? (int64_t)tile.g * p.stride_c : tile.lo * p.ldc;
      store_tile<E, STEP>(p, at, acc, m0 + wm, n0 + wn, cols, lane);
      clear();
    }
    if (!second) __builtin_amdgcn_s_barrier();
  }
};

template <class K>
__global__ __launch_bounds__(K::NT, 2) void ragged_kernel(Args p) {
  extern __shared__ __align__(1024) char ragged_smem[];
  K::run(p, ragged_smem);
}

// `tiles`: at most.
template <class K>
int launch(wgb_ctx *ctx, const Args &p, int64_t tiles) {
  if (tiles == 0) return WGB_OK;
  if (tiles > INT32_MAX) return wgb::fail(WGB_ERR_INVALID_VALUE, "grouped product: too many tiles");
  const int64_t blocks = K::kPersistent && tiles > ctx->num_cus ? ctx->num_cus : tiles;
  static const hipError_t attr =
      hipFuncSetAttribute((const void *)ragged_kernel<K>, hipFuncAttributeMaxDynamicSharedMemorySize, K::LDS);
  if (attr != hipSuccess) return wgb::fail_hip(attr, "LDS size of a grouped product");
  ragged_kernel<K><<<(unsigned)blocks, K::NT, K::LDS, ctx->stream>>>(p);
  WGB_CHECK_LAUNCH("ragged_kernel");
  return WGB_OK;
}

// Tiles that a ragged-columns launch has at most: a group of c columns has
// ceil(c / bn) column tiles, at most one of them partly filled.
template <class K>
int launch_columns(wgb_ctx *ctx, Args &p) {
  const int64_t bn = K::kBN;
  p.tiles_m = (int)((p.m + K::kBM - 1) / K::kBM);
  const int64_t across = !p.off ? (p.n + bn - 1) / bn : p.n / bn + (p.n < p.groups ? p.n : p.groups);
  return launch<K>(ctx, p, across * p.tiles_m);
}

template <class K>
int launch_k(wgb_ctx *ctx, Args &p) {
  p.tiles_m = (int)((p.m + K::kBM - 1) / K::kBM);
  p.tiles_n = (int)((p.n + K::kBN - 1) / K::kBN);
  return launch<K>(ctx, p, (int64_t)p.tiles_m * p.tiles_n * p.groups);
}

}  // namespace wgb_ragged
