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
#include "copy_plan.h"
#include "tile_order.h"

#include <atomic>
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
  // CUs of a persistent launch of 256 x 256 tiles, which leaves a last round
  // that would use at most half of them to 128 x 128 tiles; 0: no such launch
  int round;
  int pieces;     // of k that a tile of that rest is cut into at most, each a block's; their sums go to
  float *parts;   // this array, 128 x 128 a block
  int stream;  // C's columns start at 64-byte boundaries: large results bypass the caches
  int c_f32;   // C holds fp32 (else the operands' type; fp4: bf16, or f16 with c_f16)
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
// and even out the end. Either part is dealt to the XCDs in runs.
struct ColumnOrder {
  int whole, total;  // tiles: of whole columns, all
  int bn;
  int lo, hi;        // lane's group: its columns (below 2^31),
  int sum, rest;     // whole column tiles, and leftovers, up to and with it

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

  // Place of tile w < total among the column tiles of its kind (`left`: a leftover), and what is left of it in that.
  __device__ __forceinline__ int place(const Args &p, int w, bool &left, int &L) const {
    left = w >= whole;
    L = left ? wgb_tiles::xcd_remap(w - whole, total - whole) : wgb_tiles::xcd_remap(w, whole);
    return L / p.tiles_m;
  }
  // The tile, once its group is known; `past`: whole column tiles up to and with that group.
  __device__ __forceinline__ void settle(const Args &p, bool left, int L, int q, int past, Tile &t) const {
    const int tn = (int)(t.hi - t.lo) / bn;
    if (left) {
      t.tm = L - q * p.tiles_m;
      t.tn = tn;
    } else {
      wgb_tiles::logical_tile(L - (past - tn) * p.tiles_m, p.tiles_m, tn, 0, t.tm, t.tn);
    }
  }

  // Tile w of a wave (w is the same in all lanes): false if there is none.
  __device__ __forceinline__ bool find(const Args &p, int w, Tile &t) {
    if (w >= total) return false;
    bool left;
    int L;
    const int q = place(p, w, left, L);
    t.g = 0;
    t.lo = 0;
    t.hi = p.n;
    int past = (int)(p.n / bn);
    if (p.off) {
      int before = 0, rest_before = 0, g0 = 0;
      uint64_t beyond;
      for (;; g0 += 64) {
        if (p.groups > 64) scan(p, g0, before, rest_before);
        beyond = __ballot((left ? rest : sum) > q);
        if (beyond || g0 + 64 >= p.groups) break;
        before = __builtin_amdgcn_readlane(sum, 63);
        rest_before = __builtin_amdgcn_readlane(rest, 63);
      }
      if (!beyond) return false;
      const int at = __builtin_ctzll(beyond);
      t.g = g0 + at;
      t.lo = __builtin_amdgcn_readlane(lo, at);
      t.hi = __builtin_amdgcn_readlane(hi, at);
      past = __builtin_amdgcn_readlane(sum, at);
    }
    settle(p, left, L, q, past, t);
    return true;
  }

  // Each lane's tile w < total.
  __device__ __forceinline__ void find_lanes(const Args &p, int w, Tile &t) {
    bool left;
    int L;
    const int q = place(p, w, left, L);
    t.g = 0;
    t.lo = 0;
    t.hi = p.n;
    int past = (int)(p.n / bn);
    if (p.off) {
      int before = 0, rest_before = 0;
      bool open = true;
      for (int g0 = 0; g0 < p.groups; g0 += 64) {
        if (p.groups > 64) scan(p, g0, before, rest_before);
        const int count = p.groups - g0 < 64 ? p.groups - g0 : 64;
        for (int i = 0; i < count; ++i) {
          const int s = __builtin_amdgcn_readlane(sum, i), r = __builtin_amdgcn_readlane(rest, i);
          if (open && (left ? r : s) > q) {
            open = false;
            t.g = g0 + i;
            t.lo = __builtin_amdgcn_readlane(lo, i);
            t.hi = __builtin_amdgcn_readlane(hi, i);
            past = s;
          }
        }
        before = __builtin_amdgcn_readlane(sum, 63);
        rest_before = __builtin_amdgcn_readlane(rest, 63);
      }
    }
    settle(p, left, L, q, past, t);
  }
};

// The tiles of a ragged-k launch: the groups from the longest to the shortest
// (up to 64 of them, one a lane; more stay in their order), the rounds of a
// persistent launch to and fro, so that blocks come out even; each group's
// tiles are dealt to all XCDs.
struct KOrder {
  int total, per;

  __device__ __forceinline__ void init(const Args &p, int) {
    per = p.tiles_m * p.tiles_n;
    total = per * p.groups;
  }
  // Each lane's tile w < total (lanes may have the same).
  __device__ __forceinline__ void find_lanes(const Args &p, int w, Tile &t) {
    const int blocks = p.round ? p.round : (int)gridDim.x;
    const int round = w / blocks, begin = round * blocks;
    const int end = begin + blocks < total ? begin + blocks : total;
    const int at = round & 1 ? begin + end - 1 - w : w;
    const int place = at / per;
    wgb_tiles::logical_tile(wgb_tiles::xcd_remap(at - place * per, per), p.tiles_m, p.tiles_n, 0, t.tm, t.tn);
    t.g = place;
    if (p.groups > 64) {
      group_range(p.off, t.g, p.k, t.lo, t.hi);
      return;
    }
    const int lane = threadIdx.x & 63;
    int64_t l = 0, h = 0;
    if (lane < p.groups) group_range(p.off, lane, p.k, l, h);
    const int lo = (int)l, hi = (int)h, size = hi - lo;  // k is below 2^31
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const int other = __builtin_amdgcn_readlane(size, g);
      rank += other > size || (other == size && g < lane);
    }
    for (int g = 0; g < p.groups; ++g)
      if (__builtin_amdgcn_readlane(rank, g) == place) {
        t.g = g;
        t.lo = __builtin_amdgcn_readlane(lo, g);
        t.hi = __builtin_amdgcn_readlane(hi, g);
      }
  }
  // Tile w of a wave: false if there is none. A launch of its own takes the
  // groups as they are (ranking 64 of them costs every block a microsecond);
  // the rest of a persistent launch has to keep that one's order.
  __device__ __forceinline__ bool find(const Args &p, int w, Tile &t) {
    if (w >= total) return false;
    if (p.round) {
      find_lanes(p, w, t);
    } else {
      t.g = w / per;
      wgb_tiles::logical_tile(wgb_tiles::xcd_remap(w - t.g * per, per), p.tiles_m, p.tiles_n, 0, t.tm, t.tn);
      group_range(p.off, t.g, p.k, t.lo, t.hi);
    }
    t.g = __builtin_amdgcn_readfirstlane(t.g);
    t.lo = __builtin_amdgcn_readfirstlane((int)t.lo);
    t.hi = __builtin_amdgcn_readfirstlane((int)t.hi);
    return true;
  }
};

// Of `total` 256 x 256 tiles those that the persistent launch computes: whole
// rounds, and the rest if it is more than half a round.
__device__ __forceinline__ int whole_rounds(const Args &p, int total) {
  if (!p.round) return total;
  const int cut = total / p.round * p.round;
  return total - cut > p.round / 2 ? total : cut;
}

// A quarter (128 x 128) of a tile that the persistent launch left, by a block
// of the launch for those: false if there is none. Few quarters are cut along
// k, as many pieces as keep all blocks at once on the GPU: 60 of them at k =
// 4096, one a CU, take 65 us whole, for a CU's copies are the limit there.
struct Quarter {
  int at, piece, pieces;

  template <class Order>
  __device__ __forceinline__ bool find(const Args &p, Order &order, int block, bool fold, Tile &t) {
    order.init(p, 256);
    const int whole = whole_rounds(p, order.total), left = order.total - whole;
    if (left <= 0) return false;
    pieces = p.round / (2 * left);
    pieces = pieces > p.pieces ? p.pieces : pieces < 1 ? 1 : pieces;
    at = fold ? block : block / pieces;
    piece = fold ? 0 : block - at * pieces;
    if (at >= 4 * left || !order.find(p, whole + at / 4, t)) return false;
    t.tm = 2 * t.tm + (at & 1);
    t.tn = 2 * t.tn + ((at >> 1) & 1);
    return true;
  }
};

// A persistent block's tiles, one a lane: all of them are found at the start.
constexpr int kTilesPerBlock = 64;
template <class Order>
struct TileTable {
  int count;  // of this block's tiles
  int g, tm, tn, lo, hi;

  __device__ __forceinline__ void init(const Args &p, int bn) {
    Order o;
    o.init(p, bn);
    const int first = (int)blockIdx.x, step = (int)gridDim.x;
    const int total = whole_rounds(p, o.total);
    count = first < total ? (total - first + step - 1) / step : 0;
    if (count > kTilesPerBlock) count = kTilesPerBlock;  // the launch has blocks enough
    const int lane = threadIdx.x & 63;
    Tile t = {0, 0, 0, 0, 0};
    if (count > 0) o.find_lanes(p, first + (lane < count ? lane : 0) * step, t);
    g = t.g;
    tm = t.tm;
    tn = t.tn;
    lo = (int)t.lo;
    hi = (int)t.hi;
  }
  __device__ __forceinline__ bool get(int i, Tile &t) const {
    if (i >= count) return false;
    t.g = __builtin_amdgcn_readlane(g, i);
    t.tm = __builtin_amdgcn_readlane(tm, i);
    t.tn = __builtin_amdgcn_readlane(tn, i);
    t.lo = __builtin_amdgcn_readlane(lo, i);
    t.hi = __builtin_amdgcn_readlane(hi, i);
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

template <class E, int BT, bool MC, int NT>
struct Stager : CopyPlan<E::kBits, BT, MC, NT> {
  typedef CopyPlan<E::kBits, BT, MC, NT> Plan;
  using Plan::CPR;
  using Plan::EPC;
  using Plan::LOADS;
  using Plan::origin;
  using Plan::voff;
  using Plan::t;

  // k-tile kt.
  __device__ __forceinline__ void copy(char *stage, int kt, int wave) const {
    const char *from = origin + (int64_t)kt * this->step();
#pragma unroll
    for (int r = 0; r < LOADS; ++r) copy_chunks(from, voff[r], stage + wave * 1024 + r * NT * 16);
  }

  // Chunk r of k-tile kt through registers: rows past the matrix and k past
  // K read as zeros, at any alignment of the elements.
  __device__ __forceinline__ v4i load_guarded(int kt, int r) const {
    typedef typename E::chunk v4u;  // 16 bytes at the elements' alignment
    int64_t at;
    const int64_t left = this->guarded(kt, r, at);
    v4i v = {0, 0, 0, 0};
    if (left >= EPC) {
      v = *reinterpret_cast<const v4u *>(origin + at);
    } else if (left > 0) {
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

// Of a lane's chunk of which `left` elements are before the end of k: all
// ones there, zeros after.
template <class E>
__device__ __forceinline__ v4i tail_mask(int left) {
  v4i m;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (E::kBits == 32)
      m[i] = left > i ? -1 : 0;
    else
      m[i] = left >= 2 * i + 2 ? -1 : left == 2 * i + 1 ? 0xffff : 0;
  }
  return m;
}
// The operands of step s of a k-tile with `left` elements of k.
template <class E, int MB, int NB>
__device__ __forceinline__ void clear_tail(int left, int s, int lane, v4i (&a)[MB], v4i (&b)[NB]) {
  const v4i m = tail_mask<E>(left - (4 * s + (lane >> 4)) * (128 / E::kBits));
#pragma unroll
  for (int i = 0; i < MB; ++i) a[i] &= m;
#pragma unroll
  for (int j = 0; j < NB; ++j) b[j] &= m;
}

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
// two row blocks: with 8 bytes a lane 8192 x 16384 x 4096 took 4% longer.
// STREAM: non-temporal stores, for results too large for the caches (12 x 1032
// x 520 in f16, which fits, 16.7 -> 21 us) and whose columns do not cut lines
// (12872 columns of 2249 fp32 values 109 -> 168 us), in whole lines: as runs
// of 64 bytes, weight gradients of 8 x 4096 x 2048 in fp32 wrote 399 MB for the
// 268 of C and took 195 us instead of 175, forward products of 16384 columns of
// 8192 bf16 values 1020 instead of 983.
template <typename T, int MB, int NB, int STEP, bool STREAM>
__device__ __forceinline__ void epilogue(const Args &p, T *C, const f4 (&acc)[MB][NB], int64_t row0, int64_t rows,
                                         int64_t col0, int64_t cols, int lane) {
  typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  constexpr bool PAIRS = sizeof(T) == 2 && MB % 2 == 0;
  const int i16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t col = col0 + STEP * j + i16;
    const bool in = col < cols;
    if (!STREAM && !in) continue;
    T *cp = C + col * p.ldc;
    // a lane's four rows of row block i
    auto value = [&](int i) {
      const int64_t row = row0 + 16 * i + 4 * g;
      f4 x = acc[i][j];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] *= p.alpha;
      if (p.beta != 0.0f && in) {
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
    if constexpr (STREAM) {
      // two runs of 64 bytes of 16 columns become 128 bytes of 8 columns each:
      // lanes 0 - 7 of 16 give the second run, lanes 8 - 15 the first
      constexpr int ROWS = 16 / sizeof(T), BLOCKS = PAIRS ? 4 : 2;
      typedef T Run __attribute__((ext_vector_type(ROWS), aligned(sizeof(T))));
      const bool low = i16 < 8;
#pragma unroll
      for (int i = 0; i < MB; i += BLOCKS) {
        v4i x[2], y[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (PAIRS) {
            typedef uint32_t u2 __attribute__((ext_vector_type(2)));
            const u2 a = __builtin_bit_cast(u2, value(i + 2 * h)), b = __builtin_bit_cast(u2, value(i + 2 * h + 1));
            x[h] = eight_rows(a[0], a[1], b[0], b[1]);
          } else {
            x[h] = __builtin_bit_cast(v4i, value(i + h));
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int other = __builtin_amdgcn_mov_dpp(low ? x[1][c] : x[0][c], 0x128, 0xf, 0xf, true);  // lane ^ 8
          y[0][c] = low ? x[0][c] : other;
          y[1][c] = low ? other : x[1][c];
        }
        const int64_t row = row0 + 16 * i + (PAIRS ? 32 * (i16 >> 3) + 16 * (g & 1) + 8 * (g >> 1) : 16 * (i16 >> 3) + 4 * g);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t to = col0 + STEP * j + 8 * h + (i16 & 7);
          if (to >= cols) continue;
          T *at = C + to * p.ldc + row;
          const Run v = __builtin_bit_cast(Run, y[h]);
          if (row + ROWS <= rows) {
            __builtin_nontemporal_store(v, reinterpret_cast<Run *>(at));
          } else {
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
              if (row + q < rows) at[q] = v[q];
          }
        }
      }
    } else if constexpr (PAIRS) {
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
template <class E, int STEP, bool STREAM = false, int MB, int NB>
__device__ __forceinline__ void store_tile(const Args &p, int64_t at, const f4 (&acc)[MB][NB], int64_t row0, int64_t col0,
                                           int64_t cols, int lane) {
  if (E::kBits == 32 || p.c_f32) {
    epilogue<float, MB, NB, STEP, STREAM>(p, (float *)p.C + at, acc, row0, p.m, col0, cols, lane);
  } else if constexpr (E::kBits == 4) {
    if (p.c_f16)
      epilogue<_Float16, MB, NB, STEP, STREAM>(p, (_Float16 *)p.C + at, acc, row0, p.m, col0, cols, lane);
    else
      epilogue<__bf16, MB, NB, STEP, STREAM>(p, (__bf16 *)p.C + at, acc, row0, p.m, col0, cols, lane);
  } else if constexpr (E::kBits == 16) {
    epilogue<typename E::store, MB, NB, STEP, STREAM>(p, (typename E::store *)p.C + at, acc, row0, p.m, col0, cols, lane);
  }
}

// One BM x BN tile of C a block, WM x WN waves: what the larger tiles would
// leave CUs idle for. Bound by the copies into LDS, about 40 bytes a cycle and
// CU (bf16 4096^3 on 128 x 128 tiles 1.0 PFLOP/s), and with few columns (128 x
// 32 tiles) by reading A (64 experts of 2048 x 1024 in bf16, 64 columns: 27 us,
// 6.4 TB/s); in fp32 by the matrix cores (64 x 64 tiles: 1000 x 1537 x 777 in 5
// groups 31 us, 77 TFLOP/s, their last round half empty). AMC / BMC: the operand is
// row-contiguous in memory. VEC: both operands can be copied by 16-byte
// (4-byte aligned) loads at 32-bit offsets; otherwise every k-tile goes
// through registers. RK: ragged k. S: stages of LDS.
template <class E, int BM, int BN, int WM, int WN, bool AMC, bool BMC, bool VEC, bool RK, int S>
struct Kernel {
  typedef E Element;
  typedef typename std::conditional<RK, KOrder, ColumnOrder>::type Order;
  static constexpr int kBM = BM, kBN = BN, kWM = WM, kWN = WN;
  static constexpr bool kRK = RK;
  // computes what a launch of 256 x 256 tiles leaves, too
  static constexpr bool REST = BM == 128 && BN == 128 && VEC && E::kBits != 32;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
  static constexpr bool kScaled = E::kBits == 4;
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
    Order order;
    Quarter quarter = {0, 0, 1};
    if (REST && p.round) {
      if (!quarter.find(p, order, blockIdx.x, false, tile)) return;
    } else {
      order.init(p, BN);
      if (!order.find(p, blockIdx.x, tile)) return;
    }
    const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
    const int64_t cols = RK ? p.n : tile.hi - tile.lo;
    if (m0 >= p.m || n0 >= cols) return;
    int64_t K = RK ? tile.hi - tile.lo : p.k;
    if (p.alpha == 0.0f) K = 0;  // reads neither operand
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);

    f4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    int nt = (int)((K + SA::BK - 1) / SA::BK), first = 0;
    if (REST && quarter.pieces > 1) {
      const int most = (nt + quarter.pieces - 1) / quarter.pieces;
      first = quarter.piece * most;
      nt = nt - first < most ? nt - first : most;
      K -= (int64_t)first * SA::BK;
      if (K > (int64_t)most * SA::BK) K = (int64_t)most * SA::BK;
    }
    if (nt > 0) {
      SA sa;
      SB sb;
      SS ss;
      const char *A = RK ? p.A + tile.lo * p.lda : p.A + (int64_t)tile.g * p.stride_a;
      const char *B = RK ? p.B + tile.lo * p.ldb : p.B + tile.lo * p.ldb;
      sa.init(A, p.lda, m0, p.m, K, t);
      sb.init(B, p.ldb, n0, cols, K, t);
      if constexpr (REST) {
        sa.origin += first * sa.step();
        sb.origin += first * sb.step();
      }
      if constexpr (kScaled) {
        const int64_t lsa = p.lda / 16, lsb = p.ldb / 16;
        ss.init(p.scale_a + (int64_t)tile.g * (p.stride_a / 16) + m0 * lsa + first * SS::RB, lsa, p.m - m0,
                p.scale_b + (tile.lo + n0) * lsb + first * SS::RB, lsb, cols - n0, K, wave, lane);
      }
      int whole = 0;
      if constexpr (VEC) {
        whole = sa.whole_tiles();
        const int wb = sb.whole_tiles();
        whole = whole < wb ? whole : wb;
      }
      const int cut = kScaled ? 0 : (int)(K % SA::BK);  // elements of k in a cut last k-tile
      const bool soft = VEC && cut && whole == nt - 1 && sa.soft_tail() && sb.soft_tail();

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
        if (VEC && kt < whole) {
          copy(kt);
        } else if (soft) {
          char *st = smem + (kt % S) * STAGE;
          const char *fa = sa.origin + (int64_t)kt * sa.step(), *fb = sb.origin + (int64_t)kt * sb.step();
#pragma unroll
          for (int r = 0; r < SA::LOADS; ++r) copy_chunks(fa, sa.tail_voff(r), st + wave * 1024 + r * NT * 16);
#pragma unroll
          for (int r = 0; r < SB::LOADS; ++r) copy_chunks(fb, sb.tail_voff(r), st + SA::BYTES + wave * 1024 + r * NT * 16);
        } else {
          guarded(kt);
        }
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
      if (soft && nt == 1) clear_tail<E>(cut, 0, lane, xa, xb);
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
        if (soft && kt == nt - 1) clear_tail<E>(cut, 1, lane, ya, yb);
        mma(0, xa, xb, qa, qb);
        wait_barrier<0>();
        if (kt + S < nt) fill(kt + S);
        if (kt + 1 < nt) fetch(kt + 1, 0, xa, xb);
        if (soft && kt + 1 == nt - 1) clear_tail<E>(cut, 0, lane, xa, xb);
        mma(1, ya, yb, qa, qb);
        if (kt + 1 < nt) fetch_scales(kt + 1, qa, qb);
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
    const int64_t at = RK ? (int64_t)tile.g * p.stride_c : tile.lo * p.ldc;
    store_tile<E, 16>(p, at, acc, m0 + wm, n0 + wn, cols, lane);
  }
};

// Adds up the pieces of quarters that were cut along k, in their order (the
// result is the same every time): block 4 q + j column block j of each wave's
// part of quarter q.
template <class K>
struct FoldKernel {
  static constexpr int NT = K::NT, LDS = 0;

  static __device__ __forceinline__ void run(const Args &p, char *) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile tile;
    typename K::Order order;
    Quarter quarter;
    if (!quarter.find(p, order, blockIdx.x / K::NB, true, tile) || quarter.pieces == 1) return;
    const int64_t m0 = (int64_t)tile.tm * K::kBM, n0 = (int64_t)tile.tn * K::kBN;
    const int64_t cols = K::kRK ? p.n : tile.hi - tile.lo;
    if (m0 >= p.m || n0 >= cols) return;
    const int j = blockIdx.x % K::NB;
    const f4 *part = reinterpret_cast<const f4 *>(p.parts) +
                     (((int64_t)quarter.at * quarter.pieces * K::NW + wave) * K::NB + j) * (K::MB * 64) + lane;
    f4 total[K::MB][1];
#pragma unroll
    for (int i = 0; i < K::MB; ++i) total[i][0] = part[i * 64];
    for (int q = 1; q < quarter.pieces; ++q) {
      part += K::NW * K::NB * K::MB * 64;
#pragma unroll
      for (int i = 0; i < K::MB; ++i) total[i][0] += part[i * 64];
    }
    const int wm = (wave % K::kWM) * (K::kBM / K::kWM), wn = (wave / K::kWM) * (K::kBN / K::kWN);
    const int64_t at = K::kRK ? (int64_t)tile.g * p.stride_c : tile.lo * p.ldc;
    store_tile<typename K::Element, 16>(p, at, total, m0 + wm, n0 + wn + 16 * j, cols, lane);
  }
};

// The 256 x 256 tile of the large products: 8 waves of 128 x 64 each (the
// columns in blocks of 16, 64 apart), two on every SIMD, which take turns.
// Time runs in slots between barriers: while one wave of a SIMD runs the 32
// MFMAs of a step (512 cycles of the matrix core), the other reads its operands
// of the next step from LDS and issues its share of the copies. Waves 4 - 7
// run one slot behind waves 0 - 3 (k-tile k, steps 0 and 1):
//   slot           4 k             4 k + 1     4 k + 2     4 k + 3     4 k + 4
//   waves 0 - 3    read 0          multiply 0  read 1      multiply 1  read 0
//   waves 4 - 7    multiply 1 (-)  read 0      multiply 0  read 1      multiply 1
// One block a CU runs through tiles (w, w + blocks, ...), and its k-tiles are
// one stream: the copies of the next tile's first k-tiles are under way while
// a tile is finished, and one half of the waves stores its part of C while
// the other multiplies. 16-bit: A's and B's k-tiles rotate through five units
// of 32 KB, all of LDS (A 0, B 0, A 1, B 1, ...). Both units of k-tile k - 1
// are free from slot 4 k on, when waves 4 - 7 have read its step 1: either half
// of the waves issues its copies of B k + 1 in "read 0" of k and of A k + 2 in
// "read 1", and waits for them at the end of "read 1" of k (B) and of k + 1 (A),
// two and four slots later, before the first read of k + 1 and k + 2. fp4 also
// keeps scales and has four units: either half issues all of k + 1 in "read 0"
// of k and waits for all of it at the end of "read 1".
// 16-bit is bound by the matrix cores and the clock that they leave (1.7 GHz at
// 8192^3 in bf16, 735 to 780 us, 1.4 to 1.5 PFLOP/s, busy 0.76 of the time); 16 groups of 1024 columns 8192 x 16384 x 4096 in
// 830 us (A is read once for each group) and ragged ones in 980. fp4's k-tiles
// have as many bytes and as many MFMA cycles as the 16-bit ones, but the matrix
// cores are busy for 0.38 of the time (16-bit: 0.76; 4096 columns times 8192 x
// 8192 165 us, 8192^3 302 us, 3.6 PFLOP/s).
// What differs is that each k-tile waits for all its copies two slots after their
// issue, the scale reads, whose banks conflict, and registers that are spilled;
// which of them costs most has not been measured.
template <class E, bool AMC, bool BMC, bool RK>
struct TurnKernel {
  static constexpr int BM = 256, BN = 256, WM = 2, WN = 4;
  static constexpr int kBM = BM, kBN = BN;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16, STEP = 16 * WN;
  static constexpr bool kScaled = E::kBits == 4;
  typedef Stager<E, BM, AMC, NT> SA;
  typedef Stager<E, BN, BMC, NT> SB;
  typedef ScaleStager<kScaled ? BM : 64, kScaled ? BN : 64, NW> SS;
  typedef TileTable<typename std::conditional<RK, KOrder, ColumnOrder>::type> Table;
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

  // The copies of one operand, k-tile after k-tile and tile after tile.
  template <class S, bool IS_A>
  struct Stream {
    S s;
    const char *from;  // the next k-tile's first byte
    int i, kt, nt, whole, unit;
    int parts;  // of a k-tile that the tile's columns need

    // The first tile from i on that has k-tiles; nt == 0: none.
    __device__ __forceinline__ void seek(const Args &p, const Table &table, int t) {
      Tile tile;
      kt = nt = whole = 0;
      for (; table.get(i, tile); ++i) {
        const int K = depth(p, tile);
        nt = tiles_k(K);
        if (nt == 0) continue;
        parts = S::LOADS;
        if constexpr (IS_A) {
          s.init(RK ? p.A + tile.lo * p.lda : p.A + (int64_t)tile.g * p.stride_a, p.lda, (int64_t)tile.tm * BM, p.m, K, t);
        } else {
          const int64_t n0 = (int64_t)tile.tn * BN, cols = RK ? p.n : tile.hi - tile.lo;
          s.init(p.B + tile.lo * p.ldb, p.ldb, n0, cols, K, t);
          static_assert(BMC || SB::RPS == STEP, "a part is STEP columns");
          if (!BMC && cols - n0 < BN) parts = (int)((cols - n0 + STEP - 1) / STEP);
        }
        whole = s.whole_tiles();
        from = s.origin;
        break;
      }
    }
    __device__ __forceinline__ void start(const Args &p, const Table &table, int t) {
      i = 0;
      unit = IS_A ? 0 : UNIT;
      seek(p, table, t);
    }
    // k-tiles that can be copied one after the other without a look at what
    // comes: whole, and not the tile's last
    __device__ __forceinline__ int run() const { return (whole < nt - 1 ? whole : nt - 1) - kt; }
    __device__ __forceinline__ void copy(char *smem, int wave) const {
#pragma unroll
      for (int r = 0; r < S::LOADS; ++r)
        if (IS_A || r == 0 || __builtin_expect(r < parts, 1))
          copy_chunks(from, s.voff[r], smem + unit + wave * 1024 + r * NT * 16);
    }
    __device__ __forceinline__ void advance() {
      ++kt;
      from += s.step();
      unit = rotate(unit);
    }
    // The next k-tile, whatever it is: a cut one of 16-bit values goes through
    // registers.
    __device__ __forceinline__ void issue(const Args &p, const Table &table, char *smem, int t, int wave) {
      if (nt == 0) return;
      if (kt < whole) {
        copy(smem, wave);
      } else if (kScaled || (kt == nt - 1 && s.soft_tail())) {
#pragma unroll
        for (int r = 0; r < S::LOADS; ++r)
          copy_chunks(from, kScaled ? s.half_voff(r) : s.tail_voff(r), smem + unit + wave * 1024 + r * NT * 16);
      } else {
#pragma unroll
        for (int r = 0; r < S::LOADS; ++r) s.put(smem + unit, r, s.load_guarded(kt, r));
      }
      advance();
      if (kt == nt) {
        ++i;
        seek(p, table, t);
      }
    }
  };

  // The scales of both operands (fp4), alike.
  struct ScaleStream {
    SS s;
    int i, kt, nt, at;

    __device__ __forceinline__ void seek(const Args &p, const Table &table, int wave, int lane) {
      Tile tile;
      kt = nt = 0;
      for (; table.get(i, tile); ++i) {
        const int K = depth(p, tile);
        nt = tiles_k(K);
        if (nt == 0) continue;
        const int64_t lsa = p.lda / 16, lsb = p.ldb / 16;
        const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
        s.init(p.scale_a + (int64_t)tile.g * (p.stride_a / 16) + m0 * lsa, lsa, p.m - m0,
               p.scale_b + (tile.lo + n0) * lsb, lsb, tile.hi - tile.lo - n0, K, wave, lane);
        break;
      }
    }
    __device__ __forceinline__ void start(const Args &p, const Table &table, int wave, int lane) {
      i = 0;
      at = UNITS * UNIT;
      seek(p, table, wave, lane);
    }
    __device__ __forceinline__ int run() const { return nt - 1 - kt; }
    __device__ __forceinline__ void advance() {
      ++kt;
      at ^= (UNITS * UNIT) ^ (UNITS * UNIT + SS::BYTES);
    }
    __device__ __forceinline__ void issue(const Args &p, const Table &table, char *smem, int wave, int lane) {
      if (nt == 0) return;
      if (kt < nt - 1)
        s.copy(smem + at, kt);
      else
        s.put_guarded(smem + at, kt, lane);
      advance();
      if (kt == nt) {
        ++i;
        seek(p, table, wave, lane);
      }
    }
  };

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * 16;
    const bool second = wave >= NW / 2;
    Table table;
    table.init(p, BN);

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

    Stream<SA, true> ca;
    Stream<SB, false> cb;
    ScaleStream cs;
    ca.start(p, table, t);
    cb.start(p, table, t);
    if constexpr (kScaled) cs.start(p, table, wave, lane);
    auto issue_a = [&]() { ca.issue(p, table, smem, t, wave); };
    auto issue_b = [&]() { cb.issue(p, table, smem, t, wave); };
    // ahead of the first slot: A 0, B 0 and, with five units, A 1
#pragma nounroll
    for (int i = 0; i < (UNITS == 5 ? 2 : 1); ++i) {
      issue_a();
      if (i == 0) issue_b();
      if constexpr (kScaled) cs.issue(p, table, smem, wave, lane);
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
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (j == 0 || __builtin_expect(j < nb, 1))
#pragma unroll
          for (int i = 0; i < MB; ++i) E::mma(a[i], b[j], acc[i][j], s, i, qa[i / 2], j, qb[j / 2]);
      __builtin_amdgcn_s_setprio(0);
    };
    auto next_k = [&]() {
      ua = rotate(ua);
      ub = rotate(ub);
      if (kScaled) scales ^= (UNITS * UNIT) ^ (UNITS * UNIT + SS::BYTES);
    };

    Tile tile;
    for (int i = 0; table.get(i, tile); ++i) {
      const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * BN;
      const int64_t cols = RK ? p.n : tile.hi - tile.lo;
      const int K = depth(p, tile), nt = tiles_k(K);
      const int cut = kScaled ? 0 : K % SA::BK;  // elements of k in a cut last k-tile, which is not a steady one
      // column blocks in use: a group's last tile costs what its columns need
      int nb = NB;
      if (cols - n0 < BN) nb = (int)((cols - n0 + STEP - 1) / STEP);
      int kt = 0;
      while (kt < nt) {
        // The steady state: k-tiles while every copy is whole and none the
        // last of its tile.
        int count = ca.run();
        const int rb = cb.run();
        count = count < rb ? count : rb;
        if (kScaled) count = count < cs.run() ? count : cs.run();
        const int rest = nt - kt - (cut ? 1 : 0);
        count = count < rest ? count : rest;
        if (count > 0) kt += count;
        for (; count > 0; --count) {
          read(0, nb);
          if (UNITS == 4) ca.copy(smem, wave);
          cb.copy(smem, wave);
          if constexpr (kScaled) cs.s.copy(smem + cs.at, cs.kt);
          wait_barrier<63>();
          multiply(0, nb);
          cb.advance();
          if (UNITS == 4) ca.advance();
          if constexpr (kScaled) cs.advance();
          wait_barrier<63>();
          read(1, nb);
          if (UNITS == 5) ca.copy(smem, wave);
          // the next k-tile is there; the copies of A just issued may go on
          wait_barrier<UNITS == 5 ? SA::LOADS : 0>();
          multiply(1, nb);
          if (UNITS == 5) ca.advance();
          next_k();
          wait_barrier<63>();
        }
        if (kt == nt) break;
        // one k-tile, whatever it and its copies are
        const bool last = cut && kt == nt - 1;
        read(0, nb);
        if (last) clear_tail<E>(cut, 0, lane, a, b);
        if (UNITS == 4) issue_a();
        issue_b();
        if constexpr (kScaled) cs.issue(p, table, smem, wave, lane);
        wait_barrier<63>();
        multiply(0, nb);
        wait_barrier<63>();
        read(1, nb);
        if (last) clear_tail<E>(cut, 1, lane, a, b);
        if (UNITS == 5) issue_a();
        wait_barrier<0>();
        multiply(1, nb);
        next_k();
        wait_barrier<63>();
        ++kt;
      }
      const int64_t at = RK ? (int64_t)tile.g * p.stride_c : tile.lo * p.ldc;
      if (p.stream)
        store_tile<E, STEP, true>(p, at, acc, m0 + wm, n0 + wn, cols, lane);
      else
        store_tile<E, STEP, false>(p, at, acc, m0 + wm, n0 + wn, cols, lane);
      clear();
    }
    if (!second) __builtin_amdgcn_s_barrier();
  }
};

// Few columns a group (single tokens): bound by reading A once. A block has
// R row blocks and CB column blocks of 16; its eight waves share k in runs of
// 256 bytes, load both operands straight into MFMA operand registers, the next
// run ahead of the present one's MFMAs, and add their sums in LDS in the
// waves' order. A k-contiguous only. The loads take any alignment. One column
// of 8192 x 4096 fp4 weights: 5.8 us, 3.1 TB/s of the 18 MB (a launch alone
// is 2 us).
template <class E, int R, int CB>
struct SkinnyKernel {
  static constexpr int kBM = 16 * R, kBN = 16 * CB;
  static constexpr int NW = 8, NT = 64 * NW;
  static constexpr bool kScaled = E::kBits == 4;
  static constexpr int RUN = 256, STEPS = RUN / 64;  // bytes of k, MFMA steps
  static constexpr int LDS = NW * R * CB * 1024;

  struct Operands {
    v4i a[STEPS][R], b[STEPS][CB];
    v4i qa[R], qb[CB];  // the run's scales of a row: a dword a step
  };

  // Chunk at `from` of which `left` elements exist.
  static __device__ __forceinline__ v4i load_cut(const char *from, int64_t left) {
    constexpr int EPC = 128 / E::kBits;
    v4i v = {0, 0, 0, 0};
    if (left >= EPC) {
      v = *reinterpret_cast<const typename E::chunk *>(from);
    } else if (left > 0) {
      if constexpr (E::kBits == 16) {
        typedef short s8 __attribute__((ext_vector_type(8)));
        s8 s = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) s[i] = reinterpret_cast<const short *>(from)[i];
        v = __builtin_bit_cast(v4i, s);
      } else if constexpr (E::kBits == 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < left) v[i] = reinterpret_cast<const int *>(from)[i];
      }
    }
    return v;
  }

  static __device__ __forceinline__ void run(const Args &p, char *smem) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    Tile tile;
    ColumnOrder order;
    order.init(p, kBN);
    if (!order.find(p, blockIdx.x, tile)) return;
    const int64_t m0 = (int64_t)tile.tm * kBM, n0 = tile.lo + (int64_t)tile.tn * kBN;
    const int64_t K = p.alpha == 0.0f ? 0 : p.k;  // alpha == 0 reads neither operand
    const int64_t bytes = (K * E::kBits + 7) / 8;
    const int runs = (int)((bytes + RUN - 1) / RUN), whole = (int)(bytes / RUN);

    // this lane's chunk 0 of its rows and columns; past the end the last one
    // is read again (what it gives is never stored)
    const char *pa[R], *pb[CB];
    const uint8_t *sa[R], *sb[CB];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      int64_t row = m0 + 16 * r + i16;
      if (row >= p.m) row = p.m - 1;
      pa[r] = p.A + (int64_t)tile.g * p.stride_a + row * p.lda + 16 * g;
      if constexpr (kScaled) sa[r] = p.scale_a + (int64_t)tile.g * (p.stride_a / 16) + row * (p.lda / 16);
    }
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      int64_t col = n0 + 16 * c + i16;
      if (col >= tile.hi) col = tile.hi - 1;
      pb[c] = p.B + col * p.ldb + 16 * g;
      if constexpr (kScaled) sb[c] = p.scale_b + col * (p.ldb / 16);
    }
    auto load = [&](int run, Operands &o) {
      const int64_t at = (int64_t)run * RUN;
      if (run < whole) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
#pragma unroll
          for (int r = 0; r < R; ++r) o.a[s][r] = *reinterpret_cast<const typename E::chunk *>(pa[r] + at + 64 * s);
#pragma unroll
          for (int c = 0; c < CB; ++c) o.b[s][c] = *reinterpret_cast<const typename E::chunk *>(pb[c] + at + 64 * s);
        }
        if constexpr (kScaled) {
          typedef int v4d __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
          for (int r = 0; r < R; ++r) o.qa[r] = *reinterpret_cast<const v4d *>(sa[r] + at / 16);
#pragma unroll
          for (int c = 0; c < CB; ++c) o.qb[c] = *reinterpret_cast<const v4d *>(sb[c] + at / 16);
        }
      } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int64_t left = K - (at + 64 * s + 16 * g) * 8 / E::kBits;
#pragma unroll
          for (int r = 0; r < R; ++r) o.a[s][r] = load_cut(pa[r] + at + 64 * s, left);
#pragma unroll
          for (int c = 0; c < CB; ++c) o.b[s][c] = load_cut(pb[c] + at + 64 * s, left);
          if constexpr (kScaled) {
            // fp4: whole steps, K is a multiple of 128
            const bool in = at + 64 * s < bytes;
#pragma unroll
            for (int r = 0; r < R; ++r) o.qa[r][s] = in ? *reinterpret_cast<const int *>(sa[r] + at / 16 + 4 * s) : 0;
#pragma unroll
            for (int c = 0; c < CB; ++c) o.qb[c][s] = in ? *reinterpret_cast<const int *>(sb[c] + at / 16 + 4 * s) : 0;
          }
        }
      }
    };
    f4 acc[R][CB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < CB; ++c) acc[r][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const Operands &o) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < CB; ++c) {
            int qa = 0, qb = 0;
            if constexpr (kScaled) {  // the lane group's byte
              qa = (int)((uint32_t)o.qa[r][s] >> (8 * g));
              qb = (int)((uint32_t)o.qb[c][s] >> (8 * g));
            }
            E::mma(o.a[s][r], o.b[s][c], acc[r][c], 0, 0, qa, 0, qb);
          }
    };
    Operands x, y;
    int run = wave;
    if (run < runs) load(run, x);
    while (run < runs) {
      if (run + NW < runs) load(run + NW, y);
      multiply(x);
      run += NW;
      if (run >= runs) break;
      if (run + NW < runs) load(run + NW, x);
      multiply(y);
      run += NW;
    }

    // the waves' sums, one block (r, c) after the other: lane's f4 as it is
    f4 *sums = reinterpret_cast<f4 *>(smem);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < CB; ++c) sums[(wave * R * CB + r * CB + c) * 64 + lane] = acc[r][c];
    __syncthreads();
    const int64_t cols = tile.hi - n0;
#pragma unroll
    for (int q = 0; q < (R * CB + NW - 1) / NW; ++q) {
      const int at = wave + q * NW;
      if (at >= R * CB) return;
      f4 total[1][1] = {{sums[at * 64 + lane]}};
#pragma unroll
      for (int v = 1; v < NW; ++v) total[0][0] += sums[(v * R * CB + at) * 64 + lane];
      store_tile<E, 16>(p, n0 * p.ldc, total, m0 + 16 * (at / CB), 16 * (at % CB), cols, lane);
    }
  }
};

template <class K>
__global__ __launch_bounds__(K::NT, 2) void ragged_kernel(Args p) {
  extern __shared__ __align__(1024) char ragged_smem[];
  K::run(p, ragged_smem);
}

template <class K>
int launch(wgb_ctx *ctx, const Args &p, int64_t blocks) {
  if (blocks == 0) return WGB_OK;
  if (blocks > INT32_MAX) return wgb::fail(WGB_ERR_INVALID_VALUE, "grouped product: too many tiles");
  // a kernel's LDS size is allowed for each device by itself: a bit for each one where it is
  static std::atomic<uint64_t> allowed{0};
  const uint64_t device = ctx->device < 64 ? (uint64_t)1 << ctx->device : 0;
  if (!(allowed.load(std::memory_order_relaxed) & device)) {
    const hipError_t e =
        hipFuncSetAttribute((const void *)ragged_kernel<K>, hipFuncAttributeMaxDynamicSharedMemorySize, K::LDS);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return wgb::fail_hip(e, "LDS size of a grouped product");
    }
    allowed.fetch_or(device, std::memory_order_relaxed);
  }
  ragged_kernel<K><<<(unsigned)blocks, K::NT, K::LDS, ctx->stream>>>(p);
  WGB_CHECK_LAUNCH("ragged_kernel");
  return WGB_OK;
}

// Tiles that a ragged-columns launch has at most: a group of c columns has
// ceil(c / bn) column tiles, at most one of them partly filled.
inline int64_t most_columns(const Args &p, int64_t bn) {
  return !p.off ? (p.n + bn - 1) / bn : p.n / bn + (p.n < p.groups ? p.n : p.groups);
}

template <class K>
int launch_columns(wgb_ctx *ctx, Args &p) {
  p.tiles_m = (int)((p.m + K::kBM - 1) / K::kBM);
  return launch<K>(ctx, p, most_columns(p, K::kBN) * p.tiles_m);
}

template <class K>
int launch_k(wgb_ctx *ctx, Args &p) {
  p.tiles_m = (int)((p.m + K::kBM - 1) / K::kBM);
  p.tiles_n = (int)((p.n + K::kBN - 1) / K::kBN);
  return launch<K>(ctx, p, (int64_t)p.tiles_m * p.tiles_n * p.groups);
}

// Pieces that k elements are cut into at most: at least 8 k-tiles (of bk) each,
// and 3 of them, for their sums cost a launch.
inline int most_pieces(int64_t k, int bk) {
  const int64_t pieces = k / (8 * bk);
  return pieces < 3 ? 1 : pieces < 8 ? (int)pieces : 8;
}
// Bytes of Args::parts: what the rest's blocks that run at once (two a CU) may hold.
inline size_t parts_bytes(const wgb_ctx *ctx) { return (size_t)ctx->num_cus * 2 * 128 * 128 * 4; }

// `Turn` on at most `tiles` 256 x 256 tiles, a block a CU (more where one
// could not keep its tiles), then `Rest` (128 x 128 tiles, a quarter of one
// each) on what that leaves, and if that may be cut along k, their sums. Which
// tiles there are is only known on the GPU, unless `exact`. k: of a tile, to
// expect.
template <class Turn, class Rest>
int launch_rounds(wgb_ctx *ctx, Args &p, int64_t tiles, bool exact, int64_t k) {
  p.stream = ((uintptr_t)p.C & 63) == 0 && p.ldc * (p.c_f32 ? 4 : 2) % 64 == 0 && p.stride_c * (p.c_f32 ? 4 : 2) % 64 == 0;
  int64_t blocks = tiles;
  if (tiles > ctx->num_cus) {
    blocks = (tiles + kTilesPerBlock - 1) / kTilesPerBlock;
    if (blocks <= ctx->num_cus) blocks = p.round = ctx->num_cus;
  }
  int64_t rest = p.round / 2;  // at most
  if (p.round && exact) {
    const int64_t over = tiles % p.round;
    rest = over > rest ? 0 : over;
  }
  p.pieces = most_pieces(k, Rest::SA::BK);
  if (rest && exact && p.round / (2 * rest) < 3) p.pieces = 1;
  if (rest && p.pieces > 1 && !p.parts) {
    const int st = wgb::ensure_op_workspace(ctx, parts_bytes(ctx));
    if (st == WGB_ERR_ALLOC)
      p.pieces = 1;  // no memory for the sums: nothing is cut
    else if (st)
      return st;
    else
      p.parts = (float *)ctx->op_ws;
  }
  int st = launch<Turn>(ctx, p, blocks);
  if (st || !rest) return st;
  const int64_t slots = 2 * (int64_t)p.round;
  st = launch<Rest>(ctx, p, p.pieces == 1 ? 4 * rest : slots);
  if (st || p.pieces == 1) return st;
  return launch<FoldKernel<Rest>>(ctx, p, (slots / 2 < 4 * rest ? slots / 2 : 4 * rest) * Rest::NB);
}

template <class Turn, class Rest>
int launch_columns_rounds(wgb_ctx *ctx, Args &p) {
  p.tiles_m = (int)((p.m + Turn::kBM - 1) / Turn::kBM);
  return launch_rounds<Turn, Rest>(ctx, p, most_columns(p, Turn::kBN) * p.tiles_m, !p.off, p.k);
}

template <class Turn, class Rest>
int launch_k_rounds(wgb_ctx *ctx, Args &p) {
  p.tiles_m = (int)((p.m + Turn::kBM - 1) / Turn::kBM);
  p.tiles_n = (int)((p.n + Turn::kBN - 1) / Turn::kBN);
  return launch_rounds<Turn, Rest>(ctx, p, (int64_t)p.tiles_m * p.tiles_n * p.groups, true, p.k / p.groups);
}

// Estimated time of a launch of T x T tiles, to choose among sizes: `first` us
// for a tile of k = 1024 alone on its CU, `next` for each further one there
// (several small blocks run at once; 256 x 256 tiles come in whole rounds),
// and the time to write C at the 4.5 TB/s that large results reach. Measured:
//   first / next      64 x 64       128 x 128     256 x 256
//   16-bit            5.4 / 4.1     12.5 / 9.5    23.5
//   fp4               4.0 / 1.5     5.6 / 3.3     10.5
//   fp32              20 / 15.2     64 / 59.3     -
// (us on 256 CUs; bf16 1024^3 8 / 13 / 26 us, 2048^3 33 / 28 / 45 us, 8192 x
// 16384 x 4096 - / 1008 / 759 us; fp4 2048^3 19 / 13 / 25 us, 8192^3 - / 365 /
// 302 us; fp32 1024^3 25 / 68 us, 8192 x 8192 x 2048 1944 / 1891 us).
struct TileCost {
  double first, next;
};
// `tiles`: on each CU.
inline double small_time(int T, TileCost c, double tiles, double k, double c_size) {
  const double store = T * T * c_size / 17.6e3, depth = k / 1024;
  return c.first * depth + store + (tiles > 1 ? tiles - 1 : 0) * (c.next * depth + store);
}
// 256 x 256 tiles: whole rounds (fewer tiles than CUs are one, however few: 512
// x 256 x 8192 in bf16 138 us, on 64 x 64 tiles 58), then the rest as
// launch_rounds has it (cut along k, a piece more than fills its share: 60
// quarters at k = 4096 in 16 bits 30 us and 8 for the sums).
inline double rounds_time(TileCost c256, TileCost c128, double tiles, double k, double c_size, int most) {
  const double store = 256 * 256 * c_size / 17.6e3, round = c256.first * (k / 1024) + store;
  const double whole = (double)(int64_t)tiles, rest = tiles - whole;
  if (whole > 0 && rest < 0.01) return whole * round;
  if (whole > 0 && rest <= 0.17 && most > 1) {
    const double pieces = 0.5 / rest < most ? 0.5 / rest : most;
    return whole * round + (c128.first + c128.next) * (k / 1024) / pieces + 15;
  }
  return whole * round + (rest > 0.5 || whole == 0 ? round : small_time(128, c128, 4 * rest, k, c_size) + 4);
}
inline double per_cu(const wgb_ctx *ctx, const Args &p, int T, double tiles_n) {
  return (double)((p.m + T - 1) / T) * tiles_n / ctx->num_cus;
}
// Column tiles of a ragged launch to expect: every group's last one is half full.
inline double expected_columns(const Args &p, int T) {
  if (!p.off || p.groups == 1) return (double)((p.n + T - 1) / T);
  return (double)p.n / T + 0.5 * (double)(p.n < p.groups ? p.n : p.groups);
}

}  // namespace wgb_ragged
