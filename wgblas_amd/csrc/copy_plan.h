// Addresses of the copies that stage an operand's k-tiles in LDS
// (ragged_tile.h): which 16-byte chunk each thread takes, and which k-tiles
// can be copied without reading outside the matrix.
//
// Included by ragged_tile.h (device code) and compiled for the host by the CPU
// test tests/test_copy_plan.py, which defines the HIP function qualifiers away
// and checks every address against the matrix it is made for.
#pragma once

#include <stdint.h>

namespace wgb_ragged {

// k-tiles are 128 bytes of k: a whole cache line of every row. (Of 64 bytes,
// each line came from L2 twice, once for either half: 8192 x 16384 x 4096 in
// bf16 886 us, of which 180 were the copies'.)
constexpr int TB = 128;

// Chunk keys of the row-contiguous layout, for k-row r of a tile whose rows
// have `chunks` chunks: 16-bit transposing reads touch k-rows 8 g .. 8 g + 3
// (32 bytes of each), fp32 reads k-rows 4 g (64 bytes of each), 8-bit ones
// k-rows 16 g .. 16 g + 7 (16 bytes of each).
template <int BITS, int CHUNKS>
__host__ __device__ __forceinline__ int mc_key(int r) {
  if (BITS == 8) return ((r & 7) | (((r >> 4) & 1) << 3)) & (CHUNKS - 1);
  const int key = BITS == 16 ? ((r & 3) << 1) | (((r >> 3) & 1) << 3) : ((r >> 2) & 3) << 2;
  return key & (CHUNKS - 1);
}

// The chunks of a tile of BT rows of BITS-bit elements, k-contiguous or
// row-contiguous (MC), among NT threads.
template <int BITS, int BT, bool MC, int NT>
struct CopyPlan {
  static constexpr int EPC = 128 / BITS;               // elements in a 16-byte chunk
  static constexpr int BK = TB * 8 / BITS;             // elements of k in a k-tile
  static constexpr int BYTES = BT * TB;                // of a staged tile
  static constexpr int LOADS = BYTES / 16 / NT;        // chunks a thread stages
  static constexpr int CPR = MC ? BT / EPC : TB / 16;  // chunks in a staged row
  static constexpr int RPS = NT / CPR;                 // staged rows in one step of all threads
  static_assert(BYTES % (16 * NT) == 0 && NT % CPR == 0, "whole steps");

  const char *origin;    // element (row0, k = 0)
  int64_t ld;            // bytes
  int64_t rows_left;     // rows from row0 to the end of the matrix
  int64_t K;             // elements
  uint32_t voff[LOADS];  // this lane's chunks of k-tile 0, in bytes from origin
  int t;

  __host__ __device__ __forceinline__ int slot_row(int r) const { return t / CPR + r * RPS; }
  __host__ __device__ __forceinline__ int slot_chunk(int r) const {
    const int row = slot_row(r);
    return (t % CPR) ^ (MC ? mc_key<BITS, CPR>(row) : row & 7);
  }

  __host__ __device__ __forceinline__ void init(const char *P, int64_t ld_, int64_t row0, int64_t rows, int64_t K_,
                                                int t_) {
    t = t_;
    ld = ld_;
    rows_left = rows - row0;
    K = K_;
    origin = MC ? P + row0 * BITS / 8 : P + row0 * ld;
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
  // a last chunk that the end of the rows cuts reads on into the k-rows after
  // it, one where they are 16 bytes apart or more, up to EPC - 1 of them where
  // they are closer (a matrix of 1 to 3 rows). The last k-rows do not have
  // those. 8-bit columns are whole runs of 128 elements: none is cut.
  __host__ __device__ __forceinline__ int whole_tiles() const {
    const bool cut = MC && BITS != 8 && rows_left < BT;
    const int after = !cut ? 0 : ld < 16 ? EPC - 1 : 1;
    return (int)((K > after ? K - after : 0) / BK);
  }

  // Bytes from one k-tile to the next.
  __host__ __device__ __forceinline__ int64_t step() const { return MC ? BK * ld : TB; }

  // A last k-tile that K cuts can be copied too, chunks past K reading one
  // that exists: whoever reads the operands then clears what is past K
  // (tail_mask). Not where a cut chunk could reach past the matrix: at its
  // last row (k-contiguous), or with cut rows (row-contiguous). Columns of
  // 8-bit codes are whole runs of 128: no chunk is cut, and what a k-row past K
  // is multiplied with is zeros; k-contiguous ones have no cut k-tile.
  __host__ __device__ __forceinline__ bool soft_tail() const {
    return BITS == 8 ? MC : MC ? rows_left >= BT : K % EPC == 0 || (rows_left > BT && K >= EPC);
  }
  __host__ __device__ __forceinline__ uint32_t tail_voff(int r) const {
    const int left = (int)(K % BK);
    if (MC) return voff[r] - (slot_row(r) < left ? 0u : (uint32_t)(slot_row(r) * ld));
    return voff[r] - (slot_chunk(r) * EPC < left ? 0u : (uint32_t)(slot_chunk(r) * 16));
  }

  // fp4, a last k-tile of which only the first 64 bytes exist: the other four
  // chunks of a row read those again. What they hold does not matter (a code
  // is never Inf or NaN), for their scales are staged as 2^-127 in both
  // operands, and 36 * 2^-254 is nothing in fp32.
  __host__ __device__ __forceinline__ uint32_t half_voff(int r) const {
    return voff[r] - (slot_chunk(r) >= 4 ? 64u : 0u);
  }

  // Chunk r of k-tile kt: its place from origin, and how many of its elements
  // the matrix has (none or fewer than a chunk's: rows or k end before).
  __host__ __device__ __forceinline__ int64_t guarded(int kt, int r, int64_t &at) const {
    const int row = slot_row(r), chunk = slot_chunk(r);
    if (MC) {
      const int64_t kk = (int64_t)kt * BK + row;
      at = kk * ld + chunk * 16;
      return kk < K ? rows_left - (int64_t)chunk * EPC : 0;
    }
    at = row * ld + (int64_t)kt * TB + chunk * 16;
    return row < rows_left ? K - ((int64_t)kt * BK + (int64_t)chunk * EPC) : 0;
  }
};

}  // namespace wgb_ragged
