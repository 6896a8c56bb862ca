// Host build of wgblas_amd/csrc/copy_plan.h for tests/test_copy_plan_fp8.py: the copies that stage 8-bit operands, whose
// columns are whole runs of 128 codes. For every tile shape, layout and small matrix each 16-byte read of every thread and
// k-tile (a cut last one's rows past the end read others) stays inside the matrix, and every code comes from its own
// address. Prints a line for each kind of tile, "ok" and the matrices checked, or the first mistake.
#define __host__
#define __device__
#define __forceinline__ inline
#include <cstdio>

#include "../../wgblas_amd/csrc/copy_plan.h"

using namespace wgb_ragged;

namespace {

const char *const kBase = (const char *)((uintptr_t)1 << 40);

// K: of the k-contiguous layout whole runs; of the row-contiguous one any, and `rows` whole runs.
template <int BT, bool MC, int NT>
bool matrix(int64_t rows, int64_t ld, int64_t K) {
  typedef CopyPlan<8, BT, MC, NT> Plan;
  const int64_t end = MC ? (K - 1) * ld + rows : (rows - 1) * ld + K;
  for (int64_t row0 = 0; row0 < rows; row0 += BT)
    for (int t = 0; t < NT; ++t) {
      Plan p;
      p.init(kBase, ld, row0, rows, K, t);
      const int whole = p.whole_tiles(), tiles = (int)((K + Plan::BK - 1) / Plan::BK);
      if (whole != K / Plan::BK || (tiles > whole && !p.soft_tail())) return false;
      for (int kt = 0; kt < tiles; ++kt)
        for (int r = 0; r < Plan::LOADS; ++r) {
          const int64_t at = p.origin - kBase + kt * p.step() + (int64_t)(int32_t)(kt < whole ? p.voff[r] : p.tail_voff(r));
          if (at < 0 || at + 16 > end) return false;
          const int64_t slot = p.slot_row(r), chunk = p.slot_chunk(r);
          const int64_t row = row0 + (MC ? chunk * 16 : slot), k = (int64_t)kt * Plan::BK + (MC ? slot : chunk * 16);
          if (row < rows && k < K && at != (MC ? k * ld + row : row * ld + k)) return false;
        }
    }
  return true;
}

template <int BT, bool MC, int NT>
void check(const char *name) {
  int64_t done = 0;
  for (int64_t a = 1; a <= 2 * (MC ? 128 : BT) + 3; a += a < 20 ? 1 : 7)  // columns of the matrix
    for (int64_t b = 128; b <= (MC ? 2 * BT + 128 : 512); b += 128)       // codes in a column
      for (int64_t pad = 0; pad <= 256; pad += 128) {
        const int64_t rows = MC ? b : a, K = MC ? a : b;
        if (!matrix<BT, MC, NT>(rows, b + pad, K)) {
          std::printf("%s: rows %lld K %lld ld %lld\n", name, (long long)rows, (long long)K, (long long)(b + pad));
          return;
        }
        ++done;
      }
  std::printf("%s: ok %lld\n", name, (long long)done);
}

}  // namespace

int main() {
  check<32, false, 256>("32");
  check<64, false, 256>("64");
  check<64, true, 256>("64 row-contiguous");
  check<128, false, 256>("128");
  check<128, true, 256>("128 row-contiguous");
  check<256, false, 512>("256");
  check<256, true, 512>("256 row-contiguous");
  return 0;
}
