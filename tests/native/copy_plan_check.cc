// Host build of wgblas_amd/csrc/copy_plan.h (the copies that stage operands of
// the grouped and 4-bit products) for tests/test_copy_plan.py. For every tile
// shape, layout and small matrix it takes the addresses of all threads' copies
// of the k-tiles that may be copied, of a cut last one, and of the guarded
// loads, and checks that each 16-byte read stays inside the matrix and that
// every element of the matrix comes from its own address. Prints a line for
// each kind of tile, "ok" and the matrices checked, or the first mistake.
#define __host__
#define __device__
#define __forceinline__ inline
#include <cstdio>
#include <vector>

#include "../../wgblas_amd/csrc/copy_plan.h"

using namespace wgb_ragged;

namespace {

const char *const kBase = (const char *)((uintptr_t)1 << 40);

template <int BITS, int BT, bool MC, int NT>
struct Check {
  typedef CopyPlan<BITS, BT, MC, NT> Plan;
  static constexpr int EPC = Plan::EPC, BK = Plan::BK;
  int64_t rows, ld, K;  // ld in elements
  int64_t row0;
  char error[512];

  int64_t bytes(int64_t elements) const { return elements * BITS / 8; }
  int64_t end() const { return MC ? bytes((K - 1) * ld + rows) : bytes((rows - 1) * ld + K); }

  // A 16-byte read of k-tile kt by slot (t, r) at `at` from the matrix's start.
  bool read(const char *kind, const Plan &p, int kt, int r, int64_t at, int64_t size) {
    if (at >= 0 && at + size <= end()) return true;
    std::snprintf(error, sizeof(error), "%s: rows %lld ld %lld K %lld row0 %lld k-tile %d thread %d load %d reads %lld..%lld of %lld",
                  kind, (long long)rows, (long long)ld, (long long)K, (long long)row0, kt, p.t, r, (long long)at,
                  (long long)(at + size), (long long)end());
    return false;
  }
  // Where the slot's chunk has an element of the matrix, `at` has to be that element's address.
  bool own(const char *kind, const Plan &p, int kt, int r, int64_t at) {
    const int64_t slot = p.slot_row(r), chunk = p.slot_chunk(r);
    const int64_t row = row0 + (MC ? chunk * EPC : slot), k = (int64_t)kt * BK + (MC ? slot : chunk * EPC);
    if (row >= rows || k >= K || at == (MC ? bytes(k * ld + row) : bytes(row * ld + k))) return true;
    std::snprintf(error, sizeof(error), "%s: rows %lld ld %lld K %lld row0 %lld k-tile %d thread %d load %d has another's address",
                  kind, (long long)rows, (long long)ld, (long long)K, (long long)row0, kt, p.t, r);
    return false;
  }

  bool matrix() {
    for (row0 = 0; row0 < rows; row0 += BT) {
      for (int t = 0; t < NT; ++t) {
        Plan p;
        p.init(kBase, bytes(ld), row0, rows, K, t);
        const int whole = p.whole_tiles(), tiles = (int)((K + BK - 1) / BK);
        const bool soft = K % BK != 0 && whole == tiles - 1 && p.soft_tail();
        for (int kt = 0; kt < tiles; ++kt)
          for (int r = 0; r < Plan::LOADS; ++r) {
            const int64_t from = p.origin - kBase + kt * p.step();
            if (kt < whole) {
              const int64_t at = from + p.voff[r];
              if (!read("copy", p, kt, r, at, 16) || !own("copy", p, kt, r, at)) return false;
            } else if (BITS == 4) {
              const int64_t at = from + p.half_voff(r);
              if (!read("half", p, kt, r, at, 16) || !own("half", p, kt, r, at)) return false;
            } else if (soft) {
              const int64_t at = from + (int32_t)p.tail_voff(r);
              if (!read("tail", p, kt, r, at, 16) || !own("tail", p, kt, r, at)) return false;
            }
            if (BITS != 4) {  // whatever the k-tile: operands that cannot be copied go this way alone
              int64_t at;
              const int64_t left = p.guarded(kt, r, at);
              if (left <= 0) continue;
              at += p.origin - kBase;
              const int64_t n = left < EPC ? left : EPC;
              if (!read("guarded", p, kt, r, at, bytes(n)) || !own("guarded", p, kt, r, at)) return false;
            }
          }
      }
    }
    return true;
  }
};

template <int BITS, int BT, bool MC, int NT>
bool check(const char *name) {
  Check<BITS, BT, MC, NT> c;
  constexpr int EPC = 128 / BITS, BK = 128 * 8 / BITS;
  // copies start at whole dwords; fp4 columns hold whole runs of 128
  constexpr int unit = BITS == 32 ? 1 : BITS == 16 ? 2 : 128, kstep = BITS == 4 ? 128 : 1;
  std::vector<int64_t> rows, ks, pads;
  for (int64_t r = 1; r <= 2 * EPC + 2; ++r) rows.push_back(r);
  for (int64_t r : {BT - EPC - 1, BT - EPC, BT - 1, BT, BT + 1, BT + EPC - 1, 2 * BT, 2 * BT + 3}) rows.push_back(r);
  for (int64_t k = kstep; k <= 8 * kstep; k += kstep) ks.push_back(k);
  for (int64_t b : {BK, 2 * BK, 3 * BK})
    for (int64_t d = -EPC - 1; d <= EPC + 1; ++d)
      if (BITS != 4 || d % kstep == 0) ks.push_back(b + d);
  if (BITS == 4) ks.insert(ks.end(), {BK + 128, 2 * BK + 128});
  for (int64_t pad = 0; pad <= (BITS == 4 ? 128 : EPC + 1); pad += BITS == 4 ? 128 : 1) pads.push_back(pad);
  int64_t done = 0;
  for (int64_t r : rows)
    for (int64_t k : ks)
      for (int64_t pad : pads) {
        if (r <= 0 || k <= 0) continue;
        c.rows = r;
        c.K = k;
        c.ld = (MC ? r : k) + pad;
        if (c.ld % unit) continue;
        if (!c.matrix()) {
          std::printf("%s: %s\n", name, c.error);
          return false;
        }
        ++done;
      }
  std::printf("%s: ok %lld\n", name, (long long)done);
  return true;
}

}  // namespace

int main() {
  // the tiles that grouped.hip and mxfp4.hip launch: sides, waves, layouts
  check<32, 64, false, 256>("fp32 64");
  check<32, 64, true, 256>("fp32 64 row-contiguous");
  check<32, 128, false, 256>("fp32 128");
  check<32, 128, true, 256>("fp32 128 row-contiguous");
  check<32, 32, false, 256>("fp32 32");
  check<16, 64, false, 256>("16-bit 64");
  check<16, 64, true, 256>("16-bit 64 row-contiguous");
  check<16, 128, false, 256>("16-bit 128");
  check<16, 128, true, 256>("16-bit 128 row-contiguous");
  check<16, 32, false, 256>("16-bit 32");
  check<16, 256, false, 512>("16-bit 256");
  check<16, 256, true, 512>("16-bit 256 row-contiguous");
  check<4, 64, false, 256>("fp4 64");
  check<4, 128, false, 256>("fp4 128");
  check<4, 32, false, 256>("fp4 32");
  check<4, 256, false, 512>("fp4 256");
  return 0;
}
