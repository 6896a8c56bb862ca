// Routing tokens to experts: the choice of each token's experts and their
// weights (wgb_route), its gradient (wgb_route_grad), the order of the pairs
// (token, expert) by expert (wgb_route_order), and the tokens' way to the
// experts' columns and back (wgb_route_gather, wgb_route_combine,
// wgb_route_combine_grad).
//
// wgblas has no counterpart. These are what stands before and behind the
// grouped products (grouped.hip, mxfp4.hip, fp8.hip): their boundaries and
// the order of their columns are this file's results, and stay on the GPU.
#include "common.h"

#include <type_traits>

namespace {

using wgb::fail;

constexpr int kMaxExperts = 1024, kMaxTopk = 64, kMaxGroups = 64;

// ---- reductions over the lanes of a token ------------------------------------

// All lanes of each run of LPT (16 or 64) lanes get op over the run. The 16
// lanes of a DPP row are rotated onto each other; rows meet by shuffles.
template <int ROR>
__device__ __forceinline__ float ror(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + ROR, 0xf, 0xf, true));
}
template <int ROR>
__device__ __forceinline__ int ror(int x) {
  return __builtin_amdgcn_mov_dpp(x, 0x120 + ROR, 0xf, 0xf, true);
}
template <int ROR>
__device__ __forceinline__ double ror(double x) {
  typedef int i2 __attribute__((ext_vector_type(2)));
  i2 v = __builtin_bit_cast(i2, x);
  v[0] = __builtin_amdgcn_mov_dpp(v[0], 0x120 + ROR, 0xf, 0xf, true);
  v[1] = __builtin_amdgcn_mov_dpp(v[1], 0x120 + ROR, 0xf, 0xf, true);
  return __builtin_bit_cast(double, v);
}
template <int LPT, class T, class Op>
__device__ __forceinline__ T over_lanes(T x, Op op) {
  x = op(x, ror<8>(x));
  x = op(x, ror<4>(x));
  x = op(x, ror<2>(x));
  x = op(x, ror<1>(x));
  if constexpr (LPT == 64) {
    x = op(x, __shfl_xor(x, 16));
    x = op(x, __shfl_xor(x, 32));
  }
  return x;
}
struct Max {
  template <class T>
  __device__ T operator()(T a, T b) const {
    return a > b ? a : b;
  }
};
struct Sum {
  template <class T>
  __device__ T operator()(T a, T b) const {
    return a + b;
  }
};
// The lowest lane of this token's run for which `hit` holds, counted in the
// run; LPT where none.
template <int LPT>
__device__ __forceinline__ int first_lane(bool hit, int lane) {
  uint64_t b = __ballot(hit);
  if constexpr (LPT == 64) return b ? __builtin_ctzll(b) : LPT;
  const uint32_t mine = (uint32_t)(b >> (lane & 48)) & 0xffffu;
  return mine ? __builtin_ctz(mine) : LPT;
}

// ---- the choice ----------------------------------------------------------------

struct RouteArgs {
  const void *logits;
  int64_t ldl, n;
  const float *bias;
  int experts, topk, groups, top_groups, best, per;
  uint32_t magic;  // e / per = e * magic >> 20 for e < 1024
  int sigmoid, renorm;
  float scale;
  int32_t *ids;
  float *weights;
};

// A token's lanes are in one wave: what one has stored in LDS the others read
// behind this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What is compared: whole numbers in the order of fp32 values (zeros of either
// sign are equal, NaN comes after all numbers), or fp64 values themselves.
template <class F>
struct Keys;
template <>
struct Keys<float> {
  typedef int key;
  static constexpr int kNone = (int)0x80000000;  // not there
  static constexpr int kNan = kNone + 1;
  static constexpr int kPart = kNone + 2;  // of a group: a number and a NaN
  static __device__ __forceinline__ int of(float x) {
    const int b = __float_as_int(x + 0.0f);
    return x != x ? kNan : x == -__builtin_inff() ? kNone : b ^ ((b >> 31) & 0x7fffffff);
  }
  static __device__ __forceinline__ float value(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
  // of a group: half the sum of its two best (the sum may be past fp32); scores that are NaN come after all numbers there, too
  static __device__ __forceinline__ int sum(int a, int b) {
    if (a == kNone || b == kNone) return kNone;
    if (b == kNan) return a == kNan ? kNan : kPart;
    return of(0.5f * value(a) + 0.5f * value(b));
  }
};
template <>
struct Keys<double> {
  typedef double key;
  static constexpr double kNone = -__builtin_inf(), kNan = -1e300, kPart = -1e299;
  static __device__ __forceinline__ double of(double x) { return x != x ? kNan : x; }
  static __device__ __forceinline__ double sum(double a, double b) {
    if (a == kNone || b == kNone) return kNone;
    if (b == kNan) return a == kNan ? kNan : kPart;
    return a + b;
  }
};

// Room of a token in LDS: its values, and its groups' scores (fp64 ones, or fp32 ones and their sizes).
template <class F>
struct Room {
  static __host__ __device__ int values(int experts) { return (experts + 3) & ~3; }
  static __host__ __device__ size_t bytes(int experts, int groups) {
    return (values(experts) + ((groups + 3) & ~3)) * sizeof(F);
  }
};

// How far two choice values have to be apart so that fp32 tells which is the
// larger: a score is off by at most 4 units of 2^-24 (sigmoid: the exponential
// by |x| 2^-23 of itself, which p (1 - p) |x| < 0.3 makes 0.6 units, the
// reciprocal by 2; softmax: 26 with the sum's), the value by half a unit more,
// and twice that is doubled. Half the sum of two values is off by half of what
// they are, whatever it is itself: `value` is half the sum of their magnitudes
// there, for large ones of different signs leave a small sum.
__device__ __forceinline__ float unsure(float value, int sigmoid) {
  return ((sigmoid ? 4.0f : 32.0f) + fabsf(value)) * 0x1p-22f;
}

// The two best of a run of values, a >= b.
template <class K>
__device__ __forceinline__ void best_two(K &a, K &b, K x, K y) {
  const K low = a < x ? a : x;
  a = a < x ? x : a;
  b = b < y ? y : b;
  b = b < low ? low : b;
}

// What a lane knows of its values: bit j of value j.
struct Groups {
  uint32_t kept;   // in one of the top_groups best groups
  uint32_t best;   // may be one of its group's best
  bool close;      // a kept group and one that is not are too near to tell (fp32)
};

template <class F, int LPT, int PER>
__device__ __forceinline__ Groups keep_groups(const RouteArgs &p, char *room, int lane, const typename Keys<F>::key (&v)[PER]) {
  typedef typename Keys<F>::key K;
  K *values = reinterpret_cast<K *>(room), *score = values + Room<K>::values(p.experts);
  float *size = reinterpret_cast<float *>(score + ((p.groups + 3) & ~3));  // fp32: half the two values' magnitudes
  const int e0 = lane * PER, lanes = p.per / PER;  // of a group, where groups are whole lanes
  const bool two = p.best == 2 && p.per > 1;
  auto put_score = [&](int i, K a, K b) {
    score[i] = two ? Keys<F>::sum(a, b) : a;
    if constexpr (std::is_same<F, float>::value) {
      if (two) size[i] = 0.5f * fabsf(Keys<F>::value(a)) + 0.5f * fabsf(Keys<F>::value(b));
    }
  };
  Groups g = {0, (1u << PER) - 1, false};
  const bool whole = lanes * PER == p.per && (lanes & (lanes - 1)) == 0;
  if (whole) {
    K a = v[0], b = Keys<F>::kNone;
#pragma unroll
    for (int j = 1; j < PER; ++j) best_two(a, b, v[j], Keys<F>::kNone);
    for (int d = 1; d < lanes; d <<= 1) best_two(a, b, (K)__shfl_xor(a, d), (K)__shfl_xor(b, d));
    if ((lane & (lanes - 1)) == 0 && e0 < p.experts) put_score(e0 / p.per, a, b);
    if constexpr (std::is_same<F, float>::value) {
      if (b > Keys<F>::kNan) {
        const K least = Keys<F>::of(Keys<F>::value(b) - unsure(Keys<F>::value(b), p.sigmoid));
        g.best = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) g.best |= v[j] >= least ? 1u << j : 0u;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e0 + j < p.experts) values[e0 + j] = v[j];
    wave_sync();
    for (int i = lane; i < p.groups; i += LPT) {
      K a = Keys<F>::kNone, b = a;
      for (int j = 0; j < p.per; ++j) best_two(a, b, values[i * p.per + j], Keys<F>::kNone);
      put_score(i, a, b);
    }
  }
  wave_sync();
  // whether group i is kept; the least that a kept one's score may be, the most that another's may be (a score that is
  // no number is behind all others, whatever those are off by)
  float least = __builtin_inff(), next = -__builtin_inff();
  auto kept = [&](int i) {
    const K mine = score[i];
    int before = 0;
    for (int o = 0; o < p.groups; ++o) before += score[o] > mine || (score[o] == mine && o < i);
    const bool in = before < p.top_groups;
    if constexpr (std::is_same<F, float>::value) {
      if (mine > Keys<F>::kPart) {
        const float x = Keys<F>::value(mine), off = unsure(two ? size[i] : x, p.sigmoid);
        if (in)
          least = fminf(least, x - off);
        else
          next = fmaxf(next, x + off);
      }
    }
    return in;
  };
  if (whole) {
    if (e0 < p.experts && kept(e0 / p.per)) g.kept = (1u << PER) - 1;
  } else {
    int of = -1;
    bool in = false;
#pragma nounroll
    for (int j = 0; j < PER && e0 + j < p.experts; ++j) {
      const int i = (int)(((uint32_t)(e0 + j) * p.magic) >> 20);
      if (i != of) in = kept(of = i);
      g.kept |= in ? 1u << j : 0u;
    }
  }
  if constexpr (std::is_same<F, float>::value) g.close = -over_lanes<LPT>(-least, Max()) <= over_lanes<LPT>(next, Max());
  wave_sync();
  return g;
}

// The topk largest, one a round, the lowest expert of equal ones, into
// chosen[]. fp32 values that are not exact: `may` gets a lane's values that may
// be among them, and the result is whether two of them, or the last one and the
// next, are too near to tell.
template <class F, int LPT, int PER>
__device__ __forceinline__ bool choose(const RouteArgs &p, int lane, int wave_lane, typename Keys<F>::key (&v)[PER],
                                       int *chosen, uint32_t &may) {
  typedef typename Keys<F>::key K;
  bool close = false;
  K last = Keys<F>::kNone;
  may = 0;
  for (int s = 0; s <= p.topk; ++s) {
    K best = v[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) best = v[j] > best ? v[j] : best;
    const K most = over_lanes<LPT>(best, Max());
    const bool any = most != Keys<F>::kNone;
    if constexpr (std::is_same<F, float>::value) {
      if (s > 0 && any) close |= Keys<F>::value(last) - Keys<F>::value(most) <= unsure(Keys<F>::value(most), p.sigmoid);
      if (s == p.topk && close) {
        const K least = Keys<F>::of(Keys<F>::value(last) - unsure(Keys<F>::value(last), p.sigmoid));
#pragma unroll
        for (int j = 0; j < PER; ++j) may |= v[j] != Keys<F>::kNone && (last <= Keys<F>::kNan || v[j] >= least) ? 1u << j : 0u;
      }
    }
    last = any ? most : last;
    if (s == p.topk) break;
    const bool mine = any && first_lane<LPT>(best == most, wave_lane) == lane;
    // the lowest of the lane's that is the largest, as masks of lanes
    uint64_t open = __ballot(mine);
    int at = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint64_t hit = __ballot(v[j] == most) & open;
      open &= ~hit;
      const bool here = __builtin_amdgcn_inverse_ballot_w64(hit);
      v[j] = here ? Keys<F>::kNone : v[j];
      at = here ? j : at;
    }
    if (mine) may |= 1u << at;
    if (any ? mine : lane == 0) chosen[s] = any ? lane * PER + at : -1;
  }
  return close;
}

// PER values of a row from e0, `none` past its end; any alignment.
template <class T, int PER>
__device__ __forceinline__ void load_row(const T *x, int e0, int experts, float none, float (&l)[PER]) {
  if (e0 + PER <= experts) {
    struct __attribute__((packed, aligned(sizeof(T)))) V {
      T v[PER];
    };
    const V v = *reinterpret_cast<const V *>(x + e0);
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = (float)v.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = e0 + j < experts ? (float)x[e0 + j] : none;
  }
}

// The chosen experts' scores, a lane a slot: l[r] the logit of slot lane + r LPT
// or -Inf, `top` and `total` the row's of the softmax (total 1 for sigmoids).
// `relative`: to the largest of them, for weights that are divided by their sum:
// the scores themselves may all be below fp32's least number (sigmoids from -104
// down; softmax where a bias or the groups keep the largest logits out). As 64
// bits have it, what is below their least number is 0: a logit of the type's
// lowest value is a mask. A softmax with a NaN or an Inf has no scores.
constexpr float kLeastLogit = -745.0f;
template <int LPT, int SLOTS>
__device__ __forceinline__ void slot_scores(const float (&l)[SLOTS], bool sigmoid, bool relative, float top, float total,
                                            float (&w)[SLOTS]) {
  const float zero = sigmoid ? 0.0f : top;
  float shift = zero;
  if (relative) {
    float most = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < SLOTS; ++r)
      if (!(l[r] - zero < kLeastLogit)) most = fmaxf(most, l[r]);
    most = over_lanes<LPT>(most, Max());
    shift = sigmoid ? fminf(most, 0.0f) : most;
  }
#pragma unroll
  for (int r = 0; r < SLOTS; ++r) {
    const float r1 = 1.0f / (1.0f + expf(-fabsf(l[r]))), e = expf(l[r] - shift);
    w[r] = l[r] - zero < kLeastLogit ? 0.0f : sigmoid ? (l[r] < 0.0f ? e * r1 : r1) : relative ? e : e / total;
    if (l[r] != -__builtin_inff()) w[r] += total - total;
  }
}

// LPT lanes a token, PER consecutive experts a lane. A token's choice values
// stay in its lanes' registers; each round takes the largest.
//
// Scores grow with the logits, so without a bias and with groups by their best
// expert the logits themselves decide, exactly. Otherwise (WIDE) score + bias
// do, or sums of two scores, and values next to each other are told apart in 64
// bits: fp32 ones first, and where two that matter are within what those may be
// off (0.1% of tokens with 256 experts, all with equal ones), fp64 ones of the
// values that may be chosen, one at a time: few, and the code short, for it is
// seldom run and comes from beyond the instruction cache (fp64 values of all 256
// experts of such tokens alone: 10 us, for 16384 tokens that otherwise take 16).
// Bound by the rounds' compares: 22.7 us for those tokens with 8 groups and a
// bias (0.8 TB/s), 3.5 for 16 tokens of 64 experts.
template <class T, bool WIDE, int LPT, int PER>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs p) {
  constexpr int TOKENS = 256 / LPT;
  typedef typename std::conditional<WIDE, double, int>::type Widest;
  __shared__ int chosen[TOKENS][kMaxTopk];
  extern __shared__ __align__(16) char route_smem[];  // WIDE or with groups: a Room for each token
  const int lane = threadIdx.x % LPT, slot = threadIdx.x / LPT, wave_lane = threadIdx.x & 63;
  const int64_t token = (int64_t)blockIdx.x * TOKENS + slot;
  const bool here = token < p.n;
  const T *x = (const T *)p.logits + (here ? token : p.n - 1) * p.ldl;
  const int e0 = lane * PER;
  char *room = route_smem + slot * Room<Widest>::bytes(p.experts, p.groups);

  float l[PER];
  load_row<T, PER>(x, e0, p.experts, -__builtin_inff(), l);

  // softmax: the largest logit and the sum of exponentials
  float top = 0.0f, total = 1.0f;
  if (!p.sigmoid) {
    top = l[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) top = fmaxf(top, l[j]);
    top = over_lanes<LPT>(top, Max());
    if (top == -__builtin_inff()) top = 0.0f;  // no expert at all: scores of zero
    total = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) total += __expf(l[j] - top);
    total = over_lanes<LPT>(total, Sum());
    if (total == 0.0f) total = 1.0f;
  }

  int v[PER];
  uint32_t may;
  if constexpr (!WIDE) {
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = Keys<float>::of(l[j]);
    if (p.groups > 1) {
      const Groups g = keep_groups<float, LPT, PER>(p, room, lane, v);
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = g.kept >> j & 1 ? v[j] : Keys<float>::kNone;
    }
    choose<float, LPT, PER>(p, lane, wave_lane, v, chosen[slot], may);
  } else {
    float b[PER];
    if (p.bias) {
      load_row<float, PER>(p.bias, e0, p.experts, 0.0f, b);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) b[j] = 0.0f;
    }
    const float inverse = __builtin_amdgcn_rcpf(total);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float s = p.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __expf(-l[j])) : __expf(l[j] - top) * inverse;
      v[j] = l[j] == -__builtin_inff() ? Keys<float>::kNone : Keys<float>::of(s + b[j]);
    }
    // the fp64 values of those of `which`, the others none
    double w[PER];
    auto exact = [&](uint32_t which) {
      auto score = [&](float y) { return p.sigmoid ? 1.0 / (1.0 + exp(-(double)y)) : exp((double)y - (double)top); };
      double *values = reinterpret_cast<double *>(room), sum = 1.0;
      if (!p.sigmoid) {
        sum = 0.0;
#pragma nounroll
        for (int j = 0; j < PER && e0 + j < p.experts; ++j) sum += score((float)x[e0 + j]);
        sum = over_lanes<LPT>(sum, Sum());
        if (sum == 0.0) sum = 1.0;
      }
#pragma nounroll
      for (uint32_t left = e0 < p.experts ? which : 0; left; left &= left - 1) {
        const int e = e0 + __builtin_ctz(left);
        if (e < p.experts) values[e] = score((float)x[e]) / sum + (p.bias ? (double)p.bias[e] : 0.0);
      }
#pragma unroll
      for (int j = 0; j < PER; ++j)
        w[j] = (which >> j & 1) && l[j] != -__builtin_inff() ? Keys<double>::of(values[e0 + j]) : Keys<double>::kNone;
      wave_sync();
    };
    uint32_t kept = (1u << PER) - 1;
    if (p.groups > 1) {
      const Groups g = keep_groups<float, LPT, PER>(p, room, lane, v);
      kept = g.kept;
      if (__ballot(g.close)) {
        exact(g.best);
        kept = keep_groups<double, LPT, PER>(p, room, lane, w).kept;
      }
    }
    // without a bias the logits decide in the groups that stay, among scores that are numbers
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!p.bias && v[j] > Keys<float>::kNan) v[j] = Keys<float>::of(l[j]);
      v[j] = kept >> j & 1 ? v[j] : Keys<float>::kNone;
    }
    const bool close = choose<float, LPT, PER>(p, lane, wave_lane, v, chosen[slot], may);
    if (p.bias && __ballot(close)) {
      exact(may);
      choose<double, LPT, PER>(p, lane, wave_lane, w, chosen[slot], may);
    }
  }
  wave_sync();

  // the weights, a lane a choice
  float c[kMaxTopk / LPT], w[kMaxTopk / LPT], sum = 0.0f;
#pragma unroll
  for (int r = 0; r < kMaxTopk / LPT; ++r) {
    const int s = lane + r * LPT;
    c[r] = s < p.topk && chosen[slot][s] >= 0 ? (float)x[chosen[slot][s]] : -__builtin_inff();
  }
  slot_scores<LPT>(c, p.sigmoid, p.renorm, top, total, w);
#pragma unroll
  for (int r = 0; r < kMaxTopk / LPT; ++r) sum += w[r];
  if (p.renorm) {
    sum = over_lanes<LPT>(sum, Sum());
    if (sum == 0.0f) sum = 1.0f;
  } else {
    sum = 1.0f;
  }
#pragma unroll
  for (int r = 0; r < kMaxTopk / LPT; ++r) {
    const int s = lane + r * LPT;
    if (here && s < p.topk) {
      p.ids[token * p.topk + s] = chosen[slot][s];
      p.weights[token * p.topk + s] = w[r] / sum * p.scale;
    }
  }
}

template <class T, bool WIDE, int LPT, int PER>
int launch_route(wgb_ctx *ctx, const RouteArgs &p) {
  constexpr int TOKENS = 256 / LPT;
  const size_t room = WIDE ? Room<double>::bytes(p.experts, p.groups) : p.groups > 1 ? Room<int>::bytes(p.experts, p.groups) : 0;
  route_kernel<T, WIDE, LPT, PER><<<(unsigned)((p.n + TOKENS - 1) / TOKENS), 256, TOKENS * room, ctx->stream>>>(p);
  WGB_CHECK_LAUNCH("route_kernel");
  return WGB_OK;
}

template <class T, bool WIDE>
int route_sizes(wgb_ctx *ctx, const RouteArgs &p) {
  if (p.experts <= 16) return launch_route<T, WIDE, 16, 1>(ctx, p);
  if (p.experts <= 32) return launch_route<T, WIDE, 16, 2>(ctx, p);
  if (p.experts <= 64) return launch_route<T, WIDE, 16, 4>(ctx, p);
  if (p.experts <= 128) return launch_route<T, WIDE, 16, 8>(ctx, p);
  if (p.experts <= 256) return launch_route<T, WIDE, 16, 16>(ctx, p);
  if (p.experts <= 512) return launch_route<T, WIDE, 64, 8>(ctx, p);
  return launch_route<T, WIDE, 64, 16>(ctx, p);
}

template <class T>
int route(wgb_ctx *ctx, const RouteArgs &p) {
  const bool wide = p.bias || (p.groups > 1 && p.best == 2);
  return wide ? route_sizes<T, true>(ctx, p) : route_sizes<T, false>(ctx, p);
}

// ---- its gradient -----------------------------------------------------------------

struct GradArgs {
  const void *logits;
  int64_t ldl, n;
  const int32_t *ids;
  const float *dweights;
  void *dlogits;
  int64_t ldd;
  int experts, topk, sigmoid, renorm;
  float scale;
};

// With p the scores and d_s what came back for weight s (times scale): a chosen
// score's gradient is d_s; sigmoid: the chosen logits get d p (1 - p), the others
// 0; softmax: every logit p (d - sum_r d_r p_r). With renormalised weights w = p /
// S the sum of d_r w_r is taken from d_s, and p / S is w again: the chosen logits
// get w_s (d_s - sum_r d_r w_r), times 1 - p of the sigmoid, the others nothing,
// and neither S nor the scores need be in fp32's range.
// Where one expert has nearly all of the softmax or of S, that difference is of
// nearly equal numbers. The weights add up to 1, the chosen scores to 1 less the
// others' (R), so it is written as a sum that does not cancel: sum_r w_r (d_s -
// d_r), and sum_r p_r (d_s - d_r) + d_s R. An expert that is there twice has the
// sum of its slots, in their order.
// A row is read and written once, in registers (16384 rows of 128 fp32 logits:
// 7.9 us from call to call, 2.3 TB/s, and 7.1 with differences of sums; as short
// as it is, nearly half of that is the launch and the first loads' way).
template <class T, int LPT, int PER>
__global__ __launch_bounds__(256) void route_grad_kernel(GradArgs p) {
  constexpr int TOKENS = 256 / LPT, SLOTS = kMaxTopk / LPT;
  __shared__ float q[TOKENS][kMaxTopk], share[TOKENS][kMaxTopk];
  __shared__ int at[TOKENS][kMaxTopk];
  __shared__ float back[TOKENS][LPT * PER];
  const int lane = threadIdx.x % LPT, slot = threadIdx.x / LPT;
  const int64_t token = (int64_t)blockIdx.x * TOKENS + slot;
  const bool here = token < p.n;
  const int64_t row = here ? token : p.n - 1;
  const T *x = (const T *)p.logits + row * p.ldl;
  const int e0 = lane * PER;
  float l[PER];
  load_row<T, PER>(x, e0, p.experts, -__builtin_inff(), l);
  // softmax: scores; sigmoid: what an expert's slots are multiplied by
  float s[PER], slope[PER], top = 0.0f, total = 1.0f;
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float t = expf(-fabsf(l[j])), r = 1.0f / (1.0f + t);
      slope[j] = p.renorm ? (l[j] < 0.0f ? r : t * r) : t * r * r;
    }
  } else {
    top = l[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) top = fmaxf(top, l[j]);
    top = over_lanes<LPT>(top, Max());
    if (top == -__builtin_inff()) top = 0.0f;
    total = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) total += s[j] = expf(l[j] - top);
    total = over_lanes<LPT>(total, Sum());
    if (total == 0.0f) total = 1.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] /= total;
  }
  // the chosen scores: a lane a slot
  float c[SLOTS], w[SLOTS], d[SLOTS], sum = 0.0f;
  int id[SLOTS];
#pragma unroll
  for (int r = 0; r < SLOTS; ++r) {
    const int i = lane + r * LPT;
    c[r] = -__builtin_inff();
    d[r] = 0.0f;
    id[r] = i < p.topk ? p.ids[row * p.topk + i] : -1;
    if (id[r] >= p.experts) id[r] = -1;
    if (id[r] >= 0) {
      c[r] = (float)x[id[r]];
      d[r] = p.dweights[row * p.topk + i];
    }
  }
  slot_scores<LPT>(c, p.sigmoid, p.renorm, top, total, w);
  if (p.renorm) {
#pragma unroll
    for (int r = 0; r < SLOTS; ++r) sum += w[r];
    sum = over_lanes<LPT>(sum, Sum());
#pragma unroll
    for (int r = 0; r < SLOTS; ++r) w[r] /= sum == 0.0f ? 1.0f : sum;
  }
  auto each_slot = [&](auto f) {
#pragma unroll
    for (int r = 0; r < SLOTS; ++r)
      if (lane + r * LPT < p.topk) f(r, lane + r * LPT);
  };
  // sum over the slots of share (x - q)
  auto differences = [&](float x) {
    float all = 0.0f;
    for (int i = 0; i < p.topk; ++i) all = fmaf(share[slot][i], x - q[slot][i], all);
    return all;
  };
  each_slot([&](int r, int i) {
    at[slot][i] = id[r];
    q[slot][i] = d[r];
    share[slot][i] = w[r];
  });
#pragma unroll
  for (int j = 0; j < PER; ++j) back[slot][e0 + j] = 0.0f;
  wave_sync();
  if (p.renorm) {
    each_slot([&](int r, int) { d[r] = w[r] * differences(d[r]); });
    wave_sync();
    each_slot([&](int r, int i) { q[slot][i] = d[r]; });
    wave_sync();
  }
  uint32_t mine = 0;
  for (int i = 0; i < p.topk; ++i) {  // each expert's lane adds its own
    const int e = at[slot][i];
    if (e < e0 || e >= e0 + PER) continue;
    back[slot][e] += q[slot][i];
    if (mine >> (e - e0) & 1) share[slot][i] = 0.0f;  // its score counts once
    mine |= 1u << (e - e0);
  }
  float inner = 0.0f, rest = 0.0f;
  if (!p.sigmoid && !p.renorm) {
#pragma unroll
    for (int j = 0; j < PER; ++j) rest += mine >> j & 1 ? 0.0f : s[j];
    rest = over_lanes<LPT>(rest, Sum());
    wave_sync();
    each_slot([&](int r, int i) {
      d[r] = id[r] >= 0 ? back[slot][id[r]] : 0.0f;
      q[slot][i] = d[r];
      inner += share[slot][i] * d[r];
    });
    inner = over_lanes<LPT>(inner, Sum());
    wave_sync();
    each_slot([&](int r, int) {
      if (id[r] >= 0) back[slot][id[r]] = differences(d[r]) + d[r] * rest;
    });
    wave_sync();
  }
  if (!here) return;
  T out[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float g = back[slot][e0 + j];
    // (total - total: 0, or NaN where the softmax has no scores)
    const float y = p.sigmoid ? g * slope[j] : p.renorm ? g + (total - total) : s[j] * (mine >> j & 1 ? g : -inner);
    out[j] = (T)wgb::in_fp32(y * p.scale);
  }
  T *y = (T *)p.dlogits + token * p.ldd;
  if (e0 + PER <= p.experts) {
    struct __attribute__((packed, aligned(sizeof(T)))) V {
      T v[PER];
    };
    V v;
#pragma unroll
    for (int j = 0; j < PER; ++j) v.v[j] = out[j];
    *reinterpret_cast<V *>(y + e0) = v;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e0 + j < p.experts) y[e0 + j] = out[j];
  }
}

template <class T, int LPT, int PER>
int launch_grad(wgb_ctx *ctx, const GradArgs &p) {
  constexpr int TOKENS = 256 / LPT;
  route_grad_kernel<T, LPT, PER><<<(unsigned)((p.n + TOKENS - 1) / TOKENS), 256, 0, ctx->stream>>>(p);
  WGB_CHECK_LAUNCH("route_grad_kernel");
  return WGB_OK;
}

template <class T>
int grad(wgb_ctx *ctx, const GradArgs &p) {
  if (p.experts <= 16) return launch_grad<T, 16, 1>(ctx, p);
  if (p.experts <= 32) return launch_grad<T, 16, 2>(ctx, p);
  if (p.experts <= 64) return launch_grad<T, 16, 4>(ctx, p);
  if (p.experts <= 128) return launch_grad<T, 16, 8>(ctx, p);
  if (p.experts <= 256) return launch_grad<T, 16, 16>(ctx, p);
  if (p.experts <= 512) return launch_grad<T, 64, 8>(ctx, p);
  return launch_grad<T, 64, 16>(ctx, p);
}

// ---- the order by expert ------------------------------------------------------------

// A stable counting sort of the pairs. Each block has a run of `chunk` pairs:
// their counts go to counts[block][expert] (order_count_kernel), then every
// block adds up the counts before its own and of all, and places its pairs
// (order_place_kernel). A single block counts for itself: one launch (2.4 us for
// 128 pairs; 131072 pairs of 256 experts in 64 blocks: 2.1 + 7.3 us, bound by the
// ranks within a block).
__device__ __forceinline__ int expert_of(const int32_t *ids, int64_t p, int64_t end, int experts) {
  const int e = p < end ? ids[p] : -1;
  return e < experts ? e : -1;
}

__global__ __launch_bounds__(1024) void order_count_kernel(const int32_t *ids, int64_t pairs, int64_t chunk, int experts,
                                                           int32_t *counts) {
  __shared__ int32_t count[kMaxExperts];
  for (int e = threadIdx.x; e < experts; e += blockDim.x) count[e] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * chunk, end = begin + chunk < pairs ? begin + chunk : pairs;
  for (int64_t p = begin + threadIdx.x; p < end; p += blockDim.x) {
    const int e = expert_of(ids, p, end, experts);
    if (e >= 0) atomicAdd(&count[e], 1);  // whole numbers: any order gives the same
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[(int64_t)blockIdx.x * experts + e] = count[e];
}

__global__ __launch_bounds__(1024) void order_place_kernel(const int32_t *ids, int64_t pairs, int64_t chunk, int experts,
                                                           int bits, const int32_t *counts, int blocks, int64_t *offsets,
                                                           int32_t *places, int32_t *sorted) {
  // next[e]: where the block's next pair of expert e goes; in a round, of[w * experts + e] pairs of wave w's
  __shared__ int32_t next[kMaxExperts], all[kMaxExperts], sums[16];
  __shared__ __align__(16) uint16_t of[16 * kMaxExperts];
  const int t = threadIdx.x, threads = blockDim.x, lane = t & 63, wave = t >> 6, waves = threads >> 6;
  const int64_t begin = blockIdx.x * chunk, end = begin + chunk < pairs ? begin + chunk : pairs;
  int e = expert_of(ids, begin + t, end, experts);  // of the round's pair
  for (int i = t; i < experts; i += threads) next[i] = all[i] = 0;
  typedef int v4i __attribute__((ext_vector_type(4)));
  const int clear = (waves * experts * 2 + 15) / 16;
  for (int i = t; i < clear; i += threads) reinterpret_cast<v4i *>(of)[i] = v4i{0, 0, 0, 0};
  __syncthreads();
  if (blocks == 1) {
    for (int64_t p = t; p < end; p += threads) {
      const int x = expert_of(ids, p, end, experts);
      if (x >= 0) atomicAdd(&all[x], 1);
    }
  } else {
    // threads / width rows of counts at once, all of a thread's loads under way together
    const int width = 1 << bits, step = threads >> bits, x = t & (width - 1), b0 = t >> bits;
    if (x < experts) {
      int before = 0, sum = 0;
#pragma unroll 16
      for (int b = b0; b < blocks; b += step) {
        const int c = counts[(int64_t)b * experts + x];
        sum += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
      atomicAdd(&all[x], sum);
      atomicAdd(&next[x], before);
    }
  }
  __syncthreads();
  // exclusive sums of all[] over the experts, a thread each (experts <= threads)
  int mine = t < experts ? all[t] : 0, scan = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 63) sums[wave] = scan;
  __syncthreads();
  int ahead = 0, total = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) ahead += sums[w];
    total += sums[w];
  }
  if (t < experts) {
    next[t] += ahead + scan - mine;
    if (blockIdx.x == 0) offsets[t] = ahead + scan - mine;
  }
  if (t == 0 && blockIdx.x == 0) offsets[experts] = total;

  for (int64_t p0 = begin; p0 < end; p0 += threads) {
    const int64_t p = p0 + t;
    // lanes with the same expert
    uint64_t same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
    if (e >= 0 && rank == 0) of[wave * experts + e] = (uint16_t)__popcll(same);
    __syncthreads();
    int place = -1;
    if (e >= 0) {
      place = next[e] + rank;
      for (int w = 0; w < wave; ++w) place += of[w * experts + e];
      sorted[place] = (int32_t)p;
    }
    if (p < end) {
      places[p] = place;
      if (p >= total) sorted[p] = -1;  // behind the last group
    }
    if (p0 + threads >= end) break;
    e = expert_of(ids, p + threads, end, experts);
    __syncthreads();
    for (int x = t; x < experts; x += threads) {
      int here = 0;
      for (int w = 0; w < waves; ++w) {
        here += of[w * experts + x];
        of[w * experts + x] = 0;
      }
      next[x] += here;
    }
    __syncthreads();
  }
}

// ---- moving rows -----------------------------------------------------------------------

struct RowsArgs {
  int64_t d, n;
  int topk;
  const void *X, *Y;
  int64_t ldx, ldy;
  const int32_t *places;
  const float *weights;
  float beta;
  void *out;
  int64_t ldo;
  float *dweights;
  int shift;  // 2^shift threads a token
};

// STREAM: non-temporal accesses, where the rows are more than the L2 caches
// hold. With 49152 rows of 2048 bf16 values (201 MB), read in any order, their
// sums take 43 us instead of 63, the gradients 77 instead of 110.
// Only for rows at whole dwords: at halves they are slower than plain ones.
template <class T, bool STREAM>
struct Lanes {
  static constexpr int V = 16 / sizeof(T);  // elements of a 16-byte access
  typedef int Raw __attribute__((ext_vector_type(4), aligned(4)));
  typedef int Any __attribute__((ext_vector_type(4), aligned(2)));
  struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[V];
  };
  // As dwords: made values of at the load they would be waited for there.
  static __device__ __forceinline__ Raw get(const T *x) {
    if constexpr (STREAM)
      return __builtin_nontemporal_load(reinterpret_cast<const Raw *>(x));
    else
      return *reinterpret_cast<const Any *>(x);
  }
  static __device__ __forceinline__ void put(T *x, const Vec &v) {
    if constexpr (STREAM) {
      const Raw raw = __builtin_bit_cast(Raw, v);
      __builtin_nontemporal_store(raw, reinterpret_cast<Raw *>(x));
    } else {
      *reinterpret_cast<Vec *>(x) = v;
    }
  }
  static __device__ __forceinline__ void widen(const Raw &raw, float (&f)[V]) {
    const Vec v = __builtin_bit_cast(Vec, raw);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)v.v[i];
  }
  // up to `left` elements at x, as floats
  static __device__ __forceinline__ void load(const T *x, int64_t left, float (&f)[V]) {
    if (left >= V) {
      widen(get(x), f);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = i < left ? (float)x[i] : 0.0f;
    }
  }
  static __device__ __forceinline__ void store(T *x, int64_t left, const float (&f)[V]) {
    if (left >= V) {
      Vec v;
#pragma unroll
      for (int i = 0; i < V; ++i) v.v[i] = (T)wgb::in_fp32(f[i]);
      put(x, v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < left) x[i] = (T)wgb::in_fp32(f[i]);
    }
  }
};

// Up to S of a token's slots from s0 on: their columns (-1: none, or outside)
// and weights. A thread's loads of them and of their rows are under way together.
template <int S>
struct Slots {
  int64_t place[S];
  float w[S];
  __device__ __forceinline__ void load(const RowsArgs &p, int64_t token, int s0) {
    const int64_t columns = p.n * p.topk, at = token * p.topk + s0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const bool there = s0 + s < p.topk;
      place[s] = there ? p.places[at + s] : -1;
      w[s] = there && p.weights ? p.weights[at + s] : 1.0f;
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (place[s] >= columns) place[s] = -1;
  }
};
constexpr int kSlots = 8;

// Y(:, places[s, t]) = w X(:, t): a token's row is read once and stored topk
// times. Bound by those stores (8192 tokens of 2048 bf16 values, 6 times: 40 us,
// 5.9 TB/s; 32 of 4096, 8 times: 3.4 us).
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void gather_kernel(RowsArgs p) {
  typedef Lanes<T, STREAM> L;
  const int lanes = 1 << p.shift, lane = threadIdx.x & (lanes - 1);
  const int64_t token = (int64_t)blockIdx.x * (blockDim.x >> p.shift) + (threadIdx.x >> p.shift);
  if (token >= p.n) return;
  const T *x = (const T *)p.X + token * p.ldx;
  for (int64_t at = ((int64_t)blockIdx.y * lanes + lane) * L::V; at < p.d; at += (int64_t)gridDim.y * lanes * L::V) {
    float f[L::V];
    Lanes<T, false>::load(x + at, p.d - at, f);
    for (int s0 = 0; s0 < p.topk; s0 += kSlots) {
      Slots<kSlots> slots;
      slots.load(p, token, s0);
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        if (slots.place[s] < 0) continue;
        float g[L::V];
#pragma unroll
        for (int i = 0; i < L::V; ++i) g[i] = slots.w[s] * f[i];
        L::store((T *)p.out + slots.place[s] * p.ldo + at, p.d - at, g);
      }
    }
  }
}

// C(:, t) = sum over s of w Y(:, places[s, t]) + beta C(:, t), in the slots'
// order, in fp32. Bound by reading Y (those 8192 tokens: 43 us, 5.4 TB/s; those
// 32: 3.4 us).
template <class T, class C, bool STREAM>
__global__ __launch_bounds__(256) void combine_kernel(RowsArgs p) {
  typedef Lanes<T, STREAM> L;
  const int lanes = 1 << p.shift, lane = threadIdx.x & (lanes - 1);
  const int64_t token = (int64_t)blockIdx.x * (blockDim.x >> p.shift) + (threadIdx.x >> p.shift);
  if (token >= p.n) return;
  C *c = (C *)p.out + token * p.ldo;
  for (int64_t at = ((int64_t)blockIdx.y * lanes + lane) * L::V; at < p.d; at += (int64_t)gridDim.y * lanes * L::V) {
    float sum[L::V];
#pragma unroll
    for (int i = 0; i < L::V; ++i) sum[i] = 0.0f;
    const bool whole = p.d - at >= L::V;
    for (int s0 = 0; s0 < p.topk; s0 += kSlots) {
      Slots<kSlots> slots;
      slots.load(p, token, s0);
      if (whole) {
        typename L::Raw y[kSlots];
#pragma unroll
        for (int s = 0; s < kSlots; ++s)
          if (slots.place[s] >= 0) y[s] = L::get((const T *)p.Y + slots.place[s] * p.ldy + at);
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (slots.place[s] < 0) continue;
          float f[L::V];
          L::widen(y[s], f);
#pragma unroll
          for (int i = 0; i < L::V; ++i) sum[i] = fmaf(slots.w[s], f[i], sum[i]);
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (slots.place[s] < 0) continue;
          float f[L::V];
          L::load((const T *)p.Y + slots.place[s] * p.ldy + at, p.d - at, f);
#pragma unroll
          for (int i = 0; i < L::V; ++i) sum[i] = fmaf(slots.w[s], f[i], sum[i]);
        }
      }
    }
    if (p.beta != 0.0f) {
#pragma unroll
      for (int i = 0; i < L::V; ++i)
        if (at + i < p.d) sum[i] = fmaf(p.beta, (float)c[at + i], sum[i]);
    }
    if (whole) {
      struct __attribute__((packed, aligned(sizeof(C)))) Out {
        C v[L::V];
      } out;
#pragma unroll
      for (int i = 0; i < L::V; ++i) out.v[i] = (C)wgb::in_fp32(sum[i]);
      *reinterpret_cast<Out *>(c + at) = out;
    } else {
#pragma unroll
      for (int i = 0; i < L::V; ++i)
        if (at + i < p.d) c[at + i] = (C)wgb::in_fp32(sum[i]);
    }
  }
}

// dY(:, places[s, t]) = w dC(:, t) and dw[s, t] = <Y(:, places[s, t]), dC(:,
// t)>: eight slots at a time, their rows' loads under way together; the threads'
// sums are folded in a fixed order. Bound by memory (those 8192 tokens: 77 us,
// 5.7 TB/s).
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void combine_grad_kernel(RowsArgs p) {
  typedef Lanes<T, STREAM> L;
  __shared__ float sums[4][kSlots];
  const int64_t token = blockIdx.x;
  const int t = threadIdx.x;
  const T *dc = (const T *)p.X + token * p.ldx;
  for (int s0 = 0; s0 < p.topk; s0 += kSlots) {
    Slots<kSlots> slots;
    slots.load(p, token, s0);
    float dot[kSlots];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) dot[s] = 0.0f;
    for (int64_t at = (int64_t)t * L::V; at < p.d; at += (int64_t)blockDim.x * L::V) {
      float f[L::V];
      if (p.d - at >= L::V) {
        const auto own = Lanes<T, false>::get(dc + at);
        typename L::Raw y[kSlots];
#pragma unroll
        for (int s = 0; s < kSlots; ++s)
          if (slots.place[s] >= 0) y[s] = L::get((const T *)p.Y + slots.place[s] * p.ldy + at);
        L::widen(own, f);
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (slots.place[s] < 0) continue;
          float v[L::V], g[L::V];
          L::widen(y[s], v);
#pragma unroll
          for (int i = 0; i < L::V; ++i) {
            dot[s] = fmaf(v[i], f[i], dot[s]);
            g[i] = slots.w[s] * f[i];
          }
          L::store((T *)p.out + slots.place[s] * p.ldo + at, L::V, g);
        }
      } else {
        Lanes<T, false>::load(dc + at, p.d - at, f);
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (slots.place[s] < 0) continue;
          float y[L::V], g[L::V];
          L::load((const T *)p.Y + slots.place[s] * p.ldy + at, p.d - at, y);
#pragma unroll
          for (int i = 0; i < L::V; ++i) {
            dot[s] = fmaf(y[i], f[i], dot[s]);
            g[i] = slots.w[s] * f[i];
          }
          L::store((T *)p.out + slots.place[s] * p.ldo + at, p.d - at, g);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const float x = over_lanes<64>(dot[s], Sum());
      if ((t & 63) == 0) sums[t >> 6][s] = x;
    }
    __syncthreads();
    if (t < kSlots && s0 + t < p.topk) {
      float x = sums[0][t];
      for (int w = 1; w < (int)blockDim.x >> 6; ++w) x += sums[w][t];
      p.dweights[token * p.topk + s0 + t] = x;
    }
    __syncthreads();
  }
}

// Threads of a block and of a token (2^shift), and blocks along d, for rows of
// d elements of `size` bytes: 256 threads a block, or 64 where that leaves CUs
// idle (32 tokens of 4096 bf16 values).
int row_shape(const wgb_ctx *ctx, int64_t d, int64_t n, int size, int &shift, dim3 &grid) {
  const int64_t vectors = (d * size + 15) / 16;
  const int threads = n * vectors < (int64_t)ctx->num_cus * 512 ? 64 : 256, most = threads == 64 ? 6 : 8;
  shift = 0;
  while (shift < most && ((int64_t)1 << shift) < vectors) ++shift;
  const int64_t along = (vectors + ((int64_t)1 << shift) - 1) >> shift, per = threads >> shift;
  grid = dim3((unsigned)((n + per - 1) / per), (unsigned)(along < 65535 ? along : 65535));
  return threads;
}

// Whether the rows of all pairs are more than the L2 caches hold (8 of 4 MB),
// and at whole dwords: `parts`, their addresses and leading dimensions in bytes
// or'ed together.
bool streams(int type, int64_t d, int64_t n, int64_t topk, uint64_t parts) {
  return d * n * topk * (type == WGB_F32 ? 4 : 2) > (int64_t)32 << 20 && (parts & 3) == 0;
}
uint64_t part(int type, const void *p, int64_t ld) { return (uint64_t)(uintptr_t)p | (uint64_t)ld * (type == WGB_F32 ? 4 : 2); }

// f(a value of the type, std::true_type or std::false_type)
template <class F>
void with_type(int type, bool flag, F f) {
  auto call = [&](auto t) { flag ? f(t, std::true_type()) : f(t, std::false_type()); };
  if (type == WGB_F32)
    call(0.0f);
  else if (type == WGB_F16)
    call((_Float16)0.0f);
  else
    call((__bf16)0.0f);
}

// ---- checks ----------------------------------------------------------------------------

int check_type(int type) {
  if (type != WGB_F32 && type != WGB_F16 && type != WGB_BF16)
    return fail(WGB_ERR_INVALID_VALUE, "type must be WGB_F32, WGB_F16 or WGB_BF16");
  return WGB_OK;
}

int check_pairs(int64_t n, int64_t topk) {
  if (n < 0) return fail(WGB_ERR_INVALID_VALUE, "n must be non-negative");
  if (topk < 1 || topk > kMaxTopk) return fail(WGB_ERR_INVALID_VALUE, "topk must be between 1 and 64");
  if (n > INT32_MAX / topk) return fail(WGB_ERR_INVALID_VALUE, "n * topk must be below 2^31");
  return WGB_OK;
}

// A launch has fewer than 2^32 threads, of which a token has up to 256.
int check_tokens(int64_t n) {
  if (n >= (int64_t)1 << 24) return fail(WGB_ERR_INVALID_VALUE, "n must be below 2^24");
  return WGB_OK;
}

int check_choice(int64_t experts, int64_t n, int64_t topk) {
  const int st = check_pairs(n, topk);
  if (st) return st;
  if (experts < 1 || experts > kMaxExperts) return fail(WGB_ERR_INVALID_VALUE, "experts must be between 1 and 1024");
  if (topk > experts) return fail(WGB_ERR_INVALID_VALUE, "topk must be at most experts");
  return WGB_OK;
}

int check_scoring(int scoring) {
  if (scoring != WGB_SOFTMAX && scoring != WGB_SIGMOID)
    return fail(WGB_ERR_INVALID_VALUE, "scoring must be WGB_SOFTMAX or WGB_SIGMOID");
  return WGB_OK;
}

int check_rows(int type, int64_t d, int64_t n, int64_t topk) {
  int st = check_type(type);
  if (!st) st = check_pairs(n, topk);
  if (!st) st = check_tokens(n);
  if (st) return st;
  if (d < 0 || d > INT32_MAX) return fail(WGB_ERR_INVALID_VALUE, "d must be non-negative and below 2^31");
  return WGB_OK;
}

int check_ld(int64_t ld, int64_t rows, const char *what) {
  if (ld < (rows > 1 ? rows : 1))
    return fail(WGB_ERR_INVALID_VALUE, std::string(what) + " must be at least the column's length and 1");
  return WGB_OK;
}

}  // namespace

extern "C" int wgb_route(wgb_ctx *ctx, int type, int scoring, int64_t experts, int64_t n, int64_t topk,
                         const void *logits, int64_t ldl, const float *bias, int64_t groups, int64_t top_groups, int best,
                         int renorm, float scale, int32_t *ids, float *weights) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_type(type)) || (st = check_scoring(scoring)) || (st = check_choice(experts, n, topk)) ||
      (st = check_tokens(n)) || (st = check_ld(ldl, experts, "ldl")))
    return st;
  if (groups < 1 || groups > kMaxGroups || experts % groups != 0)
    return fail(WGB_ERR_INVALID_VALUE, "groups must be between 1 and 64 and divide experts");
  if (top_groups < 1 || top_groups > groups)
    return fail(WGB_ERR_INVALID_VALUE, "top_groups must be between 1 and groups");
  if (best != 1 && best != 2) return fail(WGB_ERR_INVALID_VALUE, "best must be 1 or 2");
  if (topk > experts / groups * top_groups)
    return fail(WGB_ERR_INVALID_VALUE, "topk must be at most the experts of top_groups groups");
  if (n == 0) return WGB_OK;
  if (!logits || !ids || !weights) return fail(WGB_ERR_INVALID_VALUE, "logits, ids or weights is null");
  RouteArgs p = {};
  p.logits = logits;
  p.ldl = ldl;
  p.n = n;
  p.bias = bias;
  p.experts = (int)experts;
  p.topk = (int)topk;
  p.groups = top_groups == groups ? 1 : (int)groups;  // all kept: as none
  p.top_groups = (int)top_groups;
  p.best = best;
  p.per = (int)(experts / groups);
  p.magic = ((1u << 20) + p.per - 1) / p.per;
  p.sigmoid = scoring == WGB_SIGMOID;
  p.renorm = renorm != 0;
  p.scale = scale;
  p.ids = ids;
  p.weights = weights;
  wgb::timing_begin(ctx);
  st = type == WGB_F32 ? route<float>(ctx, p) : type == WGB_F16 ? route<_Float16>(ctx, p) : route<__bf16>(ctx, p);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_route_grad(wgb_ctx *ctx, int type, int scoring, int64_t experts, int64_t n, int64_t topk,
                              const void *logits, int64_t ldl, const int32_t *ids, int renorm, float scale,
                              const float *dweights, void *dlogits, int64_t ldd) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_type(type)) || (st = check_scoring(scoring)) || (st = check_choice(experts, n, topk)) ||
      (st = check_tokens(n)) || (st = check_ld(ldl, experts, "ldl")) || (st = check_ld(ldd, experts, "ldd")))
    return st;
  if (n == 0) return WGB_OK;
  if (!logits || !ids || !dweights || !dlogits)
    return fail(WGB_ERR_INVALID_VALUE, "logits, ids, dweights or dlogits is null");
  GradArgs p = {logits, ldl, n, ids, dweights, dlogits, ldd, (int)experts, (int)topk, scoring == WGB_SIGMOID, renorm != 0,
                scale};
  wgb::timing_begin(ctx);
  st = type == WGB_F32 ? grad<float>(ctx, p) : type == WGB_F16 ? grad<_Float16>(ctx, p) : grad<__bf16>(ctx, p);
  wgb::timing_end(ctx);
  return st;
}

extern "C" int wgb_route_order(wgb_ctx *ctx, int64_t experts, int64_t n, int64_t topk, const int32_t *ids,
                               int64_t *d_offsets, int32_t *places, int32_t *pairs) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_choice(experts, n, topk))) return st;
  if (!d_offsets) return fail(WGB_ERR_INVALID_VALUE, "d_offsets is null");
  if (n > 0 && (!ids || !places || !pairs)) return fail(WGB_ERR_INVALID_VALUE, "ids, places or pairs is null");
  const int64_t count = n * topk;
  int bits = 0;
  while ((1 << bits) < experts) ++bits;
  // at most 64 blocks, each of whole rounds of 1024 pairs: every block reads all counts
  int64_t chunk = (count + 63) / 64;
  chunk = (chunk + 1023) / 1024 * 1024;
  const int blocks = count > 1024 ? (int)((count + chunk - 1) / chunk) : 1;
  int threads = 1024;
  while (blocks == 1 && threads > 64 && threads / 2 >= count && threads / 2 >= experts) threads /= 2;
  if (blocks == 1) chunk = count;
  if (blocks > 1 && (st = wgb::ensure_op_workspace(ctx, (size_t)blocks * experts * 4))) return st;
  wgb::timing_begin(ctx);
  if (blocks > 1) {
    order_count_kernel<<<blocks, 1024, 0, ctx->stream>>>(ids, count, chunk, (int)experts, (int32_t *)ctx->op_ws);
  }
  order_place_kernel<<<blocks, threads, 0, ctx->stream>>>(ids, count, chunk, (int)experts, bits, (const int32_t *)ctx->op_ws,
                                                          blocks, d_offsets, places, pairs);
  wgb::timing_end(ctx);
  WGB_CHECK_LAUNCH("order_place_kernel");
  return WGB_OK;
}

extern "C" int wgb_route_gather(wgb_ctx *ctx, int type, int64_t d, int64_t n, int64_t topk, const void *X, int64_t ldx,
                                const int32_t *places, const float *weights, void *Y, int64_t ldy) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_rows(type, d, n, topk)) || (st = check_ld(ldx, d, "ldx")) || (st = check_ld(ldy, d, "ldy"))) return st;
  if (n == 0 || d == 0) return WGB_OK;
  if (!X || !places || !Y) return fail(WGB_ERR_INVALID_VALUE, "X, places or Y is null");
  RowsArgs p = {};
  p.d = d;
  p.n = n;
  p.topk = (int)topk;
  p.X = X;
  p.ldx = ldx;
  p.places = places;
  p.weights = weights;
  p.out = Y;
  p.ldo = ldy;
  dim3 grid;
  const int threads = row_shape(ctx, d, n, type == WGB_F32 ? 4 : 2, p.shift, grid);
  wgb::timing_begin(ctx);
  with_type(type, streams(type, d, n, topk, part(type, X, ldx) | part(type, Y, ldy)), [&](auto t, auto stream) {
    gather_kernel<decltype(t), decltype(stream)::value><<<grid, threads, 0, ctx->stream>>>(p);
  });
  wgb::timing_end(ctx);
  WGB_CHECK_LAUNCH("gather_kernel");
  return WGB_OK;
}

extern "C" int wgb_route_combine(wgb_ctx *ctx, int type, int64_t d, int64_t n, int64_t topk, const void *Y, int64_t ldy,
                                 const int32_t *places, const float *weights, float beta, void *C, int64_t ldc,
                                 int ctype) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_rows(type, d, n, topk)) || (st = check_ld(ldy, d, "ldy")) || (st = check_ld(ldc, d, "ldc"))) return st;
  if (ctype != type && ctype != WGB_F32)
    return fail(WGB_ERR_INVALID_VALUE, "the type of C must be Y's type or WGB_F32");
  if (n == 0 || d == 0) return WGB_OK;
  if (!Y || !places || !C) return fail(WGB_ERR_INVALID_VALUE, "Y, places or C is null");
  RowsArgs p = {};
  p.d = d;
  p.n = n;
  p.topk = (int)topk;
  p.Y = Y;
  p.ldy = ldy;
  p.places = places;
  p.weights = weights;
  p.beta = beta;
  p.out = C;
  p.ldo = ldc;
  dim3 grid;
  const int threads = row_shape(ctx, d, n, type == WGB_F32 ? 4 : 2, p.shift, grid);
  wgb::timing_begin(ctx);
  with_type(type, streams(type, d, n, topk, part(type, Y, ldy)), [&](auto t, auto stream) {
    typedef decltype(t) T;
    if (ctype == type)
      combine_kernel<T, T, decltype(stream)::value><<<grid, threads, 0, ctx->stream>>>(p);
    else
      combine_kernel<T, float, decltype(stream)::value><<<grid, threads, 0, ctx->stream>>>(p);
  });
  wgb::timing_end(ctx);
  WGB_CHECK_LAUNCH("combine_kernel");
  return WGB_OK;
}

extern "C" int wgb_route_combine_grad(wgb_ctx *ctx, int type, int64_t d, int64_t n, int64_t topk, const void *dC,
                                      int64_t lddc, const void *Y, int64_t ldy, const int32_t *places,
                                      const float *weights, void *dY, int64_t lddy, float *dweights) {
  int st = wgb::enter(ctx);
  if (st) return st;
  if ((st = check_rows(type, d, n, topk)) || (st = check_ld(lddc, d, "lddc")) || (st = check_ld(ldy, d, "ldy")) ||
      (st = check_ld(lddy, d, "lddy")))
    return st;
  if (n == 0) return WGB_OK;
  if (!places || !weights || !dweights) return fail(WGB_ERR_INVALID_VALUE, "places, weights or dweights is null");
  if (d > 0 && (!dC || !Y || !dY)) return fail(WGB_ERR_INVALID_VALUE, "dC, Y or dY is null");
  RowsArgs p = {};
  p.d = d;
  p.n = n;
  p.topk = (int)topk;
  p.X = dC;
  p.ldx = lddc;
  p.Y = Y;
  p.ldy = ldy;
  p.places = places;
  p.weights = weights;
  p.out = dY;
  p.ldo = lddy;
  p.dweights = dweights;
  wgb::timing_begin(ctx);
  with_type(type, streams(type, d, n, topk, part(type, dC, lddc) | part(type, Y, ldy) | part(type, dY, lddy)), [&](auto t, auto stream) {
    combine_grad_kernel<decltype(t), decltype(stream)::value><<<(unsigned)n, 256, 0, ctx->stream>>>(p);
  });
  wgb::timing_end(ctx);
  WGB_CHECK_LAUNCH("combine_grad_kernel");
  return WGB_OK;
}
