// moe.hip -- what stands around the routed experts' products: the choice of each
// token's experts with their weights, and the weighted sum of their outputs.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/higgs_hip.h"
#include "hgk_common.h"
#include "hgk_host.h"

namespace hgk {
namespace {

// ---------------------------------------------------------------- routing
struct RouteArgs {
  const char* logits;
  const float* bias;
  float* weights;
  int32_t* experts;
  int64_t row;  // elements between logits of two tokens
  int64_t tokens;
  int32_t n, top_k, groups, top_groups, group_top, group_size;
  int32_t sigmoid, renormalize, group_bits, pieces, bias_pieces;
  float scale;
};

constexpr float kLog2e = 1.44269504088896341f;

// e^x to about 2^-22 of itself for x >= -87, and zero below: x log2(e) in two parts, the
// lesser one put back by its series (the product alone is off by up to 2^-17 of the
// result at x = -88).
__device__ inline float exp_f32(float x) {
  const float t = x * kLog2e, r = fmaf(x, kLog2e, -t) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return x < -150.0f ? 0.0f : fmaf(e, r * 0.693147181f, e);
}
// ... where results below 2^-126 count too, which the hardware's exp2 has as zero: those
// are 2^64 times as great until the last product, which rounds to the step of 2^-149.
__device__ inline float exp_small(float x) {
  const bool far = x < -80.0f;
  const float t = x * kLog2e, r = fmaf(x, kLog2e, -t) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(far ? t + 64.0f : t);
  return x < -150.0f ? 0.0f : fmaf(e, r * 0.693147181f, e) * (far ? 0x1p-64f : 1.0f);
}

// Value of the lane that a DPP control pairs with this one.
template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
// ... and of the lane 2^S away (4: the rows of 16 trade places, 5: the halves).
template <int S>
__device__ inline uint32_t partner(uint32_t v) {
  if constexpr (S == 0) return dpp<0xB1>(v);        // quad_perm [1,0,3,2]
  else if constexpr (S == 1) return dpp<0x4E>(v);   // quad_perm [2,3,0,1]
  else if constexpr (S == 2) return dpp<0x141>(v);  // mirrored in 8: another quad
  else if constexpr (S == 3) return dpp<0x140>(v);  // mirrored in 16: another 8
  else {
    const bool low = !(threadIdx.x & (1u << S));
    if constexpr (S == 4) {
      const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
      return low ? r[1] : r[0];
    } else {
      const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
      return low ? r[1] : r[0];
    }
  }
}
template <int S>
__device__ inline double partner(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)partner<S>((uint32_t)(b >> 32)) << 32 | partner<S>((uint32_t)b));
}
template <int S>
__device__ inline float partner(float v) { return u2f(partner<S>(f2u(v))); }

// f folded over the aligned 2^BITS lanes around this one: all get the result.
// (The mirrors pair each lane with one of the other half, which is enough once
// a half's lanes agree.)
template <int BITS, int S = 0, class V, class F>
__device__ inline V fold(V v, F f) {
  if constexpr (S >= BITS) return v;
  else return fold<BITS, S + 1>(f(v, partner<S>(v)), f);
}
template <int BITS>
__device__ inline uint32_t fold_max(uint32_t v) {
  return fold<BITS>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int BITS>
__device__ inline uint32_t fold_min(uint32_t v) {
  return fold<BITS>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// A choice as whole numbers in the same order, none of them 0 (NaN has been put
// below all others).
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = f2u(x == 0.0f ? 0.0f : x);  // one zero
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline uint64_t key_of(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x == 0.0 ? 0.0 : x);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ inline float value_of(uint32_t key) { return u2f(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// Of the 2^BITS lanes' (key, index), the index of the greatest key, the lowest
// one of several.
template <int BITS>
__device__ inline uint32_t best_of(uint32_t key, uint32_t index) {
  const uint32_t top = fold_max<BITS>(key);
  return fold_min<BITS>(key == top ? index : ~0u);
}
template <int BITS>
__device__ inline uint32_t best_of(uint64_t key, uint32_t index) {
  const uint32_t hi = (uint32_t)(key >> 32), top = fold_max<BITS>(hi);
  const uint32_t lo = hi == top ? (uint32_t)key : 0u, low = fold_max<BITS>(lo);
  return fold_min<BITS>(hi == top && lo == low ? index : ~0u);
}

// The sum of a group's two greatest choices, or its greatest: over a lane's choices,
// then over the group's 2^gbits lanes.
template <int BITS, int PER, class V>
__device__ inline V group_score(const V* c, int gbits, int group_top) {
  V b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    b2 = fmax(b2, fmin(b1, c[i]));
    b1 = fmax(b1, c[i]);
  }
  auto join = [&](V p, V q) {
    b2 = fmax(fmin(b1, p), fmax(b2, q));
    b1 = fmax(b1, p);
  };
  if (gbits > 0) join(partner<0>(b1), partner<0>(b2));
  if (gbits > 1) join(partner<1>(b1), partner<1>(b2));
  if (gbits > 2) join(partner<2>(b1), partner<2>(b2));
  if (gbits > 3) join(partner<3>(b1), partner<3>(b2));
  if constexpr (BITS > 4)
    if (gbits > 4) join(partner<4>(b1), partner<4>(b2));
  const V sum = b1 + b2;
  return group_top != 2 ? b1 : sum == sum ? sum : (V)-INFINITY;  // (infinities of both signs: NaN)
}

// The choice to the last bit: the keys hold all of it. c: -inf where a lane has no
// expert. Returns lane r's expert.
template <int BITS, int PER, class V, class E>
__device__ __forceinline__ uint32_t choose_exact(const RouteArgs& a, const V (&c)[PER], int sub, int group,
                                                           int gbits, int mine, E expert_of) {
  typedef decltype(key_of(V())) Key;
  Key key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = i < mine ? key_of(c[i]) : 0;
  if (a.top_groups < a.groups) {
    const V score = group_score<BITS, PER>(c, gbits, a.group_top);
    Key left = group < a.groups ? key_of(score) : 0;
    bool kept = false;
    for (int r = 0; r < a.top_groups; ++r)
      if (best_of<BITS>(left, (uint32_t)group) == (uint32_t)group) {
        kept = true;
        left = 0;
      }
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = kept ? key[i] : 0;
  }
  uint32_t got = 0;
  for (int r = 0; r < a.top_k; ++r) {
    Key best = 0;
    uint32_t e = ~0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      e = key[i] > best ? expert_of(i) : e;
      best = key[i] > best ? key[i] : best;
    }
    const uint32_t w = best_of<BITS>(best, e);
    if (sub == r) got = w;
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = expert_of(i) == w ? 0 : key[i];
  }
  return got;
}

// 2^BITS lanes have a token, a lane PER experts of one group: pieces of V in a row,
// side by side over the group's lanes.
//
// Where nothing is added to the scores (SUMS false) they are in the order of the
// logits, and those are compared. Else two sums may lie closer than f32 holds
// scores: their order is that of 64 bits.
//
// Both are first tried on 32-bit keys: 22 bits of the choice and the expert's number,
// so that one fold over the lanes finds the best choice with its expert, ties by the
// lower one. The next best is the greatest of (key - last best) modulo 2^32: what
// has been taken wraps to the bottom. All of a 16-bit logit is in the upper 22 bits
// of its f32 form. Other choices are brought to 2^22 equal steps of their range;
// ones that follow each other by less than the steps' and the f32 sums' errors leave
// the order open: those are put in the order of their whole choices, and where that
// is not enough (a chain of them reaches past the last one looked at, or groups'
// scores are as close) the wave takes its tokens again with whole keys.
//
// Bound by the folds' and keys' instructions. 16384 tokens of 256 experts in f32, 4
// of 8 groups, top 8, with a bias: 14.5 us, of which the reading of the logits would
// be 3; a wave a token and whole keys for all 34.0.
constexpr int kSpare = 2;
template <class T, bool SUMS, int BITS, int PER>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteArgs a) {
  constexpr int W = 1 << BITS, V = PER < 16 / T::kBytes ? PER : 16 / T::kBytes;
  constexpr bool kWhole = !SUMS && T::kBytes == 2;  // the short keys hold all
  const int sub = threadIdx.x & (W - 1);
  const int64_t token = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
  const char* row = a.logits + (token < a.tokens ? token : 0) * a.row * T::kBytes;

  // lanes of a group, and this lane's experts: its i-th is expert_of(i) for i < mine
  const int gbits = a.group_bits, group = sub >> gbits, in = sub & ((1 << gbits) - 1);
  const uint32_t e0 = group * a.group_size + in * V;
  auto place = [&](int i) { return (i / V) * (V << gbits) + i % V; };  // from e0
  auto expert_of = [&](int i) { return e0 + place(i); };
  int mine = 0;
  if (group < a.groups)
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += in * V + place(i) < a.group_size;

  float x[PER];
  if (a.pieces) {  // whole pieces, aligned
#pragma unroll
    for (int i = 0; i < PER; i += V) {
      const int64_t at = i < mine ? expert_of(i) : 0;
      if constexpr (V * T::kBytes == 16) {
        const u32x4 r = ld16<T>(row, at);
#pragma unroll
        for (int k = 0; k < V; ++k) x[i + k] = elem<T>(r, k);
      } else {
        static_assert(V * T::kBytes == 8, "pieces of 8 or 16 bytes");
        const u32x2 r = ld_raw<8>(row, at * T::kBytes);
#pragma unroll
        for (int k = 0; k < V; ++k) x[i + k] = elem<T>(r, k);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = load1<T>(row, i < mine ? expert_of(i) : 0);
  }
  float top = -INFINITY;
  uint32_t lost = 0;  // bits of the logits behind the first 22
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i >= mine || x[i] != x[i]) x[i] = -INFINITY;
    top = fmaxf(top, x[i]);
    lost |= f2u(x[i]);
  }
  top = fold<BITS>(top, [](float p, float q) { return fmaxf(p, q); });
  lost &= 0x3ffu;

  // softmax's sum, where scores themselves count
  float whole = 0.0f, e[PER];
  if (!a.sigmoid && (SUMS || !a.renormalize)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      e[i] = x[i] == -INFINITY ? 0.0f : x[i] == top ? 1.0f : exp_f32(x[i] - top);
      whole += e[i];
    }
    whole = fold<BITS>(whole, [](float p, float q) { return p + q; });
  }

  // choices, to f32's rounding
  float c[PER], bias[PER];
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < PER; ++i) bias[i] = 0.0f;
    if (a.bias && a.bias_pieces) {
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        const u32x4 r = ld16<F32>(a.bias, i < mine ? expert_of(i) : 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) bias[i + k] = u2f(r[k]);
      }
    } else if (a.bias) {
#pragma unroll
      for (int i = 0; i < PER; ++i) bias[i] = a.bias[i < mine ? expert_of(i) : 0];
    }
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        c[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[i] * -kLog2e));
    } else {
      const float r = whole > 0.0f ? __builtin_amdgcn_rcpf(whole) : 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = e[i] * r;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] += bias[i];
      if (i >= mine || c[i] != c[i]) c[i] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) c[i] = x[i];
  }
  // 22 bits of every choice: those of its f32 form, or 2^22 steps of the choices'
  // range (its upper 16, if it is greater)
  if constexpr (!kWhole && !SUMS) lost = fold<BITS>(lost, [](uint32_t p, uint32_t q) { return p | q; });
  const bool steps = SUMS || (!kWhole && lost != 0);
  float low = INFINITY, high = -INFINITY, per = 0.0f, err = 0.0f;  // err: of the sums, in f32
  if constexpr (!kWhole) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      low = fminf(low, i < mine ? c[i] : INFINITY);
      high = fmaxf(high, c[i]);
    }
    low = fold<BITS>(low, [](float p, float q) { return fminf(p, q); });
    high = fold<BITS>(high, [](float p, float q) { return fmaxf(p, q); });
    low = fmaxf(low, high - 16.0f);
    // a sigmoid is good to 2^-22 (its exponential's 2^-23 counts for a quarter, the sum
    // and the reciprocal for 2^-24 and 2^-23), a softmax score to 2^-19 (a sum of up
    // to 1024), and their sum with the bias is rounded
    if constexpr (SUMS) err = fmaxf(fabsf(low), fabsf(high)) * 0x1p-24f + (a.sigmoid ? 0x1p-22f : 0x1p-19f);
    per = high > low && high < INFINITY ? 4194200.0f / (high - low) : 0.0f;
  }
  const float margin = fmaf(2.0f * err, per, 3.0f);  // in steps: two roundings, and one (NaN beside an infinity)
  bool again = false;
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    uint32_t k = 0;
    if constexpr (!kWhole)
      if (steps) k = 2u + (uint32_t)__builtin_amdgcn_fmed3f((c[i] - low) * per, 0.0f, 4194200.0f);
    if constexpr (!SUMS)
      if (!steps) k = key_of(c[i]) >> 10;
    key[i] = i < mine ? k << 10 | (1023u - expert_of(i)) : 0u;
  }

  // groups: all but the best are taken out
  if (a.top_groups < a.groups) {
    const float score = group_score<BITS, PER>(c, gbits, a.group_top);
    uint32_t left = group < a.groups ? key_of(score) : 0u;
    bool kept = false;
    uint32_t w = 0;
    for (int r = 0; r < a.top_groups; ++r) {
      w = fold_max<BITS>(left);
      if (fold_min<BITS>(left == w ? (uint32_t)group : ~0u) == (uint32_t)group) {
        kept = true;
        left = 0;
      }
    }
    if constexpr (SUMS) {  // the best of the others
      const uint32_t next = fold_max<BITS>(left);
      const float p = value_of(w), q = value_of(next);
      if (next) again = !(p - q > fmaf(fabsf(p) + fabsf(q), 0x1p-22f, 5.0f * err));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = kept ? key[i] : 0u;
  }

  // Lane r takes the r-th best, a few more than are asked for where they may have to
  // change places. chain: how many in front of the last all leave their order open.
  const int rounds = kWhole ? a.top_k : min(a.top_k + kSpare, W);
  uint32_t expert = 0, last = 0;
  int chain = 0;
  bool swap = false, got = false;
  for (int r = 0; r < rounds; ++r) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; i += 2) best = max(best, max(key[i] - last, key[i + 1] - last));
    uint32_t w = fold_max<BITS>(best) + last;
    if (r > 0) {
      if (w >= last) w = 0;  // nothing is left
      if constexpr (!kWhole) {
        const bool open = steps && w && !((float)(last >> 10) - (float)(w >> 10) > margin);
        swap |= open && r <= a.top_k;
        chain = open ? chain + 1 : 0;
      }
    }
    if (sub == r) {
      expert = 1023u - (w & 1023u);
      got = w != 0;
    }
    last = w;
  }
  if constexpr (!kWhole) {
    // the last of them may be one of the best, and so may others behind it
    again |= last && steps && chain >= rounds - a.top_k;
    if (__any(swap)) {
      // those taken in the order of their whole choices
      typedef typename std::conditional<SUMS, double, float>::type V;
      V mine_is = got ? (V)load1<T>(row, expert) : (V)-INFINITY;
      if (mine_is != mine_is) mine_is = -INFINITY;
      if constexpr (SUMS) {
        again |= !a.sigmoid;  // (softmax: of a sum over all experts)
        mine_is = 1.0 / (1.0 + exp(-mine_is));
        if (a.bias) mine_is += (double)a.bias[got ? expert : 0];
        if (mine_is != mine_is) mine_is = -INFINITY;
      }
      int rank = 0;
      for (int r = 0; r < rounds; ++r) {
        const V other = __shfl(mine_is, r, W);
        const uint32_t of = __shfl(got ? expert : ~0u, r, W);
        rank += of != ~0u && (other > mine_is || (other == mine_is && of < expert));
      }
      // lane r takes the expert of the lane whose rank is r
      uint32_t sorted = expert;
      for (int r = 0; r < rounds; ++r) {
        const int to = __shfl(got ? rank : -1, r, W);
        const uint32_t of = __shfl(expert, r, W);
        sorted = to == sub ? of : sorted;
      }
      expert = sorted;
    }
  }
  if constexpr (!kWhole) {
    if (__any(again)) {
      if constexpr (SUMS) {
        double d[PER], sum = 0.0;
        if (a.sigmoid) {
#pragma unroll
          for (int i = 0; i < PER; ++i) d[i] = 1.0 / (1.0 + exp(-(double)x[i]));
        } else {
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            d[i] = x[i] == -INFINITY ? 0.0 : x[i] == top ? 1.0 : exp((double)x[i] - (double)top);
            sum += d[i];
          }
          sum = fold<BITS>(sum, [](double p, double q) { return p + q; });
#pragma unroll
          for (int i = 0; i < PER; ++i) d[i] = sum > 0.0 ? d[i] / sum : 0.0;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          d[i] += (double)bias[i];
          if (i >= mine || d[i] != d[i]) d[i] = -INFINITY;
        }
        expert = choose_exact<BITS, PER>(a, d, sub, group, gbits, mine, expert_of);
      } else {
        expert = choose_exact<BITS, PER>(a, c, sub, group, gbits, mine, expert_of);
      }
    }
  }

  // lane r: the weight of expert r
  const bool has = sub < a.top_k;
  float l = has ? load1<T>(row, expert) : -INFINITY, s;
  if (l != l) l = -INFINITY;
  // Scores that are renormalised are taken from the greatest of the chosen logits on:
  // all of them may be below what f32 holds (sigmoids of logits below -100, experts that
  // a bias has put in front of others with logits far above). Where even 64 bits hold
  // none of them (a logit masked by its type's lowest value) they are zero.
  constexpr float kLeast = -745.0f;  // log 2^-1074
  float most = 0.0f;
  if (a.renormalize) most = fold<BITS>(l, [](float p, float q) { return fmaxf(p, q); });
  if (a.sigmoid) {
    // of a large negative logit the exponential is the score
    const float f = exp_small(-fabsf(l)), from = most > kLeast ? fminf(most, 0.0f) : 0.0f;
    s = (l < 0.0f ? exp_small(l - from) : 1.0f) / (1.0f + f);
  } else {
    // (renormalised weights need no sum over all experts)
    const float from = a.renormalize && most - top > kLeast ? most : top;
    s = l == -INFINITY ? 0.0f : l == from ? 1.0f : exp_small(l - from);
    if (!a.renormalize) s = whole > 0.0f ? s / whole : 0.0f;
  }
  if (a.renormalize) {
    const float sum = fold<BITS>(has ? s : 0.0f, [](float p, float q) { return p + q; });
    s = sum > 0.0f ? s / sum : 0.0f;
  }
  if (has && token < a.tokens) {
    a.weights[token * a.top_k + sub] = s * a.scale;
    a.experts[token * a.top_k + sub] = (int32_t)expert;
  }
}

constexpr int kRouteExperts = 1024, kRouteTopK = 64;
constexpr int64_t kRouteBlocks = 1 << 23;  // of a launch

// How a token's experts lie on lanes: 2^bits lanes, per of them each.
struct RoutePlan {
  int bits, group_bits, per;
};
RoutePlan plan_route(int64_t groups, int64_t group_size, int64_t top_k, int bits) {
  RoutePlan p{bits, bits, 0};
  while (p.group_bits >= 0 && groups << p.group_bits > 1 << bits) --p.group_bits;
  // (with the choices looked at beyond the top_k, where there are lanes for them)
  if (p.group_bits < 0 || (bits < 6 && top_k + kSpare > 1 << bits)) return p;  // per 0: does not fit
  const int64_t lanes = 1 << p.group_bits, per = (group_size + lanes - 1) / lanes;
  // pieces of 4 to 8 are whole: such a lane has room for 4, 8 or 16
  p.per = per <= 4 ? 4 : per <= 8 ? 8 : per <= 16 ? 16 : 0;
  return p;
}

template <class T, bool SUMS, int BITS, int PER>
void launch_route(RouteArgs a, hipStream_t stream) {
  constexpr int kTokens = 256 >> BITS, V = PER < 16 / T::kBytes ? PER : 16 / T::kBytes;
  a.pieces = a.group_size % V == 0 && a.row % V == 0 &&
             (reinterpret_cast<uintptr_t>(a.logits) & (V * T::kBytes - 1)) == 0;
  a.bias_pieces = a.pieces && aligned16(a.bias);
  // (a launch has fewer than 2^32 threads)
  const int64_t tokens = a.tokens;
  for (int64_t t = 0; t < tokens; t += kRouteBlocks * kTokens) {
    RouteArgs b = a;
    b.logits += t * a.row * T::kBytes;
    b.weights += t * a.top_k;
    b.experts += t * a.top_k;
    b.tokens = std::min(tokens - t, kRouteBlocks * kTokens);
    HGK_LAUNCH((moe_route_kernel<T, SUMS, BITS, PER>), dim3((unsigned)((b.tokens + kTokens - 1) / kTokens)), dim3(256), 0,
               stream, b);
  }
}
template <class T, bool SUMS>
void route_of(const RouteArgs& a, const RoutePlan& p, hipStream_t stream) {
  if (p.bits == 4 && p.per == 4) launch_route<T, SUMS, 4, 4>(a, stream);
  else if (p.bits == 4 && p.per == 8) launch_route<T, SUMS, 4, 8>(a, stream);
  else if (p.bits == 4) launch_route<T, SUMS, 4, 16>(a, stream);
  else if (p.bits == 5) launch_route<T, SUMS, 5, 16>(a, stream);
  else if (p.per == 4) launch_route<T, SUMS, 6, 4>(a, stream);
  else launch_route<T, SUMS, 6, 16>(a, stream);
}
template <class T>
void route_as(const RouteArgs& a, const RoutePlan& p, bool sums, hipStream_t stream) {
  if (sums) route_of<T, true>(a, p, stream);
  else route_of<T, false>(a, p, stream);
}

// ---------------------------------------------------------------- the sum
struct CombineArgs {
  const char* y;
  const float* weights;
  const char* shared;
  const char* gate;
  char* out;
  int64_t y_row, shared_row, gate_row, out_row, w_row;
  int64_t tokens, hidden;
  int32_t top_k, gate_dtype;
};

__device__ inline float gate_of(const CombineArgs& a, int64_t t) {
  if (!a.gate) return 1.0f;
  const float g = load1_dt(a.gate, a.gate_dtype, t * a.gate_row);
  const float e = exp_f32(-fabsf(g));
  return (g < 0.0f ? e : 1.0f) / (1.0f + e);
}

// Block = (token, columns); a thread sums a 16-byte piece of the token's rows, up
// to kRows of them in flight. The rows are read once: past the caches.
constexpr int kCombineThreads = 64, kRows = 8;
template <class T>
__global__ __launch_bounds__(kCombineThreads) void moe_combine_kernel(CombineArgs a, uint32_t pieces, int64_t blocks) {
  constexpr int N = Vec<T>::N;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int64_t t = b / pieces, col = ((b - t * pieces) * kCombineThreads + threadIdx.x) * N;
    if (col >= a.hidden) continue;
    const float* w = a.weights + t * a.w_row;
    float sum[N] = {};
    auto add = [&](u32x4 r, float f) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = fmaf(f, elem<T>(r, e), sum[e]);
    };
    const int64_t first = t * a.top_k * a.y_row + col;
    for (int i0 = 0; i0 < a.top_k; i0 += kRows) {
      u32x4 r[kRows];
      float f[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        f[i] = i0 + i < a.top_k ? w[i0 + i] : 0.0f;
        if (f[i] != 0.0f) r[i] = ld16_nt<T>(a.y, first + (i0 + i) * a.y_row);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (f[i] != 0.0f) add(r[i], f[i]);
    }
    if (a.shared) add(ld16_nt<T>(a.shared, t * a.shared_row + col), gate_of(a, t));
    store_elems<T, N, false>(a.out, t * a.out_row + col, sum);
  }
}

// Rows that 16-byte pieces do not fit: an element a thread.
template <class T>
__global__ __launch_bounds__(kCombineThreads) void moe_combine_any_kernel(CombineArgs a, uint32_t pieces, int64_t blocks) {
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int64_t t = b / pieces, col = (b - t * pieces) * kCombineThreads + threadIdx.x;
    if (col >= a.hidden) continue;
    const float* w = a.weights + t * a.w_row;
    float sum = 0.0f;
    for (int i = 0; i < a.top_k; ++i)
      if (w[i] != 0.0f) sum = fmaf(w[i], load1<T>(a.y, (t * a.top_k + i) * a.y_row + col), sum);
    if (a.shared) sum = fmaf(gate_of(a, t), load1<T>(a.shared, t * a.shared_row + col), sum);
    store1<T>(a.out, t * a.out_row + col, sum);
  }
}

template <class T>
void combine_as(const CombineArgs& a, hipStream_t stream) {
  constexpr int N = Vec<T>::N;
  const bool whole = a.hidden % N == 0 && a.y_row % N == 0 && a.out_row % N == 0 && aligned16(a.y) &&
                     aligned16(a.out) && (!a.shared || (aligned16(a.shared) && a.shared_row % N == 0));
  const int64_t per = (int64_t)kCombineThreads * (whole ? N : 1), pieces = (a.hidden + per - 1) / per;
  const int64_t blocks = a.tokens * pieces;
  const dim3 grid((unsigned)std::min<int64_t>(blocks, 1 << 24));
  if (whole)
    HGK_LAUNCH(moe_combine_kernel<T>, grid, dim3(kCombineThreads), 0, stream, a, (uint32_t)pieces, blocks);
  else
    HGK_LAUNCH(moe_combine_any_kernel<T>, grid, dim3(kCombineThreads), 0, stream, a, (uint32_t)pieces, blocks);
}

bool is_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace hgk

using namespace hgk;

extern "C" int hgk_moe_route(int dtype, const void* logits, int64_t logits_row_stride, const float* bias, int scores,
                             int64_t tokens, int64_t n_experts, int64_t top_k, int64_t groups, int64_t top_groups,
                             int group_top, int renormalize, float scale, float* weights, int32_t* experts,
                             void* stream) {
  const char* what = "hgk_moe_route";
  clear_error();
  if (!is_float_dtype(dtype)) return fail(HGK_ERR_ARG, "%s: logits of dtype %s", what, dtype_name(dtype));
  if (scores != HGK_SCORE_SOFTMAX && scores != HGK_SCORE_SIGMOID) return fail(HGK_ERR_ARG, "%s: scores=%d", what, scores);
  if (tokens < 0 || n_experts < 1) return fail(HGK_ERR_ARG, "%s: %lld tokens, %lld experts", what, (long long)tokens, (long long)n_experts);
  if (n_experts > kRouteExperts)
    return fail(HGK_ERR_UNSUPPORTED, "%s: %lld experts (at most %d)", what, (long long)n_experts, kRouteExperts);
  if (top_k < 1 || top_k > n_experts) return fail(HGK_ERR_ARG, "%s: top_k=%lld of %lld experts", what, (long long)top_k, (long long)n_experts);
  if (top_k > kRouteTopK) return fail(HGK_ERR_UNSUPPORTED, "%s: top_k=%lld (at most %d)", what, (long long)top_k, kRouteTopK);
  if (groups < 1 || n_experts % groups || top_groups < 1 || top_groups > groups)
    return fail(HGK_ERR_ARG, "%s: %lld of %lld groups of %lld experts", what, (long long)top_groups, (long long)groups, (long long)n_experts);
  if (groups > 64) return fail(HGK_ERR_UNSUPPORTED, "%s: %lld groups (at most 64)", what, (long long)groups);
  if (top_k > top_groups * (n_experts / groups))
    return fail(HGK_ERR_ARG, "%s: top_k=%lld of %lld groups of %lld", what, (long long)top_k, (long long)top_groups, (long long)(n_experts / groups));
  if (group_top != 1 && group_top != 2) return fail(HGK_ERR_ARG, "%s: group_top=%d (1 or 2)", what, group_top);
  if (group_top > n_experts / groups && top_groups < groups)
    return fail(HGK_ERR_ARG, "%s: group_top=%d of groups of %lld", what, group_top, (long long)(n_experts / groups));
  if (!std::isfinite(scale)) return fail(HGK_ERR_ARG, "%s: scale must be finite", what);
  if (logits_row_stride < 0) return fail(HGK_ERR_ARG, "%s: negative row stride", what);
  // As few lanes a token as hold its experts: rounds of a small fold, tokens side by
  // side. (Not by the tokens' number: a token's bits are the same in every batch.)
  RoutePlan plan{};
  for (int bits = 4; bits <= 6 && !plan.per; ++bits) plan = plan_route(groups, n_experts / groups, top_k, bits);
  if (!plan.per)
    return fail(HGK_ERR_UNSUPPORTED, "%s: %lld groups of %lld experts", what, (long long)groups, (long long)(n_experts / groups));
  if (tokens > INT32_MAX) return fail(HGK_ERR_ARG, "%s: %lld tokens are too many", what, (long long)tokens);
  if (tokens == 0) return HGK_OK;
  if (!logits || !weights || !experts) return fail(HGK_ERR_ARG, "%s: null logits, weights or experts", what);
  if (!is_aligned(logits, dtype_bytes(dtype)) || !is_aligned(bias, 4) || !is_aligned(weights, 4) || !is_aligned(experts, 4))
    return fail(HGK_ERR_ARG, "%s: operands must be aligned to their elements", what);
  RouteArgs a{static_cast<const char*>(logits), bias, weights, experts, logits_row_stride, tokens, (int32_t)n_experts,
              (int32_t)top_k, (int32_t)groups, (int32_t)top_groups, group_top, (int32_t)(n_experts / groups),
              scores == HGK_SCORE_SIGMOID, renormalize != 0, plan.group_bits, 0, 0, scale};
  const bool sums = bias || (group_top == 2 && top_groups < groups);
  switch (dtype) {
    case DT_BF16: route_as<BF16>(a, plan, sums, as_stream(stream)); break;
    case DT_F16: route_as<F16>(a, plan, sums, as_stream(stream)); break;
    default: route_as<F32>(a, plan, sums, as_stream(stream)); break;
  }
  return launch_status(what);
}

extern "C" int hgk_moe_combine(int dtype, const void* y, int64_t y_row_stride, const float* weights,
                               int64_t weights_row_stride, int64_t top_k, const void* shared, int64_t shared_row_stride,
                               const void* shared_gate, int gate_dtype, int64_t gate_row_stride, void* out,
                               int64_t out_row_stride, int64_t tokens, int64_t hidden, void* stream) {
  const char* what = "hgk_moe_combine";
  clear_error();
  if (!is_float_dtype(dtype)) return fail(HGK_ERR_ARG, "%s: y of dtype %s", what, dtype_name(dtype));
  if (tokens < 0 || hidden < 0 || top_k < 1 || top_k > INT32_MAX)
    return fail(HGK_ERR_ARG, "%s: tokens=%lld, hidden=%lld, top_k=%lld", what, (long long)tokens, (long long)hidden, (long long)top_k);
  if (shared_gate && !shared) return fail(HGK_ERR_ARG, "%s: a gate without the rows that it gates", what);
  if (shared_gate && !is_float_dtype(gate_dtype)) return fail(HGK_ERR_ARG, "%s: gate of dtype %s", what, dtype_name(gate_dtype));
  if (tokens == 0 || hidden == 0) return HGK_OK;
  if (!y || !weights || !out) return fail(HGK_ERR_ARG, "%s: null y, weights or out", what);
  const int size = dtype_bytes(dtype);
  if (!is_aligned(y, size) || !is_aligned(out, size) || !is_aligned(shared, size) || !is_aligned(weights, 4) ||
      (shared_gate && !is_aligned(shared_gate, dtype_bytes(gate_dtype))))
    return fail(HGK_ERR_ARG, "%s: operands must be aligned to their elements", what);
  if (y_row_stride < 0 || weights_row_stride < 0 || (shared && shared_row_stride < 0) || (shared_gate && gate_row_stride < 0))
    return fail(HGK_ERR_ARG, "%s: negative row stride", what);
  if (tokens > 1 && out_row_stride < hidden)
    return fail(HGK_ERR_ARG, "%s: out rows overlap (stride %lld)", what, (long long)out_row_stride);
  if (tokens > INT32_MAX / top_k || hidden > INT32_MAX)
    return fail(HGK_ERR_ARG, "%s: %lld tokens of %lld rows are too many", what, (long long)tokens, (long long)top_k);
  CombineArgs a{static_cast<const char*>(y), weights, static_cast<const char*>(shared),
                static_cast<const char*>(shared_gate), static_cast<char*>(out), y_row_stride,
                shared ? shared_row_stride : 0, gate_row_stride, tokens > 1 ? out_row_stride : 0, weights_row_stride,
                tokens, hidden, (int32_t)top_k, gate_dtype};
  switch (dtype) {
    case DT_BF16: combine_as<BF16>(a, as_stream(stream)); break;
    case DT_F16: combine_as<F16>(a, as_stream(stream)); break;
    default: combine_as<F32>(a, as_stream(stream)); break;
  }
  return launch_status(what);
}
