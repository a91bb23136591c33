// moe.hip -- what stands around the routed experts' products: the choice of each
// token's experts with their weights, and the weighted sum of their outputs.
#include <algorithm>
#include <cmath>

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
  int32_t sigmoid, renormalize;
  float scale;
};

constexpr float kLog2e = 1.44269504088896341f;

// e^x to about 2^-22 of itself: x log2(e) in two parts, the lesser one put back
// by its series (the product alone is off by up to 2^-17 of the result at x = -88).
__device__ inline float exp_f32(float x) {
  const float t = x * kLog2e, r = fmaf(x, kLog2e, -t) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return x < -150.0f ? 0.0f : fmaf(e, r * 0.693147181f, e);
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

// A choice as whole numbers in the same order, none of them 0: that is a choice
// that has been taken. NaN counts as the lowest.
__device__ inline uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t b = f2u(x == 0.0f ? 0.0f : x);  // one zero
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline uint64_t key_of(double x) {
  if (x != x) x = -INFINITY;
  const uint64_t b = __builtin_bit_cast(uint64_t, x == 0.0 ? 0.0 : x);
  return b >> 63 ? ~b : b | 1ull << 63;
}

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

template <class V> struct KeyOf;
template <> struct KeyOf<float> { typedef uint32_t type; };
template <> struct KeyOf<double> { typedef uint64_t type; };

// 2^BITS lanes have a token; a lane has PER experts in a row, of one group. V:
// the type of the choices. Where nothing is added to the scores they are in the
// order of the logits, which are compared as they are; where a bias or a second
// score is added, two sums may lie closer than f32 holds scores, and are 64 bits.
// A round takes the best choice left, its expert found by two folds over the
// lanes, and the lane that had it looks for its next best.
template <class T, class V, int BITS, int PER>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteArgs a) {
  typedef typename KeyOf<V>::type Key;
  constexpr int W = 1 << BITS;
  const int sub = threadIdx.x & (W - 1);
  const int64_t token = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
  const char* row = a.logits + (token < a.tokens ? token : 0) * a.row * T::kBytes;

  // lanes of a group, and this lane's experts
  int gbits = BITS;
  while (gbits > 0 && (a.groups << gbits) > W) --gbits;
  const int group = sub >> gbits, in = (sub & ((1 << gbits) - 1)) * PER;
  const int e0 = group * a.group_size + in;
  const int mine = group < a.groups ? min(max(a.group_size - in, 0), PER) : 0;

  float x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    x[i] = i < mine ? load1<T>(row, e0 + i) : -INFINITY;
    if (x[i] != x[i]) x[i] = -INFINITY;
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) top = fmaxf(top, x[i]);
  top = fold<BITS>(top, [](float p, float q) { return fmaxf(p, q); });

  // choices
  V c[PER];
  double whole = 1.0;  // softmax: the sum over all experts
  if constexpr (sizeof(V) == 4) {
#pragma unroll
    for (int i = 0; i < PER; ++i) c[i] = x[i];
  } else {
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = 1.0 / (1.0 + exp(-(double)x[i]));
    } else {
      double part = 0.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        c[i] = x[i] == -INFINITY ? 0.0 : x[i] == top ? 1.0 : exp((double)x[i] - (double)top);
        part += c[i];
      }
      whole = fold<BITS>(part, [](double p, double q) { return p + q; });
      if (whole == 0.0) whole = 1.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] /= whole;
    }
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < mine) c[i] += (double)a.bias[e0 + i];
    }
  }
  Key key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = i < mine ? key_of(c[i]) : 0;

  // groups: all but the best are taken out
  if (a.top_groups < a.groups) {
    V b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const V v = i < mine && c[i] == c[i] ? c[i] : -INFINITY;
      b2 = fmax(b2, fmin(b1, v));
      b1 = fmax(b1, v);
    }
    auto join = [&](V p, V q) {
      b2 = fmax(fmin(b1, p), fmax(b2, q));
      b1 = fmax(b1, p);
    };
    if (gbits > 0) join(partner<0>(b1), partner<0>(b2));
    if (gbits > 1) join(partner<1>(b1), partner<1>(b2));
    if (gbits > 2) join(partner<2>(b1), partner<2>(b2));
    if (gbits > 3) join(partner<3>(b1), partner<3>(b2));
    if constexpr (BITS > 4) if (gbits > 4) join(partner<4>(b1), partner<4>(b2));
    Key left = group < a.groups ? key_of(a.group_top == 2 ? b1 + b2 : b1) : 0;
    bool kept = false;
    for (int r = 0; r < a.top_groups; ++r)
      if (best_of<BITS>(left, (uint32_t)group) == (uint32_t)group) {
        kept = true;
        left = 0;
      }
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = kept ? key[i] : 0;
  }

  Key best = 0;
  uint32_t at = 0;
  auto look = [&]() {
    best = key[0];
    at = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i) {
      at = key[i] > best ? i : at;
      best = key[i] > best ? key[i] : best;
    }
  };
  look();
  uint32_t expert = 0;
  for (int r = 0; r < a.top_k; ++r) {
    const uint32_t w = best_of<BITS>(best, e0 + at);
    if (sub == r) expert = w;
    if (w == e0 + at && best != 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = at == (uint32_t)i ? 0 : key[i];
      look();
    }
  }

  // lane r: the weight of expert r
  const bool has = sub < a.top_k;
  float l = has ? load1<T>(row, expert) : -INFINITY, s;
  if (l != l) l = -INFINITY;
  if (a.sigmoid) {
    // of a large negative logit the exponential is the score
    const float e = exp_f32(-fabsf(l));
    s = (l < 0.0f ? e : 1.0f) / (1.0f + e);
  } else {
    // (renormalised weights are of no sum over all experts)
    s = l == -INFINITY ? 0.0f : l == top ? 1.0f : exp_f32(l - top);
    if (!a.renormalize) {
      if constexpr (sizeof(V) == 4) {
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) part += x[i] == -INFINITY ? 0.0f : x[i] == top ? 1.0f : exp_f32(x[i] - top);
        part = fold<BITS>(part, [](float p, float q) { return p + q; });
        s = part > 0.0f ? s / part : 0.0f;
      } else {
        s /= (float)whole;
      }
    }
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

template <class T, class V, int BITS, int PER>
void launch_route(const RouteArgs& a, hipStream_t stream) {
  constexpr int kTokens = 256 >> BITS;
  HGK_LAUNCH((moe_route_kernel<T, V, BITS, PER>), dim3((unsigned)((a.tokens + kTokens - 1) / kTokens)), dim3(256), 0,
             stream, a);
}
template <class T, class V>
void route_of(const RouteArgs& a, hipStream_t stream) {
  // experts that a lane of 64 has, when groups keep to lanes of their own
  int lanes = 64;
  while (lanes > 1 && a.groups * lanes > 64) lanes >>= 1;
  const int per = (a.group_size + lanes - 1) / lanes;
  if (per <= 1) launch_route<T, V, 6, 1>(a, stream);
  else if (per <= 2) launch_route<T, V, 6, 2>(a, stream);
  else if (per <= 4) launch_route<T, V, 6, 4>(a, stream);
  else if (per <= 8) launch_route<T, V, 6, 8>(a, stream);
  else launch_route<T, V, 6, 16>(a, stream);
}
template <class T>
void route_as(const RouteArgs& a, bool wide, hipStream_t stream) {
  if (wide) route_of<T, double>(a, stream);
  else route_of<T, float>(a, stream);
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
constexpr int kCombineThreads = 128, kRows = 4;
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
  // lanes of a group hold at most 16 experts each
  int lanes = 64;
  while (groups * lanes > 64) lanes >>= 1;
  if ((n_experts / groups + lanes - 1) / lanes > 16)
    return fail(HGK_ERR_UNSUPPORTED, "%s: %lld groups of %lld experts", what, (long long)groups, (long long)(n_experts / groups));
  if (tokens > INT32_MAX) return fail(HGK_ERR_ARG, "%s: %lld tokens are too many", what, (long long)tokens);
  if (tokens == 0) return HGK_OK;
  if (!logits || !weights || !experts) return fail(HGK_ERR_ARG, "%s: null logits, weights or experts", what);
  if (!is_aligned(logits, dtype_bytes(dtype)) || !is_aligned(bias, 4) || !is_aligned(weights, 4) || !is_aligned(experts, 4))
    return fail(HGK_ERR_ARG, "%s: operands must be aligned to their elements", what);
  RouteArgs a{static_cast<const char*>(logits), bias, weights, experts, logits_row_stride, tokens, (int32_t)n_experts,
              (int32_t)top_k, (int32_t)groups, (int32_t)top_groups, group_top, (int32_t)(n_experts / groups),
              scores == HGK_SCORE_SIGMOID, renormalize != 0, scale};
  const bool wide = bias || (group_top == 2 && top_groups < groups);
  switch (dtype) {
    case DT_BF16: route_as<BF16>(a, wide, as_stream(stream)); break;
    case DT_F16: route_as<F16>(a, wide, as_stream(stream)); break;
    default: route_as<F32>(a, wide, as_stream(stream)); break;
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
