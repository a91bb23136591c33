// attn.hip -- attention of new tokens over a paged key-value cache.
#include <algorithm>
#include <cmath>

#include "kv.h"

namespace hgk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  KvView p;
  KvBatchView b;
  const char* q;
  char* out;
  int64_t qst[2], ost[2];  // token, head
  int32_t q_heads, group;  // group = q heads per kv head
  float scale, softcap;
  int32_t window, sinks;
  int32_t splits;  // parts of the cache; more than one: joined from the workspace
  float* part;     // [tokens * q_heads][splits][head_dim], not normalised
  float* stat;     // [tokens * q_heads][splits][2]: reference (log2 domain), sum
};

// Matrix instructions, pair packing and the non-finite test of the two types.
template <class T> struct Mx;
template <> struct Mx<BF16> {
  static __device__ inline f32x4 mma16x32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ inline f32x4 mma16x16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                     __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
};
template <> struct Mx<F16> {
  static __device__ inline f32x4 mma16x32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ inline f32x4 mma16x16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  }
};

constexpr float kLog2e = 1.44269504088896341f;

// Four 16-bit values of one column from LDS: lane l of each 16 names the row
// l/4 and the columns 4 (l%4) .. +3, and receives column l of rows 0..3.
__device__ inline u32x2 lds_transposed(const char* p) {
  typedef __attribute__((address_space(3))) s16x4* lds_p;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (lds_p)(__attribute__((address_space(3))) char*)p));
}

// The scores' scale, folded so that a raw score x (the dot product, or the
// tanh of the scaled one under a soft cap) has exp2 exponent c * x with c > 0:
// a negative scale flips q's signs, a scale of zero makes q zero.
struct Scale {
  float c, inner;      // inner: scale / softcap
  uint32_t flip, keep; // q word = (q & keep) ^ flip
};
template <bool CAP>
__device__ inline Scale fold_scale(const AttnArgs& a) {
  Scale s;
  s.flip = 0;
  s.keep = ~0u;
  if constexpr (CAP) {
    s.c = a.softcap * kLog2e;
    s.inner = a.scale / a.softcap;
  } else {
    s.inner = 0.0f;
    s.c = fabsf(a.scale) * kLog2e;
    if (a.scale < 0.0f) s.flip = 0x80008000u;
    if (s.c == 0.0f) {
      s.c = 1.0f;
      s.keep = 0u;
    }
  }
  return s;
}

// tanh from one exp2 and one reciprocal: 1 - 2 / (e^2x + 1). Its absolute
// error, a few 2^-24, is what matters for softcap * tanh as a score.
__device__ inline float fast_tanh(float x) {
  const float e = __builtin_amdgcn_exp2f(x * (2.0f * kLog2e));
  return fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
}

// The running maximum only has to keep exp2 in range, so a row's reference
// moves when a raw score passes it by more than 2^kSlack in weight, and not
// with every new maximum: f32 sums and 16-bit weights up to 2^kSlack lose nothing.
constexpr float kSlack = 8.0f;

// The reference of a row that has seen no score: below every score that can
// occur, and finite times c.
__device__ inline float lowest_ref(float c) { return -3.0e38f / fmaxf(c, 1.0f); }

// ---------------------------------------------------------------- one token
// The keys that a sequence's last token sees, as one run of n: index i is key
// i below `sinks`, and key i + skip behind them.
struct Seen {
  int32_t n, sinks, skip;
};
__device__ inline Seen seen_by_last(const AttnArgs& a, int32_t len) {
  const int64_t cap = (int64_t)a.b.width << a.p.page_shift;
  Seen s;
  if (len < 0) len = 0;
  const int32_t lo = a.window > 0 && len > a.window ? len - a.window : 0;
  s.sinks = a.sinks < lo ? a.sinks : lo;
  s.skip = lo - s.sinks;
  if (cap < len) {  // the table ends before the sequence
    len = (int32_t)cap;
    if (s.sinks > len) s.sinks = len;
  }
  s.n = s.sinks + (len > lo ? len - lo : 0);
  return s;
}

constexpr int kDecWaves = 4;

// One new token per sequence: block = (part of the cache, 16 of a kv head's
// query heads, sequence and kv head). Each wave walks its own tiles of NS * 16
// keys with a softmax of its own; nothing is shared until the end, so no wave
// waits for another.
//
// A tile's scores are S^T = K Q^T on 16x16x32 matrix instructions: keys are
// the rows, so K's 16-byte pieces go from memory straight into the operand,
// and a lane ends with 4 keys each of one head. That is also where the second
// product O^T = V^T P^T wants its weights: no weight crosses lanes. V^T comes
// through LDS (written row by row, read transposed). K and V of the next tile
// are in flight while a tile is computed.
//
// Weights are split in two 16-bit parts (hi + lo, both multiplied): the
// matrix cores have time to spare, and the result is as good as f32 weights.
template <class T, int D, int NS, bool CAP>
__global__ __launch_bounds__(64 * kDecWaves, 2) void attn_decode_kernel(AttnArgs a) {
  constexpr int kKeys = 16 * NS, kStep = D / 32, kOut = D / 16;
  // V rows 32 bytes apart in banks: 16 rows of a transposed read cover each bank twice
  constexpr int kRow = 2 * D + 32, kTile = kKeys * kRow;
  constexpr int kJoin = kDecWaves * 16 * D * 4;
  __shared__ __align__(16) char lds[kTile * kDecWaves > kJoin ? kTile * kDecWaves : kJoin];
  __shared__ float wref[kDecWaves][16], wsum[kDecWaves][16];
  __shared__ int wseen[kDecWaves];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = lane & 15, j = lane >> 4;
  const int seq = blockIdx.x / a.p.kv_heads, hk = blockIdx.x - seq * a.p.kv_heads, part = blockIdx.z;
  const int h0 = hk * a.group + blockIdx.y * 16;  // first of this block's heads
  const int heads = min(16, a.group - (int)blockIdx.y * 16);
  const Scale sc = fold_scale<CAP>(a);

  // this block's keys: whole tiles, as even as they go
  const Seen seen = seen_by_last(a, a.b.lens[seq]);
  const int tiles = (seen.n + kKeys - 1) / kKeys;
  int per = (tiles + a.splits - 1) / a.splits;
  if (per < 2 * kDecWaves) per = 2 * kDecWaves;
  const int first = min((int64_t)per * part, (int64_t)tiles);
  const int last = min(first + per, tiles);

  u32x4 qf[kStep];
  {
    const char* qp = a.q + 2 * (seq * a.qst[0] + (h0 + (m < heads ? m : 0)) * a.qst[1] + 8 * j);
#pragma unroll
    for (int s = 0; s < kStep; ++s) {
      qf[s] = *reinterpret_cast<const u32x4*>(qp + 64 * s);
      for (int w = 0; w < 4; ++w) qf[s][w] = (qf[s][w] & sc.keep) ^ sc.flip;
    }
  }

  const int32_t* table = a.b.table + (int64_t)seq * a.b.table_stride;
  const char* kbase = a.p.k + 2 * (hk * a.p.kst[2] + 8 * j);
  const char* vbase = a.p.v + 2 * (hk * a.p.vst[2] + 8 * j);
  // page of key i of the run (-1: none) and its place in the page
  auto look_up = [&](int tile, int32_t* page, int32_t* at) {
#pragma unroll
    for (int h = 0; h < NS; ++h) {
      const int i = tile * kKeys + 16 * h + m;
      page[h] = -1;
      at[h] = 0;
      if (tile < last && i < seen.n) {
        const int32_t key = i < seen.sinks ? i : i + seen.skip;
        page[h] = table[key >> a.p.page_shift];
        at[h] = key & a.p.page_mask;
      }
    }
  };
  u32x4 kr[NS][kStep], vr[NS][kStep];
  uint32_t there = 0;  // bit i: key i of the loaded tile exists
  auto load = [&](const int32_t* page, const int32_t* at) {
    there = 0;
#pragma unroll
    for (int h = 0; h < NS; ++h) {
      const bool ok = (uint32_t)page[h] < (uint32_t)a.p.n_pages;
      there |= (uint32_t)(__ballot(ok) & 0xffffu) << (16 * h);
      // a key that does not exist reads the pool's first row, and is masked below
      const int64_t pg = ok ? page[h] : 0, r = ok ? at[h] : 0;
      const char* kp = kbase + 2 * (pg * a.p.kst[0] + r * a.p.kst[1]);
      const char* vp = vbase + 2 * (pg * a.p.vst[0] + r * a.p.vst[1]);
#pragma unroll
      for (int s = 0; s < kStep; ++s) kr[h][s] = *reinterpret_cast<const u32x4*>(kp + 64 * s);
#pragma unroll
      for (int s = 0; s < kStep; ++s) vr[h][s] = *reinterpret_cast<const u32x4*>(vp + 64 * s);
    }
  };

  f32x4 o[kOut];
#pragma unroll
  for (int t = 0; t < kOut; ++t) o[t] = f32x4{0, 0, 0, 0};
  float ref = lowest_ref(sc.c), sum = 0.0f;
  const float slack = kSlack / sc.c;
  bool any = false;
  constexpr uint32_t kAll = NS == 2 ? 0xffffffffu : 0xffffu;
  char* vt = lds + wave * kTile;

  int32_t page[NS], at[NS];
  if (a.p.n_pages > 0 && first + wave < last) {
    look_up(first + wave, page, at);
    load(page, at);
    look_up(first + wave + kDecWaves, page, at);
    for (int tile = first + wave; tile < last; tile += kDecWaves) {
      // scores
      f32x4 s[NS];
#pragma unroll
      for (int h = 0; h < NS; ++h) {
        s[h] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < kStep; ++k) s[h] = Mx<T>::mma16x32(kr[h][k], qf[k], s[h]);
      }
      const uint32_t now = there;
      if (now != kAll) {  // values that do not exist must not be multiplied by their zero weight
#pragma unroll
        for (int h = 0; h < NS; ++h)
          if (!((now >> (16 * h + m)) & 1))
#pragma unroll
            for (int k = 0; k < kStep; ++k) vr[h][k] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int h = 0; h < NS; ++h)
#pragma unroll
        for (int k = 0; k < kStep; ++k)
          *reinterpret_cast<u32x4*>(vt + (16 * h + m) * kRow + 64 * k + 16 * j) = vr[h][k];
      if (tile + kDecWaves < last) {
        load(page, at);
        look_up(tile + 2 * kDecWaves, page, at);
      }
      // weights
      float x[4 * NS], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) {
        x[i] = s[i / 4][i % 4];
        if constexpr (CAP) x[i] = fast_tanh(x[i] * sc.inner);
      }
      const uint32_t mine = now >> (4 * j);  // this lane's keys: bits 0..3 and 16..19
      if (now != kAll) {
#pragma unroll
        for (int i = 0; i < 4 * NS; ++i)
          if (!((mine >> (16 * (i / 4) + i % 4)) & 1)) x[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) top = fmaxf(top, x[i]);
      if (__any(top > ref + slack)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = fmaxf(ref, top), f = __builtin_amdgcn_exp2f((ref - to) * sc.c);
        sum *= f;
#pragma unroll
        for (int t = 0; t < kOut; ++t) o[t] *= f;
        ref = to;
      }
      const float base = -ref * sc.c;
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], sc.c, base));
      if (now != kAll) {
#pragma unroll
        for (int i = 0; i < 4 * NS; ++i)
          if (!((mine >> (16 * (i / 4) + i % 4)) & 1)) x[i] = 0.0f;
      }
      any |= now != 0;
      uint32_t hi[2 * NS], lo[2 * NS];
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        sum += x[2 * i] + x[2 * i + 1];
        hi[i] = Mx<T>::pack(x[2 * i], x[2 * i + 1]);
        lo[i] = Mx<T>::pack(x[2 * i] - T::lo(hi[i]), x[2 * i + 1] - T::hi(hi[i]));
      }
      // O^T += V^T P^T
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < kOut; ++t) {
        const char* p = vt + (4 * j + m / 4) * kRow + 32 * t + 8 * (m & 3);
        const u32x2 v0 = lds_transposed(p);
        if constexpr (NS == 2) {
          const u32x2 v1 = lds_transposed(p + 16 * kRow);
          const u32x4 v = {v0[0], v0[1], v1[0], v1[1]};
          o[t] = Mx<T>::mma16x32(v, u32x4{hi[0], hi[1], hi[2], hi[3]}, o[t]);
          o[t] = Mx<T>::mma16x32(v, u32x4{lo[0], lo[1], lo[2], lo[3]}, o[t]);
        } else {
          o[t] = Mx<T>::mma16x16(v0, u32x2{hi[0], hi[1]}, o[t]);
          o[t] = Mx<T>::mma16x16(v0, u32x2{lo[0], lo[1]}, o[t]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  // join the waves
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  __syncthreads();  // every wave is done with its V tile
  float* wo = reinterpret_cast<float*>(lds) + wave * 16 * D;
#pragma unroll
  for (int t = 0; t < kOut; ++t) *reinterpret_cast<f32x4*>(wo + m * D + 16 * t + 4 * j) = o[t];
  if (lane < 16) {
    wref[wave][lane] = ref;
    wsum[wave][lane] = sum;
  }
  if (lane == 0) wseen[wave] = any;
  __syncthreads();
  bool some = false;
  for (int w = 0; w < kDecWaves; ++w) some |= wseen[w] != 0;
  for (int idx = threadIdx.x; idx < heads * (D / 2); idx += 64 * kDecWaves) {
    const int h = idx / (D / 2), d = 2 * (idx - h * (D / 2));
    float top = wref[0][h];
    for (int w = 1; w < kDecWaves; ++w) top = fmaxf(top, wref[w][h]);
    float l = 0.0f, v0 = 0.0f, v1 = 0.0f;
    for (int w = 0; w < kDecWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f((wref[w][h] - top) * sc.c);
      const float* src = reinterpret_cast<float*>(lds) + (w * 16 + h) * D + d;
      l = fmaf(wsum[w][h], f, l);
      v0 = fmaf(src[0], f, v0);
      v1 = fmaf(src[1], f, v1);
    }
    const int64_t row = (int64_t)seq * a.q_heads + h0 + h;
    if (a.splits > 1) {
      if (some) {
        float* p = a.part + (row * a.splits + part) * D + d;
        *reinterpret_cast<f32x2*>(p) = f32x2{v0, v1};
      }
      if (d == 0) {
        float* st = a.stat + 2 * (row * a.splits + part);
        st[0] = some ? top * sc.c : -INFINITY;
        st[1] = l;
      }
    } else {
      const float r = 1.0f / l;
      *reinterpret_cast<uint32_t*>(a.out + 2 * (seq * a.ost[0] + (h0 + h) * a.ost[1] + d)) =
          some ? T::pack(v0 * r, v1 * r) : 0u;
    }
  }
}

// Joins the parts of one row (token and query head) per block: out =
// sum_s 2^(ref_s - max) part_s / sum_s 2^(ref_s - max) sum_s. Parts that saw
// no key (ref = -inf) were not written.
template <class T>
__global__ __launch_bounds__(128) void attn_join_kernel(AttnArgs a) {
  const int t = blockIdx.x, h = blockIdx.y, D = a.p.head_dim, d = 2 * threadIdx.x;
  const KvSeq s = kv_seq(a.b, kv_row_owner(a.b, t));
  if (t < s.first || t >= s.first + s.n) return;
  const int64_t row = (int64_t)t * a.q_heads + h;
  const float* stat = a.stat + 2 * row * a.splits;
  float top = -INFINITY;
  for (int i = 0; i < a.splits; ++i) top = fmaxf(top, stat[2 * i]);
  if (d >= D) return;
  float l = 0.0f, v0 = 0.0f, v1 = 0.0f;
  const float* part = a.part + row * a.splits * D + d;
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) {
    if (stat[2 * i] == -INFINITY) continue;
    const float f = __builtin_amdgcn_exp2f(stat[2 * i] - top);
    const f32x2 v = *reinterpret_cast<const f32x2*>(part + (int64_t)i * D);
    l = fmaf(stat[2 * i + 1], f, l);
    v0 = fmaf(v[0], f, v0);
    v1 = fmaf(v[1], f, v1);
  }
  const float r = 1.0f / l;
  *reinterpret_cast<uint32_t*>(a.out + 2 * (t * a.ost[0] + h * a.ost[1] + d)) =
      top == -INFINITY ? 0u : T::pack(v0 * r, v1 * r);
}

// One wave per (row, query head). Lane l scores key base + l, then the lanes
// share the head's D outputs.
template <class T>
__global__ __launch_bounds__(64) void attn_simple_kernel(AttnArgs a) {
  __shared__ float qs[256], ps[64];
  const int D = a.p.head_dim, lane = threadIdx.x;
  const int t = blockIdx.x, h = blockIdx.y, hk = h / a.group;
  const int seq = kv_row_owner(a.b, t);
  const KvSeq s = kv_seq(a.b, seq);
  const int r = t - s.first;
  if (r < 0 || r >= s.n) return;
  const int64_t p64 = (int64_t)s.len - s.n + r;
  const int p = (int)p64;
  for (int d = lane; d < D; d += 64) qs[d] = load1<T>(a.q, t * a.qst[0] + h * a.qst[1] + d) * a.scale;
  __syncthreads();
  float o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
  bool any = false;
  for (int base = 0; p64 >= 0 && base <= p; base += 64) {
    const int j = base + lane;
    bool see = j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
    const int page = see ? kv_page(a.p, a.b, seq, j) : -1;
    see = page >= 0;
    float sc = -INFINITY;
    if (see) {
      const int64_t at = page * a.p.kst[0] + (j & a.p.page_mask) * a.p.kst[1] + hk * a.p.kst[2];
      sc = 0;
      for (int d = 0; d < D; ++d) sc = fmaf(qs[d], load1<T>(a.p.k, at + d), sc);
      if (a.softcap > 0) sc = a.softcap * tanhf(sc / a.softcap);
    }
    any |= __any(see);
    float mt = sc;
    for (int x = 32; x; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x));
    const float mn = fmaxf(m, mt), ref = mn == -INFINITY ? 0.f : mn;
    const float pr = see ? expf(sc - ref) : 0.f, f = expf(m - ref);
    float sum = pr;
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    l = l * f + sum;
    m = mn;
    ps[lane] = pr;
    __syncthreads();
    for (int i = 0; i < 4; ++i) o[i] *= f;
    for (int jj = 0; jj < 64; ++jj) {
      const int pg = __shfl(page, jj);
      if (pg < 0) continue;
      const int64_t at = pg * a.p.vst[0] + ((base + jj) & a.p.page_mask) * a.p.vst[1] + hk * a.p.vst[2];
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D) o[i] = fmaf(ps[jj], load1<T>(a.p.v, at + lane + 64 * i), o[i]);
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < D)
      store1<T>(a.out, t * a.ost[0] + h * a.ost[1] + lane + 64 * i, any ? o[i] / l : 0.f);
}

// Sizes shared by the call and its workspace query.
int check_sizes(const char* what, const hgk_kv_pages* pages, const hgk_kv_batch* batch, int64_t q_heads,
                int64_t window, int64_t sinks, KvView* p, KvBatchView* b) {
  if (int st = kv_check_pages(what, pages, p)) return st;
  if (int st = kv_check_batch(what, batch, b)) return st;
  if (q_heads < 1 || q_heads > 65535 || q_heads % p->kv_heads)
    return fail(HGK_ERR_ARG, "%s: %lld query heads for %d kv heads", what, (long long)q_heads, p->kv_heads);
  if ((int64_t)b->batch * p->kv_heads > INT32_MAX || (int64_t)b->tokens * q_heads > INT32_MAX)
    return fail(HGK_ERR_ARG, "%s: %lld rows of %lld heads are too many", what, (long long)b->tokens,
                (long long)q_heads);
  if (window < 0 || sinks < 0)
    return fail(HGK_ERR_ARG, "%s: window=%lld, sinks=%lld must not be negative", what, (long long)window,
                (long long)sinks);
  return HGK_OK;
}

// Parts that the cache is split into, from the sizes alone (the lengths are on
// the device): enough blocks to fill the chip, and not so many that a part
// of the longest sequence that the table holds goes below kMinPart keys.
constexpr int kMinPart = 256, kWantBlocks = 1024, kMaxSplits = 256;
int choose_splits(const KvView& p, const KvBatchView& b, int64_t blocks, int64_t window, int64_t sinks) {
  int64_t keys = (int64_t)b.width << p.page_shift;
  if (window > 0 && window < keys && sinks < keys - window) keys = window + sinks;
  int64_t s = (kWantBlocks + blocks - 1) / blocks;
  s = std::min<int64_t>(s, keys / kMinPart);
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, kMaxSplits));
}

int64_t part_bytes(int64_t rows, int splits, int64_t head_dim) {
  return splits > 1 ? rows * splits * (head_dim + 2) * 4 : 0;
}

int plan_splits(const KvView& p, const KvBatchView& b, int64_t q_heads, int64_t window, int64_t sinks) {
  if (b.starts || b.batch == 0) return 1;
  const int64_t group = q_heads / p.kv_heads;
  return choose_splits(p, b, (int64_t)b.batch * p.kv_heads * ((group + 15) / 16), window, sinks);
}

template <class T, int D, int NS>
void launch_decode(const AttnArgs& a, hipStream_t stream) {
  const dim3 grid(a.b.batch * a.p.kv_heads, (a.group + 15) / 16, a.splits), block(64 * kDecWaves);
  if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_decode_kernel<T, D, NS, true>), grid, block, 0, stream, a);
  else
    HGK_LAUNCH((attn_decode_kernel<T, D, NS, false>), grid, block, 0, stream, a);
}

template <class T>
int run(const AttnArgs& a, const char* what, hipStream_t stream) {
  if (!a.b.starts) {
    switch (a.p.head_dim) {
      case 64: launch_decode<T, 64, 2>(a, stream); break;
      case 96: launch_decode<T, 96, 2>(a, stream); break;
      case 128: launch_decode<T, 128, 2>(a, stream); break;
      default: launch_decode<T, 256, 1>(a, stream); break;
    }
  } else {
    HGK_LAUNCH(attn_simple_kernel<T>, dim3(a.b.tokens, a.q_heads), dim3(64), 0, stream, a);
  }
  if (int st = launch_status(what)) return st;
  if (a.splits == 1) return HGK_OK;
  HGK_LAUNCH(attn_join_kernel<T>, dim3(a.b.tokens, a.q_heads), dim3(128), 0, stream, a);
  return launch_status(what);
}

}  // namespace
}  // namespace hgk

using namespace hgk;

extern "C" int64_t hgk_paged_attention_workspace(const hgk_kv_pages* pages, const hgk_kv_batch* batch,
                                                 int64_t q_heads, int64_t window, int64_t sinks) {
  clear_error();
  KvView p;
  KvBatchView b;
  if (check_sizes("hgk_paged_attention_workspace", pages, batch, q_heads, window, sinks, &p, &b)) return -1;
  return part_bytes((int64_t)b.tokens * q_heads, plan_splits(p, b, q_heads, window, sinks), p.head_dim);
}

extern "C" int hgk_paged_attention(const hgk_kv_pages* pages, const hgk_kv_batch* batch, const void* q,
                                   const int64_t q_strides[2], int64_t q_heads, float scale,
                                   float softcap, int64_t window, int64_t sinks, void* out,
                                   const int64_t out_strides[2], void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const char* what = "hgk_paged_attention";
  clear_error();
  AttnArgs a;
  if (int st = check_sizes(what, pages, batch, q_heads, window, sinks, &a.p, &a.b)) return st;
  if (!std::isfinite(scale)) return fail(HGK_ERR_ARG, "%s: scale must be finite", what);
  if (!(softcap >= 0.0f) || !std::isfinite(softcap))
    return fail(HGK_ERR_ARG, "%s: softcap must be finite and not negative", what);
  if (a.b.batch == 0 || a.b.tokens == 0) return HGK_OK;
  const int64_t T = a.b.tokens, D = a.p.head_dim;
  if (int st = kv_check_rows(what, "q", q, q_strides, T, q_heads, D, false, a.qst)) return st;
  if (int st = kv_check_rows(what, "out", out, out_strides, T, q_heads, D, true, a.ost)) return st;
  a.q = static_cast<const char*>(q);
  a.out = static_cast<char*>(out);
  a.q_heads = (int32_t)q_heads;
  a.group = (int32_t)(q_heads / a.p.kv_heads);
  a.scale = scale;
  a.softcap = softcap;
  a.window = (int32_t)(window > INT32_MAX ? INT32_MAX : window);
  a.sinks = (int32_t)(sinks > INT32_MAX ? INT32_MAX : sinks);
  a.splits = plan_splits(a.p, a.b, q_heads, window, sinks);
  const int64_t need = part_bytes(T * q_heads, a.splits, D);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(HGK_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
  a.part = static_cast<float*>(workspace);
  a.stat = a.splits > 1 ? a.part + T * q_heads * a.splits * D : nullptr;
  return pages->dtype == DT_BF16 ? run<BF16>(a, what, as_stream(stream)) : run<F16>(a, what, as_stream(stream));
}
