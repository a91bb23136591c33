// attn.hip -- attention of new tokens over a paged key-value cache.
#include <algorithm>
#include <cmath>

#include "kv.h"

namespace hgk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
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
  static __device__ inline f32x16 mma32x16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
  static constexpr uint32_t kExp = 0x7f80u, kOne = 0x3f80u, k128 = 0x4300u, k16384 = 0x4680u;
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
  static __device__ inline f32x16 mma32x16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  }
  // the exponent's bits, and 1, 128 and 16384
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u, k128 = 0x5800u, k16384 = 0x7400u;
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
    s.c = fminf(a.softcap * kLog2e, 1.0e37f);
    s.inner = a.scale / a.softcap;
  } else {
    s.inner = 0.0f;
    s.c = fminf(fabsf(a.scale) * kLog2e, 1.0e37f);
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

// 2^(c (ref - to)) of a reference that moves up. Not below the smallest normal
// number: an infinite sum (of infinite values) stays infinite, and a finite
// one that far below is lost in the new one's rounding all the same.
__device__ inline float shrink(float ref, float to, float c) {
  return fmaxf(__builtin_amdgcn_exp2f((ref - to) * c), 1.2e-38f);
}

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
      if (__any(top > ref + slack)) {  // a head's own scores alone decide for it
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = top > ref + slack ? top : ref, f = shrink(ref, to, sc.c);
        sum *= f;
#pragma unroll
        for (int t = 0; t < kOut; ++t) o[t] *= f;
        ref = to;
      }
      const float base = -ref * sc.c;
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], sc.c, base));
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

// ---------------------------------------------------------------- prompts
// 16 bytes per lane from memory to LDS at dst + 16 * lane (dst is uniform):
// from base + off, or from an address of the lane's own. m0 is written inside,
// and the compiler has to know (it need not warn that nothing preserves it).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void lds_load(uint32_t dst, const char* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(dst), "v"(off), "s"(base) : "m0", "memory");
}
__device__ inline void lds_load(uint32_t dst, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(dst), "v"(p) : "m0", "memory");
}
#pragma clang diagnostic pop
__device__ inline uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// this wave's loads to LDS have landed, then the block's barrier
__device__ inline void landed_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Where the 16-byte piece c of a tile's row r lies in its row of D/8 pieces.
// Keys are read 16 rows at a time, one piece each: those go to 16 different
// places modulo 256 bytes. Values are read transposed, 4 pieces of 8 rows at a
// time: those cover 256 bytes twice.
template <int D> __device__ inline int key_place(int r, int c) {
  if constexpr (D == 64) return c ^ ((r >> 1) & 7);
  else if constexpr (D == 96) return (c + (r >> 2)) % 12;
  else return c ^ (r & 15);
}
template <int D> __device__ inline int value_place(int r, int c) {
  if constexpr (D == 64) return c ^ ((r << 1) & 4);
  else if constexpr (D == 96) return c;
  else return c ^ ((r & 3) << 2);
}
// ... and the piece that lies at place c.
template <int D> __device__ inline int key_piece(int r, int c) {
  if constexpr (D == 96) return (c + 24 - (r >> 2)) % 12;
  else return key_place<D>(r, c);
}

// The rows of a (sequence, kv head): row r is query token r / group with the
// kv head's query head r % group, so that all heads of a group, and as many
// tokens as fit, read a tile of keys once.
//
// A non-finite value in a tile that some row sees only in part: a weight of
// zero times infinity would be NaN. Such a tile's values are counted on the
// matrix cores (+inf as 1, -inf as 128, NaN as 16384, times 1 where the row
// sees the key: at most 64 keys a tile, so the sum gives the three counts
// back), and the product runs with zeros in their place.
template <class M>
__device__ inline uint32_t finite_pair(uint32_t w) {
  uint32_t m = 0;
  if ((w & M::kExp) != M::kExp) m |= 0xffffu;
  if (((w >> 16) & M::kExp) != M::kExp) m |= 0xffff0000u;
  return w & m;
}
template <class M>
__device__ inline uint32_t count_code(uint32_t h) {
  if ((h & M::kExp) != M::kExp) return 0;
  if (h & 0x7fffu & ~M::kExp) return M::k16384;
  return h & 0x8000u ? M::k128 : M::kOne;
}
template <class M>
__device__ inline uint32_t count_pair(uint32_t w) {
  return count_code<M>(w & 0xffffu) | count_code<M>(w >> 16) << 16;
}
// top bits set where a half is not finite
template <class M>
__device__ inline uint32_t odd_pair(uint32_t w) {
  constexpr uint32_t e = M::kExp | M::kExp << 16, one = (M::kExp & -M::kExp) * 0x10001u;
  return ((w & e) + one) & 0x80008000u;
}

// Block = (kv head, tile of 32 * NW rows, part of its tiles of BN keys); a wave
// has 32 rows. As in the decode kernel S^T = K Q^T and O^T = V^T P^T, here on
// 32x32x16 instructions: a lane has half the scores of one row in registers,
// its weights are the second product's operand as they stand, and a row's
// reference and sum are one register each.
//
// K and V tiles come straight from memory to LDS, double buffered: the next
// tile's loads are issued before a tile is computed, one barrier a tile.
template <class T, int D, int NW, int BN, bool CAP>
__global__ __launch_bounds__(64 * NW, 2) void attn_prompt_kernel(AttnArgs a) {
  constexpr int NT = 64 * NW, BM = 32 * NW, CH = D / 8, kUnits = BN * CH / NT;
  constexpr int kRow = 2 * D, kTile = BN * kRow;
  constexpr int KT = BN / 32, QS = D / 16, DT = D / 32;
  static_assert(BN * CH % NT == 0, "whole units per thread");
  typedef Mx<T> M;
  __shared__ __align__(16) char lds[4 * kTile];  // keys, values; keys, values
  __shared__ int odd;  // 1 + index of the last tile found to hold values that are not finite

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.x, G = a.group;

  // which sequence's tile this is: tiles are counted over the sequences, from
  // the last one on (the longest ones of a prompt first)
  int seq = -1, tile = 0;
  KvSeq s{0, 0, 0};
  {
    int want = gridDim.y - 1 - blockIdx.y, before = 0;
    for (int b0 = 0; b0 < a.b.batch; b0 += 64) {
      const int b = b0 + lane;
      const KvSeq c = b < a.b.batch ? kv_seq(a.b, b) : KvSeq{0, 0, 0};
      const int mine = (c.n * G + BM - 1) / BM;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
      }
      const uint64_t has = __ballot(before + upto > want);
      if (has) {
        const int l = __builtin_ctzll(has);
        seq = b0 + l;
        tile = want - before - __builtin_amdgcn_readlane(upto - mine, l);
        s.first = __builtin_amdgcn_readlane(c.first, l);
        s.n = __builtin_amdgcn_readlane(c.n, l);
        s.len = __builtin_amdgcn_readlane(c.len, l);
        break;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (seq < 0) return;
  const int R = s.n * G, pos0 = s.len - s.n;  // pos0 may be negative: rows in front of the sequence

  // the block's keys, in tiles of BN: those of the first `sinks`, then the window's
  const int row0 = tile * BM;
  const int p_first = pos0 + row0 / G, p_last = pos0 + (min(row0 + BM, R) - 1) / G;
  const int64_t cap = (int64_t)a.b.width << a.p.page_shift;
  const int hi = (int)min((int64_t)p_last + 1, cap);
  const int lo = a.window > 0 && p_first >= a.window ? p_first - a.window + 1 : 0;
  const int t_hi = hi > 0 ? (hi + BN - 1) / BN : 0, t_lo = lo / BN;
  const int front = min(min((min(a.sinks, lo) + BN - 1) / BN, t_lo), t_hi);
  const int tiles = a.p.n_pages > 0 ? front + max(t_hi - t_lo, 0) : 0;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int it0 = min(per * (int)blockIdx.z, tiles), it1 = min(it0 + per, tiles);
  auto tile_of = [&](int it) { return it < front ? it : t_lo + it - front; };

  // this lane's row, and the range of the wave's
  const int wrow0 = row0 + 32 * wave;
  const int row = min(wrow0 + col, R - 1);
  const int qi = row / G, head = hk * G + row - qi * G, p = pos0 + qi;
  const bool in = wrow0 + col < R;
  const int pw_first = pos0 + min(wrow0, R - 1) / G, pw_last = pos0 + min(wrow0 + 31, R - 1) / G;
  const bool idle = wrow0 >= R;

  const Scale sc = fold_scale<CAP>(a);
  u32x4 qf[QS];
  {
    const char* qp = a.q + 2 * ((int64_t)(s.first + qi) * a.qst[0] + head * a.qst[1] + 8 * half);
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      qf[i] = *reinterpret_cast<const u32x4*>(qp + 32 * i);
      for (int w = 0; w < 4; ++w) qf[i][w] = (qf[i][w] & sc.keep) ^ sc.flip;
    }
  }

  // lane l looks up key l of a tile
  const int32_t* table = a.b.table + (int64_t)seq * a.b.table_stride;
  const char* kbase = a.p.k + 2 * hk * a.p.kst[2];
  const char* vbase = a.p.v + 2 * hk * a.p.vst[2];
  auto look_up = [&](int it) -> int32_t {
    if (it >= it1) return -1;
    const int key = tile_of(it) * BN + (lane & (BN - 1));
    const int32_t page = key < hi ? table[key >> a.p.page_shift] : -1;
    return (uint32_t)page < (uint32_t)a.p.n_pages ? page : -1;
  };
  // One load instruction takes 64 pieces, of rows that lie in one page when
  // pages have 16 tokens or more: its page is then scalar, and the lanes'
  // offsets are the same for every tile. A key that does not exist reads what
  // is there (a page's end, or page 0); its score is masked and its value, if
  // not finite, taken out.
  const bool whole = a.p.page_shift >= 4 && a.p.kst[1] < (1 << 24) && a.p.vst[1] < (1 << 24);
  uint32_t koff[kUnits], voff[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u0 = i * NT + 64 * wave, u = u0 + lane, r = u / CH, c = u - r * CH, r0 = u0 / CH;
    koff[i] = 2 * ((r - r0) * (uint32_t)a.p.kst[1] + 8 * key_piece<D>(r, c));
    voff[i] = 2 * ((r - r0) * (uint32_t)a.p.vst[1] + 8 * value_place<D>(r, c));
  }
  uint64_t there = 0;  // bit i: key i of the tile being loaded exists
  auto load = [&](int it, int buf, int32_t page) {
    there = __ballot(page >= 0);
    if (page < 0) page = 0;
    const int key0 = tile_of(it) * BN;
    const uint32_t kt = lds_address(lds) + buf * 2 * kTile + 1024 * wave, vt = kt + kTile;
    if (whole) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int r0 = (i * NT + 64 * wave) / CH;
        const int64_t pg = __builtin_amdgcn_readlane(page, r0), at = (key0 + r0) & a.p.page_mask;
        lds_load(kt + 16 * NT * i, kbase + 2 * (pg * a.p.kst[0] + at * a.p.kst[1]), koff[i]);
        lds_load(vt + 16 * NT * i, vbase + 2 * (pg * a.p.vst[0] + at * a.p.vst[1]), voff[i]);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kUnits; ++i) {
        const int u = i * NT + threadIdx.x, r = u / CH, c = u - r * CH;
        const int64_t pg = __shfl(page, r), at = (key0 + r) & a.p.page_mask;
        lds_load(kt + 16 * NT * i, kbase + 2 * (pg * a.p.kst[0] + at * a.p.kst[1] + 8 * key_piece<D>(r, c)));
        lds_load(vt + 16 * NT * i, vbase + 2 * (pg * a.p.vst[0] + at * a.p.vst[1] + 8 * value_place<D>(r, c)));
      }
    }
  };
  // does some row of this range see only a part of the tile?
  auto part_seen = [&](int key0, int first, int last) {
    return !(key0 + BN - 1 <= first &&
             (a.window == 0 || key0 > last - a.window || key0 + BN - 1 < a.sinks));
  };
  // does this lane's row see key i of the tile?
  auto sees = [&](int key0, uint64_t exist, int i) {
    const int key = key0 + i;
    return key <= p && (a.window == 0 || key > p - a.window || key < a.sinks) && ((exist >> i) & 1);
  };

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = f32x16{};
  float ref = lowest_ref(sc.c), sum = 0.0f;
  const float slack = kSlack / sc.c;
  bool any = false;

  // the transposed reads: value rows 4 half + (lane % 16) / 4, and pieces of
  // 8 bytes; the place of a piece depends on the row modulo 4 alone
  const int vr = 4 * half + (lane & 15) / 4, vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  uint32_t vplace[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) vplace[t] = vr * kRow + 16 * value_place<D>(vr, 4 * t + vc) + 8 * (lane & 1);

  if (threadIdx.x == 0) odd = 0;
  int32_t page = look_up(it0);
  if (it0 < it1) load(it0, 0, page);
  page = look_up(it0 + 1);
  uint64_t now = there;
  landed_barrier();

  for (int it = it0; it < it1; ++it) {
    const int buf = (it - it0) & 1;
    char* kt = lds + buf * 2 * kTile;
    char* vt = kt + kTile;
    const int key0 = tile_of(it) * BN;
    if (it + 1 < it1) {
      load(it + 1, buf ^ 1, page);
      page = look_up(it + 2);
    }
    const bool exist = BN == 64 ? now == ~0ull : (uint32_t)now == ~0u;  // all keys of the tile do
    bool strange = false;
    if (!exist || part_seen(key0, p_first, p_last)) {
      uint32_t bits = 0;
#pragma unroll 1
      for (int i = 0; i < kUnits; ++i) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(vt + 16 * (i * NT + threadIdx.x));
        bits |= odd_pair<M>(v[0]) | odd_pair<M>(v[1]) | odd_pair<M>(v[2]) | odd_pair<M>(v[3]);
      }
      if (bits) odd = it + 1;
      __syncthreads();
      strange = odd == it + 1;
    }
    const bool none = idle || key0 > pw_last ||
                      (a.window > 0 && key0 + BN - 1 <= pw_first - a.window && key0 >= a.sinks);
    u32x4 w[2 * KT];
    if (!none) {
      f32x16 x[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        x[t] = f32x16{};
#pragma unroll
        for (int i = 0; i < QS; ++i) {
          const int r = 32 * t + col;
          const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + r * kRow + 16 * key_place<D>(r, 2 * i + half));
          x[t] = M::mma32x16(kf, qf[i], x[t]);
        }
      }
      if constexpr (CAP) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[t][e] = fast_tanh(x[t][e] * sc.inner);
      }
      if (!exist || part_seen(key0, pw_first, pw_last)) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (sees(key0, now, 32 * t + 8 * (e / 4) + 4 * half + e % 4)) any = true;
            else x[t][e] = -INFINITY;
          }
      } else {
        any = true;
      }
      float top = x[0][0];
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, x[t][e]);
      if (__any(top > ref + slack)) {  // a row's own scores alone decide for it
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = top > ref + slack ? top : ref, f = shrink(ref, to, sc.c);
        sum *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= f;
        ref = to;
      }
      const float base = -ref * sc.c;
      float add[4] = {0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float w0 = __builtin_amdgcn_exp2f(fmaf(x[t][e], sc.c, base));
          const float w1 = __builtin_amdgcn_exp2f(fmaf(x[t][e + 1], sc.c, base));
          add[(e / 2) & 3] += w0 + w1;
          w[2 * t + e / 8][(e / 2) & 3] = M::pack(w0, w1);
        }
      sum += (add[0] + add[1]) + (add[2] + add[3]);
    }
    if (strange) {
      if (!none) {
#pragma unroll 1
        for (int t = 0; t < DT; ++t) {
          f32x16 n = f32x16{};
#pragma unroll 1
          for (int k = 0; k < 2 * KT; ++k) {
            const char* vp = vt + 16 * k * kRow + vr * kRow + 16 * value_place<D>(vr, 4 * t + vc) + 8 * (lane & 1);
            const u32x2 v0 = lds_transposed(vp), v1 = lds_transposed(vp + 8 * kRow);
            uint32_t see = 0;
            for (int e = 0; e < 8; ++e)
              see |= (uint32_t)sees(key0, now, 16 * k + 8 * (e / 4) + 4 * half + e % 4) << e;
            u32x4 c = {count_pair<M>(v0[0]), count_pair<M>(v0[1]), count_pair<M>(v1[0]), count_pair<M>(v1[1])}, on;
            for (int i = 0; i < 4; ++i)
              on[i] = ((see >> (2 * i)) & 1 ? M::kOne : 0u) | ((see >> (2 * i)) & 2 ? M::kOne << 16 : 0u);
            n = M::mma32x16(c, on, n);
          }
          f32x16 f;
          for (int e = 0; e < 16; ++e) {
            const int counts = (int)n[e], nan = counts >> 14, neg = (counts >> 7) & 127, pos = counts & 127;
            f[e] = nan || (neg && pos) ? __builtin_nanf("") : neg ? -INFINITY : pos ? INFINITY : 0.0f;
          }
#pragma unroll
          for (int u = 0; u < DT; ++u)
            if (u == t) o[u] += f;
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < kUnits; ++i) {
        u32x4* v = reinterpret_cast<u32x4*>(vt + 16 * (i * NT + threadIdx.x));
        u32x4 t = *v;
        for (int j = 0; j < 4; ++j) t[j] = finite_pair<M>(t[j]);
        *v = t;
      }
      __syncthreads();
    }
    if (!none) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int k = 0; k < 2 * KT; ++k) {
          const char* vp = vt + vplace[t] + 16 * k * kRow;
          const u32x2 v0 = lds_transposed(vp), v1 = lds_transposed(vp + 8 * kRow);
          o[t] = M::mma32x16(u32x4{v0[0], v0[1], v1[0], v1[1]}, w[k], o[t]);
        }
    }
    now = there;
    landed_barrier();
  }

  sum += __shfl_xor(sum, 32);
  any |= __shfl_xor((int)any, 32) != 0;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)(s.first + qi) * a.q_heads + head) * a.splits + blockIdx.z;
    if (!in) return;
    if (half == 0) *reinterpret_cast<f32x2*>(a.stat + 2 * at) = f32x2{any ? ref * sc.c : -INFINITY, sum};
    if (!any) return;
    float* dst = a.part + at * D + 4 * half;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(dst + 32 * t + 2 * e) = f32x4{o[t][e], o[t][e + 1], o[t][e + 2], o[t][e + 3]};
    return;
  }
  // a lane has 4 of every 8 values of its row: the halves trade, for 16-byte stores
  const float r = any ? 1.0f / sum : 0.0f;
  char* dst = a.out + 2 * ((int64_t)(s.first + qi) * a.ost[0] + head * a.ost[1] + 8 * half);
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
      u32x4 v;
      for (int i = 0; i < 2; ++i) {
        const uint32_t b0 = T::pack(o[t][e + 2 * i] * r, o[t][e + 2 * i + 1] * r);
        const uint32_t b1 = T::pack(o[t][e + 4 + 2 * i] * r, o[t][e + 5 + 2 * i] * r);
        const auto x = __builtin_amdgcn_permlane32_swap(b0, b1, false, false);
        v[i] = x[0];
        v[2 + i] = x[1];
      }
      if (in) *reinterpret_cast<u32x4*>(dst + 64 * t + 4 * e) = v;
    }
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

// Rows of a block of the prompt kernel, and the most blocks' tiles that the rows can take.
int prompt_rows(int64_t head_dim) { return head_dim == 256 ? 256 : 128; }
int64_t prompt_tiles(const KvBatchView& b, int64_t group, int rows) {
  return (int64_t)b.tokens * group / rows + std::min(b.batch, b.tokens);
}

int plan_splits(const KvView& p, const KvBatchView& b, int64_t q_heads, int64_t window, int64_t sinks) {
  if (b.batch == 0 || b.tokens == 0) return 1;
  const int64_t group = q_heads / p.kv_heads;
  if (b.starts)
    return choose_splits(p, b, p.kv_heads * prompt_tiles(b, group, prompt_rows(p.head_dim)), window, sinks);
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

template <class T, int D, int NW, int BN>
void launch_prompt(const AttnArgs& a, hipStream_t stream) {
  const dim3 grid(a.p.kv_heads, prompt_tiles(a.b, a.group, 32 * NW), a.splits), block(64 * NW);
  if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_prompt_kernel<T, D, NW, BN, true>), grid, block, 0, stream, a);
  else
    HGK_LAUNCH((attn_prompt_kernel<T, D, NW, BN, false>), grid, block, 0, stream, a);
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
    switch (a.p.head_dim) {
      case 64: launch_prompt<T, 64, 4, 64>(a, stream); break;
      case 96: launch_prompt<T, 96, 4, 64>(a, stream); break;
      case 128: launch_prompt<T, 128, 4, 64>(a, stream); break;
      default: launch_prompt<T, 256, 8, 32>(a, stream); break;
    }
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
