// attn.h -- what the kernels of attention over a paged key-value cache share: the
// matrix instructions, the softmax's arithmetic, a wave's walk over a single token's
// keys and the prompts' kernel.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

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
  // Parts of the keys; more than one are joined from the workspace. Prompts: of
  // every row, [tokens * q_heads][splits]. One token: blocks that share the work,
  // [row tiles][splits][2][16].
  int32_t splits;
  float* part;  // [...][head_dim], not normalised
  float* stat;  // [...][2]: reference (log2 domain; behind a prefix a raw score), sum
};

// Of a call whose sequences share a prefix: its pages, which stand for the sequences'
// own where key < prefix; the parts that a row has of a pass of its own over those
// keys (0: there is none, and the sequences' pass takes all keys); and all parts of a
// row, which lie at [row][row_parts], the prefix's first. (Not in AttnArgs: the kernels
// without a prefix are compiled otherwise with it, and slower by up to 4 %.)
struct PrefixArgs : AttnArgs {
  const int32_t* prefix_table;
  int32_t prefix_width, prefix, pre, row_parts;
  int32_t chunk;  // single tokens: tiles of a part
};
__device__ inline int32_t prefix_of(const AttnArgs&) { return 0; }
__device__ inline int32_t prefix_of(const PrefixArgs& a) { return a.prefix; }
__device__ inline int32_t pre_of(const AttnArgs&) { return 0; }
__device__ inline int32_t pre_of(const PrefixArgs& a) { return a.pre; }
__device__ inline int32_t row_parts_of(const AttnArgs&) { return 1; }
__device__ inline int32_t row_parts_of(const PrefixArgs& a) { return a.row_parts; }

// Which keys a block takes: all of each row, of the row's own table; those of the
// shared prefix, for the rows of all sequences at once; or those behind it (all, if
// there is no pass over the prefix), with the prefix's table in front of the own one.
enum Keys { kOwn, kPrefix, kBehind };

// The prefix's table's entry for a key, and the table's of a sequence that begins with it.
__device__ inline int32_t page_of_prefix(const AttnArgs&, int32_t) { return -1; }
__device__ inline int32_t page_of_prefix(const PrefixArgs& a, int32_t key) {
  const int32_t e = key >> a.p.page_shift;
  return e < a.prefix_width ? a.prefix_table[e] : -1;
}
template <class Args>
__device__ inline int32_t page_behind(const Args& a, const int32_t* table, int32_t key) {
  if (key < prefix_of(a)) return page_of_prefix(a, key);
  const int32_t e = key >> a.p.page_shift;
  return e < a.b.width ? table[e] : -1;
}

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
  // s plus the two values of w
  static __device__ inline float add_pair(uint32_t w, float s) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, 0x3f803f80u), s, false);
  }
  // slack and bias of the weights' exponents, prompts' and single tokens'
  static constexpr float kSlack = 8.0f, kBias = 0.0f, kDecSlack = 8.0f, kDecBias = 0.0f;
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
  static __device__ inline float add_pair(uint32_t w, float s) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), s, false);
  }
  static constexpr float kSlack = 8.0f, kBias = 7.0f, kDecSlack = 0.0f, kDecBias = 15.0f;
  // the exponent's bits, and 1, 128 and 16384
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u, k128 = 0x5800u, k16384 = 0x7400u;
};

constexpr float kLog2e = 1.44269504088896341f;

// max of three as one instruction (fmaxf would first quiet each operand)
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The largest magnitude of three values, NaN if one of them is NaN.
__device__ inline float peak3(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Of this lane's value and that of the lane 32 away: the larger, and the sum.
__device__ inline float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return max3(u2f(r[0]), u2f(r[1]), u2f(r[1]));
}
__device__ inline float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return u2f(r[0]) + u2f(r[1]);
}

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
template <int CAP>
__device__ inline Scale fold_scale(const AttnArgs& a) {
  Scale s;
  s.flip = 0;
  s.keep = ~0u;
  if constexpr (CAP) {
    // (a larger cap is none to scores below 10^26)
    const float cap = fminf(a.softcap, 1.0e30f);
    s.c = cap * kLog2e;
    s.inner = fminf(fabsf(a.scale) / cap, 3.0e38f);  // a score of zero stays zero
    if (a.scale < 0.0f) s.flip = 0x80008000u;
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
// error is 2^-22 at the most, so a capped score's is softcap times that.
__device__ inline float fast_tanh(float x) {
  const float e = __builtin_amdgcn_exp2f(x * (2.0f * kLog2e));
  return fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
}

// A soft cap's form (CAP): none, up to kCapMax, and beyond. Up to kCapMax the
// scores are within 2^-16 with fast_tanh, a 32nd of an f16 rounding. Far beyond
// it the scores are a small part of the cap, and tanh has to be good to its own
// size: below 5/8 it is x + x^3 p(x^2), p of degree 4 through the function's
// values at the Chebyshev points (2^-23.5 of tanh in f32). The caps of models,
// 30 and 50, do not pay for it (8191 tokens in a window of 4096, 16/8 heads of
// 256: 580 us, with the wide form 723; eight prompts of 2048, 32/8 heads of 128:
// 418, 529). Single tokens take it for every cap: it costs them nothing.
constexpr int kNoCap = 0, kCap = 1, kWideCap = 2;
constexpr float kCapMax = 64.0f;
template <int CAP>
__device__ inline float cap_tanh(float x) {
  const float t = fast_tanh(x);
  if constexpr (CAP != kWideCap) return t;
  const float z = x * x;
  float p = fmaf(z, -0.00609671418f, 0.0209971797f);
  p = fmaf(z, p, -0.0538509078f);
  p = fmaf(z, p, 0.133327693f);
  p = fmaf(z, p, -0.333333284f);
  return fabsf(x) < 0.625f ? fmaf(x * z, p, x) : t;
}

// The running maximum only has to keep exp2 in range, so a row's reference
// moves when a raw score passes it by more than 2^slack in weight, and not with
// every new maximum. A weight carries a factor 2^bias, which the division by the
// sum takes out again. bf16 holds every weight of f32. f16 ends at 2^16 and holds
// multiples of 2^-24: its bias puts the largest weight at 2^15, so that a weight
// is off by 2^-32 of the reference's at the most (a million keys of it are 2^-12
// of the row). Single tokens, whose tiles leave the time, move their references
// with every new maximum: 2^-40.

// The reference of a row that has seen no score: below every score that can
// occur, and finite times c.
__device__ inline float lowest_ref(float c) { return -3.0e38f / fmaxf(c, 1.0f); }

// A weight is 2^(c x + base), base = bias - c ref. That product is rounded, by up to
// 2^-8 at 2^16: no matter, all of the row's weights share it. Far above, the
// rounding alone would take weights beyond f32: there a weight is 2^(c (x - ref) +
// bias), as the difference is exact next to the reference. Prompts look at the base of
// every tile; single tokens, where one more branch a tile costs 3 % of a long
// cache, at their last base and their sums, and then walk their tiles again.
constexpr float kBaseMax = 65536.0f;

// The factor 2^e of sums whose reference gives way to a greater one. Never zero:
// an infinite sum (of infinite values that a row sees) stays infinite, and of a
// finite one so little is lost in the greater one's rounding.
__device__ inline float lesser(float e) { return fmaxf(__builtin_amdgcn_exp2f(e), 1.0e-44f); }

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

// Keys of a single token's tile.
template <int D> constexpr int dec_keys() { return D == 256 ? 16 : 32; }
// Bytes of a row of values in LDS: 32 more than it has, for 16 rows of a transposed
// read to cover each bank twice.
template <int D> constexpr int dec_row() { return 2 * D + 32; }

// The sequence that has item `want` when every sequence b has count(b) items,
// one after the other, and how many lie in front of its own (seq -1: there are
// fewer). `want_of(total)` gives the item. Each wave does this for itself: a
// lane sums a run of sequences, the wave scans the sums, then the run that has
// the item.
struct Owner {
  int64_t before;
  int32_t seq;
};
__device__ inline int64_t scan64(int64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}
template <class C, class W>
__device__ inline Owner find_owner(int batch, C count, W want_of) {
  const int lane = threadIdx.x & 63, run = (batch + 63) / 64, b0 = min(lane * run, batch), b1 = min(b0 + run, batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += count(b);
  int64_t upto = scan64(mine);
  const int64_t total = __shfl(upto, 63), want = want_of(total);
  if (want < 0 || want >= total) return Owner{0, -1};
  int l = __builtin_ctzll(__ballot(upto > want));
  int64_t before = __shfl(upto - mine, l);
  if (run == 1) return Owner{before, l};
  const int stop = min((l + 1) * run, batch);
  for (int b = l * run; b < stop; b += 64) {
    mine = b + lane < stop ? count(b + lane) : 0;
    upto = scan64(mine);
    const uint64_t has = __ballot(before + upto > want);
    if (has) {
      l = __builtin_ctzll(has);
      return Owner{before + __shfl(upto - mine, l), b + l};
    }
    before += __shfl(upto, 63);
  }
  return Owner{0, -1};
}

template <int KEYS>
__device__ inline int decode_tiles(const Seen& s) { return (s.n + KEYS - 1) / KEYS; }

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
// A non-finite value in a tile that some row sees only in part, or of a key whose
// weight is too small for the type: a weight of zero times infinity would be
// NaN. Such a tile's values are counted on the matrix cores (+inf as 1, -inf as
// 128, NaN as 16384, times 1 where the row sees the key: at most 64 keys a tile,
// so the sum gives the three counts back), and the product runs with zeros in
// their place. Tiles that all rows see whole are looked at only when a block's
// sums have turned out not finite.
template <class M>
__device__ inline uint32_t finite_pair(uint32_t w) {
  uint32_t m = 0;
  if ((w & M::kExp) != M::kExp) m |= 0xffffu;
  if (((w >> 16) & M::kExp) != M::kExp) m |= 0xffff0000u;
  return w & m;
}
// top bits set where a half is not finite
template <class M>
__device__ inline uint32_t odd_pair(uint32_t w) {
  constexpr uint32_t e = M::kExp | M::kExp << 16, one = (M::kExp & -M::kExp) * 0x10001u;
  return ((w & e) + one) & 0x80008000u;
}

constexpr int kPromptRows = 128;  // rows of a block: 32 a wave

// Block = (kv head, tile of 128 rows, part of its tiles of BN keys); a wave
// has 32 rows. As in the decode kernel S^T = K Q^T and O^T = V^T P^T, here on
// 32x32x16 instructions: a lane has half the scores of one row in registers,
// its weights are the second product's operand as they stand, and a row's
// reference and sum are one register each.
//
// K and V tiles come straight from memory to LDS, double buffered: the next
// tile's loads are issued before a tile is computed, one barrier a tile.
//
// 8 sequences of 2048, 32/8 heads of 128 bf16, causal (275 GFLOP): 341 to 352
// us, 780 to 806 TFLOP/s, where a large library product reaches 1260 (a card
// that clocks lower: up to 410). With two waves a SIMD the matrix units work 42
// % of the time and the vector units 50 (a score takes a multiply-add, an exp
// and half a conversion), each wave's own step one after the other. 8191 tokens
// in a window of 4096, soft cap, 16/8 heads of 256 (412 GFLOP): 575 to 582 us;
// registers allow one wave a SIMD there, and the tile's load instructions and
// its barrier stand beside the step. Deeper rings of tiles, 256 rows a block
// and loads spread over the step were no faster.
//
// lds: prompt_lds<D>() bytes, 1024-byte aligned; words: kPromptWords. x of grid_x
// and y are the block's place, `splits` the y there are.
constexpr int kPromptWords = 2 + 2 * (2 * kPromptRows / 64);
template <int D> constexpr int prompt_lds() { return 4 * 64 * 2 * D; }
template <class T, int D, int BN, int CAP, class Args>
__device__ __forceinline__ void attn_prompt(Keys keys, const Args& a, char* lds, int* words, uint32_t x, uint32_t grid_x,
                                            int y, int splits) {
  constexpr int NT = 2 * kPromptRows, BM = kPromptRows, CH = D / 8, kUnits = BN * CH / NT;
  constexpr int kRow = 2 * D, kTile = BN * kRow;
  constexpr int KT = BN / 32, QS = D / 16, DT = D / 32, kAhead = 2;
  static_assert(BN == 64 && BN * CH % NT == 0, "two tiles of 32 keys, whole units per thread");
  typedef Mx<T> M;
  static_assert(prompt_lds<D>() == 4 * kTile, "two tiles of keys, two of values");
  int& odd = words[0];   // 1 + index of the last tile found to hold values that are not finite
  int& redo = words[1];  // a row's sums are not finite

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int place = x / a.p.kv_heads, hk = x - place * a.p.kv_heads, G = a.group;

  // which sequence's tile this is: tiles are counted over the sequences, from
  // the last one on (the longest ones of a prompt first)
  const int64_t want = grid_x / a.p.kv_heads - 1 - place;
  int seq = 0, tile = (int)want;
  KvSeq s{0, a.b.tokens, 0};  // the prefix: the rows of all sequences
  if (keys != kPrefix) {
    const Owner w = find_owner(
        a.b.batch, [&](int b) { return ((int64_t)kv_seq(a.b, b).n * G + BM - 1) / BM; }, [&](int64_t) { return want; });
    if (w.seq < 0) return;
    seq = __builtin_amdgcn_readfirstlane(w.seq);
    tile = __builtin_amdgcn_readfirstlane((int)(want - w.before));
    s = kv_seq(a.b, seq);
    s.first = __builtin_amdgcn_readfirstlane(s.first);
    s.n = __builtin_amdgcn_readfirstlane(s.n);
    s.len = __builtin_amdgcn_readfirstlane(s.len);
  }
  const int R = s.n * G, pos0 = s.len - s.n;  // pos0 may be negative: rows in front of the sequence

  const int row0 = tile * BM;
  int p_first = pos0 + row0 / G, p_last = pos0 + (min(row0 + BM, R) - 1) / G;
  // this lane's row
  const int wrow0 = row0 + 32 * wave;
  const int row = min(wrow0 + col, R - 1);
  const int qi = row / G, head = hk * G + row - qi * G;
  const bool in = wrow0 + col < R;
  int p = pos0 + qi, pw_first = 0, pw_last = 0;
  if (keys == kPrefix) {
    // every row has a sequence of its own; a row of none sees nothing
    int* const lowest_of = words + 2;
    int* const highest_of = lowest_of + NT / 64;
    const KvSeq of = kv_seq(a.b, kv_row_owner(a.b, qi));
    p = qi >= of.first && qi < of.first + of.n ? of.len - of.n + qi - of.first : -1;
    int lowest = p, highest = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {  // (the halves hold the same rows)
      lowest = min(lowest, __shfl_xor(lowest, o));
      highest = max(highest, __shfl_xor(highest, o));
    }
    pw_first = __builtin_amdgcn_readfirstlane(lowest);
    pw_last = __builtin_amdgcn_readfirstlane(highest);
    if (lane == 0) {
      lowest_of[wave] = pw_first;
      highest_of[wave] = pw_last;
    }
    __syncthreads();
    p_first = min(min(lowest_of[0], lowest_of[1]), min(lowest_of[2], lowest_of[3]));
    p_last = max(max(highest_of[0], highest_of[1]), max(highest_of[2], highest_of[3]));
    p_first = __builtin_amdgcn_readfirstlane(p_first);
    p_last = __builtin_amdgcn_readfirstlane(p_last);
  }
  // the block's keys, in tiles of BN: those of the first `sinks`, then the window's,
  // of the keys from .. cap - 1 that are the call's
  const int from = keys == kBehind && pre_of(a) > 0 ? prefix_of(a) : 0;
  const int64_t own = (int64_t)a.b.width << a.p.page_shift;
  const int64_t cap = keys == kOwn ? own : keys == kPrefix ? (int64_t)prefix_of(a) : max(own, (int64_t)prefix_of(a));
  const int hi = (int)min((int64_t)p_last + 1, cap);
  const int lo = a.window > 0 && p_first >= a.window ? p_first - a.window + 1 : 0;
  const int t_from = from / BN, t_hi = hi > 0 ? (hi + BN - 1) / BN : 0;
  const int t_lo = (keys == kBehind ? max(lo, from) : lo) / BN;
  // (at most 2^30 before it is rounded up: sinks and lo may both end at int32's end)
  int front = min((min(min(a.sinks, lo), max(hi, 0)) + BN - 1) / BN, t_lo);
  if (keys == kBehind) front = max(front - t_from, 0);
  const int tiles = a.p.n_pages > 0 ? front + max(t_hi - t_lo, 0) : 0;
  const int per = (tiles + splits - 1) / splits;
  const int it0 = min(per * y, tiles), it1 = min(it0 + per, tiles);
  auto tile_of = [&](int it) { return it < front ? t_from + it : t_lo + it - front; };
  if (keys != kPrefix) {  // the range of the wave's rows
    pw_first = pos0 + min(wrow0, R - 1) / G;
    pw_last = pos0 + min(wrow0 + 31, R - 1) / G;
  }

  const Scale sc = fold_scale<CAP>(a);

  // lane l looks up key l of a tile
  const int32_t* table = a.b.table + (int64_t)seq * a.b.table_stride;
  const char* kbase = a.p.k + 2 * hk * a.p.kst[2];
  const char* vbase = a.p.v + 2 * hk * a.p.vst[2];
  auto look_up = [&](int it) -> int32_t {
    if (it >= it1) return -1;
    const int key = tile_of(it) * BN + (lane & (BN - 1));
    if (keys == kPrefix) return key < hi ? page_of_prefix(a, key) : -1;
    if (keys == kBehind) return key >= from && key < hi ? page_behind(a, table, key) : -1;
    return key < hi ? table[key >> a.p.page_shift] : -1;
  };
  // Looked at a turn after the load was issued: a wait for it is a wait for
  // the tiles' loads before it.
  auto checked = [&](int32_t page) { return (uint32_t)page < (uint32_t)a.p.n_pages ? page : -1; };
  // One load instruction takes 64 pieces, of rows that lie in one page when
  // pages have 16 tokens or more: the address of its first row is then scalar,
  // and the lanes' offsets are the same for every tile. A key that does not
  // exist reads what is there (a page's end, or page 0); its score is masked
  // and its value, if not finite, taken out.
  const bool whole = a.p.page_shift >= 4 && a.p.kst[1] < (1 << 24) && a.p.vst[1] < (1 << 24);
  // But where the prefix ends inside such a run of rows, the rows in front of its
  // end and those behind it lie in two pages: that tile goes row by row.
  const int cut = keys == kBehind && (prefix_of(a) & 15) ? prefix_of(a) / BN : -1;
  // (rows i * NT / CH apart have the same offsets, where that is a multiple of 16)
  constexpr int kOffs = NT % (16 * CH) == 0 ? 1 : kUnits;
  uint32_t koff[kOffs], voff[kOffs];
#pragma unroll
  for (int i = 0; i < kOffs; ++i) {
    const int u0 = i * NT + 64 * wave, u = u0 + lane, r = u / CH, c = u - r * CH, r0 = u0 / CH;
    koff[i] = 2 * ((r - r0) * (uint32_t)a.p.kst[1] + 8 * key_piece<D>(r, c));
    voff[i] = 2 * ((r - r0) * (uint32_t)a.p.vst[1] + 8 * value_place<D>(r, c));
  }
  const uint32_t lds0 = lds_address(lds) + 1024 * wave;
  auto load = [&](int it, uint32_t to, int32_t page, const char* base, int64_t page_step, int64_t row_step,
                  const uint32_t* off, auto piece) {
    const int key0 = tile_of(it) * BN;
    if (page < 0) page = 0;
    if (whole && (keys != kBehind || tile_of(it) != cut)) {
      const uint64_t at = (uint64_t)(base + 2 * (page * page_step + ((key0 + lane) & a.p.page_mask) * row_step));
      const int at_lo = (int)(uint32_t)at, at_hi = (int)(uint32_t)(at >> 32);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int r0 = (i * NT + 64 * wave) / CH;
        const uint64_t row = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, r0) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane(at_lo, r0);
        lds_load(to + 16 * NT * i, (const char*)row, off[i % kOffs]);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kUnits; ++i) {
        const int u = i * NT + threadIdx.x, r = u / CH, c = u - r * CH;
        const int64_t pg = __shfl(page, r), at = (key0 + r) & a.p.page_mask;
        lds_load(to + 16 * NT * i, base + 2 * (pg * page_step + at * row_step + 8 * piece(r, c)));
      }
    }
  };
  // keys and values have two slots each: tile it0 + i lies in slot i % 2
  auto load_keys = [&](int it, int slot, int32_t page) {
    load(it, lds0 + slot * kTile, page, kbase, a.p.kst[0], a.p.kst[1], koff, key_piece<D>);
  };
  auto load_values = [&](int it, int slot, int32_t page) {
    load(it, lds0 + (2 + slot) * kTile, page, vbase, a.p.vst[0], a.p.vst[1], voff, value_place<D>);
  };
  // does some row of this range see only a part of the tile?
  auto part_seen = [&](int key0, int first, int last) {
    return !(key0 + BN - 1 <= first &&
             (a.window == 0 || key0 > last - a.window || key0 + BN - 1 < a.sinks));
  };
  // which keys of a tile this lane's row sees (bit i: key key0 + i)
  auto seen_keys = [&](int key0, uint64_t exist) {
    auto below = [&](int key) {  // the tile's keys below `key`
      const int n = key - key0;
      return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
    };
    uint64_t m = p >= 0 ? below(p + 1) & exist : 0ull;
    if (a.window > 0 && p >= a.window) m &= ~below(p - a.window + 1) | below(a.sinks);
    return m;
  };

  u32x4 qf[QS];
  auto load_rows = [&]() {  // behind the first keys' loads: one wait for both
    const char* qp = a.q + 2 * ((int64_t)(s.first + qi) * a.qst[0] + head * a.qst[1] + 8 * half);
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      qf[i] = *reinterpret_cast<const u32x4*>(qp + 32 * i);
      for (int w = 0; w < 4; ++w) qf[i][w] = (qf[i][w] & sc.keep) ^ sc.flip;
    }
  };
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = f32x16{};
  float ref = lowest_ref(sc.c), sum = 0.0f;
  const float slack = M::kSlack / sc.c;
  bool any = false;

  // A lane's places in a tile of keys (row col, piece 2 i + half) and of values
  // (row 4 half + (lane % 16) / 4, 8-byte pieces, read transposed). Rows are
  // whole multiples of 64 bytes (D = 96: 192) and the places differ by an
  // exclusive or: every piece's address is one register's, xor a constant.
  const int vr = 4 * half + (lane & 15) / 4, vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t kat = col * kRow + 16 * key_place<D>(col, half);
  const uint32_t vat = vr * kRow + 16 * value_place<D>(vr, vc) + 8 * (lane & 1);
  auto key_frag = [&](int slot, int t, int i) {
    const char* kt = lds + slot * kTile + 32 * t * kRow;
    if constexpr (D == 96) {
      const int r = 32 * t + col;
      return *reinterpret_cast<const u32x4*>(kt + col * kRow + 16 * key_place<D>(r, 2 * i + half));
    } else {
      return *reinterpret_cast<const u32x4*>(kt + (kat ^ (32 * i)));
    }
  };
  auto value_frag = [&](int slot, int t, int k) {
    const char* vt = lds + (2 + slot) * kTile + 16 * k * kRow +
                     (D == 96 ? vat + 64 * t : vat ^ (64 * t));
    const u32x2 v0 = lds_transposed(vt), v1 = lds_transposed(vt + 8 * kRow);
    return u32x4{v0[0], v0[1], v1[0], v1[1]};
  };

  // Scores of tile `it` ready in x: hides those that the wave's rows do not see,
  // and moves the references that others pass; `shrunk` is then the factor for
  // the sums so far (few tiles move any: most leave `moved` false).
  bool moved;
  float shrunk, base;  // base: of the weights' exponents, c x + base
  uint32_t see[KT];  // CAP, masked: the 32 keys' bits, at 8 (e / 4) + e % 4 for score e
  auto settle = [&](f32x16* x, int it, uint64_t exist, bool masked) {
    auto top_of = [&](const f32x16* x) {
      float part[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = max3(x[0][e], x[0][e + 4], x[0][e + 8]);
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = max3(part[e], x[0][e + 12], x[1][e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = max3(part[e], x[1][e + 4], x[1][e + 8]);
      part[0] = max3(part[0], x[1][12], x[1][13]);
      part[1] = max3(part[1], x[1][14], x[1][15]);
      return max3(max3(part[0], part[1], part[2]), part[3], part[3]);
    };
    float top;
    if (masked) {
      float hidden = -INFINITY;
      asm volatile("" : "+v"(hidden));  // no register for it but here
      const uint64_t bits = seen_keys(tile_of(it) * BN, exist) >> (4 * half);
      const bool some = (bits & 0x0f0f0f0f0f0f0f0full) != 0;
      any |= some;
      f32x16 h[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        see[t] = (uint32_t)(bits >> (32 * t));
#pragma unroll
        for (int e = 0; e < 16; ++e) h[t][e] = see[t] & (1u << (8 * (e / 4) + e % 4)) ? x[t][e] : hidden;
      }
      top = top_of(h);
      if constexpr (CAP) {
        // the scores stay: under tanh a hidden one would count, so the weights are cleared instead
        top = some ? cap_tanh<CAP>(top * sc.inner) : hidden;
      } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) x[t] = h[t];
      }
    } else {
      any = true;
      top = top_of(x);
      if constexpr (CAP) top = cap_tanh<CAP>(top * sc.inner);
    }
    moved = __any(top > ref + slack);
    if (moved) {  // a row's own scores alone decide for it
      top = halves_max(top);
      const float to = top > ref + slack ? top : ref;
      shrunk = lesser((ref - to) * sc.c);
      sum *= shrunk;
      ref = to;
    }
    base = CAP == kWideCap ? M::kBias : fmaf(-ref, sc.c, M::kBias);
    if constexpr (CAP == kNoCap) {
      if (__any(fabsf(base) > kBaseMax)) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[t][e] -= fabsf(base) > kBaseMax ? ref : 0.0f;
        base = fabsf(base) > kBaseMax ? M::kBias : base;
      }
    }
  };
  // Weights of scores 2 i and 2 i + 1, rounded to the type: by half a step, as the
  // result is (a row's error against 64 bits is 1.3 times that of weights in f32).
  // A second part, as single tokens have, would be half as many matrix
  // instructions again and a conversion a weight, where the two bound the kernel.
  // The sum takes the rounded ones, so that a row's weights add up to one as used.
  float add[4];
  auto weigh = [&](const f32x16* x, int i) {
    float s0 = x[i / 8][2 * i % 16], s1 = x[i / 8][2 * i % 16 + 1];
    if constexpr (CAP) {
      s0 = cap_tanh<CAP>(s0 * sc.inner);
      s1 = cap_tanh<CAP>(s1 * sc.inner);
    }
    if constexpr (CAP == kWideCap) {  // such scores may be past kBaseMax
      s0 -= ref;
      s1 -= ref;
    }
    const float w0 = __builtin_amdgcn_exp2f(fmaf(s0, sc.c, base));
    const float w1 = __builtin_amdgcn_exp2f(fmaf(s1, sc.c, base));
    const uint32_t pair = M::pack(w0, w1);
    add[i & 3] = M::add_pair(pair, i < 4 ? 0.0f : add[i & 3]);
    return pair;
  };
  // Sums of what is not finite among a tile's values 32 t .. 32 t + 31 that the
  // lane's row sees (`see`): zero, an infinity or NaN.
  auto odd_sum = [&](int slot, int t, uint64_t see) {
    // constants of this path, kept out of the loop's registers
    uint32_t one = M::kOne, c128 = M::k128, c16384 = M::k16384, inf = 0x7f800000u;
    asm volatile("" : "+s"(one), "+s"(c128), "+s"(c16384), "+s"(inf));
    auto code = [&](uint32_t h) {
      const uint32_t e = h & M::kExp, f = h & 0x7fffu & ~M::kExp;
      return e != M::kExp ? 0u : f ? c16384 : h & 0x8000u ? c128 : one;
    };
    f32x16 n = f32x16{};
#pragma unroll 1
    for (int k = 0; k < 2 * KT; ++k) {
      const u32x4 v = value_frag(slot, t, k);
      u32x4 c, on;
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = (uint32_t)(see >> (16 * k + 8 * (i / 2) + 2 * (i & 1)));
        c[i] = code(v[i] & 0xffffu) | code(v[i] >> 16) << 16;
        on[i] = (two & 1 ? one : 0u) | (two & 2 ? one << 16 : 0u);
      }
      n = M::mma32x16(c, on, n);
    }
    f32x16 f;
    for (int e = 0; e < 16; ++e) {
      const int counts = (int)n[e], nan = counts >> 14, neg = (counts >> 7) & 127, pos = counts & 127;
      const uint32_t bits = nan || (neg && pos) ? inf | 0x400000u : neg ? inf | 0x80000000u : pos ? inf : 0u;
      f[e] = u2f(bits);
    }
    return f;
  };
  // values of tile `it` that are not finite, where some row sees only part of the tile
  auto odd_values = [&](int it, int slot, uint64_t exist, bool all) {
    const int key0 = tile_of(it) * BN;
    if (all && !part_seen(key0, p_first, p_last)) return;
    char* vt = lds + (2 + slot) * kTile;
    uint32_t bits = 0;
#pragma unroll 1
    for (int i = 0; i < kUnits; ++i) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(vt + 16 * (i * NT + threadIdx.x));
      bits |= odd_pair<M>(v[0]) | odd_pair<M>(v[1]) | odd_pair<M>(v[2]) | odd_pair<M>(v[3]);
    }
    if (bits) odd = it + 1;
    __syncthreads();
    if (odd != it + 1) return;
    const uint64_t see = seen_keys(key0, exist) >> (4 * half);
#pragma unroll 1
    for (int t = 0; t < DT; ++t) {
      const f32x16 f = odd_sum(slot, t, see);
#pragma unroll
      for (int u = 0; u < DT; ++u)
        if (u == t) o[u] += f;
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
  };
  auto all_of = [&](uint64_t exist) { return exist == ~0ull; };

  // One step: the product of tile it - 1 with its weights w, the weights wn of
  // tile `it`, whose scores x are ready, and the scores of tile it + 1 into y:
  // independent pieces, so that the matrix cores and the vector units have
  // work side by side from every wave. The product comes first, so that w is
  // done with when y begins. Before the first tile the weights are zero; behind
  // the last one the scores are of stale keys and not used.
  // The operands of the matrix instructions are read kAhead ahead; nothing
  // moves across a pair of weights, or the reads would all come first and spill.
  constexpr int kPairs = 8 * KT, kQ = KT * QS, kP = DT * 2 * KT;
  auto step = [&](const f32x16* x, f32x16* y, const u32x4* w, u32x4* wn, int slot) {
    u32x4 f[kAhead + 1];
    auto frag = [&](int n) {
      return n < kP ? value_frag(slot ^ 1, n % DT, n / DT) : key_frag(slot ^ 1, (n - kP) / QS, (n - kP) % QS);
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) f[j] = frag(j);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = i * (kQ + kP) / kPairs; n < (i + 1) * (kQ + kP) / kPairs; ++n) {
        if (n + kAhead < kQ + kP) f[(n + kAhead) % (kAhead + 1)] = frag(n + kAhead);
        const u32x4& v = f[n % (kAhead + 1)];
        const int j = n - kP;
        if (j < 0)
          o[n % DT] = M::mma32x16(v, w[n / DT], o[n % DT]);
        else
          y[j / QS] = M::mma32x16(v, qf[j % QS], j % QS ? y[j / QS] : f32x16{});
      }
      wn[i / 4][i & 3] = weigh(x, i);
      if (i % 4 == 3) {  // here, and not where they are used
        asm volatile("" : "+v"(wn[i / 4]));
        asm volatile("" : "+v"(add[0]), "+v"(add[1]), "+v"(add[2]), "+v"(add[3]));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    sum += (add[0] + add[1]) + (add[2] + add[3]);
  };

  if (threadIdx.x == 0) odd = redo = 0;
  if (it0 < it1) {
    // pages of the tiles it, it + 1 and it + 2, and which keys of it - 1 and it exist
    int32_t page0 = look_up(it0), page1 = look_up(it0 + 1), next = look_up(it0 + 2);
    page0 = checked(page0);
    page1 = checked(page1);
    uint64_t exist = __ballot(page0 >= 0), exist1 = 0;
    load_keys(it0, 0, page0);
    if (it0 + 1 < it1) load_keys(it0 + 1, 1, page1);
    load_rows();
#pragma unroll
    for (int i = 0; i < kUnits; ++i)  // the values in front of the first tile
      *reinterpret_cast<u32x4*>(lds + 3 * kTile + 16 * (i * NT + threadIdx.x)) = u32x4{0, 0, 0, 0};
    landed_barrier();
    f32x16 xa[KT], xb[KT];
    u32x4 wa[2 * KT], wb[2 * KT];
#pragma unroll
    for (int k = 0; k < 2 * KT; ++k) wb[k] = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      xa[t] = f32x16{};
#pragma unroll
      for (int i = 0; i < QS; ++i) xa[t] = M::mma32x16(key_frag(0, t, i), qf[i], xa[t]);
    }
    __syncthreads();  // its slot is loaded again below

    auto turn = [&](f32x16* x, f32x16* y, const u32x4* w, u32x4* wn, int it, int slot) {
      asm volatile("" : "+v"(next));  // waits here if it must, in front of the tiles' loads
      const int32_t page2 = checked(next);
      next = look_up(it + 3);
      load_values(it, slot, page0);
      if (it + 2 < it1) load_keys(it + 2, slot, page2);
      page0 = page1;
      page1 = page2;
      const bool masked = !all_of(exist) || part_seen(tile_of(it) * BN, pw_first, pw_last);
      settle(x, it, exist, masked);
      if (it > it0) odd_values(it - 1, slot ^ 1, exist1, all_of(exist1));
      const float before = sum;
      step(x, y, w, wn, slot);
      if (CAP && masked) {
        sum = before;
#pragma unroll
        for (int k = 0; k < 2 * KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t two = see[k / 2] >> (16 * (k & 1) + 8 * (i / 2) + 2 * (i & 1));
            wn[k][i] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
            sum = M::add_pair(wn[k][i], sum);
          }
      }
      if (moved) {
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= shrunk;
      }
      exist1 = exist;
      exist = __ballot(page0 >= 0);
      landed_barrier();
    };
    auto drain = [&](const u32x4* w, int slot) {
      odd_values(it1 - 1, slot, exist1, all_of(exist1));
#pragma unroll
      for (int j = 0; j < kP; ++j) o[j % DT] = M::mma32x16(value_frag(slot, j % DT, j / DT), w[j / DT], o[j % DT]);
    };
    // two turns a round, so that no score or weight is moved between registers
    int it = it0;
    for (; it + 1 < it1; it += 2) {
      turn(xa, xb, wb, wa, it, 0);
      turn(xb, xa, wa, wb, it + 1, 1);
    }
    if (it < it1) {
      turn(xa, xb, wb, wa, it, 0);
      drain(wa, 0);
    } else {
      drain(wb, 1);
    }
  }
  sum = halves_sum(sum);
  any = halves_sum(any ? 1.0f : 0.0f) != 0.0f;
  // Sums that are not finite though the row's weights are: its values are not.
  bool bad;
  {
    float peak[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        peak[0] = peak3(peak[0], o[t][e], o[t][e + 1]);
        peak[1] = peak3(peak[1], o[t][e + 2], o[t][e + 3]);
      }
    bad = !(peak[0] < INFINITY && peak[1] < INFINITY) && sum > 0.0f && sum < INFINITY;
  }
  auto tell = [&]() {  // the block, whether a row is bad; without a wait for stores
    if (bad) redo = 1;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  // (in front of the stores 168 registers do for rows of 64, a third block a CU;
  // rows of 256 would move 32 of their sums to memory)
  if constexpr (D < 256) tell();
  // (a row's parts over the prefix come first)
  int64_t part_at = (int64_t)(s.first + qi) * a.q_heads + head;
  if (keys == kOwn) part_at = part_at * splits + y;
  else part_at = part_at * row_parts_of(a) + (keys == kBehind ? pre_of(a) : 0) + y;
  const bool parts = keys == kOwn ? splits > 1 : row_parts_of(a) > 1;
  char* out_row = a.out + 2 * ((int64_t)(s.first + qi) * a.ost[0] + head * a.ost[1]);
  if (parts) {
    if (in && half == 0)
      *reinterpret_cast<f32x2*>(a.stat + 2 * part_at) = f32x2{any ? (keys == kOwn ? ref * sc.c : ref) : -INFINITY, sum};
    if (in && any) {
      float* dst = a.part + part_at * D + 4 * half;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4*>(dst + 32 * t + 2 * e) = f32x4{o[t][e], o[t][e + 1], o[t][e + 2], o[t][e + 3]};
    }
  } else {
    // a lane has 4 of every 8 values of its row: the halves trade, for 16-byte stores
    const float r = any ? 1.0f / sum : 0.0f;
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
        if (in) *reinterpret_cast<u32x4*>(out_row + 16 * half + 64 * t + 4 * e) = v;
      }
  }

  // Rows over values that are not finite, of which a weight may have been rounded
  // to zero: every column that holds such a value among the keys that the row sees
  // is written again, from the counts of every tile.
  if constexpr (D == 256) tell();
  if (!redo) return;
#pragma unroll 1
  for (int t = 0; t < DT; ++t) {
    f32x16 f = f32x16{};
#pragma unroll 1
    for (int it = it0; it < it1; ++it) {
      const int32_t page = checked(look_up(it));
      const uint64_t exist = __ballot(page >= 0);
      load_values(it, 0, page);
      landed_barrier();
      f += odd_sum(0, t, seen_keys(tile_of(it) * BN, exist) >> (4 * half));
      __syncthreads();
    }
    if (!bad || !in) continue;
#pragma unroll 1
    for (int e = 0; e < 16; e += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = e == 0 ? f[i] : e == 4 ? f[4 + i] : e == 8 ? f[8 + i] : f[12 + i];
        const int d = 32 * t + 2 * e + 4 * half + i;
        if (x == 0.0f) continue;
        if (parts) a.part[part_at * D + d] = x;
        else *reinterpret_cast<uint16_t*>(out_row + 2 * d) = (uint16_t)T::pack(x, x);
      }
  }
}

// Sizes shared by the call and its workspace query.
int check_sizes(const char* what, const hgk_kv_pages* pages, const hgk_kv_batch* batch, int64_t q_heads,
                int64_t window, int64_t sinks, KvView* p, KvBatchView* b) {
  if (int st = kv_check_pages(what, pages, p)) return st;
  if (int st = kv_check_batch(what, *p, batch, b)) return st;
  if (q_heads < 1 || q_heads > 65535 || q_heads % p->kv_heads)
    return fail(HGK_ERR_ARG, "%s: %lld query heads for %d kv heads", what, (long long)q_heads, p->kv_heads);
  if ((int64_t)b->batch * p->kv_heads > INT32_MAX || (int64_t)b->tokens * q_heads > 1 << 30)
    return fail(HGK_ERR_ARG, "%s: %lld rows of %lld heads are too many", what, (long long)b->tokens,
                (long long)q_heads);
  if (window < 0 || sinks < 0)
    return fail(HGK_ERR_ARG, "%s: window=%lld, sinks=%lld must not be negative", what, (long long)window,
                (long long)sinks);
  return HGK_OK;
}

// The most tiles that the rows of a call can take.
int64_t prompt_tiles(const KvBatchView& b, int64_t group) {
  return (int64_t)b.tokens * group / kPromptRows + std::min(b.batch, b.tokens);
}

// ... and of a pass over a prefix, where a tile has rows of any sequences.
int64_t prefix_tiles(const KvBatchView& b, int64_t group) {
  return ((int64_t)b.tokens * group + kPromptRows - 1) / kPromptRows;
}

// The fewest keys of a part; the blocks that prompts are split to fill; the most parts.
constexpr int64_t kMinPart = 256, kPromptBlocks = 256;
constexpr int kMaxSplits = 64;

// The operands of both entry points checked and filled in, but for the workspace.
int check_call(const char* what, AttnArgs* a, const void* q, const int64_t q_strides[2], int64_t q_heads, float scale,
               float softcap, int64_t window, int64_t sinks, void* out, const int64_t out_strides[2]) {
  const int64_t T = a->b.tokens, D = a->p.head_dim;
  if (int st = kv_check_rows(what, "q", q, q_strides, T, q_heads, D, false, a->qst)) return st;
  if (int st = kv_check_rows(what, "out", out, out_strides, T, q_heads, D, true, a->ost)) return st;
  a->q = static_cast<const char*>(q);
  a->out = static_cast<char*>(out);
  a->q_heads = (int32_t)q_heads;
  a->group = (int32_t)(q_heads / a->p.kv_heads);
  a->scale = scale;
  a->softcap = softcap;
  a->window = (int32_t)(window >= INT32_MAX ? 0 : window);  // every key of any sequence
  a->sinks = (int32_t)(sinks > INT32_MAX ? INT32_MAX : sinks);
  if (a->p.kv_heads * (a->b.starts ? prompt_tiles(a->b, a->group) : (int64_t)a->b.batch) > kMaxBlocks)
    return fail(HGK_ERR_ARG, "%s: %lld rows are too many", what, (long long)T);
  return HGK_OK;
}
int check_scales(const char* what, float scale, float softcap) {
  if (!std::isfinite(scale)) return fail(HGK_ERR_ARG, "%s: scale must be finite", what);
  if (!(softcap >= 0.0f) || !std::isfinite(softcap))
    return fail(HGK_ERR_ARG, "%s: softcap must be finite and not negative", what);
  return HGK_OK;
}

}  // namespace
}  // namespace hgk
