// attn.h -- what the kernels of attention over a paged key-value cache share: the
// matrix instructions, the softmax's arithmetic, the keys that a token sees, how tiles
// lie in LDS, and the checks of a call.
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
// own where key < prefix; the most parts that a row has of a pass of its own over those
// keys (0: there is none, and the sequences' pass takes all keys); and the parts of a
// row that lie together, at [row][row_parts]: prompts' all, the prefix's first; single
// tokens' of the prefix, behind which their other parts lie at [chunk][head]. (Not in
// AttnArgs: the kernels without a prefix are compiled otherwise with it, and slower by
// up to 4 %.)
struct PrefixArgs : AttnArgs {
  const int32_t* prefix_table;
  int32_t prefix_width, prefix, pre, row_parts;
  // Single tokens: what their work is dealt out by, once the device has the lengths.
  // A chunk has at least `least` tiles, and else as many as give `chunks` of all
  // sequences' tiles, or `most` of the longest one's, whichever is fewer (`chunks` 0: the
  // tables have room for no more than `least`). The pass over
  // the prefix gets its share of the places on the chip by time: `pass` us of it, and
  // `own` us for a tile of the other keys, if all places were its; a part of it takes
  // `rows` blocks.
  int32_t least, most, chunks, rows, places;
  float pass, own;
  // A chunk's tiles, the prefix's parts, whether chunk i is sequence i's, and if not, of
  // each sequence the numbers of its first whole chunk and of its last one, which is shorter.
  int32_t* found;
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

// Of attn_prompt.inl: the words and the bytes of LDS that it works in.
constexpr int kPromptWords = 2 + 2 * (2 * kPromptRows / 64);
template <int D, bool TWO> constexpr bool prompt_lean() { return TWO && D == 128; }
template <int D, bool TWO> constexpr int prompt_words() {
  return kPromptWords + (prompt_lean<D, TWO>() ? 3 * 2 * kPromptRows : 0);
}
template <int D> constexpr int prompt_lds() { return 4 * 64 * 2 * D; }

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
