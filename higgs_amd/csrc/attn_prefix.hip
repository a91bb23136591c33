// attn_prefix.hip -- attention of sequences that begin with the same tokens: one
// pass over the prefix for the rows of all sequences, one over each sequence's own
// keys, and the join of a row's parts.
#include "attn.h"

namespace hgk {
namespace {

// References are raw scores here, whose differences are scaled: two products would
// each be rounded, by up to 2^-8 at 2^16.
__device__ inline float scale_of(const PrefixArgs& a) {
  return a.softcap > 0.0f ? fold_scale<1>(a).c : fold_scale<0>(a).c;
}

// The keys that a sequence's last token sees behind the prefix, or all where no pass
// takes the prefix: index i is key i + the prefix below `sinks`, and key i + skip
// behind them.
__device__ inline int32_t first_behind(const PrefixArgs& a) { return a.pre > 0 ? a.prefix : 0; }
__device__ inline Seen seen_behind(const PrefixArgs& a, int32_t len) {
  const int32_t from = first_behind(a);
  const int64_t cap = max((int64_t)a.b.width << a.p.page_shift, (int64_t)a.prefix);
  if (len < 0) len = 0;
  const int32_t lo = a.window > 0 && len > a.window ? len - a.window : 0;
  const int32_t end = (int32_t)min((int64_t)len, cap), at = max(lo, from);
  Seen s;
  s.sinks = max(min(min(a.sinks, lo), end) - from, 0);
  s.skip = at - s.sinks;
  s.n = s.sinks + max(end - at, 0);
  return s;
}

// Sums of 16 heads over some keys. A lane has 4 values, 16 t + 4 (lane / 16) .., of head
// lane % 16.
template <int D> struct DecodeSums {
  f32x4 o[D / 16];
  float ref, sum;
  bool any;  // has the wave seen a key?
};

// One wave's walk over the tiles first, first + STEP, ... below last of a run of n
// keys of a kv head; key_of(i) is the position of key i, page_of(position) its page.
template <class T, int D, int CAP, int STEP, class Key, class Page>
__device__ __forceinline__ DecodeSums<D> decode_walk(const PrefixArgs& a, const Scale& sc, const u32x4 (&qf)[D / 32],
                                                     int hk, int first, int last, int n, char* vt, Key key_of,
                                                     Page page_of) {
  constexpr int NS = dec_keys<D>() / 16, kKeys = 16 * NS, kStep = D / 32, kOut = D / 16, kRow = dec_row<D>();
  const int lane = threadIdx.x & 63, m = lane & 15, j = lane >> 4;
  const char* kbase = a.p.k + 2 * (hk * a.p.kst[2] + 8 * j);
  const char* vbase = a.p.v + 2 * (hk * a.p.vst[2] + 8 * j);
  const int begin = first;
#include "attn_walk.inl"
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  DecodeSums<D> acc;
#pragma unroll
  for (int t = 0; t < kOut; ++t) acc.o[t] = o[t];
  acc.ref = ref;
  acc.sum = sum;
  acc.any = any;
  return acc;
}

// Did this lane's head's scores not fit the weights' form, or are its sums not finite?
template <int D>
__device__ __forceinline__ bool decode_odd(const Scale& sc, const DecodeSums<D>& x) {
  float peak = x.sum;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) peak = peak3(peak3(peak, x.o[t][0], x.o[t][1]), x.o[t][2], x.o[t][3]);
  return x.any && !(fabsf(x.ref * sc.c) <= kBaseMax && peak < INFINITY);
}

// Such heads' keys once more. qp: the lane's head's q from its quarter of D on. Returns
// the head's reference and sum.
template <class T, int D, int CAP, int STEP, class Key, class Page>
__device__ __forceinline__ f32x2 decode_again(const PrefixArgs& a, const Scale& sc, const char* qp, int hk, int first,
                                              int last, int n, Key key_of, Page page_of, float (&acc)[D / 4]) {
  constexpr int kKeys = dec_keys<D>();
  const int j = (threadIdx.x & 63) >> 4;
  const int begin = first;
#include "attn_again.inl"
  return f32x2{r, l};
}

// How single tokens' work is dealt out. The tables say how long sequences may become,
// not how long they are, so every block finds out from the lengths what a chunk of own
// keys has and how many parts the prefix has: it sums the sequences' tiles by itself,
// which takes 1 to 2 us beside its first loads. (64 sequences of up to 1500 tokens behind
// 8192, 16/2 heads of 256: 63 to 65 us in tables of 9696 to 131072 tokens, where a
// split by the tables' width takes 3 to 6 times as long in wide ones as in tight ones;
// 512 of up to 100 behind 2048, 32/8 heads of 128, one of them of 30000: 119 us, by
// the width 1640, without the shared prefix 549. It costs batches of many short
// sequences: 1000 of up to 200 behind 1000, 32/8 heads of 128: 139 us for 130.)
constexpr int kOwnParts = 192;  // of a row
struct Shares {
  int chunk, pre;
  bool direct;  // no sequence has more than a chunk: chunk i is sequence i's
};
// Whole chunks, and last ones that are shorter: of a thread's sequences and those of the
// threads in front of it in the wave, and of each wave's.
struct Chunks {
  int whole, last;
};
struct DealLds {
  Chunks upto[64 * kDecWaves], all[kDecWaves];
  float total[kDecWaves];
  int longest[kDecWaves];
};

// v of the lane that a DPP control names, 0 where there is none or the row of 16 is not in ROWS.
template <int CTRL, int ROWS = 0xf>
__device__ inline int from_lane(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, ROWS == 0xf); }
// f over the lanes up to each one: in its row (from 1, 2, 4 and 8 lanes below), then
// from the rows' last lanes. (0 is f's neutral value.)
template <class F>
__device__ inline int wave_scan(int v, F f) {
  v = f(v, from_lane<0x111>(v));
  v = f(v, from_lane<0x112>(v));
  v = f(v, from_lane<0x114>(v));
  v = f(v, from_lane<0x118>(v));
  v = f(v, from_lane<0x142, 0xa>(v));
  return f(v, from_lane<0x143, 0xc>(v));
}
__device__ inline int wave_sums(int v) {
  return wave_scan(v, [](int a, int b) { return a + b; });
}

template <int KEYS>
__device__ __forceinline__ Shares shares_of(const PrefixArgs& a, DealLds& lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float total = 0.0f;
  int longest = 0;
  for (int64_t i0 = threadIdx.x; i0 < a.b.batch; i0 += 4 * 64 * kDecWaves) {
    int32_t len[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) len[k] = a.b.lens[min(i0 + k * 64 * kDecWaves, (int64_t)a.b.batch - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = i0 + k * 64 * kDecWaves < a.b.batch ? decode_tiles<KEYS>(seen_behind(a, len[k])) : 0;
      total += (float)n;
      longest = max(longest, n);
    }
  }
  total = u2f((uint32_t)wave_scan((int)f2u(total), [](int p, int q) { return (int)f2u(u2f(p) + u2f(q)); }));
  longest = wave_scan(longest, [](int p, int q) { return max(p, q); });
  if (lane == 63) {
    lds.total[wave] = total;
    lds.longest[wave] = longest;
  }
  __syncthreads();
  total = lds.total[0] + lds.total[1] + lds.total[2] + lds.total[3];
  longest = max(max(lds.longest[0], lds.longest[1]), max(lds.longest[2], lds.longest[3]));
  static_assert(kDecWaves == 4, "four waves' sums");
  // more than total / chunks, whatever the sums' roundings (2^23 sequences: 2^15 a thread)
  const int even = (int)fminf(total * 1.01f / a.chunks, 1e9f) + 1, fine = (longest + a.most - 1) / a.most;
  Shares s;
  s.chunk = max(max(a.least, min(even, fine)), (longest + kOwnParts - 1) / kOwnParts);
  const int blocks = (int)(a.places * a.pass / (a.pass + total * a.own));
  s.pre = min(max((blocks + a.rows - 1) / a.rows, 1), a.pre);
  if (s.pre > 1) {  // no more than share the prefix's tiles out
    const int tiles = (a.prefix + 63) / 64, per = (tiles + s.pre - 1) / s.pre;
    s.pre = (tiles + per - 1) / per;
  }
  s.chunk = __builtin_amdgcn_readfirstlane(s.chunk);
  s.pre = __builtin_amdgcn_readfirstlane(s.pre);
  s.direct = __builtin_amdgcn_readfirstlane(longest) <= s.chunk;
  return s;
}

// Where the tables have room for no more than a chunk, that is known without the lengths.
__device__ inline bool known_direct(const PrefixArgs& a) { return a.chunks == 0; }

template <int KEYS>
__device__ inline Chunks chunks_of(const PrefixArgs& a, const Shares& s, int seq) {
  const int tiles = decode_tiles<KEYS>(seen_behind(a, a.b.lens[seq])), whole = tiles / s.chunk;
  return Chunks{whole, tiles > whole * s.chunk};
}
// A thread has a run of this many sequences.
__device__ inline int deal_run(const PrefixArgs& a) { return (a.b.batch + 64 * kDecWaves - 1) / (64 * kDecWaves); }
template <int KEYS>
__device__ __forceinline__ void deal(const PrefixArgs& a, const Shares& s, DealLds& lds) {
  const int run = deal_run(a);
  const int64_t i0 = (int64_t)threadIdx.x * run;
  Chunks mine{0, 0};
  for (int64_t i = i0; i < min(i0 + run, (int64_t)a.b.batch); ++i) {
    const Chunks c = chunks_of<KEYS>(a, s, (int)i);
    mine.whole += c.whole;
    mine.last += c.last;
  }
  const Chunks upto{wave_sums(mine.whole), wave_sums(mine.last)};
  lds.upto[threadIdx.x] = upto;
  if ((threadIdx.x & 63) == 63) lds.all[threadIdx.x >> 6] = upto;
  __syncthreads();
}

// Chunk `want` of those that there are, sequence by sequence, the whole ones first and
// then the sequences' last ones: its sequence, and a whole one's place among the sequence's.
// (In the order of the sequences alone short chunks end up beside long ones, and blocks wait.)
struct Chunk {
  int seq, at;
  bool whole;
};
template <int KEYS>
__device__ __forceinline__ Chunk find_chunk(const PrefixArgs& a, const Shares& s, const DealLds& lds, int want) {
  const int lane = threadIdx.x & 63, run = deal_run(a);
  const int wholes = lds.all[0].whole + lds.all[1].whole + lds.all[2].whole + lds.all[3].whole;
  const bool whole = want < wholes;
  auto of = [&](const Chunks& c) { return whole ? c.whole : c.last; };
  int at = whole ? want : want - wholes, wave = 0;
  while (wave < kDecWaves - 1 && at >= of(lds.all[wave])) at -= of(lds.all[wave++]);
  const int upto = of(lds.upto[64 * wave + lane]);
  const int owner = __builtin_ctzll(__ballot(upto > at));  // (there is one: want is below the sum)
  if (owner > 0) at -= __builtin_amdgcn_readlane(upto, owner - 1);
  int seq = 64 * wave + owner;
  if (run > 1) {
    const int stop = (int)min((int64_t)(seq + 1) * run, (int64_t)a.b.batch);
    for (seq *= run; seq < stop; seq += 64) {
      const int mine = seq + lane < stop ? of(chunks_of<KEYS>(a, s, seq + lane)) : 0, sums = wave_sums(mine);
      const uint64_t past = __ballot(sums > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        at -= __builtin_amdgcn_readlane(sums - mine, l);
        seq += l;
        break;
      }
      at -= __builtin_amdgcn_readlane(sums, 63);
    }
  }
  return Chunk{__builtin_amdgcn_readfirstlane(seq), __builtin_amdgcn_readfirstlane(at), whole};
}

// Single tokens' own keys: WAVES waves have the tiles first .. last - 1 of a (sequence,
// kv head), for 16 of its query heads from 16 y on. One wave makes a part of it, to_part
// for head 0 of the sequence; all of a block's make the rows.
// lds: behind_lds<D, WAVES>() bytes, 16-byte aligned.
template <int D, int WAVES> constexpr int behind_lds() {
  constexpr int kTiles = kDecWaves * dec_keys<D>() * dec_row<D>(), kJoin = WAVES > 1 ? kDecWaves * 16 * D * 4 : 0;
  return kTiles > kJoin ? kTiles : kJoin;
}
template <class T, int D, int CAP, int WAVES>
__device__ __forceinline__ void attn_behind(const PrefixArgs& a, char* lds, int seq, const Seen& seen, int hk, int y,
                                            int first, int last, int64_t to_part) {
  constexpr int kStep = D / 32, kTile = dec_keys<D>() * dec_row<D>();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, j = lane >> 4, step = WAVES > 1 ? wave : 0;

  const Scale sc = fold_scale<CAP>(a);
  const int heads = min(16, a.group - y * 16), h0 = hk * a.group + y * 16;
  const char* qp = a.q + 2 * (seq * a.qst[0] + (h0 + (m < heads ? m : 0)) * a.qst[1]);
  u32x4 qf[kStep];
#pragma unroll
  for (int s = 0; s < kStep; ++s) {
    qf[s] = *reinterpret_cast<const u32x4*>(qp + 64 * s + 16 * j);
    for (int w = 0; w < 4; ++w) qf[s][w] = (qf[s][w] & sc.keep) ^ sc.flip;
  }
  const int32_t* table = a.b.table + (int64_t)seq * a.b.table_stride;
  const int32_t from = first_behind(a);
  auto key_of = [&](int i) { return i < seen.sinks ? i + from : i + seen.skip; };
  auto page_of = [&](int32_t key) { return page_behind(a, table, key); };
  const DecodeSums<D> x = decode_walk<T, D, CAP, WAVES>(a, sc, qf, hk, first + step, last, seen.n, lds + wave * kTile,
                                                        key_of, page_of);

  // the keys of heads that the walk's form does not fit once more: the head's sums
  // in f32, a quarter of D in each of its lanes
  bool again = decode_odd(sc, x);
  float acc[D / 4];
  f32x2 rl = {x.ref, x.sum};
  if (__any(again)) {
    int mine = again;
    mine |= __shfl_xor(mine, 16);
    mine |= __shfl_xor(mine, 32);
    again = mine != 0;
    const f32x2 other = decode_again<T, D, CAP, WAVES>(a, sc, qp + 2 * j * (D / 4), hk, first + step, last, seen.n, key_of,
                                                       page_of, acc);
    if (again) rl = other;
  }

  if constexpr (WAVES == 1) {
    if (m >= heads) return;
    const int64_t to = to_part + h0 + m;
    float* part = a.part + to * D;
    if (j == 0) *reinterpret_cast<f32x2*>(a.stat + 2 * to) = f32x2{x.any ? rl[0] : -INFINITY, rl[1]};
    if (again) {
#pragma unroll
      for (int d = 0; d < D / 4; ++d) part[j * (D / 4) + d] = acc[d];
    } else {
#pragma unroll
      for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4*>(part + 16 * t + 4 * j) = x.o[t];
    }
  } else {
    char* out = a.out + 2 * (seq * a.ost[0] + h0 * a.ost[1]);
    __shared__ float wref[kDecWaves][16], wsum[kDecWaves][16];
    __shared__ int wseen[kDecWaves];
    __syncthreads();  // every wave is done with its V tile
    float* wo = reinterpret_cast<float*>(lds) + wave * 16 * D + m * D;
    if (again) {
#pragma unroll
      for (int d = 0; d < D / 4; ++d) wo[j * (D / 4) + d] = acc[d];
    } else {
#pragma unroll
      for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4*>(wo + 16 * t + 4 * j) = x.o[t];
    }
    if (lane < 16) {
      wref[wave][lane] = rl[0];
      wsum[wave][lane] = rl[1];
    }
    if (lane == 0) wseen[wave] = x.any;
    __syncthreads();
    bool some = false;
    for (int w = 0; w < kDecWaves; ++w) some |= wseen[w] != 0;
    for (int idx = threadIdx.x; idx < heads * (D / 2); idx += 64 * kDecWaves) {
      const int h = idx / (D / 2), d = 2 * (idx - h * (D / 2));
      float top = wref[0][h];
      for (int w = 1; w < kDecWaves; ++w) top = fmaxf(top, wref[w][h]);
      float l = 0.0f, v0 = 0.0f, v1 = 0.0f;
      for (int w = 0; w < kDecWaves; ++w) {
        const float f = lesser((wref[w][h] - top) * sc.c);
        const float* src = reinterpret_cast<float*>(lds) + (w * 16 + h) * D + d;
        l = fmaf(wsum[w][h], f, l);
        v0 = fmaf(src[0], f, v0);
        v1 = fmaf(src[1], f, v1);
      }
      const float r = 1.0f / l;
      *reinterpret_cast<uint32_t*>(out + 2 * (h * a.ost[1] + d)) = some ? T::pack(v0 * r, v1 * r) : 0u;
    }
  }
}

// The chunks of block `block` of `blocks`, a wave each at a time.
template <class T, int D, int CAP>
__device__ __forceinline__ void attn_dealt(const PrefixArgs& a, char* lds, DealLds& shared, const Shares& s, int block,
                                           int blocks) {
  constexpr int kKeys = dec_keys<D>();
  if (block == 0 && threadIdx.x == 0) {
    a.found[0] = s.chunk;
    a.found[2] = s.direct;
    if (!known_direct(a)) a.found[1] = s.pre;
  }
  const int heads16 = (a.group + 15) / 16, walks = a.p.kv_heads * heads16;
  int n = a.b.batch;
  if (!s.direct) {
    deal<kKeys>(a, s, shared);
    n = 0;
    for (int w = 0; w < kDecWaves; ++w) n += shared.all[w].whole + shared.all[w].last;
    n = __builtin_amdgcn_readfirstlane(n);
  }
  const int64_t own = (int64_t)a.b.tokens * a.q_heads * a.pre;  // parts of the prefix
#pragma unroll 1
  for (int u = block * kDecWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < n * walks;
       u += blocks * kDecWaves) {
    const int c = u / walks, of = u - c * walks, hk = of / heads16;
    Chunk k{c, 0, false};
    if (!s.direct) k = find_chunk<kKeys>(a, s, shared, c);
    Seen seen = seen_behind(a, a.b.lens[k.seq]);
    seen.n = __builtin_amdgcn_readfirstlane(seen.n);
    const int tiles = decode_tiles<kKeys>(seen);
    if (!s.direct) {
      if (!k.whole) k.at = tiles / s.chunk;
      if (of == 0 && (threadIdx.x & 63) == 0 && (!k.whole || k.at == 0)) a.found[3 + 2 * (int64_t)k.seq + !k.whole] = c;
    }
    const int first = k.at * s.chunk;
    if (first < tiles)
      attn_behind<T, D, CAP, 1>(a, lds, k.seq, seen, hk, of - hk * heads16, first, min(tiles, first + s.chunk),
                                own + (int64_t)c * a.q_heads);
  }
}

// Without a pass: a block a (sequence, kv head), which makes the rows, or chunks.
template <class T, int D, int CAP>
__global__ __launch_bounds__(64 * kDecWaves, 2) void attn_behind_kernel(PrefixArgs a) {
  __shared__ __align__(16) char lds[behind_lds<D, kDecWaves>()];
  const int seq = blockIdx.x / a.p.kv_heads, hk = blockIdx.x - seq * a.p.kv_heads;
  Seen seen = seen_behind(a, a.b.lens[seq]);
  seen.n = __builtin_amdgcn_readfirstlane(seen.n);
  attn_behind<T, D, CAP, kDecWaves>(a, lds, seq, seen, hk, blockIdx.y, 0, decode_tiles<dec_keys<D>()>(seen), 0);
}
template <class T, int D, int CAP>
__global__ __launch_bounds__(64 * kDecWaves, 2) void attn_dealt_kernel(PrefixArgs a) {
  __shared__ __align__(16) char lds[behind_lds<D, 1>()];
  __shared__ DealLds shared;
  Shares s{a.least, 0, true};
  if (!known_direct(a)) s = shares_of<dec_keys<D>()>(a, shared);
  attn_dealt<T, D, CAP>(a, lds, shared, s, blockIdx.x, gridDim.x);
}

// A block of the prompts' kernel, over the prefix's keys or those behind them.
template <class T, int D, int BN, int CAP, bool TWO>
__device__ __forceinline__ void attn_prompt(Keys keys, const PrefixArgs& a, char* lds, int* words, uint32_t x,
                                            uint32_t grid_x, int y, int splits) {
#include "attn_prompt.inl"
}

// Which rows and which part of its keys block `id` of the pass over the prefix takes.
// The blocks of a part are put on one XCD, whose L2 then holds its keys, where the
// parts share out evenly.
struct PrefixBlock {
  int x, grid_x, split;
};
__device__ inline PrefixBlock prefix_block(const PrefixArgs& a, int id, int blocks, int splits) {
  const int parts = splits * a.p.kv_heads, places = blocks / parts;
  int part = id / places, place = id - part * places;
  if (parts % 8 == 0) {
    const int k = id >> 3;
    part = k / places * 8 + (id & 7);
    place = k % places;
  }
  const int split = part / a.p.kv_heads, hk = part - split * a.p.kv_heads;
  return PrefixBlock{place * a.p.kv_heads + hk, places * a.p.kv_heads, split};
}

// Both passes of single tokens in one launch: the blocks that take the prefix, which
// the matrix instructions bound, and then those of the sequences' own keys, which the
// memory does, so that either finds CUs, or places on them, that the other leaves.
// With the join, in us: 256 sequences of up to 200 tokens behind 4001, 32/8 heads of
// 128 (17 GFLOP, 126 MB): 62; 64 of up to 1500 behind 8192, 16/2 heads of 256 (9 GFLOP,
// 117 MB): 59 (with weights in one part 56 and 54, and as two launches 73 and 76); every
// sequence over a table of its own (paged_attention's kernels): 497 and 151.
template <class T, int D, int CAP>
__global__ __launch_bounds__(2 * kPromptRows, D == 256 ? 1 : 2) void attn_shared_kernel(PrefixArgs a, int own_blocks) {
  static_assert(2 * kPromptRows == 64 * kDecWaves && prompt_lds<D>() >= behind_lds<D, 1>(), "one kind of block");
  __shared__ __align__(1024) char lds[prompt_lds<D>()];
  __shared__ DealLds shared;
  const int id = blockIdx.x;
  const int most = a.rows * a.pre;  // blocks of the prefix
  const bool known = known_direct(a);
  Shares s{a.least, 1, true};
  if (id < most ? a.pre > 1 : !known) s = shares_of<dec_keys<D>()>(a, shared);
  const int prefix_blocks = a.rows * s.pre;
  if (known && id == 0 && threadIdx.x == 0) a.found[1] = s.pre;
  if (id < most && id < prefix_blocks) {
    __shared__ int words[prompt_words<D, true>()];
    const PrefixBlock block = prefix_block(a, id, prefix_blocks, s.pre);
    constexpr Keys keys = kPrefix;
    constexpr bool TWO = true;
    constexpr int BN = 64;
    const uint32_t x = block.x, grid_x = block.grid_x;
    const int y = block.split, splits = s.pre;
#include "attn_prompt.inl"
  } else {
    // Blocks that the prefix does not take are the first ones of the own keys, where they
    // have worked that out; as many others then stay behind.
    const int block = known ? id - most : id - prefix_blocks;
    if (block < 0 || block >= own_blocks) return;
    attn_dealt<T, D, CAP == kNoCap ? kNoCap : kWideCap>(a, lds, shared, s, block, own_blocks);
  }
}

// Both passes of prompts in one launch. 32 sequences of up to 33 + 100 tokens behind
// 16384, 32/8 heads of 128 f16 (148 GFLOP): 217 us with the join, 681 TFLOP/s.
template <class T, int D, int CAP>
__global__ __launch_bounds__(2 * kPromptRows, D == 256 ? 1 : 2) void attn_shared_prompt_kernel(PrefixArgs a,
                                                                                                 int prefix_blocks,
                                                                                                 int behind_x) {
  __shared__ __align__(1024) char lds[prompt_lds<D>()];
  __shared__ int words[kPromptWords];
  const int id = blockIdx.x, b = id - prefix_blocks;
  const bool prefix = b < 0;
  PrefixBlock p{b % behind_x, behind_x, b / behind_x};
  if (prefix) p = prefix_block(a, id, prefix_blocks, a.pre);
  attn_prompt<T, D, 64, CAP, false>(prefix ? kPrefix : kBehind, a, lds, words, p.x, p.grid_x, p.split,
                             prefix ? a.pre : a.splits);
}

// out = sum_i w_i part_i / sum_i w_i sum_i over the parts of a row (token and query
// head), w_i = 2^(c (ref_i - max)); parts that saw no key (ref = -inf) hold nothing.
// SINGLE: of single tokens, which have the prefix's parts and those of the chunks
// that their sequence fills, and whose two passes' weights have biases of their own.
// G groups of D/4 threads share a row's parts, a thread has 4 values of it. The
// parts' factors are worked out once, side by side, and kept in LDS.
constexpr int kMaxParts = 256;
template <int D, int G, bool SINGLE> constexpr int join_parts() {
  return G == 1 ? SINGLE ? 1 : 4 : !SINGLE && G == 2 ? 16 : kMaxParts;
}
template <class T, int D, int G, bool SINGLE>
__global__ __launch_bounds__(256) void attn_prefix_join_kernel(PrefixArgs a, uint32_t rows) {
  constexpr uint32_t kLanes = D / 4, kRows = 256 / (kLanes * G), kShare = kLanes * G;
  constexpr bool kFew = SINGLE && G == 1;
  __shared__ f32x4 vs[kRows][G][kLanes];
  __shared__ float refs[kRows][join_parts<D, G, SINGLE>()], sums[kRows][join_parts<D, G, SINGLE>()];
  const uint32_t mine = threadIdx.x / kShare, in = threadIdx.x - mine * kShare, g = in / kLanes, c = in - g * kLanes;
  const uint32_t row = blockIdx.x * kRows + mine;
  const bool work = mine < kRows && row < rows;
  const int t = work ? row / a.q_heads : 0, h = work ? row - (uint32_t)t * a.q_heads : 0;
  const float c2 = scale_of(a);
  int n = 0, pre = 0, whole = 0, first = 0, last = 0;
  bool owned = false;
  if (work) {
    if constexpr (SINGLE) {
      const int tiles = decode_tiles<dec_keys<D>()>(seen_behind(a, a.b.lens[t])), chunk = a.found[0];
      pre = a.pre > 0 ? a.found[1] : 0;
      whole = tiles / chunk;
      n = pre + whole;
      n += tiles > whole * chunk;
      first = last = t;
      if (!a.found[2]) {
        if (whole > 0) first = a.found[3 + 2 * (int64_t)t];
        if (tiles > whole * chunk) last = a.found[3 + 2 * (int64_t)t + 1];
      }
      owned = true;
    } else {
      const KvSeq s = kv_seq(a.b, kv_row_owner(a.b, t));
      owned = t >= s.first && t < s.first + s.n;
      n = owned ? a.row_parts : 0;
    }
  }
  // where the row's part i lies
  auto place = [&](int i) -> int64_t {
    if (!SINGLE || i < pre) return (int64_t)row * a.row_parts + i;
    const int chunk = i - pre < whole ? first + i - pre : last;
    return (int64_t)rows * a.pre + (int64_t)chunk * a.q_heads + h;
  };
  const f32x2* stat = reinterpret_cast<const f32x2*>(a.stat);
  const float* part = a.part + 4 * c;
  float top = -INFINITY, sum = 0.0f;
  f32x4 v = {0, 0, 0, 0};
  auto factor = [&](int i, float ref) {
    const float bias = SINGLE && i < pre ? Mx<T>::kDecBias - Mx<T>::kBias : 0.0f;
    return ref == -INFINITY ? 0.0f : lesser((ref - top) * c2 + bias);
  };
  auto add = [&](int i, float f) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(part + place(i) * D);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(f == 0.0f ? 0.0f : x[e], f, v[e]);  // (0: it is not written)
  };
  if constexpr (kFew) {  // rows may have more parts than LDS holds for all of a block's: every thread for itself
#pragma unroll 8
    for (int i = 0; i < n; ++i) top = fmaxf(top, stat[place(i)][0]);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const f32x2 st = stat[place(i)];
      const float f = factor(i, st[0]);
      sum += f == 0.0f ? 0.0f : st[1] * f;
      add(i, f);
    }
  } else {
    for (int i = in; i < n; i += kShare) {
      const f32x2 st = stat[place(i)];
      refs[mine][i] = st[0];
      sums[mine][i] = st[1];
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) top = fmaxf(top, refs[mine][i]);
    __syncthreads();
    for (int i = in; i < n; i += kShare) {
      const float f = factor(i, refs[mine][i]);
      refs[mine][i] = f;
      sums[mine][i] = f == 0.0f ? 0.0f : sums[mine][i] * f;
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) sum += sums[mine][i];
#pragma unroll 4
    for (int i = g; i < n; i += G) add(i, refs[mine][i]);
  }
  if constexpr (G > 1) {
    if (mine < kRows) vs[mine][g][c] = v;
    __syncthreads();
    if (g > 0 || mine >= kRows) return;
#pragma unroll
    for (int i = 1; i < G; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += vs[mine][i][c][e];
  }
  if (!owned) return;
  const float r = 1.0f / sum;
  u32x2 w = {0u, 0u};
  if (top != -INFINITY) w = u32x2{T::pack(v[0] * r, v[1] * r), T::pack(v[2] * r, v[3] * r)};
  *reinterpret_cast<u32x2*>(a.out + 2 * (t * a.ost[0] + h * a.ost[1] + 4 * c)) = w;
}

// The split of a call: from the sizes alone, but for single tokens' chunks and parts of
// the prefix, of which it gives the bounds and the rules.
//
// A pass over the prefix costs the writing and joining of its parts, a launch, so it
// has to save the reading of 40 MB: below, the sequences read the prefix one by one,
// much of it from the caches (8 sequences behind 1000 tokens, 8 kv heads of 64, 14 MB:
// 20 us with the pass, 14.7 without; 16 behind 2000, 8 of 128, 123 MB: 18.3, 32.8).
constexpr int64_t kPassBytes = 40 << 20;
struct SharedPlan {
  int pre, splits;   // parts of the prefix at the most (single tokens) or exactly; of prompts' own keys
  bool dealt;        // single tokens whose own keys are dealt out in chunks
  int64_t most_chunks;
  int own_blocks, least, most, chunks, rows, places, likely;  // likely: parts of a row, for the join
  float pass, own;
  int64_t parts(const KvBatchView& b, int64_t q_heads) const {
    if (!dealt) return pre + splits > 1 ? (pre + splits) * (int64_t)b.tokens * q_heads : 0;
    return (pre * (int64_t)b.tokens + most_chunks) * q_heads;
  }
  int64_t bytes(const KvBatchView& b, int64_t q_heads, int64_t head_dim) const {
    const int64_t n = parts(b, q_heads) * (head_dim + 2) * 4;
    return dealt ? (n + (3 + 2 * (int64_t)b.batch) * 4 + 15) / 16 * 16 : n;
  }
};
// Blocks of own keys: two turns of those that the chip has room for.
constexpr int64_t kOwnBlocks = 1024;
SharedPlan plan_shared(const KvView& p, const KvBatchView& b, int64_t prefix, int64_t q_heads, int64_t window,
                       int64_t sinks) {
  SharedPlan s{};
  s.splits = 1;
  if (b.batch == 0 || b.tokens == 0) return s;
  const int64_t group = q_heads / p.kv_heads, width = (int64_t)b.width << p.page_shift;
  const int64_t seen = window > 0 && window < prefix && sinks < prefix - window ? window + sinks : prefix;
  const int64_t rows = p.kv_heads * prefix_tiles(b, group);
  // Places on the chip, shared out by the two passes' work: a tile of 64 keys takes 3.6 us
  // of a block with rows of 256, one a CU, and 0.85 us and 2.1 a 128 values of narrower
  // ones, two a CU; own keys come at 5 TB/s.
  s.places = p.head_dim == 256 ? 256 : 512;
  s.pass = (float)((double)rows * prefix / 64 * (p.head_dim == 256 ? 3.6 : 0.85 + 2.1 * p.head_dim / 128) / s.places);
  if ((double)(b.batch - 1) * std::min(seen, width) * p.kv_heads * p.head_dim >= kPassBytes / 4)
    s.pre = (int)std::clamp<int64_t>(b.starts ? s.places / rows : (s.places + rows - 1) / rows, 1,
                                     std::max<int64_t>(std::min<int64_t>(prefix / kMinPart, kMaxSplits), 1));
  int64_t rest = std::max(width, prefix) - (s.pre > 0 ? prefix : 0);
  if (window > 0 && window < rest && sinks < rest - window) rest = window + sinks;
  if (b.starts) {
    const int64_t n = std::min(kPromptBlocks / (p.kv_heads * prompt_tiles(b, group)), rest / kMinPart);
    s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(n, kMaxSplits));
    return s;
  }
  const int64_t keys = p.head_dim == 256 ? 16 : 32, all = std::max<int64_t>((rest + keys - 1) / keys, 1);
  const int64_t walks = p.kv_heads * ((group + 15) / 16), pairs = b.batch * walks;
  if (s.pre == 0 && rest * p.head_dim <= (pairs >= 256 ? 1 << 17 : 1 << 16)) return s;
  s.dealt = true;
  s.rows = (int)rows;
  s.own = (float)((double)keys * p.kv_heads * p.head_dim * 4 / 5e6);
  // Chunks of as many tiles as leave 4096 waves if all sequences are as long as the
  // longest, two turns of those that the chip has room for (rows of 256: four), or 2048 in
  // all, if those are shorter. (Measured with weights in one part: 100 of up to 1500 behind
  // 2048, 24/8 heads of 96: 114 us with half as many waves, 82, 80 with twice as many; 64
  // behind 6000, 16/8 of 256: 116, 103, 101; 64 of up to 3000 behind 8192, 32/8 of 128: 111,
  // 98, 95. Rows of 64 are joined for as long as they are walked: half as many; 200 of up
  // to 1500 behind 4096, 32/8 heads: 99, 107, 105. Nor do few tiles of many pairs gain: 256
  // of up to 200 behind 4001, 32/8 of 128: 57, 58.)
  const int64_t units = p.head_dim > 64 ? 4096 : 2048;
  s.least = pairs >= 1024 ? 8 : 4;
  s.most = (int)std::max<int64_t>(units / pairs, 1);
  s.chunks = (int)std::max<int64_t>(units / 2 / walks, 1);
  // a chunk has no fewer tiles than one of the two rules gives: what there can be of them
  s.most_chunks = std::min(std::max(s.chunks + (int64_t)b.batch, (int64_t)b.batch * s.most),
                           b.batch * ((all + s.least - 1) / s.least));
  if (all <= s.least) s.chunks = 0;  // a sequence has no more than a chunk
  s.own_blocks = (int)std::min((s.most_chunks * walks + kDecWaves - 1) / kDecWaves, kOwnBlocks);
  s.likely = (int)((s.pre + 1) / 2 + 1 + units / 2 / pairs);
  return s;
}
int check_prefix(const char* what, const KvView& p, int64_t width, int64_t prefix) {
  if (prefix < 0 || width < 0 || prefix > (int64_t)1 << 30 || width > (int64_t)1 << (30 - p.page_shift))
    return fail(HGK_ERR_ARG, "%s: a prefix of %lld tokens on %lld pages", what, (long long)prefix, (long long)width);
  if (((prefix + p.page_mask) >> p.page_shift) > width)
    return fail(HGK_ERR_ARG, "%s: %lld pages of %d tokens do not hold a prefix of %lld", what, (long long)width,
                p.page_mask + 1, (long long)prefix);
  return HGK_OK;
}

template <class T, int D>
void launch_behind(const PrefixArgs& a, hipStream_t stream) {
  const dim3 grid(a.b.batch * a.p.kv_heads, (a.group + 15) / 16), block(64 * kDecWaves);
  if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_behind_kernel<T, D, kWideCap>), grid, block, 0, stream, a);
  else
    HGK_LAUNCH((attn_behind_kernel<T, D, kNoCap>), grid, block, 0, stream, a);
}

template <class T, int D>
void launch_dealt(const PrefixArgs& a, int blocks, hipStream_t stream) {
  if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_dealt_kernel<T, D, kWideCap>), dim3(blocks), dim3(64 * kDecWaves), 0, stream, a);
  else
    HGK_LAUNCH((attn_dealt_kernel<T, D, kNoCap>), dim3(blocks), dim3(64 * kDecWaves), 0, stream, a);
}

template <class T, int D, bool SINGLE>
void launch_prefix_join(const PrefixArgs& a, int parts, hipStream_t stream) {
  constexpr int kGroups = 256 / (D / 4);
  const uint32_t rows = (uint32_t)a.b.tokens * a.q_heads;
  auto grid = [&](int g) { const uint32_t n = kGroups / g; return dim3((rows + n - 1) / n); };
  if (parts > 16)
    HGK_LAUNCH((attn_prefix_join_kernel<T, D, kGroups, SINGLE>), grid(kGroups), dim3(256), 0, stream, a, rows);
  else if (parts > 4)
    HGK_LAUNCH((attn_prefix_join_kernel<T, D, 2, SINGLE>), grid(2), dim3(256), 0, stream, a, rows);
  else
    HGK_LAUNCH((attn_prefix_join_kernel<T, D, 1, SINGLE>), grid(1), dim3(256), 0, stream, a, rows);
}

template <class T, int D>
void launch_shared(const PrefixArgs& a, int own_blocks, hipStream_t stream) {
  const dim3 grid(a.rows * a.pre + own_blocks), block(2 * kPromptRows);
  if (a.softcap > kCapMax)
    HGK_LAUNCH((attn_shared_kernel<T, D, kWideCap>), grid, block, 0, stream, a, own_blocks);
  else if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_shared_kernel<T, D, kCap>), grid, block, 0, stream, a, own_blocks);
  else
    HGK_LAUNCH((attn_shared_kernel<T, D, kNoCap>), grid, block, 0, stream, a, own_blocks);
}

template <class T, int D>
void launch_shared_prompts(const PrefixArgs& a, hipStream_t stream) {
  const int prefix = (int)(a.p.kv_heads * prefix_tiles(a.b, a.group) * a.pre);
  const int behind = (int)(a.p.kv_heads * prompt_tiles(a.b, a.group));
  const dim3 grid(prefix + behind * a.splits), block(2 * kPromptRows);
  if (a.softcap > kCapMax)
    HGK_LAUNCH((attn_shared_prompt_kernel<T, D, kWideCap>), grid, block, 0, stream, a, prefix, behind);
  else if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_shared_prompt_kernel<T, D, kCap>), grid, block, 0, stream, a, prefix, behind);
  else
    HGK_LAUNCH((attn_shared_prompt_kernel<T, D, kNoCap>), grid, block, 0, stream, a, prefix, behind);
}

template <class T, int D>
int run_of(const PrefixArgs& a, const SharedPlan& s, const char* what, hipStream_t stream) {
  if (a.b.starts) {
    launch_shared_prompts<T, D>(a, stream);
  } else if (!s.dealt) {
    launch_behind<T, D>(a, stream);
  } else if (a.pre > 0) {
    launch_shared<T, D>(a, s.own_blocks, stream);
  } else {
    launch_dealt<T, D>(a, s.own_blocks, stream);
  }
  if (int st = launch_status(what)) return st;
  if (s.dealt) launch_prefix_join<T, D, true>(a, s.likely, stream);
  else if (a.row_parts > 1) launch_prefix_join<T, D, false>(a, a.row_parts, stream);
  else return HGK_OK;
  return launch_status(what);
}

template <class T>
int run(const PrefixArgs& a, const SharedPlan& s, const char* what, hipStream_t stream) {
  switch (a.p.head_dim) {
    case 64: return run_of<T, 64>(a, s, what, stream);
    case 96: return run_of<T, 96>(a, s, what, stream);
    case 128: return run_of<T, 128>(a, s, what, stream);
    default: return run_of<T, 256>(a, s, what, stream);
  }
}

}  // namespace
}  // namespace hgk

using namespace hgk;

extern "C" int64_t hgk_shared_prefix_attention_workspace(const hgk_kv_pages* pages, const hgk_kv_batch* batch,
                                                         int64_t prefix_width, int64_t prefix_len, int64_t q_heads,
                                                         int64_t window, int64_t sinks) {
  const char* what = "hgk_shared_prefix_attention_workspace";
  clear_error();
  KvView p;
  KvBatchView b;
  if (check_sizes(what, pages, batch, q_heads, window, sinks, &p, &b)) return -1;
  if (check_prefix(what, p, prefix_width, prefix_len)) return -1;
  return plan_shared(p, b, prefix_len, q_heads, window, sinks).bytes(b, q_heads, p.head_dim);
}

extern "C" int hgk_shared_prefix_attention(const hgk_kv_pages* pages, const hgk_kv_batch* batch,
                                           const int32_t* prefix_table, int64_t prefix_width, int64_t prefix_len,
                                           const void* q, const int64_t q_strides[2], int64_t q_heads, float scale,
                                           float softcap, int64_t window, int64_t sinks, void* out,
                                           const int64_t out_strides[2], void* workspace, int64_t workspace_bytes,
                                           void* stream) {
  const char* what = "hgk_shared_prefix_attention";
  clear_error();
  PrefixArgs a{};
  if (int st = check_sizes(what, pages, batch, q_heads, window, sinks, &a.p, &a.b)) return st;
  if (int st = check_prefix(what, a.p, prefix_width, prefix_len)) return st;
  if (int st = check_scales(what, scale, softcap)) return st;
  if (a.b.batch == 0 || a.b.tokens == 0) return HGK_OK;
  if (prefix_len > 0 && !prefix_table) return fail(HGK_ERR_ARG, "%s: null prefix table", what);
  if (int st = check_call(what, &a, q, q_strides, q_heads, scale, softcap, window, sinks, out, out_strides)) return st;
  const SharedPlan s = plan_shared(a.p, a.b, prefix_len, q_heads, window, sinks);
  const int64_t blocks =
      a.p.kv_heads * (s.pre * prefix_tiles(a.b, a.group) +
                      s.splits * (a.b.starts ? prompt_tiles(a.b, a.group) : a.b.batch * (int64_t)((a.group + 15) / 16)));
  if (blocks > kMaxBlocks)
    return fail(HGK_ERR_ARG, "%s: %lld rows are too many", what, (long long)a.b.tokens);
  const int64_t need = s.bytes(a.b, q_heads, a.p.head_dim), parts = s.parts(a.b, q_heads);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(HGK_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
  a.prefix_table = prefix_table;
  a.prefix_width = (int32_t)prefix_width;
  a.prefix = (int32_t)prefix_len;
  a.pre = s.pre;
  a.splits = s.splits;
  a.row_parts = s.dealt ? s.pre : s.pre + s.splits;
  a.least = s.least;
  a.most = s.most;
  a.chunks = s.chunks;
  a.rows = s.rows;
  a.places = s.places;
  a.pass = softcap > 0.0f ? 1.3f * s.pass : s.pass;  // (the tanh)
  a.own = s.own;
  a.part = static_cast<float*>(workspace);
  a.stat = parts > 0 ? a.part + parts * a.p.head_dim : nullptr;
  a.found = s.dealt ? reinterpret_cast<int32_t*>(a.stat + 2 * parts) : nullptr;
  return pages->dtype == DT_BF16 ? run<BF16>(a, s, what, as_stream(stream))
                                 : run<F16>(a, s, what, as_stream(stream));
}
