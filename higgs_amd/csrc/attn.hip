// attn.hip -- attention of new tokens over a paged key-value cache.
#include "attn.h"

namespace hgk {
namespace {

// The fewest tiles that a block of single tokens takes (two a wave).
constexpr int kDecMinTiles = 2 * kDecWaves;
constexpr int kDecJoinBlocks = 2048;  // of the join, about: 2048 sequences get a block each

// The tiles of all (sequence, kv head) pairs, one after the other, are dealt out
// to the blocks in equal runs, whatever the lengths: no block is left with a
// long sequence, and a short one in a wide table is still spread. A run may end
// in the middle of a pair; its part is then joined with the neighbours' by
// attn_decode_join_kernel.
__device__ inline int64_t decode_share(int64_t total, int blocks) {
  return max((total + blocks - 1) / blocks, (int64_t)kDecMinTiles);
}

// One new token per sequence: block = (16 of a kv head's query heads; a run of
// tiles, or with one part a (sequence, kv head)). Each wave walks its own tiles
// of NS * 16 keys with a softmax of its own; nothing is shared until a pair's
// end, so no wave waits for another.
//
// Bound by the reading of the cache. 64 ragged sequences of up to 32768 tokens,
// 16/2 heads of 256 bf16 (2.2 GB): 392 us with the join, 5.5 TB/s, where a
// streaming read reaches 6.1; a block per (pair, fixed part) took 527 us, its
// longest pair last. One sequence of 131071, 32/8 heads of 128: 107 us, 5.0
// TB/s. One of 127: 11 us, a launch and a chain of dependent loads.
template <class T, int D, int CAP>
__global__ __launch_bounds__(64 * kDecWaves, 2) void attn_decode_kernel(AttnArgs a) {
  constexpr int NS = dec_keys<D>() / 16, kKeys = 16 * NS, kStep = D / 32, kOut = D / 16;
  // V rows 32 bytes apart in banks: 16 rows of a transposed read cover each bank twice
  constexpr int kRow = 2 * D + 32, kTile = kKeys * kRow;
  constexpr int kJoin = kDecWaves * 16 * D * 4;
  __shared__ __align__(16) char lds[kTile * kDecWaves > kJoin ? kTile * kDecWaves : kJoin];
  __shared__ float wref[kDecWaves][16], wsum[kDecWaves][16];
  __shared__ int wseen[kDecWaves];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = lane & 15, j = lane >> 4;
  const Scale sc = fold_scale<CAP>(a);
  const int heads = min(16, a.group - (int)blockIdx.y * 16);

  // the pair's sequence, and what its last token sees; the tiles in front of the sequence's, and this run
  int32_t of_seq, of_tiles;
  Seen of_seen;
  int64_t before = 0, at_tile = 0, end_tile = 0;
  if (a.splits > 1) {
    const Owner w = find_owner(
        a.b.batch,
        [&](int b) { return (int64_t)decode_tiles<kKeys>(seen_by_last(a, a.b.lens[b])) * a.p.kv_heads; },
        [&](int64_t total) {
          const int64_t share = decode_share(total, a.splits);
          at_tile = blockIdx.x * share;
          end_tile = min(at_tile + share, total);
          return at_tile;
        });
    if (w.seq < 0) return;
    of_seq = w.seq;
    before = w.before;
  } else {
    of_seq = blockIdx.x / a.p.kv_heads;
  }
  of_seen = seen_by_last(a, a.b.lens[of_seq]);
  of_tiles = decode_tiles<kKeys>(of_seen);
  for (bool head_of_run = true;; head_of_run = false) {
    // this pair, and the tiles of it that fall to this block
    const int seq = __builtin_amdgcn_readfirstlane(of_seq), tiles = __builtin_amdgcn_readfirstlane(of_tiles);
    const Seen seen{__builtin_amdgcn_readfirstlane(of_seen.n), __builtin_amdgcn_readfirstlane(of_seen.sinks),
                    __builtin_amdgcn_readfirstlane(of_seen.skip)};
    int hk, first, last;
    if (a.splits > 1) {
      hk = (int)((at_tile - before) / tiles);
      first = (int)(at_tile - before - (int64_t)hk * tiles);
      last = (int)min((int64_t)tiles, first + end_tile - at_tile);
    } else {
      hk = blockIdx.x - seq * a.p.kv_heads;
      first = 0;
      last = tiles;
    }
    hk = __builtin_amdgcn_readfirstlane(hk);
    first = __builtin_amdgcn_readfirstlane(first);
    last = __builtin_amdgcn_readfirstlane(last);
    const bool whole = first == 0 && last == tiles;
    const int h0 = hk * a.group + blockIdx.y * 16;  // first of this block's heads

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
    constexpr int STEP = kDecWaves;
    const int begin = first + wave, n = seen.n;
    auto key_of = [&](int i) { return i < seen.sinks ? i : i + seen.skip; };
    auto page_of = [&](int32_t key) { return table[key >> a.p.page_shift]; };
    char* vt = lds + wave * kTile;
#include "attn_walk.inl"

    // join the waves
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    // Did this head's scores fit the weights' form, and are its sums finite?
    bool again;
    {
      float peak = sum;
#pragma unroll
      for (int t = 0; t < kOut; ++t) peak = peak3(peak3(peak, o[t][0], o[t][1]), o[t][2], o[t][3]);
      again = any && !(fabsf(ref * sc.c) <= kBaseMax && peak < INFINITY);
    }
    __syncthreads();  // every wave is done with its V tile
    float* wo = reinterpret_cast<float*>(lds) + wave * 16 * D;
#pragma unroll
    for (int t = 0; t < kOut; ++t) *reinterpret_cast<f32x4*>(wo + m * D + 16 * t + 4 * j) = o[t];
    if (lane < 16) {
      wref[wave][lane] = ref;
      wsum[wave][lane] = sum;
    }
    if (lane == 0) wseen[wave] = any;
    if (__any(again)) {
      int mine = again;
      mine |= __shfl_xor(mine, 16);
      mine |= __shfl_xor(mine, 32);
      again = mine != 0;  // all lanes of the head
      const char* qp = a.q + 2 * (seq * a.qst[0] + (h0 + (m < heads ? m : 0)) * a.qst[1] + j * (D / 4));
      float acc[D / 4];
#include "attn_again.inl"
      if (again) {
#pragma unroll
        for (int d = 0; d < D / 4; ++d) wo[m * D + j * (D / 4) + d] = acc[d];
        if (j == 0) {
          wref[wave][m] = r;
          wsum[wave][m] = l;
        }
      }
    }
    __syncthreads();
    bool some = false;
    for (int w = 0; w < kDecWaves; ++w) some |= wseen[w] != 0;
    // a part of the run's first pair, or of its last
    const int64_t slot = (((int64_t)blockIdx.y * a.splits + blockIdx.x) * 2 + (head_of_run ? 0 : 1)) * 16;
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
      if (whole) {
        const float r = 1.0f / l;
        *reinterpret_cast<uint32_t*>(a.out + 2 * (seq * a.ost[0] + (h0 + h) * a.ost[1] + d)) =
            some ? T::pack(v0 * r, v1 * r) : 0u;
      } else {
        *reinterpret_cast<f32x2*>(a.part + (slot + h) * D + d) = f32x2{v0, v1};
        if (d == 0)
          *reinterpret_cast<f32x2*>(a.stat + 2 * (slot + h)) = f32x2{some ? top * sc.c : -INFINITY, l};
      }
    }
    if (a.splits == 1) return;
    // the run's next pair: the sequence's next head, or the next sequence that sees anything
    at_tile += last - first;
    if (at_tile >= end_tile) return;
    if (at_tile - before >= (int64_t)tiles * a.p.kv_heads) {
      before = at_tile;
      do {
        if (++of_seq >= a.b.batch) return;
        of_seen = seen_by_last(a, a.b.lens[of_seq]);
        of_tiles = decode_tiles<kKeys>(of_seen);
      } while (of_tiles == 0);
    }
    __syncthreads();  // the waves' sums are read; V tiles may be written again
  }
}

// Joins the parts of a (sequence, query head): out = sum 2^(ref - max) part /
// sum 2^(ref - max) sum over the blocks whose runs meet in its pair (parts that
// saw no key have ref = -inf). Pairs that one block had are written already;
// a sequence that sees nothing gets its zeros here. A block has the query heads
// blockIdx.y, blockIdx.y + gridDim.y, ...: with many sequences most pairs are
// written already, and counting the sequences' tiles is what a block costs
// (1024 sequences of up to 512 tokens in a wide table, 32 query heads: a block
// per head 63 us, two blocks a sequence 20 us).
template <class T, int D>
__global__ __launch_bounds__(256) void attn_decode_join_kernel(AttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 vs[kGroups][kLanes];
  __shared__ float ls[kGroups];
  const int seq = blockIdx.x;
  const int tiles = decode_tiles<dec_keys<D>()>(seen_by_last(a, a.b.lens[seq]));
  const int g = threadIdx.x / kLanes, c = threadIdx.x - g * kLanes;
  char* out = a.out + 2 * (seq * a.ost[0] + 4 * c);
  if (tiles == 0) {
    if (g == 0)
      for (int h = blockIdx.y; h < a.q_heads; h += gridDim.y)
        *reinterpret_cast<u32x2*>(out + 2 * h * a.ost[1]) = u32x2{0u, 0u};
    return;
  }
  // all tiles, and those in front of the sequence's
  __shared__ int64_t part_total[4], part_before[4];
  int64_t total = 0, before = 0;
  for (int b = threadIdx.x; b < a.b.batch; b += 256) {
    const int64_t n = decode_tiles<dec_keys<D>()>(seen_by_last(a, a.b.lens[b]));
    total += n;
    if (b < seq) before += n;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    total += __shfl_xor(total, o);
    before += __shfl_xor(before, o);
  }
  if ((threadIdx.x & 63) == 0) {
    part_total[threadIdx.x >> 6] = total;
    part_before[threadIdx.x >> 6] = before;
  }
  __syncthreads();
  total = (part_total[0] + part_total[1] + part_total[2] + part_total[3]) * a.p.kv_heads;
  before = (part_before[0] + part_before[1] + part_before[2] + part_before[3]) * a.p.kv_heads;
  const int64_t share = decode_share(total, a.splits);
  for (int h = blockIdx.y; h < a.q_heads; h += gridDim.y) {
    const int hk = h / a.group, in = h - hk * a.group;
    const int64_t t0 = before + (int64_t)hk * tiles;
    const int b0 = (int)(t0 / share), b1 = (int)((t0 + tiles - 1) / share);
    if (b0 == b1) continue;
    auto slot = [&](int b) {
      return (((int64_t)(in >> 4) * a.splits + b) * 2 + (b * share < t0 ? 1 : 0)) * 16 + (in & 15);
    };
    const f32x2* stat = reinterpret_cast<const f32x2*>(a.stat);
    float top = -INFINITY, l = 0.0f;
    for (int b = b0 + (threadIdx.x & 63); b <= b1; b += 64) top = fmaxf(top, stat[slot(b)][0]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    f32x4 v = {0, 0, 0, 0};
    __syncthreads();  // the last head's parts are read
    if (g < kGroups) {
#pragma unroll 4
      for (int b = b0 + g; b <= b1; b += kGroups) {
        const int64_t at = slot(b);
        const f32x2 st = stat[at];
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + at * D + 4 * c);
        const float f = st[0] == -INFINITY ? 0.0f : lesser(st[0] - top);
        l = fmaf(st[1], f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
      }
      vs[g][c] = v;
      if (c == 0) ls[g] = l;
    }
    __syncthreads();
    if (g > 0) continue;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) {
      l += ls[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += vs[i][c][e];
    }
    const float r = 1.0f / l;
    u32x2 w = {0u, 0u};
    if (top != -INFINITY) w = u32x2{T::pack(v[0] * r, v[1] * r), T::pack(v[2] * r, v[3] * r)};
    *reinterpret_cast<u32x2*>(out + 2 * h * a.ost[1]) = w;
  }
}

// Joins the parts of rows (token and query head): out =
// sum_s 2^(ref_s - max) part_s / sum_s 2^(ref_s - max) sum_s. Parts that saw
// no key (ref = -inf) were not written. A thread has 4 values of a row; G
// groups of D/4 threads share a row's parts, and a block has the rows that fit
// 256 threads (many rows of few parts: G = 1; few rows of many: one row a block).
// Bound by the reading of the parts, which the prompt kernel has just written.
template <class T, int D, int G>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, uint32_t rows) {
  constexpr uint32_t kLanes = D / 4, kRows = 256 / (kLanes * G);
  __shared__ f32x4 vs[G][kLanes];
  __shared__ float ls[G];
  const uint32_t mine = threadIdx.x / kLanes, c = threadIdx.x - mine * kLanes, g = G > 1 ? mine : 0;
  const uint32_t row = G > 1 ? blockIdx.x : blockIdx.x * kRows + mine;
  const bool work = mine < G * kRows && row < rows;
  const int t = row / a.q_heads, h = row - (uint32_t)t * a.q_heads;
  const KvSeq s = work ? kv_seq(a.b, kv_row_owner(a.b, t)) : KvSeq{0, 0, 0};
  const bool owned = t >= s.first && t < s.first + s.n;
  const f32x2* stat = reinterpret_cast<const f32x2*>(a.stat) + (int64_t)row * a.splits;
  float top = -INFINITY, l = 0.0f;
  f32x4 v = {0, 0, 0, 0};
  if (owned) {
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, stat[i][0]);
    const float* part = a.part + (int64_t)row * a.splits * D + 4 * c;
#pragma unroll 4
    for (int i = g; i < a.splits; i += G) {
      const f32x2 st = stat[i];
      if (st[0] == -INFINITY) continue;
      const float f = lesser(st[0] - top);
      const f32x4 x = *reinterpret_cast<const f32x4*>(part + (int64_t)i * D);
      l = fmaf(st[1], f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
    }
  }
  if constexpr (G > 1) {
    if (mine < G) {
      vs[g][c] = v;
      if (c == 0) ls[g] = l;
    }
    __syncthreads();
    if (mine > 0) return;
#pragma unroll
    for (int i = 1; i < G; ++i) {
      l += ls[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += vs[i][c][e];
    }
  }
  if (!owned) return;
  const float r = 1.0f / l;
  u32x2 w = {0u, 0u};
  if (top != -INFINITY) w = u32x2{T::pack(v[0] * r, v[1] * r), T::pack(v[2] * r, v[3] * r)};
  *reinterpret_cast<u32x2*>(a.out + 2 * (t * a.ost[0] + h * a.ost[1] + 4 * c)) = w;
}

// How the keys are split, from the sizes alone (the lengths are on the device).
// One token a sequence: see decode_blocks. Prompts: the parts of every row's tiles, as many as fill the
// chip, and not so many that a part goes below kMinPart keys. Writing and
// joining the parts costs as much as half the work of a few hundred blocks, so
// rows are split only where they make less than half a block a CU (ragged turns
// over 20000 tokens, 250 blocks: unsplit 41 us, in two 43, in three 50).

// Blocks that share out the tiles of single tokens; 1: a block per pair and no
// join. That is for caches whose longest pair, as the table and the window allow
// it, is a block's work of about 20 us, or half of that where the pairs are fewer
// than the CUs: finding the run, the ends of pairs inside it and the join cost
// more than unequal pairs (in us, ragged lengths, a block per pair and dealt out:
// 256 pairs of up to 1024 keys of 128 values 23, 33; 1024 pairs of up to 512 33,
// 65; 512 pairs of up to 2048 keys of 64 36, 47; past the rule 256 pairs of up to
// 2048 keys of 256 74, 64; 64 of 1024 of 128 21, 18).
// Rows of 256 values take two blocks a CU (64 sequences of 16384 tokens, 2 kv
// heads: 378 us, one: 417). Rows up to 128 stream better from one (32 sequences
// of 8192, 8 kv heads of 64: 106 us, two: 127), until the pairs are so many that
// a run holds several and the gaps between them show (64 sequences, 8 kv heads of
// 64, ragged up to 4096: 82 us, two: 70; all 4096 long: 107, two: 125).
int decode_blocks(const KvView& p, const KvBatchView& b, int64_t keys) {
  const int64_t pairs = (int64_t)b.batch * p.kv_heads;
  if (keys * p.head_dim <= (pairs >= 256 ? 1 << 17 : 1 << 16)) return 1;
  return p.head_dim == 256 || pairs >= 512 ? 512 : 256;
}
int plan_splits(const KvView& p, const KvBatchView& b, int64_t q_heads, int64_t window, int64_t sinks) {
  if (b.batch == 0 || b.tokens == 0) return 1;
  const int64_t group = q_heads / p.kv_heads;
  int64_t keys = (int64_t)b.width << p.page_shift;
  if (window > 0 && window < keys && sinks < keys - window) keys = window + sinks;
  if (!b.starts) return decode_blocks(p, b, keys);
  const int64_t s = std::min(kPromptBlocks / (p.kv_heads * prompt_tiles(b, group)), keys / kMinPart);
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, kMaxSplits));
}

// Rows of the workspace: parts of head_dim values, and two statistics each.
int64_t part_rows(const KvView& p, const KvBatchView& b, int64_t q_heads, int splits) {
  if (splits == 1) return 0;
  if (b.starts) return (int64_t)b.tokens * q_heads * splits;
  return (q_heads / p.kv_heads + 15) / 16 * splits * 2 * 16;
}

template <class T, int D>
void launch_decode(const AttnArgs& a, hipStream_t stream) {
  const unsigned blocks = a.splits > 1 ? a.splits : a.b.batch * a.p.kv_heads;
  const dim3 grid(blocks, (a.group + 15) / 16), block(64 * kDecWaves);
  if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_decode_kernel<T, D, kWideCap>), grid, block, 0, stream, a);
  else
    HGK_LAUNCH((attn_decode_kernel<T, D, kNoCap>), grid, block, 0, stream, a);
  if (a.splits > 1)
    HGK_LAUNCH((attn_decode_join_kernel<T, D>),
               dim3(a.b.batch, std::clamp<int>(kDecJoinBlocks / a.b.batch, 1, a.q_heads)), dim3(256), 0, stream, a);
}

template <class T, int D, int BN, int CAP>
__global__ __launch_bounds__(2 * kPromptRows, D == 256 ? 1 : 2) void attn_prompt_kernel(AttnArgs a) {
  __shared__ __align__(1024) char lds[prompt_lds<D>()];
  __shared__ int words[kPromptWords];
  constexpr Keys keys = kOwn;
  constexpr bool TWO = false;
  const uint32_t x = blockIdx.x, grid_x = gridDim.x;
  const int y = blockIdx.y, splits = a.splits;
#include "attn_prompt.inl"
}

template <class T, int D, int BN>
void launch_prompt(const AttnArgs& a, hipStream_t stream) {
  const dim3 grid(a.p.kv_heads * prompt_tiles(a.b, a.group), a.splits), block(2 * kPromptRows);
  if (a.softcap > kCapMax)
    HGK_LAUNCH((attn_prompt_kernel<T, D, BN, kWideCap>), grid, block, 0, stream, a);
  else if (a.softcap > 0.0f)
    HGK_LAUNCH((attn_prompt_kernel<T, D, BN, kCap>), grid, block, 0, stream, a);
  else
    HGK_LAUNCH((attn_prompt_kernel<T, D, BN, kNoCap>), grid, block, 0, stream, a);
}

template <class T, int D>
void launch_join(const AttnArgs& a, hipStream_t stream) {
  constexpr int kGroups = 256 / (D / 4);
  const uint32_t rows = (uint32_t)a.b.tokens * a.q_heads;
  if (a.splits > 8)
    HGK_LAUNCH((attn_join_kernel<T, D, kGroups>), dim3(rows), dim3(256), 0, stream, a, rows);
  else
    HGK_LAUNCH((attn_join_kernel<T, D, 1>), dim3((rows + kGroups - 1) / kGroups), dim3(256), 0, stream, a, rows);
}

template <class T>
int run(const AttnArgs& a, const char* what, hipStream_t stream) {
  if (!a.b.starts) {
    switch (a.p.head_dim) {
      case 64: launch_decode<T, 64>(a, stream); break;
      case 96: launch_decode<T, 96>(a, stream); break;
      case 128: launch_decode<T, 128>(a, stream); break;
      default: launch_decode<T, 256>(a, stream); break;
    }
  } else {
    switch (a.p.head_dim) {
      case 64: launch_prompt<T, 64, 64>(a, stream); break;
      case 96: launch_prompt<T, 96, 64>(a, stream); break;
      case 128: launch_prompt<T, 128, 64>(a, stream); break;
      default: launch_prompt<T, 256, 64>(a, stream); break;
    }
  }
  if (int st = launch_status(what)) return st;
  if (a.splits == 1 || !a.b.starts) return HGK_OK;
  switch (a.p.head_dim) {
    case 64: launch_join<T, 64>(a, stream); break;
    case 96: launch_join<T, 96>(a, stream); break;
    case 128: launch_join<T, 128>(a, stream); break;
    default: launch_join<T, 256>(a, stream); break;
  }
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
  return part_rows(p, b, q_heads, plan_splits(p, b, q_heads, window, sinks)) * (p.head_dim + 2) * 4;
}

extern "C" int hgk_paged_attention(const hgk_kv_pages* pages, const hgk_kv_batch* batch, const void* q,
                                   const int64_t q_strides[2], int64_t q_heads, float scale,
                                   float softcap, int64_t window, int64_t sinks, void* out,
                                   const int64_t out_strides[2], void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const char* what = "hgk_paged_attention";
  clear_error();
  AttnArgs a{};
  if (int st = check_sizes(what, pages, batch, q_heads, window, sinks, &a.p, &a.b)) return st;
  if (int st = check_scales(what, scale, softcap)) return st;
  if (a.b.batch == 0 || a.b.tokens == 0) return HGK_OK;
  if (int st = check_call(what, &a, q, q_strides, q_heads, scale, softcap, window, sinks, out, out_strides)) return st;
  const int64_t D = a.p.head_dim;
  a.splits = plan_splits(a.p, a.b, q_heads, window, sinks);
  const int64_t rows = part_rows(a.p, a.b, q_heads, a.splits), need = rows * (D + 2) * 4;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(HGK_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
  a.part = static_cast<float*>(workspace);
  a.stat = rows > 0 ? a.part + rows * D : nullptr;
  return pages->dtype == DT_BF16 ? run<BF16>(a, what, as_stream(stream))
                                 : run<F16>(a, what, as_stream(stream));
}
