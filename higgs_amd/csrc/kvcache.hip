// kvcache.hip -- the paged key-value cache: new tokens' keys and values into
// their pages, and copies of whole pages. Both only move bytes, so the memory
// bounds them (and the call itself where they are few): 16-byte accesses, a
// thread's loads in front of its stores.
#include <algorithm>
#include <new>
#include <vector>

#include "kv.h"

namespace hgk {

int kv_check_pages(const char* what, const hgk_kv_pages* p, KvView* out) {
  if (!p) return fail(HGK_ERR_ARG, "%s: null pages", what);
  if (p->dtype != DT_BF16 && p->dtype != DT_F16)
    return fail(HGK_ERR_UNSUPPORTED, "%s: pages of dtype %s (bf16 or f16 only)", what, dtype_name(p->dtype));
  if (p->page_size < 1 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)))
    return fail(HGK_ERR_ARG, "%s: page_size=%d must be a power of two in 1..65536", what, p->page_size);
  if (p->n_pages < 0 || p->n_pages > INT32_MAX)
    return fail(HGK_ERR_ARG, "%s: n_pages=%lld out of range", what, (long long)p->n_pages);
  if (p->kv_heads < 1 || p->kv_heads > 65535)
    return fail(HGK_ERR_ARG, "%s: kv_heads=%lld out of range", what, (long long)p->kv_heads);
  if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128 && p->head_dim != 256)
    return fail(HGK_ERR_UNSUPPORTED, "%s: head_dim=%lld (64, 96, 128 or 256)", what, (long long)p->head_dim);
  if (p->n_pages > 0) {
    if (!p->k || !p->v) return fail(HGK_ERR_ARG, "%s: null pages", what);
    if (!aligned16(p->k) || !aligned16(p->v))
      return fail(HGK_ERR_ARG, "%s: pages must be 16-byte aligned", what);
  }
  const int64_t extent[3] = {p->n_pages, p->page_size, p->kv_heads};
  for (int i = 0; i < 3; ++i) {
    // an axis of one element is never stepped along
    out->kst[i] = extent[i] > 1 ? p->k_strides[i] : 0;
    out->vst[i] = extent[i] > 1 ? p->v_strides[i] : 0;
    if (out->kst[i] < 0 || out->vst[i] < 0 || (out->kst[i] & 7) || (out->vst[i] & 7))
      return fail(HGK_ERR_ARG, "%s: page strides must be multiples of 8 elements", what);
  }
  out->k = static_cast<const char*>(p->k);
  out->v = static_cast<const char*>(p->v);
  out->n_pages = (int32_t)p->n_pages;
  out->page_shift = __builtin_ctz((unsigned)p->page_size);
  out->page_mask = p->page_size - 1;
  out->kv_heads = (int32_t)p->kv_heads;
  out->head_dim = (int32_t)p->head_dim;
  return HGK_OK;
}

int kv_check_batch(const char* what, const KvView& p, const hgk_kv_batch* b, KvBatchView* out) {
  if (!b) return fail(HGK_ERR_ARG, "%s: null batch", what);
  if (b->batch < 0 || b->batch > kMaxBlocks || b->tokens < 0 || b->tokens > INT32_MAX)
    return fail(HGK_ERR_ARG, "%s: batch=%lld, tokens=%lld out of range", what, (long long)b->batch,
                (long long)b->tokens);
  if (!b->q_starts && b->tokens != b->batch)
    return fail(HGK_ERR_ARG, "%s: %lld rows for %lld sequences of one token", what,
                (long long)b->tokens, (long long)b->batch);
  if (b->table_width < 0 || b->table_width > INT32_MAX || b->table_stride < 0)
    return fail(HGK_ERR_ARG, "%s: bad table width or stride", what);
  if (b->table_width > (int64_t)1 << (30 - p.page_shift))
    return fail(HGK_ERR_ARG, "%s: a table of %lld pages of %d tokens is too wide (2^30 tokens)", what,
                (long long)b->table_width, p.page_mask + 1);
  if (b->batch > 0 && b->tokens > 0 && (!b->kv_lens || (!b->block_table && b->table_width > 0)))
    return fail(HGK_ERR_ARG, "%s: null table or lengths", what);
  out->table = b->block_table;
  out->lens = b->kv_lens;
  out->starts = b->q_starts;
  out->table_stride = b->table_stride;
  out->width = (int32_t)b->table_width;
  out->batch = (int32_t)b->batch;
  out->tokens = (int32_t)b->tokens;
  return HGK_OK;
}

namespace {
// Do rows of `d` elements, stepped along these axes, lie on each other? (Taken to
// where an axis's step does not clear the whole of the axes with smaller ones.)
bool rows_overlap(const int64_t* stride, const int64_t* extent, int axes, int64_t d) {
  int order[4] = {0, 1, 2, 3};
  std::sort(order, order + axes, [&](int x, int y) { return stride[x] < stride[y]; });
  __int128 span = d;
  for (int i = 0; i < axes; ++i) {
    const int x = order[i];
    if (extent[x] <= 1) continue;
    if (stride[x] < span) return true;
    span += (__int128)stride[x] * (extent[x] - 1);
  }
  return false;
}
}  // namespace

int kv_check_rows(const char* what, const char* name, const void* p, const int64_t strides[2],
                  int64_t tokens, int64_t heads, int64_t head_dim, bool written, int64_t out[2]) {
  if (!p || !strides) return fail(HGK_ERR_ARG, "%s: null %s", what, name);
  if (!aligned16(p)) return fail(HGK_ERR_ARG, "%s: %s must be 16-byte aligned", what, name);
  const int64_t extent[2] = {tokens, heads};
  for (int i = 0; i < 2; ++i) {
    out[i] = extent[i] > 1 ? strides[i] : 0;
    if (out[i] < 0 || (out[i] & 7))
      return fail(HGK_ERR_ARG, "%s: %s strides must be multiples of 8 elements", what, name);
  }
  if (written && rows_overlap(out, extent, 2, head_dim))
    return fail(HGK_ERR_ARG, "%s: %s rows overlap (strides %lld, %lld)", what, name, (long long)out[0],
                (long long)out[1]);
  return HGK_OK;
}

int kv_check_written_pages(const char* what, const KvView& p) {
  const int64_t extent[3] = {p.n_pages, (int64_t)p.page_mask + 1, p.kv_heads};
  if (rows_overlap(p.kst, extent, 3, p.head_dim) || rows_overlap(p.vst, extent, 3, p.head_dim))
    return fail(HGK_ERR_ARG, "%s: rows of the pages overlap", what);
  return HGK_OK;
}

namespace {

constexpr int kThreads = 256;

struct RowsView {
  const char* k;
  const char* v;
  int64_t kst[2], vst[2];  // token, head
};

// Do the key pages lie on the value pages? Of pools with the same strides: they
// are then one array with an axis of two more.
bool pools_meet(const KvView& p) {
  if (!std::equal(p.kst, p.kst + 3, p.vst)) return false;
  const int64_t apart = p.k < p.v ? p.v - p.k : p.k - p.v;
  const __int128 span = (__int128)p.kst[0] * (p.n_pages - 1) + (__int128)p.kst[1] * p.page_mask +
                        (__int128)p.kst[2] * (p.kv_heads - 1) + p.head_dim;
  if (apart / 2 >= span) return false;  // two arrays
  const int64_t st[4] = {p.kst[0], p.kst[1], p.kst[2], apart / 2};
  const int64_t extent[4] = {p.n_pages, (int64_t)p.page_mask + 1, p.kv_heads, 2};
  return rows_overlap(st, extent, 4, p.head_dim);
}
// Values that are the keys, in pages that are the keys' pages: written twice alike.
bool same_rows(const KvView& p, const RowsView& x) {
  return p.k == p.v && x.k == x.v && x.kst[0] == x.vst[0] && x.kst[1] == x.vst[1];
}

// Block = `per` tokens. Their places are worked out once, by a thread each (a
// search of the starts, the length, the table: dependent loads), and kept in
// LDS; then all threads move the tokens' 2 * Hk * D/8 16-byte units, keys and
// values, U at a time with the loads in front of the stores. k and v are read
// past the caches, the pages are not written past them: the attention over them
// comes next. 16384 tokens of 8 heads of 128 (134 MB read and written, nothing
// cached): 32 us, 4.2 TB/s; with every thread looking up its own units 51 us.
// With `slots` the places are given.
constexpr int kMaxTokens = 16;
template <bool SLOTS>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvView p, KvBatchView b, RowsView x,
                                                             uint32_t units, uint32_t chunks, int per,
                                                             const int64_t* slots) {
  __shared__ int32_t page_of[kMaxTokens], at_of[kMaxTokens];
  const int t0 = blockIdx.x * per, n = min(per, b.tokens - t0);
  if constexpr (SLOTS) {
    if ((int)threadIdx.x < n) {
      const int64_t slot = slots[t0 + threadIdx.x], page = slot >> p.page_shift;
      page_of[threadIdx.x] = page >= 0 && page < p.n_pages ? (int32_t)page : -1;
      at_of[threadIdx.x] = (int32_t)(slot & p.page_mask);
    }
  } else if ((int)threadIdx.x < n) {
    const int t = t0 + threadIdx.x, seq = kv_row_owner(b, t);
    const KvSeq s = kv_seq(b, seq);
    const int r = t - s.first;
    const int64_t pos = (int64_t)s.len - s.n + r;
    const bool mine = r >= 0 && r < s.n && pos >= 0;
    page_of[threadIdx.x] = mine ? kv_page(p, b, seq, (int32_t)pos) : -1;
    at_of[threadIdx.x] = mine ? (int32_t)pos & p.page_mask : 0;
  }
  __syncthreads();
  constexpr int U = 4;
  const uint32_t total = n * units;
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += U * kThreads) {
    u32x4 val[U];
    char* dst[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t idx = i0 + i * kThreads, tok = idx / units;
      dst[i] = nullptr;
      if (idx >= total || page_of[tok] < 0) continue;
      uint32_t u = idx - tok * units;
      const bool is_v = u >= units / 2;
      if (is_v) u -= units / 2;
      const uint32_t h = u / chunks, c = u - h * chunks;
      const int64_t* ps = is_v ? p.vst : p.kst;
      const int64_t* xs = is_v ? x.vst : x.kst;
      val[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(
          (is_v ? x.v : x.k) + 2 * ((int64_t)(t0 + tok) * xs[0] + h * xs[1] + 8 * (int64_t)c)));
      dst[i] = const_cast<char*>(is_v ? p.v : p.k) +
               2 * (page_of[tok] * ps[0] + at_of[tok] * ps[1] + h * ps[2] + 8 * (int64_t)c);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (dst[i]) *reinterpret_cast<u32x4*>(dst[i]) = val[i];
  }
}

constexpr int kPairs = 256;
struct PagePairs {
  int32_t src[kPairs], dst[kPairs];
};

struct CopyView {
  char* base[2];
  int64_t layer[2], page[2], token[2], head[2];  // strides in elements
  uint32_t chunks, heads, units;                 // per page and pool
  int whole;                                     // a page is one run of units
};

// Block (x, pair, layer and pool): U units per thread, kThreads apart, read and
// written past the caches (a forked or compacted page is not read at once). 80
// pages of 32 KB in 12 layers (126 MB read and written): 23 us, 5.5 TB/s; through
// the caches 29 us. The pairs travel as kernel arguments: checked on the host,
// and a captured call keeps them.
template <int U>
__global__ __launch_bounds__(kThreads) void kv_copy_kernel(CopyView c, PagePairs pairs) {
  const int pool = blockIdx.z & 1;
  const int pair = blockIdx.y;
  char* base = c.base[pool] + 2 * ((int64_t)(blockIdx.z >> 1) * c.layer[pool]);
  const char* src = base + 2 * (pairs.src[pair] * c.page[pool]);
  char* dst = base + 2 * (pairs.dst[pair] * c.page[pool]);
  u32x4 v[U];
  int64_t off[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = (blockIdx.x * U + i) * kThreads + threadIdx.x;
    if (c.whole) {
      off[i] = 16 * (int64_t)u;
    } else {
      const uint32_t row = u / c.chunks, t = row / c.heads;
      off[i] = 2 * (t * c.token[pool] + (row - t * c.heads) * c.head[pool] + 8 * (int64_t)(u - row * c.chunks));
    }
    if (u < c.units) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + off[i]));
  }
#pragma unroll
  for (int i = 0; i < U; ++i)
    if ((blockIdx.x * U + i) * kThreads + threadIdx.x < c.units)
      __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4*>(dst + off[i]));
}

// One run of page_size * kv_heads * head_dim elements, token- or head-major.
bool whole_page(const int64_t st[3], const hgk_kv_pages* p) {
  const int64_t d = p->head_dim, ps = p->page_size, h = p->kv_heads;
  return (st[1] == h * d && (h == 1 || st[2] == d)) || (st[2] == ps * d && (ps == 1 || st[1] == d)) ||
         (ps == 1 && (h == 1 || st[2] == d)) || (h == 1 && st[1] == d);
}

}  // namespace
}  // namespace hgk

using namespace hgk;

namespace {
// The call's operands checked, and the launch; `b` holds at least the tokens.
int append(const char* what, const KvView& p, const KvBatchView& b, const void* k, const int64_t k_strides[2],
           const void* v, const int64_t v_strides[2], const int64_t* slots, void* stream) {
  if (int st = kv_check_written_pages(what, p)) return st;
  RowsView x{static_cast<const char*>(k), static_cast<const char*>(v), {}, {}};
  if (int st = kv_check_rows(what, "k", k, k_strides, b.tokens, p.kv_heads, p.head_dim, false, x.kst)) return st;
  if (int st = kv_check_rows(what, "v", v, v_strides, b.tokens, p.kv_heads, p.head_dim, false, x.vst)) return st;
  if (pools_meet(p) && !same_rows(p, x))
    return fail(HGK_ERR_ARG, "%s: the key pages and the value pages overlap", what);
  const uint32_t chunks = p.head_dim / 8;
  const int64_t units = 2 * (int64_t)p.kv_heads * chunks;
  if (units > INT32_MAX / kMaxTokens) return fail(HGK_ERR_ARG, "%s: too many kv heads", what);
  // a token a block until the chip is full of blocks, then 16
  const int per = b.tokens <= 2048 ? 1 : kMaxTokens;
  const int64_t blocks = (b.tokens + (int64_t)per - 1) / per;
  if (blocks > kMaxBlocks) return fail(HGK_ERR_ARG, "%s: %d rows are too many", what, b.tokens);
  if (slots)
    HGK_LAUNCH(kv_append_kernel<true>, dim3((unsigned)blocks), dim3(kThreads), 0, as_stream(stream), p, b, x,
               (uint32_t)units, chunks, per, slots);
  else
    HGK_LAUNCH(kv_append_kernel<false>, dim3((unsigned)blocks), dim3(kThreads), 0, as_stream(stream), p, b, x,
               (uint32_t)units, chunks, per, slots);
  return launch_status(what);
}
}  // namespace

extern "C" int hgk_kv_append(const hgk_kv_pages* pages, const hgk_kv_batch* batch, const void* k,
                             const int64_t k_strides[2], const void* v, const int64_t v_strides[2],
                             void* stream) {
  clear_error();
  KvView p;
  KvBatchView b;
  if (int st = kv_check_pages("hgk_kv_append", pages, &p)) return st;
  if (int st = kv_check_batch("hgk_kv_append", p, batch, &b)) return st;
  if (b.batch == 0 || b.tokens == 0 || p.n_pages == 0) return HGK_OK;
  return append("hgk_kv_append", p, b, k, k_strides, v, v_strides, nullptr, stream);
}

extern "C" int hgk_kv_append_slots(const hgk_kv_pages* pages, const int64_t* slots, int64_t tokens, const void* k,
                                   const int64_t k_strides[2], const void* v, const int64_t v_strides[2],
                                   void* stream) {
  const char* what = "hgk_kv_append_slots";
  clear_error();
  KvView p;
  if (int st = kv_check_pages(what, pages, &p)) return st;
  if (tokens < 0 || tokens > INT32_MAX) return fail(HGK_ERR_ARG, "%s: tokens=%lld out of range", what, (long long)tokens);
  if (tokens == 0 || p.n_pages == 0) return HGK_OK;
  if (!slots || (reinterpret_cast<uintptr_t>(slots) & 7)) return fail(HGK_ERR_ARG, "%s: null or unaligned slots", what);
  KvBatchView b{};
  b.tokens = (int32_t)tokens;
  return append(what, p, b, k, k_strides, v, v_strides, slots, stream);
}

extern "C" int hgk_kv_copy_pages(const hgk_kv_pages* pages, int64_t layers,
                                 const int64_t layer_strides[2], const int32_t* src,
                                 const int32_t* dst, int64_t n, void* stream) {
  const char* what = "hgk_kv_copy_pages";
  clear_error();
  KvView p;
  if (int st = kv_check_pages(what, pages, &p)) return st;
  if (layers < 0 || layers > 32767) return fail(HGK_ERR_ARG, "%s: layers=%lld out of range", what, (long long)layers);
  if (n < 0) return fail(HGK_ERR_ARG, "%s: n=%lld", what, (long long)n);
  if (n > 0 && (!src || !dst)) return fail(HGK_ERR_ARG, "%s: null page list", what);
  if (layers > 1 && (!layer_strides || layer_strides[0] < 0 || layer_strides[1] < 0 ||
                     (layer_strides[0] & 7) || (layer_strides[1] & 7)))
    return fail(HGK_ERR_ARG, "%s: layer strides must be multiples of 8 elements", what);
  for (int64_t i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= p.n_pages || dst[i] < 0 || dst[i] >= p.n_pages)
      return fail(HGK_ERR_ARG, "%s: pair %lld (%d to %d) outside the %d pages", what, (long long)i,
                  src[i], dst[i], p.n_pages);
  try {
    std::vector<int32_t> d(dst, dst + n);
    std::sort(d.begin(), d.end());
    const auto twice = std::adjacent_find(d.begin(), d.end());
    if (twice != d.end()) return fail(HGK_ERR_ARG, "%s: page %d is a destination twice", what, *twice);
    for (int64_t i = 0; i < n; ++i)
      if (std::binary_search(d.begin(), d.end(), src[i]))
        return fail(HGK_ERR_ARG, "%s: page %d is a source and a destination", what, src[i]);
  } catch (const std::bad_alloc&) {
    return fail(HGK_ERR_ARG, "%s: no host memory to check %lld pairs", what, (long long)n);
  }
  if (n == 0 || layers == 0) return HGK_OK;
  if (int st = kv_check_written_pages(what, p)) return st;
  const int64_t extent[4] = {p.n_pages, (int64_t)p.page_mask + 1, p.kv_heads, layers};
  const int64_t ks[4] = {p.kst[0], p.kst[1], p.kst[2], layers > 1 ? layer_strides[0] : 0};
  const int64_t vs[4] = {p.vst[0], p.vst[1], p.vst[2], layers > 1 ? layer_strides[1] : 0};
  if (rows_overlap(ks, extent, 4, p.head_dim) || rows_overlap(vs, extent, 4, p.head_dim))
    return fail(HGK_ERR_ARG, "%s: the layers' pages overlap", what);
  CopyView c;
  c.base[0] = static_cast<char*>(pages->k);
  c.base[1] = static_cast<char*>(pages->v);
  const int64_t* st[2] = {p.kst, p.vst};
  for (int i = 0; i < 2; ++i) {
    c.layer[i] = layers > 1 ? layer_strides[i] : 0;
    c.page[i] = st[i][0];
    c.token[i] = st[i][1];
    c.head[i] = st[i][2];
  }
  c.chunks = p.head_dim / 8;
  c.heads = p.kv_heads;
  const int64_t units = (int64_t)pages->page_size * p.kv_heads * c.chunks;
  if (units > INT32_MAX) return fail(HGK_ERR_ARG, "%s: a page of %lld units is too large", what, (long long)units);
  c.units = (uint32_t)units;
  c.whole = whole_page(st[0], pages) && whole_page(st[1], pages);
  constexpr int U = 2;
  const unsigned gx = (unsigned)((units + kThreads * U - 1) / (kThreads * U));
  PagePairs pairs;
  for (int64_t at = 0; at < n; at += kPairs) {
    const int m = (int)std::min<int64_t>(kPairs, n - at);
    std::copy(src + at, src + at + m, pairs.src);
    std::copy(dst + at, dst + at + m, pairs.dst);
    HGK_LAUNCH(kv_copy_kernel<U>, dim3(gx, m, (unsigned)(2 * layers)), dim3(kThreads), 0,
               as_stream(stream), c, pairs);
    if (int e = launch_status(what)) return e;
  }
  return HGK_OK;
}
