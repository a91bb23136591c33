// kv.h -- the paged key-value cache as the kernels see it: the pool's and the
// batch's layout, passed by value, and the checks that the entry points share.
#pragma once

#include "../../include/higgs_hip.h"
#include "hgk_common.h"
#include "hgk_host.h"

namespace hgk {

struct KvView {
  const char* k;
  const char* v;
  int64_t kst[3], vst[3];  // page, token, head (elements)
  int32_t n_pages, page_shift, page_mask;
  int32_t kv_heads, head_dim;
};

struct KvBatchView {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;  // null: one row per sequence
  int64_t table_stride;
  int32_t width;  // table entries per sequence
  int32_t batch, tokens;
};

// Rows [first, first + n) of a sequence and its length (a negative one counts
// as none). Whatever the arrays hold, the rows lie within the packed array.
struct KvSeq {
  int32_t first, n, len;
};

__host__ __device__ inline KvSeq kv_seq(const KvBatchView& b, int seq) {
  KvSeq s;
  s.len = b.lens[seq] < 0 ? 0 : b.lens[seq];
  if (!b.starts) {
    s.first = seq;
    s.n = seq < b.tokens ? 1 : 0;
    return s;
  }
  const int32_t lo = b.starts[seq], hi = b.starts[seq + 1];
  if (lo < 0 || hi > b.tokens || lo >= hi) {
    s.first = 0;
    s.n = 0;
  } else {
    s.first = lo;
    s.n = hi - lo;
  }
  return s;
}

// Page of key position `pos` (>= 0) of a sequence: -1 where the table has none.
__host__ __device__ inline int32_t kv_page(const KvView& p, const KvBatchView& b, int seq, int32_t pos) {
  const int32_t e = pos >> p.page_shift;
  if (e >= b.width) return -1;
  const int32_t page = b.table[(int64_t)seq * b.table_stride + e];
  return (uint32_t)page < (uint32_t)p.n_pages ? page : -1;
}

// Sequence that owns row t of the packed array, if one does: the last b with
// starts[b] <= t (0 where there is none).
__host__ __device__ inline int kv_row_owner(const KvBatchView& b, int t) {
  if (!b.starts) return t;
  int lo = 0, hi = b.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Checks of the pool and the batch; on success the views are filled in.
int kv_check_pages(const char* what, const hgk_kv_pages* p, KvView* out);
int kv_check_batch(const char* what, const KvView& p, const hgk_kv_batch* b, KvBatchView* out);

// A grid of 256-thread blocks has at most this many (2^31 threads).
constexpr int64_t kMaxBlocks = 1 << 23;

// A [tokens, heads, head_dim] operand: pointer and strides usable by 16-byte
// accesses (the stride of an axis of one element is not looked at, and comes
// out as 0); rows that are written may not lie on each other.
int kv_check_rows(const char* what, const char* name, const void* p, const int64_t strides[2],
                  int64_t tokens, int64_t heads, int64_t head_dim, bool written, int64_t out[2]);
// The same of pages that a call writes to.
int kv_check_written_pages(const char* what, const KvView& p);

}  // namespace hgk
