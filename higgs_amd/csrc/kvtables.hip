// kvtables.hip -- pages given out to sequences and taken back on the GPU, with the
// tables, starts, positions and places that a call over the new tokens needs, so
// that a step whose lengths only the GPU knows needs no host.
#include <algorithm>

#include "kv.h"

namespace hgk {
namespace {

constexpr int kPlanThreads = 1024, kMaxRows = 1 << 18, kFill = 256, kNear = 4096;
// Calls in one launch: at most so many sequences (releases of named ones: fewer),
// resident ones and blocks.
constexpr int kOneBatch = 1024, kOneNamed = 640, kOneRows = 1 << 15, kOneBlocks = 512;

struct TablesView {
  int32_t* table;
  const int32_t* lens;
  int32_t* free_pages;
  const int32_t* n_free;
  int64_t stride;
  int32_t rows, width, n_pages, shift;
};

struct PlanArgs {
  TablesView t;
  const int32_t* seqs;    // rows of the batch; null: row i is sequence i
  const int32_t* counts;  // new tokens, or (release) the tokens that stay; null: 0
  const int32_t* owned;   // release: pages at a row's front that are not its own; null: 0
  int32_t batch, tokens, release;
  int32_t* lens_out;
  int32_t* n_free_out;
  int32_t* kv_lens;
  int32_t* q_starts;
  int32_t* status;
  int32_t* page_starts;  // [batch + 1] pages that go to, or come from, the sequences before each
};

// Pages that hold so many tokens; past 2^30 of them, which no table has, 2^30 + 1.
__device__ inline int32_t pages_of(const TablesView& t, int64_t tokens) {
  return (int32_t)min((tokens + (1 << t.shift) - 1) >> t.shift, (int64_t)(1 << 30) + 1);
}

// What sequence i of the batch asks for.
struct Ask {
  int32_t row, old, pages, tokens, status;  // row -1: none
  int64_t now;
};
__device__ inline Ask ask_of(const PlanArgs& a, int i) {
  Ask k{a.seqs ? a.seqs[i] : i, 0, 0, 0, 0, 0};
  if ((uint32_t)k.row >= (uint32_t)a.t.rows) return Ask{-1, 0, 0, 0, HGK_TABLES_SEQUENCE, 0};
  const int32_t n = a.counts ? a.counts[i] : 0;
  k.old = max(a.t.lens[k.row], 0);
  if (a.release) {
    k.now = min(max(n, 0), k.old);
    const int32_t had = pages_of(a.t, k.old), first = max(pages_of(a.t, k.now), a.owned ? a.owned[k.row] : 0);
    k.pages = max(had - first, 0);
    if (had > a.t.width) k.status |= HGK_TABLES_WIDTH;
  } else {
    k.tokens = max(n, 0);
    k.now = (int64_t)k.old + k.tokens;
    const int32_t has = pages_of(a.t, k.now);
    k.pages = has - pages_of(a.t, k.old);
    if (n < 0) k.status |= HGK_TABLES_SEQUENCE;
    if (has > a.t.width) k.status |= HGK_TABLES_WIDTH;
  }
  return k;
}

struct Pair {
  int64_t pages, tokens;
};
__device__ inline int64_t shift_up(int64_t v, int by) { return __shfl_up(v, by); }

// What a block finds out about a call: a thread has the run i0 .. i1 - 1 of the
// batch's sequences; the pages and tokens of all in front of it, and of all.
struct Sums {
  int i0, i1;
  int32_t status, n_free;
  Pair before, total;
};
template <int THREADS, int ROWS>
__device__ inline Sums sums_of(const PlanArgs& a) {
  constexpr int kWaves = THREADS / 64;
  __shared__ uint32_t named[ROWS / 32];
  __shared__ int64_t wave_pages[kWaves], wave_tokens[kWaves];
  __shared__ int32_t bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (a.batch + THREADS - 1) / THREADS;
  Sums s;
  s.i0 = min(tid * run, a.batch);
  s.i1 = min(s.i0 + run, a.batch);
  s.n_free = min(max(*a.t.n_free, 0), a.t.n_pages);
  if (tid == 0) bad = 0;
  if (a.seqs)
    for (int w = tid; w < (a.t.rows + 31) / 32; w += THREADS) named[w] = 0;
  __syncthreads();
  Pair mine{0, 0};
  int32_t status = 0;
  for (int i = s.i0; i < s.i1; ++i) {
    const Ask k = ask_of(a, i);
    mine.pages += k.pages;
    mine.tokens += k.tokens;
    status |= k.status;
    if (a.seqs && k.row >= 0 && (atomicOr(&named[k.row >> 5], 1u << (k.row & 31)) >> (k.row & 31)) & 1)
      status |= HGK_TABLES_SEQUENCE;
  }
  Pair upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t p = shift_up(upto.pages, o), t = shift_up(upto.tokens, o);
    if (lane >= o) {
      upto.pages += p;
      upto.tokens += t;
    }
  }
  if (lane == 63) {
    wave_pages[wave] = upto.pages;
    wave_tokens[wave] = upto.tokens;
  }
  if (status) atomicOr(&bad, status);
  __syncthreads();
  s.before = Pair{upto.pages - mine.pages, upto.tokens - mine.tokens};
  s.total = Pair{0, 0};
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) {
      s.before.pages += wave_pages[w];
      s.before.tokens += wave_tokens[w];
    }
    s.total.pages += wave_pages[w];
    s.total.tokens += wave_tokens[w];
  }
  s.status = bad;
  if (s.total.pages > (a.release ? a.t.n_pages - s.n_free : s.n_free)) s.status |= HGK_TABLES_PAGES;
  if (s.total.tokens > a.tokens) s.status |= HGK_TABLES_TOKENS;
  return s;
}

// Writes the new state and the sequences' small results, by one block. The state may
// be written where it was read: each of its values is read by the thread that writes
// it, or before a barrier.
template <int THREADS>
__device__ inline void write_plan(const PlanArgs& a, const Sums& s) {
  const bool go = s.status == 0;
  if (a.lens_out != a.t.lens) {
    for (int r = threadIdx.x; r < a.t.rows; r += THREADS) a.lens_out[r] = a.t.lens[r];
    __syncthreads();
  }
  Pair before = s.before;
  for (int i = s.i0; i < s.i1; ++i) {
    const Ask k = ask_of(a, i);
    a.page_starts[i] = go ? (int32_t)before.pages : 0;
    if (!a.release) {
      a.q_starts[i] = go ? (int32_t)before.tokens : 0;
      a.kv_lens[i] = go ? (int32_t)k.now : k.old;
    }
    if (go) a.lens_out[k.row] = (int32_t)k.now;
    before.pages += k.pages;
    before.tokens += k.tokens;
  }
  if (threadIdx.x == 0) {
    a.page_starts[a.batch] = go ? (int32_t)s.total.pages : 0;
    if (!a.release) a.q_starts[a.batch] = go ? (int32_t)s.total.tokens : 0;
    const int32_t moved = go ? (int32_t)s.total.pages : 0;
    *a.n_free_out = s.n_free + (a.release ? moved : -moved);
    *a.status = s.status;
  }
}

// The first of two launches: what the second one's blocks read.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a) {
  write_plan<kPlanThreads>(a, sums_of<kPlanThreads, kMaxRows>(a));
}

struct ExtendArgs {
  PlanArgs p;
  int64_t* slots;
  int32_t* positions;
  int32_t* block_table;  // null: the tables themselves
  int64_t block_stride;
  int32_t token_blocks, row_blocks, blocks;  // blocks over tokens; of a row of block_table; all
};

// The page of entry e of a sequence that had `had` pages and whose new ones begin
// at `from` of the call's: they come from the top of the stack downwards.
__device__ inline int32_t entry_of(const PlanArgs& a, int32_t top, int32_t row, int32_t had, int32_t from, int32_t e) {
  return e < had ? a.t.table[row * a.t.stride + e] : a.t.free_pages[top - 1 - (from + e - had)];
}

// What the blocks of a call read of its sequences: the pages and tokens in front of
// each, and its row; the length is worked out of them.
struct Seqs {
  const int32_t* pages;   // [batch + 1]
  const int32_t* tokens;  // [batch + 1]
  int32_t top;            // free pages before the call
};

// Block `block` over the tokens, each thread with one: its sequence, position and place;
// the first token of a page writes the page into the table. Then blocks over the
// rows of the batch's own table, if it has one. old(i, row): sequence i's tokens
// before the call.
template <class Old>
__device__ inline void extend_block(const ExtendArgs& x, int block, const Seqs& q, Old old) {
  const PlanArgs& a = x.p;
  if (block < x.token_blocks) {
    const int t = block * kFill + threadIdx.x;
    if (t >= a.tokens) return;
    if (t >= q.tokens[a.batch]) {
      x.slots[t] = -1;
      x.positions[t] = 0;
      return;
    }
    int lo = 0, hi = a.batch;  // the last sequence that starts at t or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (q.tokens[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int32_t row = a.seqs ? a.seqs[lo] : lo, had = old(lo, row), pos = had + t - q.tokens[lo];
    const int32_t e = pos >> a.t.shift, at = pos & ((1 << a.t.shift) - 1);
    const int32_t page = entry_of(a, q.top, row, pages_of(a.t, had), q.pages[lo], e);
    if (at == 0) a.t.table[row * a.t.stride + e] = page;
    x.slots[t] = ((int64_t)page << a.t.shift) + at;
    x.positions[t] = pos;
    return;
  }
  const int b = block - x.token_blocks, i = b / x.row_blocks;
  const int e = (b - i * x.row_blocks) * kFill + threadIdx.x;
  if (e >= a.t.width) return;
  const int32_t row = a.seqs[i];
  int32_t page = -1;
  if ((uint32_t)row < (uint32_t)a.t.rows) {
    const int32_t had = old(i, row);
    if (e < pages_of(a.t, (int64_t)had + q.tokens[i + 1] - q.tokens[i]))
      page = entry_of(a, q.top, row, pages_of(a.t, had), q.pages[i], e);
  }
  x.block_table[i * x.block_stride + e] = page;
}
__global__ __launch_bounds__(kFill) void kv_extend_kernel(ExtendArgs x) {
  const PlanArgs& a = x.p;
  // the starts, where they fit: a search is a chain of reads
  __shared__ int32_t near[kNear + 1];
  const bool cached = a.batch <= kNear && (int)blockIdx.x < x.token_blocks;
  if (cached) {
    for (int i = threadIdx.x; i <= a.batch; i += kFill) near[i] = a.q_starts[i];
    __syncthreads();
  }
  const Seqs q{a.page_starts, cached ? near : a.q_starts, *a.n_free_out + a.page_starts[a.batch]};
  extend_block(x, blockIdx.x, q, [&](int i, int32_t) { return a.kv_lens[i] - (q.tokens[i + 1] - q.tokens[i]); });
}

// Block = sequence: its pages that are no longer needed go on the stack, in order.
__device__ inline void release_row(const PlanArgs& a, int i, int32_t keeps, int32_t from, int32_t n, int32_t base) {
  if (n == 0) return;
  const int32_t row = a.seqs ? a.seqs[i] : i, first = max(pages_of(a.t, keeps), a.owned ? a.owned[row] : 0);
  for (int j = threadIdx.x; j < n; j += kFill) a.t.free_pages[base + from + j] = a.t.table[row * a.t.stride + first + j];
}
__global__ __launch_bounds__(kFill) void kv_release_kernel(PlanArgs a) {
  const int i = blockIdx.x;
  const int32_t from = a.page_starts[i], n = a.page_starts[i + 1] - from;
  if (n > 0)
    release_row(a, i, a.lens_out[a.seqs ? a.seqs[i] : i], from, n, *a.n_free_out - a.page_starts[a.batch]);
}

// A call in one launch: every block works the sums out for itself, and the state must
// not be written where other blocks still read it. In us, in a graph, in one launch and
// in two: 64 sequences given a token each 4.4, 6.3; 512 6.1, 8.3; 1000 8.6, 9.5; up to 64
// tokens each 4.5, 7.5; 6.2, 9.0; 8.8, 10.3. Releases 3.6, 6.3; 5.0, 6.6; 7.4, 7.6; of
// named ones, which are looked up and marked in every block, 64 of 96 4.1, 6.6; 512 of
// 768 6.2, 7.4; 768 of 1152 8.8, 7.9; 1000 of 1500 10.3, 8.7. (In place, always two.)
template <bool RELEASE>
__global__ __launch_bounds__(kFill) void kv_one_kernel(ExtendArgs x) {
  __shared__ int32_t pages[kOneBatch + 1], tokens[kOneBatch + 1];
  const PlanArgs& a = x.p;
  const Sums s = sums_of<kFill, kOneRows>(a);
  const bool go = s.status == 0;
  Pair before = s.before;
  for (int i = s.i0; i < s.i1; ++i) {
    const Ask k = ask_of(a, i);
    pages[i] = go ? (int32_t)before.pages : 0;
    tokens[i] = go ? (int32_t)before.tokens : 0;
    before.pages += k.pages;
    before.tokens += k.tokens;
  }
  if (threadIdx.x == 0) {
    pages[a.batch] = go ? (int32_t)s.total.pages : 0;
    tokens[a.batch] = go ? (int32_t)s.total.tokens : 0;
  }
  if (blockIdx.x == 0) write_plan<kFill>(a, s);
  __syncthreads();
  if constexpr (RELEASE) {
    for (int i = blockIdx.x; i < a.batch; i += gridDim.x)
      if (pages[i + 1] > pages[i])
        release_row(a, i, (int32_t)ask_of(a, i).now, pages[i], pages[i + 1] - pages[i], s.n_free);
  } else if ((int)blockIdx.x < x.blocks) {
    const Seqs q{pages, tokens, s.n_free};
    extend_block(x, blockIdx.x, q, [&](int, int32_t row) { return max(a.t.lens[row], 0); });
  }
}

int check_tables(const char* what, const hgk_kv_tables* t, int64_t batch, TablesView* out) {
  if (!t) return fail(HGK_ERR_ARG, "%s: null tables", what);
  if (t->page_size < 1 || t->page_size > 65536 || (t->page_size & (t->page_size - 1)))
    return fail(HGK_ERR_ARG, "%s: page_size=%d must be a power of two in 1..65536", what, t->page_size);
  if (t->rows < 0 || batch < 0) return fail(HGK_ERR_ARG, "%s: %lld rows, batch=%lld", what, (long long)t->rows, (long long)batch);
  if (t->rows > kMaxRows) return fail(HGK_ERR_UNSUPPORTED, "%s: %lld rows (at most %d)", what, (long long)t->rows, kMaxRows);
  if (t->n_pages < 0 || t->n_pages > INT32_MAX) return fail(HGK_ERR_ARG, "%s: n_pages=%lld out of range", what, (long long)t->n_pages);
  out->shift = __builtin_ctz((unsigned)t->page_size);
  if (t->table_width < 0 || t->table_stride < 0 || (t->rows > 1 && t->table_stride < t->table_width))
    return fail(HGK_ERR_ARG, "%s: bad table width or stride", what);
  if (t->table_width > (int64_t)1 << (30 - out->shift))
    return fail(HGK_ERR_ARG, "%s: a table of %lld pages of %d tokens is too wide (2^30 tokens)", what,
                (long long)t->table_width, t->page_size);
  if ((t->rows > 0 && (!t->lens || (t->table_width > 0 && !t->tables))) || (t->n_pages > 0 && !t->free_pages) || !t->n_free)
    return fail(HGK_ERR_ARG, "%s: null table, lengths, free pages or their number", what);
  out->table = t->tables;
  out->lens = t->lens;
  out->free_pages = t->free_pages;
  out->n_free = t->n_free;
  out->stride = t->rows > 1 ? t->table_stride : 0;
  out->rows = (int32_t)t->rows;
  out->width = (int32_t)t->table_width;
  out->n_pages = (int32_t)t->n_pages;
  return HGK_OK;
}

int check_batch(const char* what, const TablesView& t, const int32_t* seqs, int64_t batch) {
  if (!seqs && batch != t.rows && batch != 0)
    return fail(HGK_ERR_ARG, "%s: %lld sequences of %d rows need their rows' numbers", what, (long long)batch, t.rows);
  if (batch > t.rows) return fail(HGK_ERR_ARG, "%s: %lld sequences of %d rows", what, (long long)batch, t.rows);
  return HGK_OK;
}

// One launch is faster, and the state is not written in place.
bool in_one(const PlanArgs& a) {
  return a.batch <= (a.release && a.seqs ? kOneNamed : kOneBatch) && a.t.rows <= kOneRows && a.lens_out != a.t.lens && a.n_free_out != a.t.n_free;
}

}  // namespace
}  // namespace hgk

using namespace hgk;

extern "C" int hgk_kv_extend(const hgk_kv_tables* tables, const int32_t* seqs, const int32_t* counts, int64_t batch,
                             int64_t tokens, int32_t* lens_out, int32_t* n_free_out, int32_t* kv_lens,
                             int32_t* q_starts, int64_t* slots, int32_t* positions, int32_t* block_table,
                             int64_t block_table_stride, int32_t* status, int32_t* workspace, void* stream) {
  const char* what = "hgk_kv_extend";
  clear_error();
  PlanArgs a{};
  if (int st = check_tables(what, tables, batch, &a.t)) return st;
  if (int st = check_batch(what, a.t, seqs, batch)) return st;
  if (tokens < 0 || tokens > 1 << 30) return fail(HGK_ERR_ARG, "%s: tokens=%lld out of range", what, (long long)tokens);
  if ((batch > 0 && (!counts || !kv_lens)) || (a.t.rows > 0 && !lens_out) || !n_free_out || !q_starts || !status || !workspace ||
      (tokens > 0 && (!slots || !positions)))
    return fail(HGK_ERR_ARG, "%s: null counts or output", what);
  if (block_table && !seqs) return fail(HGK_ERR_ARG, "%s: a table of the batch's own needs the rows' numbers", what);
  if (block_table && batch > 1 && block_table_stride < a.t.width)
    return fail(HGK_ERR_ARG, "%s: rows of the batch's table overlap (stride %lld)", what, (long long)block_table_stride);
  a.seqs = seqs;
  a.counts = counts;
  a.batch = (int32_t)batch;
  a.tokens = (int32_t)tokens;
  a.lens_out = lens_out;
  a.n_free_out = n_free_out;
  a.kv_lens = kv_lens;
  a.q_starts = q_starts;
  a.status = status;
  a.page_starts = workspace;
  ExtendArgs x{a, slots, positions, block_table, block_table_stride, (int32_t)((tokens + kFill - 1) / kFill),
               (a.t.width + kFill - 1) / kFill, 0};
  const int64_t blocks = x.token_blocks + (block_table ? batch * x.row_blocks : 0);
  if (blocks > kMaxBlocks) return fail(HGK_ERR_ARG, "%s: %lld rows of %d pages are too many", what, (long long)batch, a.t.width);
  x.blocks = (int32_t)blocks;
  if (in_one(a) && blocks <= kOneBlocks) {
    HGK_LAUNCH(kv_one_kernel<false>, dim3((unsigned)std::max<int64_t>(blocks, 1)), dim3(kFill), 0, as_stream(stream), x);
    return launch_status(what);
  }
  HGK_LAUNCH(kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), a);
  if (int st = launch_status(what)) return st;
  if (blocks == 0) return HGK_OK;
  HGK_LAUNCH(kv_extend_kernel, dim3((unsigned)blocks), dim3(kFill), 0, as_stream(stream), x);
  return launch_status(what);
}

extern "C" int hgk_kv_release(const hgk_kv_tables* tables, const int32_t* seqs, const int32_t* keep,
                              const int32_t* owned_from, int64_t batch, int32_t* lens_out, int32_t* n_free_out,
                              int32_t* status, int32_t* workspace, void* stream) {
  const char* what = "hgk_kv_release";
  clear_error();
  PlanArgs a{};
  if (int st = check_tables(what, tables, batch, &a.t)) return st;
  if (int st = check_batch(what, a.t, seqs, batch)) return st;
  if ((a.t.rows > 0 && !lens_out) || !n_free_out || !status || !workspace) return fail(HGK_ERR_ARG, "%s: null output", what);
  a.seqs = seqs;
  a.counts = keep;
  a.owned = owned_from;
  a.batch = (int32_t)batch;
  a.release = 1;
  a.lens_out = lens_out;
  a.n_free_out = n_free_out;
  a.status = status;
  a.page_starts = workspace;
  if (in_one(a)) {
    ExtendArgs x{};
    x.p = a;
    const int64_t blocks = std::clamp<int64_t>(batch, 1, kOneBlocks);
    HGK_LAUNCH(kv_one_kernel<true>, dim3((unsigned)blocks), dim3(kFill), 0, as_stream(stream), x);
    return launch_status(what);
  }
  HGK_LAUNCH(kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), a);
  if (int st = launch_status(what)) return st;
  if (batch == 0) return HGK_OK;
  HGK_LAUNCH(kv_release_kernel, dim3((unsigned)batch), dim3(kFill), 0, as_stream(stream), a);
  return launch_status(what);
}
