// attn.hip -- attention of new tokens over a paged key-value cache.
#include <cmath>

#include "kv.h"

namespace hgk {
namespace {

struct AttnArgs {
  KvView p;
  KvBatchView b;
  const char* q;
  char* out;
  int64_t qst[2], ost[2];  // token, head
  int32_t q_heads, group;  // group = q heads per kv head
  float scale, softcap;
  int32_t window, sinks;
};

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
  if (window < 0 || sinks < 0)
    return fail(HGK_ERR_ARG, "%s: window=%lld, sinks=%lld must not be negative", what, (long long)window,
                (long long)sinks);
  return HGK_OK;
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
  return 0;
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
  const dim3 grid((unsigned)a.b.tokens, (unsigned)q_heads);
  if (pages->dtype == DT_BF16)
    HGK_LAUNCH(attn_simple_kernel<BF16>, grid, dim3(64), 0, as_stream(stream), a);
  else
    HGK_LAUNCH(attn_simple_kernel<F16>, grid, dim3(64), 0, as_stream(stream), a);
  return launch_status(what);
}
