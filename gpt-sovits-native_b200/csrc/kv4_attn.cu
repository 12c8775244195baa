// kv4_attn.cu — attention over the paged 4-bit KV cache (gsvk_kv4_attention).
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4.cuh"

namespace gsvk {

namespace {

struct AttnArgs {
  const uint8_t* pages;
  size_t page_bytes;
  int n_pages, shift, kv_heads;
  const uint16_t* q;
  size_t q_stride;
  uint16_t* out;
  size_t out_stride;
  int heads, group, n_tokens, n_seq, max_blocks;
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* prefix;
  const int32_t* table;
  float scale_log2;  // scale * log2(e)
};

constexpr int kSimpleWarps = 4;

// One warp per (row, query head): 32 keys at a time, a lane to a key for the
// scores and to head_dim / 32 dimensions for the sums.
template <int HD>
__global__ void __launch_bounds__(kSimpleWarps * 32) kv4_attn_rows_kernel(const AttnArgs a) {
  __shared__ float s_q[kSimpleWarps][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kSimpleWarps + warp;
  if (item >= static_cast<long long>(a.n_tokens) * a.heads) return;
  const int t = static_cast<int>(item / a.heads), head = static_cast<int>(item % a.heads);
  int lo = 0, hi = a.n_seq + 1;  // the last request starting at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.q_start[mid] <= t) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  if (lo >= a.n_seq || t < a.q_start[0]) return;  // a row of no request
  const int len = a.kv_len[lo], n = a.q_start[lo + 1] - a.q_start[lo];
  int limit = len - n + (t - a.q_start[lo]) + 1;
  if (a.prefix) limit = max(limit, a.prefix[lo]);
  limit = max(0, min(limit, min(len, a.max_blocks << a.shift)));
  const uint16_t* q = a.q + static_cast<size_t>(t) * a.q_stride + static_cast<size_t>(head) * HD;
  float qsum = 0.f;
  for (int d = lane; d < HD; d += 32) {
    const float x = h2f(q[d]);
    s_q[warp][d] = x;
    qsum += x;
  }
  qsum = warp_sum(qsum);
  __syncwarp();
  const size_t head_off = static_cast<size_t>(head / a.group) * kv4_head_bytes(a.shift, HD);
  const int32_t* row = a.table + static_cast<size_t>(lo) * a.max_blocks;
  float m = -INFINITY, l = 0.f, acc[HD / 32] = {};
  for (int j0 = 0; j0 < limit; j0 += 32) {
    const int j = j0 + lane;
    const int page = j < limit ? row[j >> a.shift] : -1;
    const bool live = page >= 0 && page < a.n_pages;
    const uint8_t* b = a.pages + static_cast<size_t>(live ? page : 0) * a.page_bytes + head_off;
    const int at = j & ((1 << a.shift) - 1);
    float s = -INFINITY;
    uint32_t vp = 0;
    if (live) {
      float dot = 0.f;
      for (int i = 0; i < HD / 8; ++i) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(b + at * (HD / 2) + i * 4);
        for (int u = 0; u < 8; ++u) dot = fmaf(s_q[warp][8 * i + u], float((w >> (4 * u)) & 15u), dot);
      }
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(b + kv4_k_par(a.shift, HD) + at * 4);
      vp = *reinterpret_cast<const uint32_t*>(b + kv4_v_par(a.shift, HD) + at * 4);
      s = fmaf(h2f(uint16_t(kp)), dot, h2f(uint16_t(kp >> 16)) * qsum) * a.scale_log2;
    }
    const float mn = fmaxf(m, warp_max(s));
    const float ref = mn == -INFINITY ? 0.f : mn;  // no key seen yet
    const float keep = exp2f(m - ref), p = exp2f(s - ref);
    m = mn;
    l = fmaf(l, keep, p);
    for (int i = 0; i < HD / 32; ++i) acc[i] *= keep;
    for (int u = 0; u < 32; ++u) {
      const float pu = __shfl_sync(0xffffffffu, p, u);
      const uint32_t par = __shfl_sync(0xffffffffu, vp, u);
      const unsigned long long bu = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(b), u);
      const int pos = (j0 + u) & ((1 << a.shift) - 1);
      if (pu == 0.f) continue;
      const uint8_t* c = reinterpret_cast<const uint8_t*>(bu) + kv4_v_codes(a.shift, HD) + pos * (HD / 2);
      for (int i = 0; i < HD / 32; ++i) {
        const int d = lane + 32 * i;
        const float code = float((c[d >> 1] >> (4 * (d & 1))) & 15);
        acc[i] = fmaf(pu, fmaf(h2f(uint16_t(par)), code, h2f(uint16_t(par >> 16))), acc[i]);
      }
    }
  }
  l = warp_sum(l);
  uint16_t* o = a.out + static_cast<size_t>(t) * a.out_stride + static_cast<size_t>(head) * HD;
  for (int i = 0; i < HD / 32; ++i) o[lane + 32 * i] = f2h(l > 0.f || l != l ? acc[i] / l : 0.f);
}

}  // namespace
}  // namespace gsvk

using namespace gsvk;

extern "C" {

size_t gsvk_kv4_attention_workspace(size_t n_seq, size_t n_tokens, size_t heads, size_t kv_heads,
                                    size_t head_dim) {
  if (n_seq == 0 || n_seq > 16384 || kv_heads == 0 || kv_heads > 1024 || heads % kv_heads ||
      heads == 0 || heads > 65536 || n_tokens > 0x7fffffff ||
      (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return 0;
  return 256;
}

int gsvk_kv4_attention(const gsvk_kv4_attention_args* g, gsvk_stream_t stream) {
  if (!g) return fail(GSVK_ERR_INVALID, "kv4_attention: null arguments");
  if (int rc = kv4_check(&g->cache, "kv4_attention")) return rc;
  if (g->n_tokens == 0) return GSVK_OK;
  if (!g->q || !g->out || !g->q_start || !g->kv_len || !g->block_table || !g->workspace)
    return fail(GSVK_ERR_INVALID, "kv4_attention: null pointer");
  if (g->heads == 0 || g->n_seq == 0 || g->max_blocks == 0)
    return fail(GSVK_ERR_INVALID, "kv4_attention: zero size");
  if (g->heads % g->cache.kv_heads)
    return fail(GSVK_ERR_INVALID, "kv4_attention: %zu query heads over %d kv heads", g->heads,
                g->cache.kv_heads);
  const int shift = kv4_page_shift(g->cache.page_size), hd = g->cache.head_dim;
  const size_t need = gsvk_kv4_attention_workspace(g->n_seq, g->n_tokens, g->heads,
                                                   g->cache.kv_heads, hd);
  if (need == 0 || g->max_blocks > (0x7fffff00u >> shift))
    return fail(GSVK_ERR_UNSUPPORTED, "kv4_attention: too many requests, rows, heads or blocks");
  if (g->workspace_bytes < need)
    return fail(GSVK_ERR_INVALID, "kv4_attention: workspace of %zu bytes, %zu needed",
                g->workspace_bytes, need);
  const size_t width = g->heads * hd;
  if (g->n_tokens > 1 && (g->q_stride < width || g->out_stride < width))
    return fail(GSVK_ERR_INVALID, "kv4_attention: row stride below %zu", width);
  if (!aligned16(g->q) || !aligned16(g->out) || g->q_stride % 8 || g->out_stride % 8 ||
      (reinterpret_cast<uintptr_t>(g->workspace) & 255u))
    return fail(GSVK_ERR_ALIGN, "kv4_attention: rows not in whole 16 bytes or workspace not 256-byte aligned");
  AttnArgs a{};
  a.pages = g->cache.pages;
  a.page_bytes = gsvk_kv4_page_bytes(g->cache.page_size, g->cache.kv_heads, hd);
  a.n_pages = static_cast<int>(g->cache.n_pages);
  a.shift = shift;
  a.kv_heads = g->cache.kv_heads;
  a.q = g->q;
  a.q_stride = g->q_stride;
  a.out = g->out;
  a.out_stride = g->out_stride;
  a.heads = static_cast<int>(g->heads);
  a.group = a.heads / a.kv_heads;
  a.n_tokens = static_cast<int>(g->n_tokens);
  a.n_seq = static_cast<int>(g->n_seq);
  a.max_blocks = static_cast<int>(g->max_blocks);
  a.q_start = g->q_start;
  a.kv_len = g->kv_len;
  a.prefix = g->prefix;
  a.table = g->block_table;
  a.scale_log2 = g->scale * 1.4426950408889634f;
  const size_t items = g->n_tokens * g->heads;
  const unsigned blocks = ceil_div(items, kSimpleWarps);
  cudaStream_t st = as_cuda(stream);
  if (hd == 32) kv4_attn_rows_kernel<32><<<blocks, kSimpleWarps * 32, 0, st>>>(a);
  if (hd == 64) kv4_attn_rows_kernel<64><<<blocks, kSimpleWarps * 32, 0, st>>>(a);
  if (hd == 128) kv4_attn_rows_kernel<128><<<blocks, kSimpleWarps * 32, 0, st>>>(a);
  return check_launch("kv4_attn_rows_kernel");
}

}  // extern "C"
