// kv_plan.cu — page plan of a serving step (gsvk_kv_plan) and the return of
// finished requests' pages (gsvk_kv_release).
//
// A plan is two prefix sums over the requests (packed rows, pages needed) and
// a map from every packed row to its slot.  The sums are a chain of dependent
// barriers over a few KB, so what bounds the kernel is latency: launch, one
// load of the lengths, one block-wide scan, one more load per row.  Every CTA
// therefore repeats the scan for itself (16 KB of lengths from L2 at 4096
// requests) instead of waiting for another CTA's, keeps both sums in shared
// memory, and takes a contiguous share of the rows and of the granted pages,
// each located by binary search.  Where a result is an input's own buffer (a
// step in place), the CTA that draws the last ticket writes the results, when
// every other one has read the inputs; else the first CTA does, without a ticket.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4.cuh"

namespace gsvk {

namespace {

constexpr int kPlanThreads = 1024;
constexpr size_t kPlanMaxSeq = 16384;
// Rows one CTA maps before another is launched: 4,096 requests, 260,000 rows, take 7.2 us, with 512 rows 7.4, with 2,048
// 9.0 and with 8,192 18.5; a step of 64 rows, one CTA either way, 3.9.
constexpr int kPlanRowsPerCta = 256;

struct PlanArgs {
  int n_seq, max_blocks, n_pages, page_shift;
  long long max_tokens;
  const int32_t* ctx;
  const int32_t* add;
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* q_start;
  int32_t* kv_len;
  int64_t* slots;
  int32_t* free_left;
  int32_t* refused;
  int32_t* ticket;
  int in_place;  // kv_len or free_left is an input too
};

__device__ __forceinline__ long long warp_incl_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Exclusive block-wide prefixes of N values (kPlanThreads threads); total receives the sums.
template <int N>
__device__ __forceinline__ void block_excl_scan(long long* v, long long (*sh)[32], long long* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long inc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) inc[k] = warp_incl_scan(v[k], lane);
  __syncthreads();  // sh is free again
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (lane == 31) sh[k][warp] = inc[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const long long w = warp_incl_scan(sh[k][lane], lane);  // 32 warps: every warp scans their sums
    total[k] = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    v[k] = inc[k] - v[k] + (warp ? before : 0);
  }
}

// The last i in [0, n) with start[i] <= x (start ascending, start[0] = 0); of
// equal starts the last, so requests without rows or pages are stepped over.
__device__ __forceinline__ int find_owner(const int32_t* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// What request i adds and needs.  Lengths are clamped before any sum, so no
// input overflows one: rows past max_tokens are worth max_tokens + 1.
struct Need {
  long long rows;
  int pages;
  bool valid;
};
__device__ __forceinline__ Need need_of(const PlanArgs& a, int i) {
  Need r{0, 0, true};
  const int c = a.ctx[i], n = a.add[i];
  r.rows = n > 0 ? n : 0;
  const long long end = static_cast<long long>(c) + n;
  r.valid = c >= 0 && n >= 0 && end <= (static_cast<long long>(a.max_blocks) << a.page_shift);
  if (r.valid) {
    const int p = (1 << a.page_shift) - 1;
    r.pages = static_cast<int>(((end + p) >> a.page_shift) - ((static_cast<long long>(c) + p) >> a.page_shift));
  }
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* s_row = plan_smem;             // [n_seq + 1] first row (clamped to max_tokens + 1)
  int32_t* s_page = plan_smem + a.n_seq + 1;  // [n_seq] pages before; bitwise not of it: refused
  __shared__ long long sh[2][32];
  __shared__ int s_last, s_refused, s_taken;
  const int tid = threadIdx.x;
  const int per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * per, a.n_seq), i1 = min(i0 + per, a.n_seq);
  const int free_count = min(max(*a.free_count, 0), a.n_pages);
  if (tid == 0) s_refused = s_taken = 0;

  long long before[2] = {0, 0}, total[2];  // rows, pages
  for (int i = i0; i < i1; ++i) {
    const Need q = need_of(a, i);
    before[0] += q.rows;
    before[1] += q.pages;
  }
  block_excl_scan<2>(before, sh, total);
  const long long cap = a.max_tokens, total_rows = total[0];
  long long row = before[0], page = before[1];
  if (total_rows > cap) {  // those that end past the last row need no pages: their sum again, without them
    long long r = row, pages = 0;
    for (int i = i0; i < i1; ++i) {
      const Need q = need_of(a, i);
      r += q.rows;
      if (r <= cap) pages += q.pages;
    }
    block_excl_scan<1>(&pages, sh, total);
    page = pages;
  }
  int refused = 0, taken = 0;
  for (int i = i0; i < i1; ++i) {
    const Need q = need_of(a, i);
    s_row[i] = static_cast<int>(min(row, cap + 1));
    row += q.rows;
    const int need = row <= cap ? q.pages : 0;
    const bool ok = q.valid && row <= cap && (need == 0 || page + need <= free_count);
    const int first = static_cast<int>(min(page, static_cast<long long>(free_count)));
    s_page[i] = ok ? first : ~first;
    page += need;
    if (!ok) ++refused;
    if (ok && need) taken = static_cast<int>(page);  // granted ones are those before the first shortage
  }
  refused = __reduce_add_sync(0xffffffffu, refused);
  taken = __reduce_max_sync(0xffffffffu, taken);
  if ((tid & 31) == 0) {  // s_refused and s_taken were set before the sums' barriers
    if (refused) atomicAdd(&s_refused, refused);
    atomicMax(&s_taken, taken);
  }
  if (tid == 0) s_row[a.n_seq] = static_cast<int>(min(total_rows, cap + 1));
  __syncthreads();

  const int live_rows = static_cast<int>(min(total_rows, cap));
  const int mask = (1 << a.page_shift) - 1;
  const long long gt = static_cast<long long>(gridDim.x) * kPlanThreads;
  const long long g0 = static_cast<long long>(blockIdx.x) * kPlanThreads + tid;
  for (long long t = g0; t < a.max_tokens; t += gt) {
    int64_t slot = -1;
    if (t < live_rows) {
      const int i = find_owner(s_row, a.n_seq, static_cast<int>(t));
      const int before = s_page[i];
      if (before >= 0) {
        const int c = a.ctx[i];
        const int pos = c + static_cast<int>(t) - s_row[i];
        const int blk = pos >> a.page_shift;
        const int have = (c + mask) >> a.page_shift;
        const int page = blk < have
                             ? a.table[static_cast<size_t>(i) * a.max_blocks + blk]
                             : a.free_pages[free_count - 1 - (before + blk - have)];
        if (page >= 0 && page < a.n_pages)
          slot = (static_cast<int64_t>(page) << a.page_shift) + (pos & mask);
      }
    }
    a.slots[t] = slot;
  }
  // the granted pages into the table: a warp to a request
  for (int i = static_cast<int>(blockIdx.x) * (kPlanThreads / 32) + (tid >> 5); i < a.n_seq;
       i += static_cast<int>(gridDim.x) * (kPlanThreads / 32)) {
    const int before = s_page[i];
    if (before < 0) continue;
    const int c = a.ctx[i];
    const int have = (c + mask) >> a.page_shift;
    const int end = (c + a.add[i] + mask) >> a.page_shift;
    for (int b = have + (tid & 31); b < end; b += 32)
      a.table[static_cast<size_t>(i) * a.max_blocks + b] =
          a.free_pages[free_count - 1 - (before + b - have)];
  }

  if (!a.in_place) {
    if (blockIdx.x != 0) return;
  } else if (gridDim.x > 1) {
    __syncthreads();  // this CTA has read its lengths and the free count
    if (tid == 0) {
      __threadfence();
      s_last = atomicAdd(a.ticket, 1) == static_cast<int>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!s_last) return;
  } else {
    __syncthreads();
  }
  for (int i = tid; i < a.n_seq; i += kPlanThreads) {
    const int c = a.ctx[i];
    a.q_start[i] = s_row[i];
    a.kv_len[i] = s_page[i] >= 0 ? c + a.add[i] : max(c, 0);
  }
  if (tid == 0) {
    a.q_start[a.n_seq] = s_row[a.n_seq];
    *a.free_left = free_count - s_taken;
    *a.refused = s_refused;
    if (a.in_place && gridDim.x > 1) *a.ticket = 0;
  }
}

// One CTA: the places of the returned pages are a prefix sum over the
// requests.  A warp walks a request's row 32 entries at a time, once to count
// and once to move.
__global__ void __launch_bounds__(kPlanThreads)
    kv_release_kernel(int n_seq, int max_blocks, int n_pages, int page_shift,
                      const int32_t* __restrict__ done, int32_t* __restrict__ len,
                      int32_t* __restrict__ table, int32_t* __restrict__ free_pages,
                      int32_t* __restrict__ free_count) {
  extern __shared__ int32_t rel_smem[];  // [n_seq] pages returned, then their first place
  __shared__ long long sh[1][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mask = (1 << page_shift) - 1;
  const int count = min(max(*free_count, 0), n_pages);
  const auto blocks_of = [&](int i) {
    const int n = done[i] ? max(len[i], 0) : 0;
    return static_cast<int>(
        min((static_cast<long long>(n) + mask) >> page_shift, static_cast<long long>(max_blocks)));
  };
  for (int i = warp; i < n_seq; i += kPlanThreads / 32) {
    const int n = blocks_of(i);
    const int32_t* row = table + static_cast<size_t>(i) * max_blocks;
    int found = 0;
    for (int b = 0; b < n; b += 32) {
      const int page = b + lane < n ? row[b + lane] : -1;
      found += __popc(__ballot_sync(0xffffffffu, page >= 0 && page < n_pages));
    }
    if (lane == 0) rel_smem[i] = found;
  }
  __syncthreads();
  const int per = (n_seq + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * per, n_seq), i1 = min(i0 + per, n_seq);
  long long mine = 0, total;
  for (int i = i0; i < i1; ++i) mine += rel_smem[i];
  block_excl_scan<1>(&mine, sh, &total);
  long long at = count + mine;
  for (int i = i0; i < i1; ++i) {
    const int found = rel_smem[i];
    rel_smem[i] = static_cast<int>(min(at, static_cast<long long>(n_pages)));
    at += found;
  }
  __syncthreads();
  for (int i = warp; i < n_seq; i += kPlanThreads / 32) {
    const int n = blocks_of(i);
    int32_t* row = table + static_cast<size_t>(i) * max_blocks;
    unsigned to = static_cast<unsigned>(rel_smem[i]);  // up to n_pages and a row more: past 2^31 - 1
    for (int b = 0; b < n; b += 32) {
      const int page = b + lane < n ? row[b + lane] : -1;
      const bool ok = page >= 0 && page < n_pages;
      const unsigned m = __ballot_sync(0xffffffffu, ok);
      const unsigned place = to + __popc(m & ((1u << lane) - 1u));
      if (ok && place < static_cast<unsigned>(n_pages)) free_pages[place] = page;
      if (b + lane < n) row[b + lane] = -1;
      to += __popc(m);
    }
    __syncwarp();  // every lane has read len[i]
    if (lane == 0 && done[i]) len[i] = 0;
  }
  if (tid == 0) *free_count = static_cast<int>(min(count + total, static_cast<long long>(n_pages)));
}

}  // namespace
}  // namespace gsvk

using namespace gsvk;

extern "C" {

int gsvk_kv_plan(const gsvk_kv_plan_args* g, gsvk_stream_t stream) {
  if (!g || !g->ctx_len || !g->new_len || !g->block_table || !g->free_pages || !g->free_count ||
      !g->q_start || !g->kv_len || !g->slots || !g->free_left || !g->refused || !g->workspace)
    return fail(GSVK_ERR_INVALID, "kv_plan: null pointer");
  if (g->n_seq == 0 || g->max_blocks == 0 || g->n_pages == 0 || g->max_tokens == 0)
    return fail(GSVK_ERR_INVALID, "kv_plan: zero size");
  const int shift = kv4_page_shift(g->page_size);
  if (shift < 0) return fail(GSVK_ERR_UNSUPPORTED, "kv_plan: page size %d", g->page_size);
  if (g->n_seq > kPlanMaxSeq || g->n_pages > 0x7fffffff || g->max_tokens > 0x7ffffffe ||
      g->max_blocks > (0x7fffff00u >> shift))  // positions rounded up to a page stay below 2^31
    return fail(GSVK_ERR_UNSUPPORTED, "kv_plan: too many requests, pages or tokens");
  PlanArgs a{static_cast<int>(g->n_seq), static_cast<int>(g->max_blocks),
             static_cast<int>(g->n_pages), shift, static_cast<long long>(g->max_tokens),
             g->ctx_len, g->new_len, g->block_table, g->free_pages, g->free_count, g->q_start,
             g->kv_len, g->slots, g->free_left, g->refused, g->workspace,
             g->kv_len == g->ctx_len || g->kv_len == g->new_len || g->free_left == g->free_count};
  const size_t smem = 2 * (g->n_seq + 1) * sizeof(int32_t);
  if (smem > 48 * 1024)
    if (int rc = check_cuda(cudaFuncSetAttribute(kv_plan_kernel,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)),
                            "cudaFuncSetAttribute(kv_plan)"))
      return rc;
  const unsigned grid = std::max(1u, std::min<unsigned>(ceil_div(g->max_tokens, kPlanRowsPerCta),
                                                        static_cast<unsigned>(sm_count())));
  kv_plan_kernel<<<grid, kPlanThreads, smem, as_cuda(stream)>>>(a);
  return check_launch("kv_plan_kernel");
}

int gsvk_kv_release(size_t n_seq, size_t max_blocks, size_t n_pages, int page_size,
                    const int32_t* done, int32_t* len, int32_t* block_table, int32_t* free_pages,
                    int32_t* free_count, gsvk_stream_t stream) {
  if (!done || !len || !block_table || !free_pages || !free_count)
    return fail(GSVK_ERR_INVALID, "kv_release: null pointer");
  if (n_seq == 0 || max_blocks == 0 || n_pages == 0)
    return fail(GSVK_ERR_INVALID, "kv_release: zero size");
  const int shift = kv4_page_shift(page_size);
  if (shift < 0) return fail(GSVK_ERR_UNSUPPORTED, "kv_release: page size %d", page_size);
  if (n_seq > kPlanMaxSeq || n_pages > 0x7fffffff || max_blocks > (0x7fffff00u >> shift))
    return fail(GSVK_ERR_UNSUPPORTED, "kv_release: too many requests or pages");
  const size_t smem = n_seq * sizeof(int32_t);
  if (smem > 48 * 1024)
    if (int rc = check_cuda(cudaFuncSetAttribute(kv_release_kernel,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)),
                            "cudaFuncSetAttribute(kv_release)"))
      return rc;
  kv_release_kernel<<<1, kPlanThreads, smem, as_cuda(stream)>>>(
      static_cast<int>(n_seq), static_cast<int>(max_blocks), static_cast<int>(n_pages), shift, done,
      len, block_table, free_pages, free_count);
  return check_launch("kv_release_kernel");
}

}  // extern "C"
