// kv4_attn.cuh — what the kernels of the 4-bit cache's attention share.
#pragma once

#include "kv4.cuh"
#include "tma.cuh"

namespace gsvk {

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
  int* tickets;      // of the items that several warps share
  float* parts;      // their records
  uint32_t* status;
  int most_rows;     // rows of a request (to a kv head) that the few-row kernel takes
};

// One request's rows and the keys they see.
struct Request {
  int q0, n, len, prefix;
};
__device__ __forceinline__ Request request_of(const AttnArgs& a, int s) {
  Request r;
  r.q0 = a.q_start[s];
  r.n = min(a.q_start[s + 1], a.n_tokens) - r.q0;
  if (r.q0 < 0) r.n = 0;
  r.len = a.kv_len[s];
  r.prefix = a.prefix ? a.prefix[s] : 0;
  return r;
}
// Keys that query row `row` of a request's kv head sees (64-bit on the way: lengths are the caller's).
__device__ __forceinline__ int limit_of(const AttnArgs& a, const Request& q, int row) {
  const int r = q.n == 1 || a.group == 1 ? (q.n == 1 ? 0 : row) : row / a.group;
  const long long causal = static_cast<long long>(q.len) - q.n + r + 1;
  const long long see = max(causal, static_cast<long long>(q.prefix));
  const long long have = min(q.len, a.max_blocks << a.shift);
  return static_cast<int>(max(0LL, min(see, have)));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Where query row `row` of a request's kv head goes.
__device__ __forceinline__ uint16_t* out_row(const AttnArgs& a, const Request& rq, int head, int row, int hd) {
  const int r = rq.n == 1 ? 0 : row / a.group;
  return a.out + static_cast<size_t>(rq.q0 + r) * a.out_stride +
         static_cast<size_t>(head * a.group + row - r * a.group) * hd;
}

// Attention of the requests with more than a.most_rows rows to a kv head (kv4_prompt.cu).
int kv4_prompt_run(const AttnArgs& a, int head_dim, cudaStream_t st);

}  // namespace gsvk
