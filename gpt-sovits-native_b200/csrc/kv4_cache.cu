// kv4_cache.cu — rows into and out of the paged 4-bit KV cache
// (gsvk_kv4_append, gsvk_kv4_read; the value rules are in include/gsvk.h).
//
// Both are one pass over the data: append reads K and V once (4 head_dim
// bytes per token and head in fp16) and writes head_dim + 8, read the
// reverse, so HBM bounds them at length and launch latency at a decode step.
// A row (one token, one head) is spread over head_dim / 8 lanes with 8
// values, one 16-byte load and one 32-bit word of codes each: its extremes
// are a butterfly over those lanes, loads are whole contiguous warps of the
// input, and codes leave as runs of head_dim / 2 bytes.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4.cuh"

namespace gsvk {

int kv4_check(const gsvk_kv4_cache* c, const char* who) {
  if (!c || !c->pages || c->n_pages == 0) return fail(GSVK_ERR_INVALID, "%s: empty cache", who);
  if (gsvk_kv4_page_bytes(c->page_size, c->kv_heads, c->head_dim) == 0)
    return fail(GSVK_ERR_UNSUPPORTED, "%s: page size %d, %d kv heads of %d", who, c->page_size,
                c->kv_heads, c->head_dim);
  if (c->n_pages > 0x7fffffff) return fail(GSVK_ERR_UNSUPPORTED, "%s: too many pages", who);
  if (!aligned16(c->pages)) return fail(GSVK_ERR_ALIGN, "%s: pages not 16-byte aligned", who);
  return GSVK_OK;
}

namespace {

constexpr int kRowThreads = 256;

struct RowArgs {
  uint8_t* pages;
  long long n_slots;  // pages * page size
  size_t page_bytes;
  int shift, heads;
  const int64_t* slots;
  long long rows;  // tokens * heads
};

// 8 values of a row as fp32.
__device__ __forceinline__ void load8(const uint16_t* p, float* f) {
  unpack8(ld_stream_u4(p), f);
}
__device__ __forceinline__ void load8(const float* p, float* f) {
  const uint4 a = ld_stream_u4(p), b = ld_stream_u4(p + 4);
  f[0] = __uint_as_float(a.x);
  f[1] = __uint_as_float(a.y);
  f[2] = __uint_as_float(a.z);
  f[3] = __uint_as_float(a.w);
  f[4] = __uint_as_float(b.x);
  f[5] = __uint_as_float(b.y);
  f[6] = __uint_as_float(b.z);
  f[7] = __uint_as_float(b.w);
}

// Codes of 8 of a row's values (spread over L lanes) and its parameters.
template <int L>
__device__ __forceinline__ uint32_t quantise8(const float* x, uint32_t* par) {
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad |= !(fabsf(x[i]) < 65520.f);  // NaN, infinite, or rounds to an fp16 infinity
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad |= __shfl_xor_sync(0xffffffffu, bad, o) != 0;
  }
  const uint16_t low16 = f2h(lo), step16 = f2h(__fdiv_rn(hi - lo, 15.f));
  const float low = h2f(low16), step = h2f(step16);
  uint32_t w = 0;
  if (step > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = rintf(__fdiv_rn(x[i] - low, step));
      w |= static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f)) << (4 * i);
    }
  }
  *par = step16 | static_cast<uint32_t>(low16) << 16;
  if (bad) {
    w = 0;
    *par = 0x7fff7fffu;  // NaN, NaN
  }
  return w;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kRowThreads)
    kv4_append_kernel(const RowArgs a, const T* __restrict__ k, size_t k_stride,
                      const T* __restrict__ v, size_t v_stride) {
  constexpr int L = HD / 8;
  const long long row = (static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  // a warp's lanes all shuffle: those past the end repeat the last row and write nothing
  const long long r = min(row, a.rows - 1);
  const long long t = r / a.heads;
  const int h = static_cast<int>(r - t * a.heads);
  float xk[8], xv[8];
  load8(k + t * k_stride + static_cast<size_t>(h) * HD + part * 8, xk);
  load8(v + t * v_stride + static_cast<size_t>(h) * HD + part * 8, xv);
  const int64_t slot = a.slots[t];
  uint32_t pk, pv;
  const uint32_t wk = quantise8<L>(xk, &pk);
  const uint32_t wv = quantise8<L>(xv, &pv);
  if (row >= a.rows || slot < 0 || slot >= a.n_slots) return;
  const int at = static_cast<int>(slot & ((1 << a.shift) - 1));
  uint8_t* b = a.pages + static_cast<size_t>(slot >> a.shift) * a.page_bytes +
               static_cast<size_t>(h) * kv4_head_bytes(a.shift, HD);
  *reinterpret_cast<uint32_t*>(b + at * (HD / 2) + part * 4) = wk;
  *reinterpret_cast<uint32_t*>(b + kv4_v_codes(a.shift, HD) + at * (HD / 2) + part * 4) = wv;
  if (part == 0) {
    *reinterpret_cast<uint32_t*>(b + kv4_k_par(a.shift, HD) + at * 4) = pk;
    *reinterpret_cast<uint32_t*>(b + kv4_v_par(a.shift, HD) + at * 4) = pv;
  }
}

// The top level may lie above fp16's range (a step rounded up): held at its
// greatest value.  NaN passes.
__device__ __forceinline__ float in_range(float x) {
  return fabsf(x) > 65504.f ? copysignf(65504.f, x) : x;
}
// 8 codes -> fp16 values, rounded once.
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t par) {
  const float step = h2f(static_cast<uint16_t>(par)), low = h2f(static_cast<uint16_t>(par >> 16));
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = f2h2(in_range(fmaf(step, static_cast<float>((w >> (8 * i)) & 15u), low)),
                in_range(fmaf(step, static_cast<float>((w >> (8 * i + 4)) & 15u), low)));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int HD>
__global__ void __launch_bounds__(kRowThreads)
    kv4_read_kernel(const RowArgs a, uint16_t* __restrict__ k, size_t k_stride,
                    uint16_t* __restrict__ v, size_t v_stride) {
  constexpr int L = HD / 8;
  const long long r = (static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  if (r >= a.rows) return;
  const long long t = r / a.heads;
  const int h = static_cast<int>(r - t * a.heads);
  const int64_t slot = a.slots[t];
  uint4 yk = make_uint4(0, 0, 0, 0), yv = yk;
  if (slot >= 0 && slot < a.n_slots) {
    const int at = static_cast<int>(slot & ((1 << a.shift) - 1));
    const uint8_t* b = a.pages + static_cast<size_t>(slot >> a.shift) * a.page_bytes +
                       static_cast<size_t>(h) * kv4_head_bytes(a.shift, HD);
    const uint32_t wk = *reinterpret_cast<const uint32_t*>(b + at * (HD / 2) + part * 4);
    const uint32_t wv = *reinterpret_cast<const uint32_t*>(b + kv4_v_codes(a.shift, HD) +
                                                           at * (HD / 2) + part * 4);
    yk = values8(wk, *reinterpret_cast<const uint32_t*>(b + kv4_k_par(a.shift, HD) + at * 4));
    yv = values8(wv, *reinterpret_cast<const uint32_t*>(b + kv4_v_par(a.shift, HD) + at * 4));
  }
  if (k) *reinterpret_cast<uint4*>(k + t * k_stride + static_cast<size_t>(h) * HD + part * 8) = yk;
  if (v) *reinterpret_cast<uint4*>(v + t * v_stride + static_cast<size_t>(h) * HD + part * 8) = yv;
}

// Checks and fills what append and read share; *blocks receives the grid.
int row_args(const gsvk_kv4_cache* c, const int64_t* slots, size_t n_tokens, const char* who,
             RowArgs* a, unsigned* blocks) {
  if (int rc = kv4_check(c, who)) return rc;
  if (!slots && n_tokens) return fail(GSVK_ERR_INVALID, "%s: null slots", who);
  const size_t lanes = static_cast<size_t>(c->head_dim) / 8;
  if (n_tokens > 0x7fffffff ||
      n_tokens * c->kv_heads * lanes > static_cast<size_t>(0x7fffffff) * kRowThreads)
    return fail(GSVK_ERR_UNSUPPORTED, "%s: too many tokens", who);
  a->pages = c->pages;
  a->shift = kv4_page_shift(c->page_size);
  a->n_slots = static_cast<long long>(c->n_pages) << a->shift;
  a->page_bytes = gsvk_kv4_page_bytes(c->page_size, c->kv_heads, c->head_dim);
  a->heads = c->kv_heads;
  a->slots = slots;
  a->rows = static_cast<long long>(n_tokens) * c->kv_heads;
  *blocks = ceil_div(static_cast<size_t>(a->rows) * lanes, kRowThreads);
  return GSVK_OK;
}

template <typename T>
int append_run(const RowArgs& a, int hd, const void* k, size_t ks, const void* v, size_t vs,
               unsigned blocks, cudaStream_t st) {
  const T* kt = static_cast<const T*>(k);
  const T* vt = static_cast<const T*>(v);
  if (hd == 32) kv4_append_kernel<32><<<blocks, kRowThreads, 0, st>>>(a, kt, ks, vt, vs);
  if (hd == 64) kv4_append_kernel<64><<<blocks, kRowThreads, 0, st>>>(a, kt, ks, vt, vs);
  if (hd == 128) kv4_append_kernel<128><<<blocks, kRowThreads, 0, st>>>(a, kt, ks, vt, vs);
  return check_launch("kv4_append_kernel");
}

}  // namespace
}  // namespace gsvk

using namespace gsvk;

extern "C" {

size_t gsvk_kv4_page_bytes(int page_size, int kv_heads, int head_dim) {
  const int shift = kv4_page_shift(page_size);
  if (shift < 0 || kv_heads < 1 || kv_heads > 1024 ||
      (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return 0;
  return static_cast<size_t>(kv_heads) * kv4_head_bytes(shift, head_dim);
}

int gsvk_kv4_append(const gsvk_kv4_cache* c, const void* k, size_t k_stride, const void* v,
                    size_t v_stride, int is_f32, const int64_t* slots, size_t n_tokens,
                    gsvk_stream_t stream) {
  RowArgs a;
  unsigned blocks = 0;
  if (int rc = row_args(c, slots, n_tokens, "kv4_append", &a, &blocks)) return rc;
  if (n_tokens == 0) return GSVK_OK;
  if (!k || !v) return fail(GSVK_ERR_INVALID, "kv4_append: null rows");
  const size_t unit = is_f32 ? 4 : 8, width = static_cast<size_t>(c->kv_heads) * c->head_dim;
  if (n_tokens > 1 && (k_stride < width || v_stride < width))
    return fail(GSVK_ERR_INVALID, "kv4_append: row stride below %zu", width);
  if (!aligned16(k) || !aligned16(v) || k_stride % unit || v_stride % unit)
    return fail(GSVK_ERR_ALIGN, "kv4_append: rows not in whole 16 bytes");
  return is_f32 ? append_run<float>(a, c->head_dim, k, k_stride, v, v_stride, blocks, as_cuda(stream))
                : append_run<uint16_t>(a, c->head_dim, k, k_stride, v, v_stride, blocks,
                                       as_cuda(stream));
}

int gsvk_kv4_read(const gsvk_kv4_cache* c, const int64_t* slots, size_t n_tokens, uint16_t* k,
                  size_t k_stride, uint16_t* v, size_t v_stride, gsvk_stream_t stream) {
  RowArgs a;
  unsigned blocks = 0;
  if (int rc = row_args(c, slots, n_tokens, "kv4_read", &a, &blocks)) return rc;
  if (n_tokens == 0) return GSVK_OK;
  if (!k && !v) return fail(GSVK_ERR_INVALID, "kv4_read: no output");
  const size_t width = static_cast<size_t>(c->kv_heads) * c->head_dim;
  if (n_tokens > 1 && ((k && k_stride < width) || (v && v_stride < width)))
    return fail(GSVK_ERR_INVALID, "kv4_read: row stride below %zu", width);
  if ((k && (!aligned16(k) || k_stride % 8)) || (v && (!aligned16(v) || v_stride % 8)))
    return fail(GSVK_ERR_ALIGN, "kv4_read: rows not in whole 16 bytes");
  cudaStream_t st = as_cuda(stream);
  if (c->head_dim == 32) kv4_read_kernel<32><<<blocks, kRowThreads, 0, st>>>(a, k, k_stride, v, v_stride);
  if (c->head_dim == 64) kv4_read_kernel<64><<<blocks, kRowThreads, 0, st>>>(a, k, k_stride, v, v_stride);
  if (c->head_dim == 128)
    kv4_read_kernel<128><<<blocks, kRowThreads, 0, st>>>(a, k, k_stride, v, v_stride);
  return check_launch("kv4_read_kernel");
}

}  // extern "C"
