// kv4_cache.cu — rows into and out of the paged 4-bit KV cache
// (gsvk_kv4_append, gsvk_kv4_read; the value rules are in include/gsvk.h).
//
// Both are one pass over the data: append reads K and V once (4 head_dim
// bytes per token and head in fp16) and writes head_dim + 8, read the
// reverse.  30,566 tokens, 8 heads of 128: append takes 49.5 us (3.2 TB/s: 22 instructions a
// value fill 78 % of the issue slots), read 34.7 us (4.6 TB/s), one behind the other 82; of 64
// tokens, 16 heads of 32, 2.2, 1.8 and 4.0 us, launch latency.
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
  int tokens;
  int units;     // 16-byte units of a token's row: heads * head_dim / 8
  int per_block; // tokens of a CTA; where a token has more units than a CTA threads, gridDim.y CTAs share it
};
// This thread's token and unit within its row; false past either's end.
__device__ __forceinline__ bool place_of(const RowArgs& a, int* t, int* u) {
  const int k = static_cast<int>(threadIdx.x) / a.units;  // 0 where a token fills the CTA
  *t = static_cast<int>(blockIdx.x) * a.per_block + k;
  *u = static_cast<int>(threadIdx.x) - k * a.units + static_cast<int>(blockIdx.y) * kRowThreads;
  return k < a.per_block && *t < a.tokens && *u < a.units;
}

// 8 values of a row as fp32, and the extremes of the row, which is spread over L lanes.  A NaN makes both NaN.
template <int L>
__device__ __forceinline__ void load8(const uint16_t* p, float* f, float* lo, float* hi) {
  const uint4 v = ld_stream_u4(p);
  unpack8(v, f);
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const __half2 least = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
  const __half2 most = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  // the least value and the greatest, negated: one shuffle for both
  __half2 m = __hmin2_nan(__lows2half2(least, __hneg2(most)), __highs2half2(least, __hneg2(most)));
#pragma unroll
  for (int o = 1; o < L; o <<= 1) m = __hmin2_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  *lo = __low2float(m);
  *hi = -__high2float(m);
}
template <int L>
__device__ __forceinline__ void load8(const float* p, float* f, float* lo, float* hi) {
  const uint4 a = ld_stream_u4(p), b = ld_stream_u4(p + 4);
  f[0] = __uint_as_float(a.x);
  f[1] = __uint_as_float(a.y);
  f[2] = __uint_as_float(a.z);
  f[3] = __uint_as_float(a.w);
  f[4] = __uint_as_float(b.x);
  f[5] = __uint_as_float(b.y);
  f[6] = __uint_as_float(b.z);
  f[7] = __uint_as_float(b.w);
  float least = f[0], most = f[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    least = min_nan(least, f[i]);
    most = max_nan(most, f[i]);
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) {
    least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, o));
    most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  *lo = least;
  *hi = most;
}

// Codes of 8 of a row's values and its parameters.  HALF: fp16 values, of which none is below low.
template <bool HALF>
__device__ __forceinline__ uint32_t quantise8(const float* x, float lo, float hi, uint32_t* par) {
  const uint16_t low16 = f2h(lo), step16 = f2h(__fdiv_rn(hi - lo, 15.f));
  const float low = h2f(low16), step = h2f(step16);
  *par = step16 | static_cast<uint32_t>(low16) << 16;
  if (!(fmaxf(-lo, hi) < 65520.f) || lo != lo) {  // infinite, rounds to an fp16 infinity, or NaN
    *par = 0x7fff7fffu;                            // NaN, NaN
    return 0;
  }
  if (!(step > 0.f)) return 0;
  // (x - low) * (1 / step) is within 6e-6 of the quotient (where that is below 16: the others are clamped either way);
  // further than 1e-5 from a tie it rounds like the quotient, else the division itself is made.  A sum with 1.5 2^23 is
  // rounded to an integer, to even, with the code in its low bits.
  constexpr float kRound = 12582912.f;
  float per_step;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(per_step) : "f"(step));
  const uint64_t minus_low = pair(-low, -low), per2 = pair(per_step, per_step);
  const uint64_t up = pair(kRound, kRound), down = pair(-kRound, -kRound), minus = pair(-1.f, -1.f);
  float c[8], far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float2 q = unpair(mul2(add2(pair(x[i], x[i + 1]), minus_low), per2));
    if (!HALF) q = make_float2(fmaxf(q.x, 0.f), fmaxf(q.y, 0.f));
    const uint64_t q2 = pair(fminf(q.x, 15.f), fminf(q.y, 15.f)), c2 = add2(q2, up);
    const float2 off = unpair(fma2(add2(c2, down), minus, q2)), r = unpair(c2);
    c[i] = r.x;
    c[i + 1] = r.y;
    far = fmaxf(fmaxf(far, fabsf(off.x)), fabsf(off.y));
  }
  if (!(far < 0.49999f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = fminf(fmaxf(__fdiv_rn(x[i] - low, step), 0.f), 15.f) + kRound;
  }
  uint32_t w = 0, bits = 0;  // sums of the bits, less those of the eight 1.5 2^23
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w += __float_as_uint(c[i]) << (4 * i);
    bits += 0x4b400000u << (4 * i);
  }
  return w - bits;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kRowThreads)
    kv4_append_kernel(const RowArgs a, const T* __restrict__ k, size_t k_stride,
                      const T* __restrict__ v, size_t v_stride) {
  constexpr int L = HD / 8;
  int t, u;
  const bool there = place_of(a, &t, &u);
  if (!there) t = u = 0;  // all lanes shuffle: these repeat the first row and write nothing
  const int h = u / L, part = u % L;
  float xk[8], xv[8], lo_k, hi_k, lo_v, hi_v;
  load8<L>(k + t * k_stride + u * 8, xk, &lo_k, &hi_k);
  load8<L>(v + t * v_stride + u * 8, xv, &lo_v, &hi_v);
  const int64_t slot = a.slots[t];
  uint32_t pk, pv;
  const uint32_t wk = quantise8<sizeof(T) == 2>(xk, lo_k, hi_k, &pk);
  const uint32_t wv = quantise8<sizeof(T) == 2>(xv, lo_v, hi_v, &pv);
  if (!there || slot < 0 || slot >= a.n_slots) return;
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

// 8 codes -> fp16 values: step * code + low as one fused fp16 operation, rounded once.  The top level may
// lie above fp16's range (a step rounded up): held at its greatest value.  NaN passes.
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t par) {
  const __half2 p = *reinterpret_cast<const __half2*>(&par);
  const __half2 step = __low2half2(p), low = __high2half2(p);
  const __half2 top = __float2half2_rn(65504.f), bias = __float2half2_rn(1024.f);
  uint32_t y[4];  // values k and k + 4
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t c = (w >> (4 * k) & 0x000f000fu) | 0x64006400u;  // 1024 + code
    const __half2 v = __hmin2_nan(__hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), bias), step, low), top);
    y[k] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                    __byte_perm(y[2], y[3], 0x7632));
}

template <int HD>
__global__ void __launch_bounds__(kRowThreads)
    kv4_read_kernel(const RowArgs a, uint16_t* __restrict__ k, size_t k_stride,
                    uint16_t* __restrict__ v, size_t v_stride) {
  constexpr int L = HD / 8;
  int t, u;
  if (!place_of(a, &t, &u)) return;
  const int h = u / L, part = u % L;
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
  if (k) *reinterpret_cast<uint4*>(k + t * k_stride + u * 8) = yk;
  if (v) *reinterpret_cast<uint4*>(v + t * v_stride + u * 8) = yv;
}

// Checks and fills what append and read share; *grid receives the launch's.
int row_args(const gsvk_kv4_cache* c, const int64_t* slots, size_t n_tokens, const char* who,
             RowArgs* a, dim3* grid) {
  if (int rc = kv4_check(c, who)) return rc;
  if (!slots && n_tokens) return fail(GSVK_ERR_INVALID, "%s: null slots", who);
  if (n_tokens > 0x7fffffff) return fail(GSVK_ERR_UNSUPPORTED, "%s: too many tokens", who);
  a->pages = c->pages;
  a->shift = kv4_page_shift(c->page_size);
  a->n_slots = static_cast<long long>(c->n_pages) << a->shift;
  a->page_bytes = gsvk_kv4_page_bytes(c->page_size, c->kv_heads, c->head_dim);
  a->heads = c->kv_heads;
  a->slots = slots;
  a->tokens = static_cast<int>(n_tokens);
  a->units = c->kv_heads * (c->head_dim / 8);
  a->per_block = std::max(1, kRowThreads / a->units);
  *grid = dim3(ceil_div(n_tokens, a->per_block), ceil_div(a->units, kRowThreads));
  return GSVK_OK;
}

template <typename T>
int append_run(const RowArgs& a, int hd, const void* k, size_t ks, const void* v, size_t vs,
               dim3 blocks, cudaStream_t st) {
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
  dim3 blocks;
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
  dim3 blocks;
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
