// gemm_i8.cu — row quantiser and matrix product in 8-bit integers with scales
// per row of A (token) and of B (output channel): gsvk_quantize_rows_i8,
// gsvk_gemm_i8.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "tma.cuh"

namespace gsvk {

namespace {

// ------------------------------------------------------------ row quantiser
__device__ __forceinline__ float as_f32(uint16_t v) { return h2f(v); }
__device__ __forceinline__ float as_f32(float v) { return v; }

// One warp per row: the maximum, then the codes (the row is in L1 by then).
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T* __restrict__ x, size_t ldx, long long rows, int n,
                         int8_t* __restrict__ q, size_t ldq, float* __restrict__ scale) {
  const long long r = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  const T* xr = x + r * ldx;
  float top = 0.f;
  bool bad = false;
  for (int i = lane; i < n; i += 32) {
    const float v = fabsf(as_f32(xr[i]));
    bad |= !(v <= 3.402823466e38f);
    top = fmaxf(top, v);
  }
  top = warp_max(top);
  bad = __any_sync(0xffffffffu, bad);
  const float s = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(top, 127.f);
  for (int i = lane; i < n; i += 32)
    q[r * ldq + i] = s > 0.f ? static_cast<int8_t>(rintf(__fdiv_rn(as_f32(xr[i]), s))) : 0;
  if (lane == 0) scale[r] = s;
}

// ----------------------------------------------------------------- products
struct I8Epilogue {
  const float* a_scale;
  const float* b_scale;
  const float* bias;
  const float* residual;
  float* c32;
  uint16_t* c16;
  long long ld_res, ld_c32, ld_c16;
  int act;
  float slope;
};

__device__ __forceinline__ float i8_value(int acc, float sa, float sb, float bias, const I8Epilogue& e) {
  return apply_act(fmaf(static_cast<float>(acc), sa * sb, bias), e.act, e.slope);
}

// Operands in any layout: one thread to an output, bytes in order.
__global__ void __launch_bounds__(256)
    gemm_i8_simt_kernel(const int8_t* __restrict__ a, long long lda, const int8_t* __restrict__ b,
                        long long ldb, long long M, int N, int K, const I8Epilogue e) {
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long m = at / N;
  const int n = static_cast<int>(at - m * N);
  if (m >= M) return;
  int acc = 0;
  for (int k = 0; k < K; ++k)
    acc += static_cast<int>(a[m * lda + k]) * static_cast<int>(b[n * ldb + k]);
  float y = i8_value(acc, e.a_scale[m], e.b_scale[n], e.bias ? e.bias[n] : 0.f, e);
  if (e.residual) y += e.residual[m * e.ld_res + n];
  if (e.c32) e.c32[m * e.ld_c32 + n] = y;
  if (e.c16) e.c16[m * e.ld_c16 + n] = f2h(y);
}

}  // namespace
}  // namespace gsvk

using namespace gsvk;

extern "C" {

int gsvk_quantize_rows_i8(const void* x, int is_f32, size_t rows, size_t n, size_t ldx, int8_t* q,
                          size_t ldq, float* scale, gsvk_stream_t stream) {
  if (rows == 0) return GSVK_OK;
  if (!x || !q || !scale || n == 0) return fail(GSVK_ERR_INVALID, "quantize_rows_i8: null pointer or empty row");
  if (!ldx) ldx = n;
  if (!ldq) ldq = n;
  if (rows > 1 && (ldx < n || ldq < n)) return fail(GSVK_ERR_INVALID, "quantize_rows_i8: leading dimension below %zu", n);
  if (n > 0x7fffffc0 || rows > 0x7fffffff) return fail(GSVK_ERR_UNSUPPORTED, "quantize_rows_i8: too big");
  const unsigned blocks = ceil_div(rows, 8);
  if (is_f32)
    quantize_rows_kernel<<<blocks, 256, 0, as_cuda(stream)>>>(static_cast<const float*>(x), ldx, rows, (int)n, q, ldq, scale);
  else
    quantize_rows_kernel<<<blocks, 256, 0, as_cuda(stream)>>>(static_cast<const uint16_t*>(x), ldx, rows, (int)n, q, ldq, scale);
  return check_launch("quantize_rows_kernel");
}

int gsvk_gemm_i8(const gsvk_gemm_i8_args* g, gsvk_stream_t stream) {
  if (g && g->M == 0) return GSVK_OK;
  if (!g || !g->a || !g->b || !g->a_scale || !g->b_scale || (!g->c && !g->c_f16))
    return fail(GSVK_ERR_INVALID, "gemm_i8: null pointer");
  if (g->N == 0 || g->K == 0) return fail(GSVK_ERR_INVALID, "gemm_i8: zero size");
  if (g->M > 0x7fffff00 || g->N > 0x7fffff00 || g->K >= 131072)
    return fail(GSVK_ERR_UNSUPPORTED, "gemm_i8: %zu x %zu x %zu (K below 131072: 32-bit sums)", g->M, g->N, g->K);
  const size_t lda = g->lda ? g->lda : g->K, ldb = g->ldb ? g->ldb : g->K;
  const size_t ldc = g->ldc ? g->ldc : g->N, ldh = g->ldc_f16 ? g->ldc_f16 : g->N;
  const size_t ldr = g->ld_res ? g->ld_res : g->N;
  if ((g->M > 1 && lda < g->K) || (g->N > 1 && ldb < g->K) || (g->M > 1 && (ldc < g->N || ldh < g->N || ldr < g->N)))
    return fail(GSVK_ERR_INVALID, "gemm_i8: a leading dimension is below its row");
  if (g->act < GSVK_ACT_NONE || g->act > GSVK_ACT_TANH) return fail(GSVK_ERR_INVALID, "gemm_i8: bad act");
  I8Epilogue e{g->a_scale, g->b_scale, g->bias, g->residual, g->c, g->c_f16,
               (long long)ldr, (long long)ldc, (long long)ldh, g->act, g->slope};
  const size_t outs = g->M * g->N;
  if (ceil_div(outs, 256) > 0x7fffffff) return fail(GSVK_ERR_UNSUPPORTED, "gemm_i8: too big");
  gemm_i8_simt_kernel<<<ceil_div(outs, 256), 256, 0, as_cuda(stream)>>>(
      g->a, (long long)lda, g->b, (long long)ldb, (long long)g->M, (int)g->N, (int)g->K, e);
  return check_launch("gemm_i8_simt_kernel");
}

}  // extern "C"
