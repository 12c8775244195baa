// kv4.cuh — the paged 4-bit KV cache as its kernels see it (layout and value
// rules: include/gsvk.h).
#pragma once

#include "common.cuh"

namespace gsvk {

// log2 of a supported page size, -1 for another.
inline int kv4_page_shift(int page_size) {
  return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}

// Byte offsets within one kv head's part of a page of 2^shift tokens.
__host__ __device__ __forceinline__ int kv4_head_bytes(int shift, int hd) { return (hd + 8) << shift; }
__host__ __device__ __forceinline__ int kv4_v_codes(int shift, int hd) { return (hd >> 1) << shift; }
__host__ __device__ __forceinline__ int kv4_k_par(int shift, int hd) { return hd << shift; }
__host__ __device__ __forceinline__ int kv4_v_par(int shift, int hd) { return (hd + 4) << shift; }

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ float2 unpair(uint64_t d) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(d));
  return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The host's check of a cache handed over the C ABI; GSVK_OK or an error.
int kv4_check(const gsvk_kv4_cache* c, const char* who);

}  // namespace gsvk
