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

// The host's check of a cache handed over the C ABI; GSVK_OK or an error.
int kv4_check(const gsvk_kv4_cache* c, const char* who);

}  // namespace gsvk
