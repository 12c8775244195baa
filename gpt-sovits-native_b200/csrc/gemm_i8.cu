// gemm_i8.cu — row quantiser and matrix product in 8-bit integers with scales
// per row of A (token) and of B (output channel): gsvk_quantize_rows_i8,
// gsvk_gemm_i8.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "tma.cuh"

namespace gsvk {

namespace {

// ------------------------------------------------------------ row quantiser
// Memory bounds it (3 bytes a value in fp16): a row's values are read once in
// 16-byte vectors, kept in registers between the maximum and the codes (kept in
// cache for rows longer than THREADS lanes hold), and leave 8 codes at a time.
// Short rows take a warp each, long ones a CTA.
__device__ __forceinline__ float as_f32(uint16_t v) { return h2f(v); }
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ void load8(const uint16_t* p, float* f) { unpack8(ld_stream_u4(p), f); }
__device__ __forceinline__ void load8(const float* p, float* f) {
  const uint4 a = ld_stream_u4(p), b = ld_stream_u4(p + 4);
  const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
}

// One code by division.  Where the scale is a few units of fp32's last place the quotient may pass 127.
__device__ __forceinline__ float code_of(float x, float s) { return fminf(fmaxf(__fdiv_rn(x, s), -127.f), 127.f); }
// 8 codes of a row with scale s > 0.  x * (1 / s) is within 1e-4 of the quotient (below 128): further than that from a tie
// it rounds like the quotient, else the division itself is made, as for a scale so small that its inverse is infinite.  A
// sum with 1.5 2^23 is rounded to an integer, to even, with the code as its low byte.
__device__ __forceinline__ uint2 codes8(const float* x, float s, float per_s) {
  constexpr float kRound = 12582912.f;
  float c[8], far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = x[i] * per_s;
    c[i] = q + kRound;
    far = fmaxf(far, fabsf(q - (c[i] - kRound)));
  }
  if (!(far < 0.4998f) || per_s > 3.0e38f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code_of(x[i], s) + kRound;
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(__float_as_uint(c[4 * i]), __float_as_uint(c[4 * i + 1]), 0x0040),
                       __byte_perm(__float_as_uint(c[4 * i + 2]), __float_as_uint(c[4 * i + 3]), 0x0040), 0x5410);
  return make_uint2(w[0], w[1]);
}

// THREADS threads to a row, 256 / THREADS rows to a CTA; KEEP: vectors of 8 that a thread keeps.  VEC: rows of whole vectors.
template <int THREADS, int KEEP, bool VEC, typename T>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T* __restrict__ x, size_t ldx, long long rows, int n, int8_t* __restrict__ q,
                         size_t ldq, float* __restrict__ scale) {
  __shared__ float s_top[8];
  const int tid = threadIdx.x % THREADS;
  const long long r = static_cast<long long>(blockIdx.x) * (256 / THREADS) + threadIdx.x / THREADS;
  if (r >= rows) return;  // whole warps
  griddep_wait();
  griddep_launch_dependents();
  const T* xr = x + r * ldx;
  int8_t* qr = q + r * ldq;
  const int whole = VEC ? n / 8 : 0;  // vectors; what is left is taken singly
  float kept[KEEP][8], top = 0.f;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int i = k * THREADS + tid;
    if (i < whole) {
      load8(xr + 8 * i, kept[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(kept[k][j]));
    }
  }
  for (int i = KEEP * THREADS + tid; i < whole; i += THREADS) {
    float f[8];
    load8(xr + 8 * i, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(f[j]));
  }
  for (int i = 8 * whole + tid; i < n; i += THREADS) top = max_nan(top, fabsf(as_f32(xr[i])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (THREADS > 32) {
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = max_nan(top, s_top[w]);
  }
  const float s = top <= 3.402823466e38f ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fffffff);
  if (tid == 0) scale[r] = s;
  const bool some = s > 0.f;
  const float per_s = __frcp_rn(some ? s : 1.f);
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int i = k * THREADS + tid;
    if (i < whole) *reinterpret_cast<uint2*>(qr + 8 * i) = some ? codes8(kept[k], s, per_s) : make_uint2(0, 0);
  }
  for (int i = KEEP * THREADS + tid; i < whole; i += THREADS) {
    float f[8];
    load8(xr + 8 * i, f);
    *reinterpret_cast<uint2*>(qr + 8 * i) = some ? codes8(f, s, per_s) : make_uint2(0, 0);
  }
  for (int i = 8 * whole + tid; i < n; i += THREADS)
    qr[i] = some ? static_cast<int8_t>(rintf(code_of(as_f32(xr[i]), s))) : 0;
}

template <typename T>
int quantize_run(const T* x, size_t ldx, size_t rows, int n, int8_t* q, size_t ldq, float* scale, cudaStream_t st) {
  const bool vec = aligned16(x) && (rows == 1 || ldx * sizeof(T) % 16 == 0) &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && (rows == 1 || ldq % 8 == 0);
  const auto go = [&](auto kernel, int per) {
    return launch_pdl(kernel, dim3(ceil_div(rows, per)), dim3(256), 0, st, "quantize_rows_kernel", x, ldx,
                      static_cast<long long>(rows), n, q, ldq, scale);
  };
  // A warp holds rows of up to 1024 values; longer ones, and rows too few to fill the GPU by warps, take a CTA.  4,096
  // rows of 1,024 with the product behind: 31.9 us by warps, 35.6 by CTAs; 64 rows of 512: 5.6 and 5.3.
  const bool cta = n > 1024 || (n > 256 && rows < static_cast<size_t>(8 * sm_count()));
  if (!vec) return cta ? go(quantize_rows_kernel<256, 1, false, T>, 1) : go(quantize_rows_kernel<32, 1, false, T>, 8);
  return cta ? go(quantize_rows_kernel<256, 2, true, T>, 1) : go(quantize_rows_kernel<32, 4, true, T>, 8);
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

// GELU of two values, two to an operation: gelu_erf's q = Phi(-|x|) (common.cuh) as x Phi(x) = max(x, 0) - |x| q, with |x|
// no further than q's polynomial follows it.  So infinity times 0 does not make NaN of the limits (infinity and 0), and past
// 5.5, where the result is below 1.1e-7, the bound takes back part of what q is too large by.  NaN stays.
__device__ __forceinline__ void gelu2(float& v0, float& v1) {
  const uint64_t x = pair(v0, v1);
  const float u0 = fminf(fabsf(v0), 5.5f), u1 = fminf(fabsf(v1), 5.5f);
  const uint64_t u = pair(u0, u1);
  uint64_t h = pair(-1.725302567e-08f, -1.725302567e-08f);
  h = fma2(h, u, pair(5.477549507e-07f, 5.477549507e-07f));
  h = fma2(h, u, pair(-7.458289474e-06f, -7.458289474e-06f));
  h = fma2(h, u, pair(5.484473149e-05f, 5.484473149e-05f));
  h = fma2(h, u, pair(-2.005067072e-04f, -2.005067072e-04f));
  h = fma2(h, u, pair(-1.761470485e-04f, -1.761470485e-04f));
  h = fma2(h, u, pair(7.180649787e-03f, 7.180649787e-03f));
  h = fma2(h, u, pair(-5.261564627e-02f, -5.261564627e-02f));
  h = fma2(h, u, pair(2.621913850e-01f, 2.621913850e-01f));
  h = fma2(h, u, pair(-1.151113272e+00f, -1.151113272e+00f));
  h = fma2(h, u, pair(-9.999998212e-01f, -9.999998212e-01f));
  const float2 e = unpair(fma2(mul2(x, x), pair(-0.721347520444f, -0.721347520444f), h));
  float q0, q1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(q0) : "f"(e.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(q1) : "f"(e.y));
  v0 = fmaf(-u0, q0, max_nan(v0, 0.f));
  v1 = fmaf(-u1, q1, max_nan(v1, 0.f));
}
// ReLU that keeps the NaN of a bad row's scale, which v > 0 ? v : 0 would make an ordinary 0.
__device__ __forceinline__ float relu_nan(float v) { return max_nan(v, 0.f); }
__device__ __forceinline__ float i8_value(int acc, float sa, float sb, float bias, const I8Epilogue& e) {
  float y = fmaf(static_cast<float>(acc), sa * sb, bias), same = y;
  if (e.act == GSVK_ACT_RELU) return relu_nan(y);
  if (e.act != GSVK_ACT_GELU_ERF) return apply_act(y, e.act, e.slope);
  gelu2(y, same);
  return y;
}

// ------------------------------------------------------------- tensor cores
// One persistent CTA per SM over 128 x BN output tiles.  Warp 0 loads K blocks
// of 128 bytes of A and B by TMA into 128-byte swizzled stages, warp 1 issues
// tcgen05.mma.kind::i8 (M 128, N BN, K 32; exact 32-bit sums in TMEM, two
// accumulators of BN columns), and the epilogue warps turn one accumulator
// into outputs while the next one fills.  TMA fills what lies past M, N and K
// with zeros, so no size is special.
//
// Epilogue: a lane owns a row, 32 columns at a time.  Column scales and biases
// reach it as broadcasts from a small shared-memory table per warp; results
// go to a swizzled 32 x 32 tile, which leaves by a TMA store, or, where the
// output's columns or stride are not whole 16 bytes, row by row.
constexpr int kI8BM = 128;
constexpr int kI8BK = 128;  // bytes of K per stage
constexpr int kI8MaxStages = 8;

// Four epilogue warps (a tile's rows) to every 32 columns, at most 16: with 8 at 256 columns the epilogue took twice as
// long as the products (encoder layer with GELU: 34 against 17 us).
template <int BN>
constexpr int kI8EpiWarps = BN >= 128 ? 16 : BN / 8;
template <int BN>
constexpr int kI8Threads = 64 + 32 * kI8EpiWarps<BN>;

struct I8Problem {
  int M, N, K, m_tiles, n_tiles, stages;
  int buffers;       // staged tiles of an epilogue warp and type: 1 or 2
  int tma32, tma16;  // outputs that leave by TMA
};

// tcgen05 instruction descriptor of kind::i8: signed 8-bit A and B, K-major, 32-bit integer D.
__host__ __device__ constexpr uint32_t idesc_i8(uint32_t M, uint32_t N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

constexpr int kI8Tile32 = 32 * 128, kI8Tile16 = 32 * 64;  // bytes of a staged 32 x 32 tile
// 16-byte unit j of row r of a staged tile, in the swizzle of its TMA store.
__device__ __forceinline__ uint8_t* unit32(uint8_t* tile, int r, int j) {
  return tile + r * 128 + ((j ^ (r & 7)) << 4);
}
__device__ __forceinline__ uint8_t* unit16(uint8_t* tile, int r, int j) {
  return tile + r * 64 + ((j ^ ((r >> 1) & 3)) << 4);
}

__device__ __forceinline__ void gelu16(float* v) {
#pragma unroll
  for (int j = 0; j < 16; j += 2) gelu2(v[j], v[j + 1]);
}

template <int BN>
__global__ void __launch_bounds__(kI8Threads<BN>, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tm32, const __grid_constant__ CUtensorMap tm16,
                   const I8Problem prob, const I8Epilogue epi, uint32_t* status) {
  constexpr uint32_t kABytes = kI8BM * kI8BK, kBBytes = BN * kI8BK;
  constexpr uint32_t kTmemCols = 2 * BN;
  constexpr int kEpi = kI8EpiWarps<BN>;
  const I8Problem p = prob;
  const I8Epilogue e = epi;
  extern __shared__ uint8_t i8_raw[];
  uint8_t* smem = align_smem<1024>(i8_raw);
  uint8_t* sA = smem;
  uint8_t* sB = sA + p.stages * kABytes;
  uint8_t* sOut = sB + p.stages * kBBytes;  // per epilogue warp: fp32 and fp16 tiles, as far as needed
  const int out_bytes = p.buffers * ((e.c32 ? kI8Tile32 : 0) + (e.c16 ? kI8Tile16 : 0));
  __shared__ uint64_t full[kI8MaxStages], empty[kI8MaxStages], tfull[2], tempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float2 s_col[kEpi][32];  // column scale and bias of a warp's chunk
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = p.m_tiles * p.n_tiles;
  const int kbn = (p.K + kI8BK - 1) / kI8BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kEpi);
    }
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    if (p.tma32) prefetch_tmap(&tm32);
    if (p.tma16) prefetch_tmap(&tm16);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  griddep_wait();  // operands may come from the previous kernel (the row quantiser)
  griddep_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, loaded = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        const int mt = tile / p.n_tiles, nt = tile - mt * p.n_tiles;
        for (int kb = 0; kb < kbn; ++kb) {
          if (!mbar_wait(&empty[s], ph, status)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], kABytes + kBBytes);
          tma_load_2d(sA + s * kABytes, &tmA, &full[s], kb * kI8BK, mt * kI8BM);
          tma_load_2d(sB + s * kBBytes, &tmB, &full[s], kb * kI8BK, nt * BN);
          loaded = min(loaded + 1, p.stages);
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // A wait ran out: leave once the loads in flight have landed (the last use of each stage, newest last).
      for (int i = 0; !ok && i < loaded; ++i) {
        const int last = s - 1 - i;
        mbar_wait(&full[last < 0 ? last + p.stages : last], last < 0 ? ph : ph ^ 1u, status);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(kI8BM, BN);
      // descriptors of stage 0; others lie at offsets in 16 bytes
      const uint64_t a0 = smem_desc(smem_u32(sA), 1024, 2), b0 = smem_desc(smem_u32(sB), 1024, 2);
      int s = 0, tl = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++tl) {
        const int acc = tl & 1;
        if (!mbar_wait(&tempty[acc], (static_cast<uint32_t>(tl >> 1) & 1u) ^ 1u, status)) break;
        tc_fence_after();
        for (int kb = 0; kb < kbn; ++kb) {
          if (!mbar_wait(&full[s], ph, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a = a0 + s * (kABytes / 16), b = b0 + s * (kBBytes / 16);
#pragma unroll
          for (int j = 0; j < kI8BK / 32; ++j)
            tc_mma_i8(tmem + acc * BN, a + 2 * j, b + 2 * j, idesc, (kb | j) ? 1u : 0u);
          tc_commit(&empty[s]);
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit(&tfull[acc]);
      }
    }
  } else {
    const int w = warp - 2, quarter = warp & 3;  // TMEM lanes 32 quarter .. + 31
    constexpr int kSpan = BN / (kEpi / 4);
    const int cbeg = (w >> 2) * kSpan;
    uint8_t* out32 = sOut + w * out_bytes;
    uint8_t* out16 = out32 + (e.c32 ? p.buffers * kI8Tile32 : 0);
    int turn = 0, tl = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++tl) {
      const int mt = tile / p.n_tiles, nt = tile - mt * p.n_tiles;
      const int acc = tl & 1;
      const int row0 = mt * kI8BM + quarter * 32, row = row0 + lane;
      const float sa = row < p.M ? e.a_scale[row] : 0.f;
      const auto column = [&](int c) {
        const int n = nt * BN + c + lane;
        return n < p.N ? make_float2(__ldg(e.b_scale + n), e.bias ? __ldg(e.bias + n) : 0.f) : make_float2(0.f, 0.f);
      };
      float2 col = column(cbeg);
      if (!mbar_wait(&tfull[acc], static_cast<uint32_t>(tl >> 1) & 1u, status)) break;
      tc_fence_after();
#pragma unroll 1
      for (int c0 = cbeg; c0 < cbeg + kSpan; c0 += 32) {
        const int n0 = nt * BN + c0;
        if (n0 >= p.N) break;
        s_col[w][lane] = col;
        if (c0 + 32 < cbeg + kSpan) col = column(c0 + 32);
        uint8_t* t32 = out32 + (turn & (p.buffers - 1)) * kI8Tile32;
        uint8_t* t16 = out16 + (turn & (p.buffers - 1)) * kI8Tile16;
        const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * BN + c0;
        // the stores that read this turn's tiles are done with them
        if (lane == 0 && (p.tma32 || p.tma16)) {
          if (p.buffers == 2) {
            bulk_wait_read<1>();
          } else {
            bulk_wait_read<0>();
          }
        }
        __syncwarp();
#pragma unroll 1
        for (int q = 0; q < 2; ++q) {  // 16 columns at a time
          uint32_t r[16];
          tmem_ld16(from + 16 * q, r);
          tmem_ld_wait();
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float4 c = *reinterpret_cast<const float4*>(&s_col[w][16 * q + j]);
            const uint64_t a2 = pair(static_cast<float>(static_cast<int>(r[j])), static_cast<float>(static_cast<int>(r[j + 1])));
            const float2 y = unpair(fma2(a2, mul2(pair(sa, sa), pair(c.x, c.z)), pair(c.y, c.w)));
            v[j] = y.x;
            v[j + 1] = y.y;
          }
          if (e.act == GSVK_ACT_GELU_ERF) {
            gelu16(v);
          } else if (e.act == GSVK_ACT_RELU) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = relu_nan(v[j]);
          } else {
            act_array<16>(v, e.act, e.slope);
          }
          if (e.residual && row < p.M) {
            const float* res = e.residual + row * e.ld_res + n0 + 16 * q;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (n0 + 16 * q + j < p.N) v[j] += res[j];
          }
          if (e.c32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(unit32(t32, lane, 4 * q + j)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
          if (e.c16) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              *reinterpret_cast<uint4*>(unit16(t16, lane, 2 * q + j)) =
                  make_uint4(f2h2(v[8 * j], v[8 * j + 1]), f2h2(v[8 * j + 2], v[8 * j + 3]),
                             f2h2(v[8 * j + 4], v[8 * j + 5]), f2h2(v[8 * j + 6], v[8 * j + 7]));
          }
        }
        if (p.tma32 || p.tma16) fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0 && row0 < p.M) {
          if (p.tma32) tma_store_2d(&tm32, t32, n0, row0);
          if (p.tma16) tma_store_2d(&tm16, t16, n0, row0);
        }
        if (lane == 0 && (p.tma32 || p.tma16)) bulk_commit();
        if ((e.c32 && !p.tma32) || (e.c16 && !p.tma16)) {  // row by row, a lane to a column
          const int rows = min(32, p.M - row0);
          if (n0 + lane < p.N) {
#pragma unroll 8
            for (int i = 0; i < rows; ++i) {
              if (e.c32 && !p.tma32)
                e.c32[(row0 + i) * e.ld_c32 + n0 + lane] =
                    *reinterpret_cast<const float*>(unit32(t32, i, lane >> 2) + 4 * (lane & 3));
              if (e.c16 && !p.tma16)
                e.c16[(row0 + i) * e.ld_c16 + n0 + lane] =
                    *reinterpret_cast<const uint16_t*>(unit16(t16, i, lane >> 3) + 2 * (lane & 7));
            }
          }
          __syncwarp();
        }
        ++turn;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

int i8_map(CUtensorMap* m, const int8_t* base, size_t rows, size_t K, size_t ld, int box_rows) {
  const uint64_t dims[2] = {K, rows};
  const uint64_t strides[1] = {ld};
  const uint32_t box[2] = {kI8BK, static_cast<uint32_t>(box_rows)};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int BN>
int launch_i8(const gsvk_gemm_i8_args* g, size_t lda, size_t ldb, const I8Epilogue& e, cudaStream_t st) {
  I8Problem p{};
  p.M = static_cast<int>(g->M);
  p.N = static_cast<int>(g->N);
  p.K = static_cast<int>(g->K);
  p.m_tiles = (p.M + kI8BM - 1) / kI8BM;
  p.n_tiles = (p.N + BN - 1) / BN;
  CUtensorMap ta, tb, t32{}, t16{};
  int rc = i8_map(&ta, g->a, g->M, g->K, lda, kI8BM);
  if (!rc) rc = i8_map(&tb, g->b, g->N, g->K, ldb, BN);
  // a TMA store writes whole 16 bytes of a row: the columns have to be, beside the stride
  const uint64_t odims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)};
  const uint32_t box[2] = {32, 32};
  if (!rc && e.c32 && aligned16(e.c32) && e.ld_c32 % 4 == 0 && p.N % 4 == 0) {
    const uint64_t str[1] = {static_cast<uint64_t>(e.ld_c32) * 4};
    rc = encode_tiled(&t32, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, e.c32, odims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    p.tma32 = 1;
  }
  if (!rc && e.c16 && aligned16(e.c16) && e.ld_c16 % 8 == 0 && p.N % 8 == 0) {
    const uint64_t str[1] = {static_cast<uint64_t>(e.ld_c16) * 2};
    rc = encode_tiled(&t16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, e.c16, odims, str, box, CU_TENSOR_MAP_SWIZZLE_64B);
    p.tma16 = 1;
  }
  if (rc) return rc;
  constexpr size_t kLimit = 227 * 1024 - 6144;  // barriers and column tables are static
  // one staged tile where fp32 ones would leave too little for the operands
  p.buffers = e.c32 ? 1 : 2;
  const size_t staging = static_cast<size_t>(kI8EpiWarps<BN>) * p.buffers * ((e.c32 ? kI8Tile32 : 0) + (e.c16 ? kI8Tile16 : 0));
  const size_t stage = (kI8BM + BN) * kI8BK;
  const int kbn = (p.K + kI8BK - 1) / kI8BK;
  p.stages = static_cast<int>(std::min<size_t>(kI8MaxStages, (kLimit - 1024 - staging) / stage));
  // no more stages than this CTA has K blocks to load
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  const long long rounds = (tiles + sm_count() - 1) / sm_count();
  p.stages = static_cast<int>(std::max<long long>(1, std::min<long long>(p.stages, rounds * kbn)));
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    rc = check_cuda(cudaFuncSetAttribute(gemm_i8_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(kLimit)),
                    "cudaFuncSetAttribute(gemm_i8)");
    if (rc) return rc;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const size_t smem = 1024 + p.stages * stage + staging;
  return launch_pdl(gemm_i8_kernel<BN>, dim3(static_cast<unsigned>(std::min<long long>(tiles, sm_count()))),
                    dim3(kI8Threads<BN>), smem, st, "gemm_i8_kernel", ta, tb, t32, t16, p, e, device_status());
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
  return is_f32 ? quantize_run(static_cast<const float*>(x), ldx, rows, (int)n, q, ldq, scale, as_cuda(stream))
                : quantize_run(static_cast<const uint16_t*>(x), ldx, rows, (int)n, q, ldq, scale, as_cuda(stream));
}

int gsvk_gemm_i8(const gsvk_gemm_i8_args* g, gsvk_stream_t stream) {
  if (g && g->M == 0) return GSVK_OK;
  if (!g || !g->a || !g->b || !g->a_scale || !g->b_scale || (!g->c && !g->c_f16))
    return fail(GSVK_ERR_INVALID, "gemm_i8: null pointer");
  if (g->N == 0 || g->K == 0) return fail(GSVK_ERR_INVALID, "gemm_i8: zero size");
  // a grid of the CUDA-core kernel, and 128 x 32 tiles of the other, count up to 2^31 - 1; M N is below 2^62
  if (g->M > 0x7fffff00 || g->N > 0x7fffff00 || g->K >= 131072 || (g->M * g->N + 255) / 256 > 0x7fffffff)
    return fail(GSVK_ERR_UNSUPPORTED, "gemm_i8: %zu x %zu x %zu (K below 131072: 32-bit sums)", g->M, g->N, g->K);
  const size_t lda = g->lda ? g->lda : g->K, ldb = g->ldb ? g->ldb : g->K;
  const size_t ldc = g->ldc ? g->ldc : g->N, ldh = g->ldc_f16 ? g->ldc_f16 : g->N;
  const size_t ldr = g->ld_res ? g->ld_res : g->N;
  if ((g->M > 1 && lda < g->K) || (g->N > 1 && ldb < g->K) || (g->M > 1 && (ldc < g->N || ldh < g->N || ldr < g->N)))
    return fail(GSVK_ERR_INVALID, "gemm_i8: a leading dimension is below its row");
  if (g->act < GSVK_ACT_NONE || g->act > GSVK_ACT_TANH) return fail(GSVK_ERR_INVALID, "gemm_i8: bad act");
  I8Epilogue e{g->a_scale, g->b_scale, g->bias, g->residual, g->c, g->c_f16,
               (long long)ldr, (long long)ldc, (long long)ldh, g->act, g->slope};
  cudaStream_t st = as_cuda(stream);
  if (gsvk_available() && aligned16(g->a) && aligned16(g->b) && (lda % 16 == 0 || g->M == 1) && (ldb % 16 == 0 || g->N == 1)) {
    // one row: any stride will do
    const size_t sa = g->M == 1 ? (g->K + 15) / 16 * 16 : lda, sb = g->N == 1 ? (g->K + 15) / 16 * 16 : ldb;
    // The widest tile whose tiles still fill the GPU: each A byte then feeds the most columns.  4,096 x 4,096 with K of
    // 1,024 and 4,096: 25 and 68 us at 256 columns, 29 and 82 at 128, at 64 45 (K of 1,024 with GELU; 31 at 256 and 128,
    // which the epilogue bounds).  64 x 1,536 x 512: 5.3 us at 32, 5.4 at 64, 5.9 at 128; 500 x 1,025 x 512: 6.6, 6.9, 7.7.
    const size_t m_tiles = (g->M + kI8BM - 1) / kI8BM, sms = static_cast<size_t>(sm_count());
    if (m_tiles * ((g->N + 255) / 256) >= sms) return launch_i8<256>(g, sa, sb, e, st);
    if (m_tiles * ((g->N + 127) / 128) >= sms) return launch_i8<128>(g, sa, sb, e, st);
    if (m_tiles * ((g->N + 63) / 64) >= sms) return launch_i8<64>(g, sa, sb, e, st);
    return launch_i8<32>(g, sa, sb, e, st);
  }
  const size_t outs = g->M * g->N;
  gemm_i8_simt_kernel<<<ceil_div(outs, 256), 256, 0, st>>>(
      g->a, (long long)lda, g->b, (long long)ldb, (long long)g->M, (int)g->N, (int)g->K, e);
  return check_launch("gemm_i8_simt_kernel");
}

}  // extern "C"
