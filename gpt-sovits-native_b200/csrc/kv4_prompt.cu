// kv4_prompt.cu — attention over the paged 4-bit KV cache for requests with
// many new tokens (prompts, chunks of prompts): 128-row tiles on tcgen05.
//
// A CTA owns 128 query rows (new token, query head of the group) of one
// (request, kv head) and walks the keys they see in tiles of 64, with two CTAs
// on an SM so that one's softmax covers the other's waits.  Roles:
//   warps 0-3   softmax: a thread to a row (its TMEM lane)
//   warps 4-7   unpack a tile's codes into fp16 operand tiles, and its parameters
//   warp 8      copies the tile's pages into shared memory (cp.async.bulk)
//   warp 9      issues the MMAs:  S = Q C_k^T  and  O += W C_v, W from TMEM
// The scores of tile i + 1 are computed while the softmax works on tile i (two
// score buffers; the weights overwrite the scores they come from).
//
// Mathematics.  With k_j = a_j c_j + b_j and v_j = s_j e_j + f_j (step, code,
// low), c and e the codes,
//   z_j = a_j (q.c_j) + b_j sum(q),          p_j = 2^(z_j - reference)
// so the score MMAs multiply codes, which are exact in fp16 (c as the
// subnormal c 2^-24, one AND for two of them), and q is not rounded.  The
// values go in two ways:
//   head_dim 32, 64: v_j as the sum of two fp16 numbers, side by side as
//     2 head_dim columns of one operand (an MMA of 128 x 128 takes the 67 clocks that one of
//     128 x 64 takes: measured), so the weights are p_j and need no
//     parameters of the key;
//   head_dim 128, where that would double the MMAs:
//     sum_j p_j v_j = sum_j (p_j s_j) (e_j - 8) + sum_j p_j (f_j + 8 s_j).
// Either way the one rounding to fp16 beside the result's is that of the
// weights: 2^-11 of the values (centred ones for head_dim 128).
// The reference is the row's maximum as of the last time that it grew by 2^8:
// until then the weights stay in fp16's range and the sums in TMEM are left
// alone.  Values (steps) are divided by a power of two, the same for all rows.
//
// What bounds it: per 128 x 64 scores an SM's 16 exponentials a clock take 512
// clocks, the MMAs 8 x 67 at head_dim 64, and the keys' parameters, which every
// thread reads from shared memory (8 bytes a score, 128 bytes a clock), another 512.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4_attn.cuh"

namespace gsvk {

namespace {

constexpr int kPRows = 128, kPTile = 64;
constexpr int kPThreads = 384;
constexpr int kPRegs = 80, kPRegsSoftmax = 136, kPRegsUnpack = 56, kPRegsRest = 40;
static_assert(kPRegsSoftmax + kPRegsUnpack + kPRegsRest <= 3 * kPRegs, "register shares exceed the launch's");
constexpr uint32_t kPTmemCols = 256;  // scores at 0 and 64, sums at 128

// What the softmax needs of a tile's keys.
struct alignas(16) TileParams {
  float a[kPTile], b[kPTile];
  float s[kPTile], f[kPTile];  // head_dim 128
  float unit, rescale;         // the values' unit, and the previous tile's over it
  uint32_t page_ok;
};

template <int HD>
constexpr bool kPSplit = HD <= 64;  // values as two fp16 numbers
template <int HD>
constexpr int kPCols = kPSplit<HD> ? 2 * HD : HD;  // columns of the value operand and of the sums
template <int HD>
constexpr int kPRaw = HD == 128 ? 3 : 4;  // raw tiles in flight
template <int HD>
constexpr int kPValues = HD == 128 ? 1 : 2;  // unpacked value tiles
template <int HD>
constexpr int kPQBytes = kPRows * HD * 2;
template <int HD>
constexpr int kPOpBytes = kPTile * HD * 2;
template <int HD>
constexpr int kPValBytes = kPTile * kPCols<HD> * 2;
template <int HD>
constexpr int kPRawBytes = kPTile * (HD + 8);
template <int HD>
constexpr int kPSmem = 1024 + kPQBytes<HD> + 2 * kPOpBytes<HD> + kPValues<HD> * kPValBytes<HD> + kPRaw<HD> * kPRawBytes<HD> +
                       2 * static_cast<int>(sizeof(TileParams));

// 16-byte unit u of row r of an operand tile with COLS columns: rows of 64 values in the 128-byte swizzle, 128
// columns as two slabs of `rows` rows, 32 as 64-byte rows in the 64-byte swizzle.
template <int COLS>
__device__ __forceinline__ uint32_t unit_at(int r, int u, int rows) {
  if constexpr (COLS == 32) return r * 64 + ((u ^ ((r >> 1) & 3)) << 4);
  return (u >> 3) * rows * 128 + r * 128 + (((u & 7) ^ (r & 7)) << 4);
}
// Operand descriptor; lbo: bytes between 64-column slabs of an operand that is contiguous along M or N.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo, uint32_t swizzle) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32 | 1ull << 46 | static_cast<uint64_t>(swizzle) << 61;
}
// A from TMEM: D[tmem] (+)= A[tmem] * B[smem desc].
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// N consecutive words of shared memory, in as few loads as they allow (aligned to their size, at most 16 bytes).
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

__device__ __forceinline__ int prompt_blocks(const AttnArgs& a, int s) {
  const Request q = request_of(a, s);
  const int rows = q.n * a.group;
  return rows > a.most_rows ? (rows + kPRows - 1) / kPRows : 0;
}

template <int HD>
__global__ void __launch_bounds__(kPThreads, 2) kv4_prompt_kernel(const AttnArgs a) {
  constexpr int kRaw = kPRaw<HD>, kV = kPValues<HD>;
  extern __shared__ uint8_t prompt_raw[];
  uint8_t* smem = align_smem<1024>(prompt_raw);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + kPQBytes<HD>;
  uint8_t* sV = sK + 2 * kPOpBytes<HD>;
  uint8_t* sRaw = sV + kV * kPValBytes<HD>;
  TileParams* par = reinterpret_cast<TileParams*>(sRaw + kRaw * kPRawBytes<HD>);
  __shared__ uint64_t raw_full[kRaw], raw_free[kRaw], k_full[2], k_free[2], v_full[kV], v_free[kV];
  __shared__ uint64_t par_full[2], par_free[2], s_full[2], p_full[2], o_done, all_done;
  __shared__ uint32_t raw_ok[kRaw];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_before[kPThreads / 32 + 1], s_seq, s_block;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // the row block of this CTA: blocks of all requests in reverse, so that the longest of a request come first
  {
    const int per = (a.n_seq + kPThreads - 1) / kPThreads;
    const int r0 = min(tid * per, a.n_seq), r1 = min(r0 + per, a.n_seq);
    int mine = 0;
    for (int s = r0; s < r1; ++s) mine += prompt_blocks(a, s);
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) s_before[warp + 1] = inc;
    if (tid == 0) s_before[0] = 0;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kPThreads / 32; ++w) {
      const int c = s_before[w + 1];
      if (w < warp) before += c;
      total += c;
    }
    const int want = total - 1 - static_cast<int>(blockIdx.x) / a.kv_heads;
    if (want < 0) {  // the whole CTA: the grid is an upper bound
      griddep_wait();
      return;
    }
    int left = want - (before + inc - mine);
    if (left >= 0 && left < mine) {
      int s = r0, nb = prompt_blocks(a, s);
      while (left >= nb) {
        left -= nb;
        nb = prompt_blocks(a, ++s);
      }
      s_seq = s;
      s_block = left;
    }
  }
  if (tid == 0) {
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_free[i], 1);
      mbar_init(&par_full[i], 4);
      mbar_init(&par_free[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    for (int i = 0; i < kV; ++i) {
      mbar_init(&v_full[i], 4);
      mbar_init(&v_free[i], 1);
    }
    mbar_init(&o_done, 1);
    mbar_init(&all_done, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&tmem_slot, kPTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int seq = s_seq, block = s_block, head = static_cast<int>(blockIdx.x) % a.kv_heads;
  const Request req = request_of(a, seq);
  const int all = req.n * a.group, row0 = block * kPRows;
  const int keys = limit_of(a, req, min(row0 + kPRows, all) - 1);
  const int tiles = max(1, (keys + kPTile - 1) / kPTile);
  const int sub_shift = min(a.shift, 6), subs = kPTile >> sub_shift;

  if (warp < 4) {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsSoftmax));
    const int row = row0 + tid;
    const bool live_row = row < all;
    const int limit = limit_of(a, req, min(row, all - 1));
    const int least = __reduce_min_sync(0xffffffffu, limit);
    float qsum = 0.f;
    {
      const int r = live_row ? row / a.group : 0;
      const uint16_t* src = a.q + static_cast<size_t>(req.q0 + r) * a.q_stride +
                            static_cast<size_t>(head * a.group + (live_row ? row - r * a.group : 0)) * HD;
#pragma unroll
      for (int u = 0; u < HD / 8; ++u) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (live_row) x = *reinterpret_cast<const uint4*>(src + 8 * u);
        float f[8];
        unpack8(x, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) qsum += f[i];
        // the order of a word's nibbles: 0 4, 1 5, 2 6, 3 7
        *reinterpret_cast<uint4*>(sQ + unit_at<HD>(tid, u, kPRows)) =
            make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                       __byte_perm(x.y, x.w, 0x7632));
      }
    }
    fence_proxy_async_shared();
    asm volatile("bar.sync 1, 160;" ::: "memory");  // with the MMA warp: Q is there
    const uint64_t qs = pair(qsum, qsum);
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    float ref = -INFINITY, unit = 0.f;
    uint64_t l2 = 0, pb2 = 0;
    bool ok = true;
    for (int i = 0; i < tiles; ++i) {
      const int buf = i & 1;
      const uint32_t ph = static_cast<uint32_t>(i >> 1) & 1u;
      const TileParams& t = par[buf];
      if (!mbar_wait(&par_full[buf], ph, a.status) || !mbar_wait(&s_full[buf], ph, a.status)) ok = false;
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      uint32_t r[kPTile];
#pragma unroll
      for (int c = 0; c < kPTile; c += 16) tmem_ld16(tmem + lanes + buf * kPTile + c, r + c);
      tmem_ld_wait();
      uint64_t z[kPTile / 2];
#pragma unroll
      for (int j = 0; j < kPTile; j += 4) {
        const ulonglong2 ta = *reinterpret_cast<const ulonglong2*>(t.a + j), tb = *reinterpret_cast<const ulonglong2*>(t.b + j);
        z[j / 2] = fma2(pair(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), ta.x, mul2(tb.x, qs));
        z[j / 2 + 1] = fma2(pair(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), ta.y, mul2(tb.y, qs));
      }
      const uint32_t page_ok = t.page_ok;
      if (i * kPTile + kPTile > least || page_ok != (1u << subs) - 1u) {
        const int see = limit - i * kPTile;
#pragma unroll
        for (int j = 0; j < kPTile; j += 2) {
          float2 v = unpair(z[j / 2]);
          if (j >= see || !(page_ok >> (j >> sub_shift) & 1u)) v.x = -INFINITY;
          if (j + 1 >= see || !(page_ok >> ((j + 1) >> sub_shift) & 1u)) v.y = -INFINITY;
          z[j / 2] = pair(v.x, v.y);
        }
      }
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < kPTile / 2; ++j) {
        const float2 v = unpair(z[j]);
        tops[j & 3] = fmaxf(fmaxf(tops[j & 3], v.x), v.y);
      }
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      unit = t.unit;
      if (i == 0) {
        ref = top;
      } else if (__any_sync(0xffffffffu, top > ref + 8.f || t.rescale != 1.f)) {
        // a new reference or unit: bring the sums to it.  (These scores vouch for the sums of tile i - 2 and those
        // of tile i wait for this thread, so the barrier is in one of two phases.)
        if (!mbar_wait(&o_done, static_cast<uint32_t>(i - 1) & 1u, a.status)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const float to = fmaxf(ref, top);
        const float keep = to == -INFINITY ? 1.f : ex2(ref - to);
        ref = to;
        l2 = mul2(l2, pair(keep, keep));
        pb2 = mul2(pb2, pair(keep, keep));
        const float by = keep * t.rescale;
#pragma unroll 1
        for (int c = 0; c < kPCols<HD>; c += 16) {
          uint32_t o[16];
          tmem_ld16(tmem + lanes + 128 + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
          tmem_st16(tmem + lanes + 128 + c, o);
        }
        tmem_st_wait();
      }
      const float base = ref == -INFINITY ? 0.f : ref;
      const uint64_t nb = pair(-base, -base);
      uint32_t w[kPTile / 2];
#pragma unroll
      for (int j = 0; j < kPTile / 2; ++j) {
        const float2 d = unpair(add2(z[j], nb));
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        const uint64_t p = pair(e.x, e.y);
        l2 = add2(l2, p);
        if constexpr (kPSplit<HD>) {
          w[j] = f2h2(e.x, e.y);
        } else {
          pb2 = fma2(p, *reinterpret_cast<const uint64_t*>(t.f + 2 * j), pb2);
          const float2 x = unpair(mul2(p, *reinterpret_cast<const uint64_t*>(t.s + 2 * j)));
          w[j] = f2h2(x.x, x.y);
        }
      }
      tmem_st16(tmem + lanes + buf * kPTile, w);
      tmem_st16(tmem + lanes + buf * kPTile + 16, w + 16);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&p_full[buf]);
        mbar_arrive(&par_free[buf]);
      }
    }
    if (ok && !mbar_wait(&all_done, 0, a.status)) ok = false;
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const float2 ls = unpair(l2), ps = unpair(pb2);
      const float l = ls.x + ls.y, pb = ps.x + ps.y;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t* out = out_row(a, req, head, live_row ? row : row0, HD);
#pragma unroll
      for (int c = 0; c < HD; c += 16) {
        uint32_t o[16];
        tmem_ld16(tmem + lanes + 128 + c, o);
        if constexpr (kPSplit<HD>) {
          uint32_t second[16];
          tmem_ld16(tmem + lanes + 128 + HD + c, second);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(second[k]));
        }
        tmem_ld_wait();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float v[8];  // the columns' order is the nibbles': 0 4 1 5 2 6 3 7
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[(k >> 1) + 4 * (k & 1)] = l == 0.f ? 0.f : fmaf(__uint_as_float(o[8 * u + k]), unit, pb) * inv;
          if (live_row)
            *reinterpret_cast<uint4*>(out + c + 8 * u) =
                make_uint4(f2h2(v[0], v[1]), f2h2(v[2], v[3]), f2h2(v[4], v[5]), f2h2(v[6], v[7]));
        }
      }
    }
    tc_fence_before();
  } else if (warp < 8) {
    // ----------------------------------------------------------------- unpack
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsUnpack));
    const int me = tid - 128, key = me >> 1, half = me & 1;  // two threads to a key
    const int sub_bytes = kv4_head_bytes(sub_shift, HD), sub_mask = (1 << sub_shift) - 1;
    float unit = 0.f, per_unit = 0.f;
    for (int i = 0; i < tiles; ++i) {
      const int rs = i % kRaw, buf = i & 1, vb = i % kV;
      const uint32_t ph = static_cast<uint32_t>(i >> 1) & 1u;
      bool ok = mbar_wait(&raw_full[rs], static_cast<uint32_t>(i / kRaw) & 1u, a.status) &&
                mbar_wait(&k_free[buf], ph ^ 1u, a.status) && mbar_wait(&par_free[buf], ph ^ 1u, a.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint8_t* raw = sRaw + rs * kPRawBytes<HD>;
      const uint32_t page_ok = raw_ok[rs];
      const uint8_t* sub = raw + (key >> sub_shift) * sub_bytes;
      const int at = key & sub_mask;
      uint32_t words[HD / 16];  // this thread's half of a key's codes
      load_words<HD / 16>(sub + at * (HD / 2) + half * (HD / 4), words);
#pragma unroll
      for (int u = 0; u < HD / 16; ++u) {
        const uint32_t x = words[u];
        *reinterpret_cast<uint4*>(sK + buf * kPOpBytes<HD> + unit_at<HD>(key, half * (HD / 16) + u, kPTile)) =
            make_uint4(x & 0x000f000fu, x >> 4 & 0x000f000fu, x >> 8 & 0x000f000fu, x >> 12 & 0x000f000fu);
      }
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(sub + kv4_k_par(sub_shift, HD) + at * 4);
      const uint32_t vp = *reinterpret_cast<const uint32_t*>(sub + kv4_v_par(sub_shift, HD) + at * 4);
      float vs = h2f(static_cast<uint16_t>(vp)), vf = h2f(static_cast<uint16_t>(vp >> 16));
      const bool seen = i * kPTile + key < keys && (page_ok >> (key >> sub_shift) & 1u);
      const bool number = fabsf(fmaf(15.f, vs, vf)) <= 3.0e38f;
      if (!seen || !number) vs = vf = 0.f;  // whatever the page holds there
      // What sets the unit: the greatest value (split) or step of the tile; each warp works it out for all 64 keys.
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j = lane + 32 * c;
        const uint32_t p = *reinterpret_cast<const uint32_t*>(raw + (j >> sub_shift) * sub_bytes +
                                                              kv4_v_par(sub_shift, HD) + (j & sub_mask) * 4);
        const float st = h2f(static_cast<uint16_t>(p)), lo = h2f(static_cast<uint16_t>(p >> 16));
        const float m = kPSplit<HD> ? fmaxf(fabsf(lo), fabsf(fmaf(15.f, st, lo))) : fabsf(st);
        if (i * kPTile + j < keys && (page_ok >> (j >> sub_shift) & 1u) && fabsf(fmaf(15.f, st, lo)) <= 3.0e38f)
          most = fmaxf(most, m);
      }
      most = warp_max(most);
      // a unit holds until something passes four times it
      float rescale = 1.f;
      if (most > 4.f * unit) {
        const float next = __uint_as_float((__float_as_uint(most) & 0x7f800000u) + 0x00800000u);
        rescale = unit / next;
        unit = next;
        per_unit = 1.f / next;  // a power of two: exact
      }
      if (half == 0) {
        TileParams& t = par[buf];
        // Values that are not numbers reach the rows that see them by their score, which a row that does not see the
        // key replaces.
        t.a[key] = !seen ? 0.f : number ? h2f(static_cast<uint16_t>(kp)) * (a.scale_log2 * 16777216.f) : __int_as_float(0x7fffffff);
        t.b[key] = !seen ? 0.f : h2f(static_cast<uint16_t>(kp >> 16)) * a.scale_log2;
        if constexpr (!kPSplit<HD>) {
          t.s[key] = vs * per_unit;
          t.f[key] = fmaf(8.f, vs, vf);
        }
        if (me == 0) {
          t.unit = unit;
          t.rescale = rescale;
          t.page_ok = page_ok;
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[buf]);
        mbar_arrive(&par_full[buf]);
      }
      ok = mbar_wait(&v_free[vb], (static_cast<uint32_t>(i / kV) & 1u) ^ 1u, a.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      load_words<HD / 16>(sub + kv4_v_codes(sub_shift, HD) + at * (HD / 2) + half * (HD / 4), words);
      uint8_t* val = sV + vb * kPValBytes<HD>;
      const uint64_t s2 = pair(vs * per_unit, vs * per_unit), f2 = pair(vf * per_unit, vf * per_unit);
#pragma unroll
      for (int u = 0; u < HD / 16; ++u) {
        uint32_t y[4], y2[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t c = (words[u] >> (4 * k) & 0x000f000fu) | 0x64006400u;  // 1024 + code
          if constexpr (kPSplit<HD>) {
            // two codes as fp32: 2^23 + code, less 2^23
            const uint64_t e = add2(pair(__uint_as_float((words[u] >> (4 * k) & 15u) | 0x4b000000u),
                                         __uint_as_float((words[u] >> (4 * k + 16) & 15u) | 0x4b000000u)),
                                    pair(-8388608.f, -8388608.f));
            const uint64_t v = fma2(e, s2, f2);
            const float2 x = unpair(v);
            const __half2 h = __floats2half2_rn(x.x, x.y);
            const float2 b = __half22float2(h);
            const float2 r = unpair(add2(v, pair(-b.x, -b.y)));
            y[k] = *reinterpret_cast<const uint32_t*>(&h);
            y2[k] = f2h2(r.x, r.y);
          } else {
            const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&c),
                                      __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));  // code - 8
            y[k] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        const int unit_no = half * (HD / 16) + u;
        *reinterpret_cast<uint4*>(val + unit_at<kPCols<HD>>(key, unit_no, kPTile)) = make_uint4(y[0], y[1], y[2], y[3]);
        if constexpr (kPSplit<HD>)
          *reinterpret_cast<uint4*>(val + unit_at<kPCols<HD>>(key, HD / 8 + unit_no, kPTile)) =
              make_uint4(y2[0], y2[1], y2[2], y2[3]);
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[vb]);
        mbar_arrive(&raw_free[rs]);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsRest));
    if (warp == 8) {
      // ------------------------------------------------------------------ load
      const auto page_of = [&](int tile) {
        const int j = tile * kPTile + (lane << sub_shift);
        return lane < subs && tile < tiles && j < keys
                   ? a.table[static_cast<size_t>(seq) * a.max_blocks + (j >> a.shift)]
                   : -1;
      };
      int page = page_of(0), next = page_of(1);
      const int bytes = kv4_head_bytes(sub_shift, HD);
      int i = 0;
      bool ok = true;
      for (; i < tiles; ++i) {
        const int rs = i % kRaw;
        const int later = page_of(i + 2);
        ok = mbar_wait(&raw_free[rs], (static_cast<uint32_t>(i / kRaw) & 1u) ^ 1u, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool there = page >= 0 && page < a.n_pages;
        const uint32_t mask = __ballot_sync(0xffffffffu, there);
        if (lane == 0) {
          raw_ok[rs] = mask;
          mbar_arrive_expect_tx(&raw_full[rs], __popc(mask) * bytes);
        }
        __syncwarp();
        if (there) {
          const uint8_t* src = a.pages + static_cast<size_t>(page) * a.page_bytes +
                               static_cast<size_t>(head) * kv4_head_bytes(a.shift, HD);
          uint8_t* dst = sRaw + rs * kPRawBytes<HD> + lane * bytes;
          if (a.shift <= 6) {
            bulk_load(dst, src, bytes, &raw_full[rs]);
          } else {  // half of a page of 128: its four parts
            const int part = i & 1, codes = kv4_v_codes(6, HD);
            bulk_load(dst, src + part * codes, codes, &raw_full[rs]);
            bulk_load(dst + codes, src + kv4_v_codes(7, HD) + part * codes, codes, &raw_full[rs]);
            bulk_load(dst + kv4_k_par(6, HD), src + kv4_k_par(7, HD) + part * 256, 256, &raw_full[rs]);
            bulk_load(dst + kv4_v_par(6, HD), src + kv4_v_par(7, HD) + part * 256, 256, &raw_full[rs]);
          }
        }
        page = next;
        next = later;
      }
      if (!ok)  // a wait ran out: leave once the copies in flight have landed
        for (int k = max(0, i - kRaw); k < i; ++k)
          mbar_wait(&raw_full[k % kRaw], static_cast<uint32_t>(k / kRaw) & 1u, a.status);
    } else if (warp == 9) {
      // ------------------------------------------------------------------- MMA
      asm volatile("bar.sync 1, 160;" ::: "memory");
      tc_fence_after();
      if (lane == 0) {
        constexpr uint32_t sw = HD == 32 ? 4 : 2, sbo = HD == 32 ? 512 : 1024;  // value rows: 128 bytes
        constexpr uint32_t idesc_s = idesc_f16_f32(kPRows, kPTile);
        constexpr uint32_t idesc_o = idesc_f16_f32(kPRows, kPCols<HD>) | 1u << 16;  // B contiguous along N
        const uint32_t q = smem_u32(sQ), k = smem_u32(sK), v = smem_u32(sV);
        bool ok = true;
        for (int i = 0; i <= tiles && ok; ++i) {
          if (i < tiles) {
            const int buf = i & 1;
            if (!mbar_wait(&k_full[buf], static_cast<uint32_t>(i >> 1) & 1u, a.status)) break;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
              const uint32_t slab = j >> 2, in = (j & 3) * 32;  // 16 values are 32 bytes
              tc_mma_f16(tmem + buf * kPTile, operand_desc(q + slab * (kPRows * 128) + in, 16, sbo, sw),
                         operand_desc(k + buf * kPOpBytes<HD> + slab * (kPTile * 128) + in, 16, sbo, sw), idesc_s, j ? 1u : 0u);
            }
            tc_commit(&s_full[buf]);
            tc_commit(&k_free[buf]);
          }
          if (i > 0) {
            const int p = i - 1, buf = p & 1, vb = p % kV;
            ok = mbar_wait(&v_full[vb], static_cast<uint32_t>(p / kV) & 1u, a.status) &&
                 mbar_wait(&p_full[buf], static_cast<uint32_t>(p >> 1) & 1u, a.status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < kPTile / 16; ++j)
              tc_mma_f16_ts(tmem + 128, tmem + buf * kPTile + j * 8,
                            operand_desc(v + vb * kPValBytes<HD> + j * 16 * 128, kPTile * 128, 1024, 2), idesc_o,
                            (p | j) ? 1u : 0u);
            tc_commit(&v_free[vb]);
            tc_commit(&o_done);
            if (i == tiles) tc_commit(&all_done);
          }
        }
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kPTmemCols);
  }
  griddep_wait();  // the few-row kernel's end: what follows in the stream waits for both
}

template <int HD>
int launch_prompt(const AttnArgs& a, cudaStream_t st) {
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    cudaFuncAttributes at{};
    if (int rc = check_cuda(cudaFuncGetAttributes(&at, kv4_prompt_kernel<HD>), "cudaFuncGetAttributes(kv4_prompt)"))
      return rc;
    // the roles' register shares come out of the launch's
    if (at.numRegs * 3 < kPRegsSoftmax + kPRegsUnpack + kPRegsRest)
      return fail(GSVK_ERR_UNSUPPORTED, "kv4_prompt_kernel: built with %d registers", at.numRegs);
    if (int rc = check_cuda(cudaFuncSetAttribute(kv4_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kPSmem<HD>),
                            "cudaFuncSetAttribute(kv4_prompt)"))
      return rc;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  // no more row blocks than full ones and one for each request that has any
  const long long rows = static_cast<long long>(a.n_tokens) * a.group;
  const long long blocks = rows / kPRows + std::min<long long>(a.n_seq, rows / (a.most_rows + 1));
  if (blocks == 0) return GSVK_OK;
  if (blocks * a.kv_heads > 0x7fffffff) return fail(GSVK_ERR_UNSUPPORTED, "kv4_attention: too many rows");
  return launch_pdl(kv4_prompt_kernel<HD>, dim3(static_cast<unsigned>(blocks * a.kv_heads)), dim3(kPThreads),
                    kPSmem<HD>, st, "kv4_prompt_kernel", a);
}

}  // namespace

int kv4_prompt_run(const AttnArgs& a, int head_dim, cudaStream_t st) {
  return head_dim == 32 ? launch_prompt<32>(a, st) : head_dim == 64 ? launch_prompt<64>(a, st) : launch_prompt<128>(a, st);
}

}  // namespace gsvk
