// kv4_prompt.cu — attention over the paged 4-bit KV cache for requests with
// many new tokens (prompts, chunks of prompts): 128-row tiles on tcgen05.
//
// An item is 256 query rows (two blocks of 128) of one (request, kv head), its
// unit of work a tile of 128 of the keys they see (head_dim 128: 64).  One
// persistent CTA per SM takes an equal run of the line of units (kv4_attn.cuh),
// so no SM waits for the longest item, and the loads and the unpacking of an
// item overlap the end of the last.  A run's first and last item may be shared with
// other CTAs: the warp that finishes its 32 rows last joins the pieces.  (With a
// CTA to an item, starting and ending them cost 126 of 390 us on 50 blocks of 16 heads.)  Roles:
//   warps 0-3, 4-7  softmax of the first and the second block: a thread to a row (its TMEM lane)
//   warps 8-11      unpack a tile's codes into fp16 operands
//   warp 12         copies the tile's pages into shared memory (cp.async.bulk)
//   warp 13         issues the MMAs:  S = Q K^T  and  O += W V, W from TMEM over the scores it came from
// While the tensor cores work on one block's products, the other block's
// softmax runs; what is unpacked serves both.
//
// Mathematics.  k_j = a c + b (step, codes, low), so q.k_j = q.(a c) + sum(q) b.
// a c takes 15 bits: it goes in as the sum of two fp16 numbers, one product
// and one fused product for two codes, and b as one more column of K against
// sum(q), which is two columns of Q.  So no score is rounded below fp32
// (K as one fp16 number would move each by 2^-12 |q||k|).
// v_j goes in as two fp16 parts at head_dim 32 and 64, side by side as
// 2 head_dim columns of the value operand (an MMA of 128 x 128 takes the 67
// clocks that one of 128 x 64 takes: measured).  At head_dim 128 that would double the MMAs:
//   sum_j p_j v_j = sum_j (p_j s_j) (e_j - 8) + sum_j p_j (f_j + 8 s_j)
// there, with the codes e - 8 as the operand and the last sum in the softmax.
// Either way the one rounding to fp16 beside the result's is that of the
// weights: 2^-11 of the values (centred within 8 steps at head_dim 128).
// p_j = 2^(z_j - reference); the reference is the row's maximum as of the last
// time that it grew by 2^8: until then the weights stay in fp16's range and the
// sums in TMEM are left alone.  K and V (s) are divided by a power of two, that
// of K by tile, that of V the same for all rows.
//
// What bounds it, per 256 x 128 scores at head_dim 64: 2 x (9 + 8) MMAs of 67 clocks = 2,278, 32,768
// exponentials at 16 a clock = 2,048, 5,400 warp instructions at 4 a clock.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4_attn.cuh"

namespace gsvk {

namespace {

constexpr int kPBlock = 128, kPRows = 2 * kPBlock;  // rows of a softmax group and of a CTA
constexpr int kPThreads = 512;
constexpr int kPRegs = 128, kPRegsSoftmax = 152, kPRegsUnpack = 96, kPRegsRest = 112;
static_assert(2 * kPRegsSoftmax + kPRegsUnpack + kPRegsRest <= 4 * kPRegs, "register shares exceed the launch's");
constexpr uint32_t kPTmemCols = 512;

template <int HD>
constexpr bool kPSplit = HD <= 64;  // values as two fp16 numbers
template <int HD>
constexpr int kPTile = HD <= 64 ? 128 : 64;  // keys
template <int HD>
constexpr int kPTileShift = HD <= 64 ? 7 : 6;
template <int HD>
constexpr int kPCols = kPSplit<HD> ? 2 * HD : HD;  // columns of the value operand and of the sums

// What the softmax needs of a tile's keys.
template <int HD>
struct alignas(16) TileParams {
  float s[kPSplit<HD> ? 4 : kPTile<HD>], f[kPSplit<HD> ? 4 : kPTile<HD>];  // head_dim 128
  float score;          // scores' unit: z = S * score
  float unit, rescale;  // the values' unit, and the previous tile's over it
  uint32_t page_ok;
};

constexpr int kPRaw = 3;  // raw tiles in flight
template <int HD>
constexpr int kPQBytes = kPRows * HD * 2;
template <int HD>
constexpr int kPHalfBytes = kPTile<HD> * HD * 2;  // one part of a c
template <int HD>
constexpr int kPKeyBytes = 2 * kPHalfBytes<HD> + kPTile<HD> * 32;  // both, and 16 columns for b
template <int HD>
constexpr int kPValBytes = kPTile<HD> * kPCols<HD> * 2;
template <int HD>
constexpr int kPRawBytes = kPTile<HD> * (HD + 8);
template <int HD>
constexpr int kPSmem = 1024 + kPQBytes<HD> + kPRows * 32 + 2 * kPKeyBytes<HD> + 2 * kPValBytes<HD> + kPRaw * kPRawBytes<HD> +
                       2 * static_cast<int>(sizeof(TileParams<HD>));

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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// N consecutive words of shared memory, in as few loads as they allow (aligned to their size, at most 16 bytes).
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
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

// Eight codes w of a row, times s, as the sum of two fp16 numbers, in the order of the word's nibbles:
// 0 4, 1 5, 2 6, 3 7.
__device__ __forceinline__ void two_parts(uint32_t w, __half2 s, uint4* first, uint4* second) {
  const __half2 less = __halves2half2(__ushort_as_half(0x6400), __ushort_as_half(0x6400));
  uint32_t y[4], z[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t c = (w >> (4 * k) & 0x000f000fu) | 0x64006400u;  // 1024 + code
    const __half2 e = __hsub2(*reinterpret_cast<const __half2*>(&c), less);
    const __half2 h = __hmul2(e, s), r = __hfma2(e, s, __hneg2(h));  // exact: 15 bits in all
    y[k] = *reinterpret_cast<const uint32_t*>(&h);
    z[k] = *reinterpret_cast<const uint32_t*>(&r);
  }
  *first = make_uint4(y[0], y[1], y[2], y[3]);
  *second = make_uint4(z[0], z[1], z[2], z[3]);
}
// The same plus `low`.  The sum's rounding error is that of Knuth's two-sum, exact too.
__device__ __forceinline__ void two_parts(uint32_t w, __half2 s, __half2 low, uint4* first, uint4* second) {
  const __half2 less = __halves2half2(__ushort_as_half(0x6400), __ushort_as_half(0x6400));
  uint32_t y[4], z[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t c = (w >> (4 * k) & 0x000f000fu) | 0x64006400u;
    const __half2 e = __hsub2(*reinterpret_cast<const __half2*>(&c), less);
    const __half2 h = __hmul2(e, s), r = __hfma2(e, s, __hneg2(h));
    const __half2 sum = __hadd2(h, low), b = __hsub2(sum, h);
    const __half2 rest = __hadd2(__hadd2(__hsub2(h, __hsub2(sum, b)), __hsub2(low, b)), r);
    y[k] = *reinterpret_cast<const uint32_t*>(&sum);
    z[k] = *reinterpret_cast<const uint32_t*>(&rest);
  }
  *first = make_uint4(y[0], y[1], y[2], y[3]);
  *second = make_uint4(z[0], z[1], z[2], z[3]);
}
// Row r of a 16-column operand in the 32-byte swizzle: its first two columns, the others 0.
__device__ __forceinline__ void put_two(uint8_t* tile, int r, float x, float y) {
  const int flip = (r >> 2) & 1;
  *reinterpret_cast<uint4*>(tile + r * 32 + (flip << 4)) = make_uint4(f2h2(x, y), 0, 0, 0);
  *reinterpret_cast<uint4*>(tile + r * 32 + ((flip ^ 1) << 4)) = make_uint4(0, 0, 0, 0);
}

// The power of two above x > 0, and one over it (1 for 0).
__device__ __forceinline__ float unit_above(float x, float* per_unit) {
  const float u = x > 0.f ? __uint_as_float((__float_as_uint(x) & 0x7f800000u) + 0x00800000u) : 1.f;
  *per_unit = __uint_as_float(0x7f000000u - __float_as_uint(u));
  return u;
}

template <int HD>
constexpr int kPRecord = HD + 4;  // floats of a row's piece: reference, sum, (pad); values.  Four of each row, then four of each ...
constexpr int kPMaxPieces = 16;   // CTAs that share an item

template <int HD>
using PromptLine = Line<kPRows, kPTile<HD>, true>;

// A warp's 32 rows of queries (from row `row` of the request's kv head) into registers: HD / 8 lanes read a row, so
// that a load takes whole lines, and rows lie 256 / HD apart.
template <int HD>
__device__ __forceinline__ void fetch_queries(const AttnArgs& a, const Request& rq, int head, int row, uint4* x) {
  constexpr int kLanes = HD / 8, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, all = rq.n * a.group;
  row += lane / kLanes;
  // token and head of the group by steps
  int r = a.group == 1 ? row : row / a.group, h = row - r * a.group;
  const int r_step = a.group == 1 ? kRows : kRows / a.group, h_step = kRows - r_step * a.group;
  const uint16_t* src = a.q + static_cast<size_t>(head * a.group) * HD + 8 * (lane % kLanes);
#pragma unroll
  for (int i = 0; i < kLanes; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (row < all) x[i] = *reinterpret_cast<const uint4*>(src + static_cast<size_t>(rq.q0 + r) * a.q_stride + h * HD);
    row += kRows;
    r += r_step;
    h += h_step;
    if (h >= a.group) {
      h -= a.group;
      ++r;
    }
  }
}
// And from there to rows `at` .. of the operand tile, in the order of a word's nibbles, and their sums.
template <int HD>
__device__ __forceinline__ void put_queries(const uint4* x, uint32_t sign, uint8_t* sQ, uint8_t* sS, int at) {
  constexpr int kLanes = HD / 8, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, u = lane % kLanes;
  int to = at + lane / kLanes;
#pragma unroll
  for (int i = 0; i < kLanes; ++i, to += kRows) {
    float f[8];
    unpack8(x[i], f);
    float sum = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // 0 4, 1 5, 2 6, 3 7
    *reinterpret_cast<uint4*>(sQ + (to >> 7) * (kPQBytes<HD> / 2) + unit_at<HD>(to & 127, u, kPBlock)) =
        make_uint4(__byte_perm(x[i].x, x[i].z, 0x5410) ^ sign, __byte_perm(x[i].x, x[i].z, 0x7632) ^ sign,
                   __byte_perm(x[i].y, x[i].w, 0x5410) ^ sign, __byte_perm(x[i].y, x[i].w, 0x7632) ^ sign);
    // sum(q) / 128, which fp16 holds, and 2^11 times what that leaves; against 128 b and b / 16
    if (sign) sum = -sum;
    const float first = h2f(f2h(sum * 0.0078125f));
    if (u == 0) put_two(sS, to, first, fmaf(sum, 0.0078125f, -first) * 2048.f);
  }
  fence_proxy_async_shared();
}

// 8 values of a row, whole -> fp16.
__device__ __forceinline__ void put8(uint16_t* out, const float* v) {
  *reinterpret_cast<uint4*>(out) = make_uint4(f2h2(v[0], v[1]), f2h2(v[2], v[3]), f2h2(v[4], v[5]), f2h2(v[6], v[7]));
}

template <int HD>
__global__ void __launch_bounds__(kPThreads, 1) kv4_prompt_kernel(const AttnArgs a) {
  constexpr int kT = kPTile<HD>, kTs = kPTileShift<HD>;
  constexpr uint32_t kO = 256;  // TMEM column of the sums: block 0 there, block 1 at + 128; scores of block b at 128 b
  using L = PromptLine<HD>;
  extern __shared__ uint8_t prompt_raw[];
  uint8_t* smem = align_smem<1024>(prompt_raw);
  uint8_t* sQ = smem;
  uint8_t* sS = sQ + kPQBytes<HD>;  // sum(q): 16 columns
  uint8_t* sK = sS + kPRows * 32;
  uint8_t* sV = sK + 2 * kPKeyBytes<HD>;
  uint8_t* sRaw = sV + 2 * kPValBytes<HD>;
  TileParams<HD>* par = reinterpret_cast<TileParams<HD>*>(sRaw + kPRaw * kPRawBytes<HD>);
  // Buffers of a tile, which the tiles of a run take in turn whatever their item,
  __shared__ uint64_t raw_full[kPRaw], raw_free[kPRaw], k_full[2], k_free[2], v_full[2], v_free[2];
  __shared__ uint64_t par_full[2], par_free[2], most_full[2];
  // and what belongs to a block of rows: a phase for each of its tiles, or of its items.
  __shared__ uint64_t s_full[2], p_half[2], p_full[2], q_full[2], o_full[2], o_free[2];
  __shared__ uint32_t raw_ok[kPRaw];
  __shared__ __align__(16) float2 s_most[2][4];
  __shared__ uint32_t tmem_slot;
  __shared__ typename L::template Runs<kPThreads> runs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  L::template measure<kPThreads>(a, runs, static_cast<int>(gridDim.x), kPMaxPieces);
  const int me = static_cast<int>(blockIdx.x);
  const long long u0 = me * runs.share, u1 = min(runs.before[kPThreads], u0 + runs.share);
  if (u0 >= u1) {  // the whole CTA
    griddep_wait();
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kPRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_free[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_free[i], 1);
      mbar_init(&par_full[i], 4);
      mbar_init(&par_free[i], 8);
      mbar_init(&most_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_half[i], 4);
      mbar_init(&q_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 4);
    }
    fence_barrier_init();
  }
  if (warp == 13) {
    tmem_alloc(&tmem_slot, kPTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // every warp walks the run by itself
  const int share = static_cast<int>(runs.share), run = static_cast<int>(u1 - u0);
  typename L::Cursor at = L::template place<kPThreads>(a, runs, u0);
  const int sub_shift = min(a.shift, kTs), subs = kT >> sub_shift;
  // softmax groups of an item with rows
  const auto blocks_of = [&](const typename L::Cursor& c) { return c.req.n * a.group - c.block * kPRows > kPBlock ? 2 : 1; };
  int g = 0;  // tiles of the run so far

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsSoftmax));
    const int block = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t scores = tmem + lanes + block * 128, sums = tmem + lanes + kO + block * 128;
    int mine = 0, items = 0;  // this block's tiles and items so far
    int item_start = -at.tile;
    bool ok = true;
    const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // scores are taken with a positive scale
    if (block < blocks_of(at)) {
      uint4 x[HD / 8];
      fetch_queries<HD>(a, at.req, at.head, at.block * kPRows + warp * 32, x);
      put_queries<HD>(x, sign, sQ, sS, warp * 32);
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[block]);
    }
    while (g < run && ok) {

      const int all = at.req.n * a.group, row = at.block * kPRows + tid;
      const bool live_row = row < all, active = block < blocks_of(at);
      const int limit = limit_of(a, at.req, min(row, all - 1));
      const int least = __reduce_min_sync(0xffffffffu, limit);
      const int t0 = at.tile, t1 = min(at.tiles, t0 + run - g);
      float ref = -INFINITY, unit = 0.f;
      uint64_t l2 = 0, pb2 = 0;
      for (int i = t0; i < t1; ++i, ++g) {
        const TileParams<HD>& t = par[g & 1];
        ok = mbar_wait(&par_full[g & 1], static_cast<uint32_t>(g >> 1) & 1u, a.status) &&
             (!active || mbar_wait(&s_full[block], static_cast<uint32_t>(mine) & 1u, a.status));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (!active) {
          if (lane == 0) mbar_arrive(&par_free[g & 1]);
          continue;
        }
        ++mine;
        tc_fence_after();
        const float score = t.score, rescale = t.rescale;
        const uint32_t page_ok = t.page_ok;
        unit = t.unit;
        // Two passes over the scores in loops of a few dozen instructions: three roles share the instruction caches.
        const bool mask = i * kT + kT > least || page_ok != (1u << subs) - 1u;
        const int see = limit - i * kT;
        // The 16 scores of a lane that keys c .. c + 15 have (one page's), hidden ones as minus infinity.
        const auto hide = [&](int c, uint32_t* r) {
          const int n = (page_ok >> (c >> sub_shift) & 1u) ? see - c : 0;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j >= n) r[j] = 0xff800000u;
        };
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < kT; c += 32) {
          uint32_t r[32];
          tmem_ld16(scores + c, r);
          tmem_ld16(scores + c + 16, r + 16);
          tmem_ld_wait();
          if (mask) {
            hide(c, r);
            hide(c + 16, r + 16);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            tops[(j >> 1) & 3] = fmaxf(fmaxf(tops[(j >> 1) & 3], __uint_as_float(r[j])), __uint_as_float(r[j + 1]));
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * score;
        if (i == t0) {
          ref = top;
        } else if (__any_sync(0xffffffffu, top > ref + 8.f || rescale != 1.f)) {
          // a new reference or unit: bring the sums to it (these scores were issued after the last sums)
          const float to = fmaxf(ref, top);
          const float keep = to == -INFINITY ? 1.f : ex2(ref - to);
          ref = to;
          l2 = mul2(l2, pair(keep, keep));
          pb2 = mul2(pb2, pair(keep, keep));
          const float by = keep * rescale;
#pragma unroll 1
          for (int c = 0; c < kPCols<HD>; c += 16) {
            uint32_t o[16];
            tmem_ld16(sums + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
            tmem_st16(sums + c, o);
          }
          tmem_st_wait();
        }
        const float base = ref == -INFINITY ? 0.f : ref;
        const uint64_t nb = pair(-base, -base), sc = pair(score, score);
        uint64_t more = 0;  // a second sum: the distance between dependent additions
#pragma unroll 1
        for (int c = 0; c < kT; c += 16) {
          uint32_t r[16], w[8];
          tmem_ld16(scores + c, r);
          tmem_ld_wait();
          if (mask) hide(c, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 d = unpair(fma2(pair(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), sc, nb));
            const float2 e = make_float2(ex2(d.x), ex2(d.y));
            const uint64_t p = pair(e.x, e.y);
            if (j & 1) {
              more = add2(more, p);
            } else {
              l2 = add2(l2, p);
            }
            if constexpr (kPSplit<HD>) {
              w[j] = f2h2(e.x, e.y);
            } else {
              pb2 = fma2(p, *reinterpret_cast<const uint64_t*>(t.f + c + 2 * j), pb2);
              const float2 x = unpair(mul2(p, *reinterpret_cast<const uint64_t*>(t.s + c + 2 * j)));
              w[j] = f2h2(x.x, x.y);
            }
          }
          tmem_st8(scores + c / 2, w);  // over scores that have been read
          if (kT == 128 && c == 48) {   // half of the weights: their products may begin
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[block]);
          }
        }
        l2 = add2(l2, more);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&p_full[block]);
          mbar_arrive(&par_free[g & 1]);
        }
      }
      if (!ok) break;
      // the next item's queries, over those that the last scores have used, while the last sums are made
      const typename L::Cursor done = at;
      if (g < run) {
        at.next_item(a);
        if (block < blocks_of(at)) {
          uint4 x[HD / 8];
          fetch_queries<HD>(a, at.req, at.head, at.block * kPRows + warp * 32, x);
          put_queries<HD>(x, sign, sQ, sS, warp * 32);
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[block]);
        }
      }
      const int start = item_start;
      item_start += done.tiles;
      if (!active) continue;
      ok = mbar_wait(&o_full[block], static_cast<uint32_t>(items) & 1u, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ++items;
      tc_fence_after();
      const bool whole = t0 == 0 && t1 == done.tiles;
      const int first = me - (start < 0 ? (share - 1 - start) / share : 0), last = me + (start + done.tiles - 1) / share;
      const float2 ls = unpair(l2), ps = unpair(pb2);
      const float l = ls.x + ls.y, pb = ps.x + ps.y;
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      uint16_t* out = out_row(a, done.req, done.head, live_row ? row : all - 1, HD);
      // a CTA's records: its last item's, if that goes on in the next CTA, then its first's
      float4* record = reinterpret_cast<float4*>(a.long_parts + (static_cast<size_t>(me) * 2 + (me == first ? 0 : 1)) * kPRows * kPRecord<HD>) + tid;
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t o[16];
        tmem_ld16(sums + c, o);
        if constexpr (kPSplit<HD>) {
          uint32_t second[16];
          tmem_ld16(sums + HD + c, second);
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
          if (whole) {
            if (live_row) put8(out + c + 8 * u, v);
          } else {
            record[(1 + c / 4 + 2 * u) * kPRows] = make_float4(v[0], v[1], v[2], v[3]);
            record[(2 + c / 4 + 2 * u) * kPRows] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[block]);
      if (!whole) {
        *record = make_float4(ref, l, 0.f, 0.f);
        __threadfence();
        __syncwarp();
        int* ticket = a.long_tickets + first * 8 + warp;  // of these 32 rows
        int n = 0;
        if (lane == 0) n = atomicAdd(ticket, 1);
        n = __shfl_sync(0xffffffffu, n, 0);
        if (n == last - first) {  // the others' pieces are there: join them in the order of their keys
          __threadfence();
          if (lane == 0) *ticket = 0;
          constexpr int kSet = kPRows * kPRecord<HD> / 4;  // vectors of a CTA's record
          const float4* p0 = reinterpret_cast<const float4*>(a.long_parts) + static_cast<size_t>(first) * 2 * kSet + tid;
          const float4* p1 = p0 + kSet;  // the other CTAs': their second records
          const int pieces = last - first + 1;
          float top = -INFINITY, sum = 0.f;
#pragma unroll 4
          for (int k = 0; k < pieces; ++k) top = fmaxf(top, (k ? p1 + static_cast<size_t>(k) * 2 * kSet : p0)->x);
          const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
          for (int k = 0; k < pieces; ++k) {
            const float4 ml = *(k ? p1 + static_cast<size_t>(k) * 2 * kSet : p0);
            sum = fmaf(ex2(ml.x - base), ml.y, sum);
          }
          const float by = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
          for (int c = 0; c < HD; c += 8) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
            for (int k = 0; k < pieces; ++k) {
              const float4* p = k ? p1 + static_cast<size_t>(k) * 2 * kSet : p0;
              const float w = ex2(p->x - base);
              const float4 x = p[(1 + c / 4) * kPRows], y = p[(2 + c / 4) * kPRows];
              v[0] = fmaf(w, x.x, v[0]);
              v[1] = fmaf(w, x.y, v[1]);
              v[2] = fmaf(w, x.z, v[2]);
              v[3] = fmaf(w, x.w, v[3]);
              v[4] = fmaf(w, y.x, v[4]);
              v[5] = fmaf(w, y.y, v[5]);
              v[6] = fmaf(w, y.z, v[6]);
              v[7] = fmaf(w, y.w, v[7]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = sum == 0.f ? 0.f : v[k] * by;
            if (live_row) put8(out + c, v);
          }
        }
      }
    }
    tc_fence_before();
  } else if (warp < 12) {
    // ----------------------------------------------------------------- unpack
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsUnpack));
    constexpr int kPer = 128 / kT;           // threads to a key
    constexpr int kWords = HD / 8 / kPer;    // words of codes of a thread
    constexpr int kStep = 1;
    const int me_key = tid - 256, key = me_key / kPer, part = me_key % kPer;
    const int sub_bytes = kv4_head_bytes(sub_shift, HD), sub_mask = (1 << sub_shift) - 1;
    const int at_sub = (key >> sub_shift) * sub_bytes, at_key = key & sub_mask;
    bool ok = true;
    while (g < run && ok) {
      float unit = 0.f, per_unit = 0.f;
      const int keys = at.keys, t1 = min(at.tiles, at.tile + run - g);
      for (int i = at.tile; i < t1; ++i, ++g) {
        const int rs = g % kPRaw, buf = g & 1;
        const uint32_t ph = static_cast<uint32_t>(g >> 1) & 1u;
        ok = mbar_wait(&raw_full[rs], static_cast<uint32_t>(g / kPRaw) & 1u, a.status) &&
             mbar_wait(&k_free[buf], ph ^ 1u, a.status) && mbar_wait(&par_free[buf], ph ^ 1u, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t page_ok = raw_ok[rs];
        const uint8_t* sub = sRaw + rs * kPRawBytes<HD> + at_sub;
        const uint32_t kp = *reinterpret_cast<const uint32_t*>(sub + kv4_k_par(sub_shift, HD) + at_key * 4);
        const uint32_t vp = *reinterpret_cast<const uint32_t*>(sub + kv4_v_par(sub_shift, HD) + at_key * 4);
        const uint8_t* key_codes = sub + at_key * (HD / 2) + part * (kWords * 4);
        const uint8_t* value_codes = key_codes + kv4_v_codes(sub_shift, HD);
        float ks = h2f(static_cast<uint16_t>(kp)), kl = h2f(static_cast<uint16_t>(kp >> 16));
        float vs = h2f(static_cast<uint16_t>(vp)), vf = h2f(static_cast<uint16_t>(vp >> 16));
        // What lies past every row's limit or in a page that is not there counts as zero.  Keys or values that are
        // not numbers reach the rows that see them by their scores, which a row that does not see the key replaces.
        const bool seen = i * kT + key < keys && (page_ok >> (key >> sub_shift) & 1u);
        const bool number = fabsf(ks) + fabsf(kl) + fabsf(vs) + fabsf(vf) <= 3.0e38f;
        if (!seen || !number) ks = kl = vs = vf = 0.f;
        // the units: the greatest key and value (or 16 steps; for head_dim 128 the greatest step) of the tile
        {
          const float mk = warp_max(fmaxf(fabsf(kl), 16.f * ks));
          const float mv = warp_max(kPSplit<HD> ? fmaxf(fabsf(vf), 16.f * vs) : vs);
          if (lane == 0) {
            s_most[buf][warp - 8] = make_float2(mk, mv);
            mbar_arrive(&most_full[buf]);
          }
          ok = mbar_wait(&most_full[buf], ph, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        const float4 m0 = *reinterpret_cast<const float4*>(&s_most[buf][0]), m1 = *reinterpret_cast<const float4*>(&s_most[buf][2]);
        const float most_k = fmaxf(fmaxf(m0.x, m0.z), fmaxf(m1.x, m1.z)), most_v = fmaxf(fmaxf(m0.y, m0.w), fmaxf(m1.y, m1.w));
        float per_key;
        const float key_unit = unit_above(most_k, &per_key);
        float rescale = 1.f;  // the values' unit holds until something passes four times it
        if (most_v > 4.f * unit) {
          const float before = unit;
          unit = unit_above(most_v, &per_unit);
          rescale = before * per_unit;
        }
        uint8_t* keys_at = sK + buf * kPKeyBytes<HD>;
        {
          const __half2 s2 = __float2half2_rn(ks * per_key);
#pragma unroll 1
          for (int u = 0; u < kWords; u += kStep) {
            uint32_t w[kStep];
            load_words<kStep>(key_codes + 4 * u, w);
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
              uint4 first, second;
              two_parts(w[k], s2, &first, &second);
              const uint32_t to = unit_at<HD>(key, part * kWords + u + k, kT);
              *reinterpret_cast<uint4*>(keys_at + to) = first;
              *reinterpret_cast<uint4*>(keys_at + kPHalfBytes<HD> + to) = second;
            }
          }
        }
        {
          TileParams<HD>& t = par[buf];
          if (part == 0) {
            const float low = seen && !number ? __int_as_float(0x7fffffff) : kl * per_key;
            put_two(keys_at + 2 * kPHalfBytes<HD>, key, low * 128.f, low * 0.0625f);
            if constexpr (!kPSplit<HD>) {
              t.s[key] = vs * per_unit;
              t.f[key] = fmaf(8.f, vs, vf);
            }
          }
          if (me_key == 0) {
            t.score = fmaxf(fabsf(a.scale_log2) * key_unit, 1e-30f);  // not 0, which a hidden score could not be scaled by
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
        ok = mbar_wait(&v_free[buf], ph ^ 1u, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        {
          uint8_t* dst = sV + buf * kPValBytes<HD>;
          const __half2 s2 = __float2half2_rn(vs * per_unit), low2 = __float2half2_rn(vf * per_unit);
#pragma unroll 1
          for (int u = 0; u < kWords; u += kStep) {
            uint32_t w[kStep];
            load_words<kStep>(value_codes + 4 * u, w);
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
              const int to = part * kWords + u + k;
              uint4 first, second;
              if constexpr (kPSplit<HD>) {
                two_parts(w[k], s2, low2, &first, &second);
                *reinterpret_cast<uint4*>(dst + unit_at<kPCols<HD>>(key, HD / 8 + to, kT)) = second;
              } else {
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint32_t c = (w[k] >> (4 * j) & 0x000f000fu) | 0x64006400u;
                  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&c),
                                            __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));  // code - 8
                  y[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
                first = make_uint4(y[0], y[1], y[2], y[3]);
              }
              *reinterpret_cast<uint4*>(dst + unit_at<kPCols<HD>>(key, to, kT)) = first;
            }
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&v_full[buf]);
          mbar_arrive(&raw_free[rs]);
        }
      }
      if (ok && g < run) at.next_item(a);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsRest));
    if (warp == 12) {
      // ------------------------------------------------------------------ load
      const int bytes = kv4_head_bytes(sub_shift, HD);
      const auto page_of = [&]() {
        const int j = at.tile * kT + (lane << sub_shift);
        return lane < subs && j < at.keys ? a.table[static_cast<size_t>(at.seq) * a.max_blocks + (j >> a.shift)] : -1;
      };
      int page = page_of();
      bool ok = true;
      for (; g < run; ++g) {
        const int rs = g % kPRaw;
        ok = mbar_wait(&raw_free[rs], (static_cast<uint32_t>(g / kPRaw) & 1u) ^ 1u, a.status);
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
                               static_cast<size_t>(at.head) * kv4_head_bytes(a.shift, HD);
          uint8_t* dst = sRaw + rs * kPRawBytes<HD> + lane * bytes;
          if (a.shift <= kTs) {
            bulk_load(dst, src, bytes, &raw_full[rs]);
          } else {  // half of a page of 128: its four parts
            const int part = at.tile & 1, codes = kv4_v_codes(6, HD);
            bulk_load(dst, src + part * codes, codes, &raw_full[rs]);
            bulk_load(dst + codes, src + kv4_v_codes(7, HD) + part * codes, codes, &raw_full[rs]);
            bulk_load(dst + kv4_k_par(6, HD), src + kv4_k_par(7, HD) + part * 256, 256, &raw_full[rs]);
            bulk_load(dst + kv4_v_par(6, HD), src + kv4_v_par(7, HD) + part * 256, 256, &raw_full[rs]);
          }
        }
        if (g + 1 < run) {
          if (++at.tile == at.tiles) at.next_item(a);
          page = page_of();
        }
      }
      if (!ok)  // a wait ran out: leave once the copies in flight have landed
        for (int k = max(0, g - kPRaw); k < g; ++k)
          mbar_wait(&raw_full[k % kPRaw], static_cast<uint32_t>(k / kPRaw) & 1u, a.status);
    } else if (warp == 13) {
      // ------------------------------------------------------------------- MMA
      constexpr uint32_t sw = HD == 32 ? 4 : 2, sbo = HD == 32 ? 512 : 1024;  // value rows: 128 bytes
      constexpr uint32_t idesc_s = idesc_f16_f32(kPBlock, kT);
      constexpr uint32_t idesc_o = idesc_f16_f32(kPBlock, kPCols<HD>) | 1u << 16;  // B contiguous along N
      // operand descriptors of the first buffers; others lie at offsets in 16 bytes, which no field overflows on
      const uint64_t q0 = operand_desc(smem_u32(sQ), 16, sbo, sw), k0 = operand_desc(smem_u32(sK), 16, sbo, sw);
      const uint64_t qs0 = operand_desc(smem_u32(sS), 16, 256, 6);
      const uint64_t ks0 = operand_desc(smem_u32(sK) + 2 * kPHalfBytes<HD>, 16, 256, 6);
      const uint64_t v0 = operand_desc(smem_u32(sV), kT * 128, 1024, 2);
      const auto scores = [&](int tile, int b, bool last) {
        const uint64_t q = q0 + b * (kPQBytes<HD> / 32), k = k0 + (tile & 1) * (kPKeyBytes<HD> / 16);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < HD / 16; ++j)  // 16 values are 32 bytes
            tc_mma_f16(tmem + b * 128, q + (j >> 2) * (kPBlock * 8) + (j & 3) * 2,
                       k + h * (kPHalfBytes<HD> / 16) + (j >> 2) * (kT * 8) + (j & 3) * 2, idesc_s, (h | j) ? 1u : 0u);
        tc_mma_f16(tmem + b * 128, qs0 + b * (kPBlock * 2), ks0 + (tile & 1) * (kPKeyBytes<HD> / 16), idesc_s, 1u);
        tc_commit(&s_full[b]);
        if (last) tc_commit(&k_free[tile & 1]);
      };
      int tiles[2] = {0, 0}, items[2] = {0, 0};  // of each block so far
      bool ok = true;
      while (g < run && ok) {
        const int blocks = blocks_of(at), t1 = min(at.tiles, at.tile + run - g), end = g + t1 - at.tile;
        if (lane == 0) {
          ok = mbar_wait(&k_full[g & 1], static_cast<uint32_t>(g >> 1) & 1u, a.status);
          for (int b = 0; b < blocks && ok; ++b) {
            ok = mbar_wait(&q_full[b], static_cast<uint32_t>(items[b]) & 1u, a.status);
            if (!ok) break;
            tc_fence_after();
            scores(g, b, b == blocks - 1);
          }
          bool fresh = true;
          for (int i = g; i < end && ok; ++i) {
            ok = mbar_wait(&v_full[i & 1], static_cast<uint32_t>(i >> 1) & 1u, a.status) &&
                 (i + 1 == end || mbar_wait(&k_full[(i + 1) & 1], static_cast<uint32_t>((i + 1) >> 1) & 1u, a.status));
            for (int b = 0; b < blocks && ok; ++b) {
              const uint64_t v = v0 + (i & 1) * (kPValBytes<HD> / 16);
              const uint32_t weights = tmem + b * 128, sums = weights + kO;
              // the weights (the first half before the second), and for an item's first tile the sums' columns
              if (fresh) ok = mbar_wait(&o_free[b], (static_cast<uint32_t>(items[b]) & 1u) ^ 1u, a.status);
              if (kT == 128) {
                ok = ok && mbar_wait(&p_half[b], static_cast<uint32_t>(tiles[b]) & 1u, a.status);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < kT / 32; ++j)
                  tc_mma_f16_ts(sums, weights + j * 8, v + j * 128, idesc_o, fresh && j == 0 ? 0u : 1u);
              }
              ok = ok && mbar_wait(&p_full[b], static_cast<uint32_t>(tiles[b]) & 1u, a.status);
              if (!ok) break;
              ++tiles[b];
              tc_fence_after();
#pragma unroll
              for (int j = kT == 128 ? kT / 32 : 0; j < kT / 16; ++j)
                tc_mma_f16_ts(sums, weights + j * 8, v + j * 128, idesc_o, fresh && j == 0 ? 0u : 1u);
              if (b == blocks - 1) tc_commit(&v_free[i & 1]);
              if (i + 1 < end) {
                scores(i + 1, b, b == blocks - 1);  // over the weights just read: MMAs run in order
              } else {
                tc_commit(&o_full[b]);
                ++items[b];
              }
            }
            fresh = false;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        g = end;
        if (ok && g < run) at.next_item(a);
      }
    }
  }
  __syncthreads();
  if (warp == 13) {
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
    if (at.numRegs * 4 < 2 * kPRegsSoftmax + kPRegsUnpack + kPRegsRest)
      return fail(GSVK_ERR_UNSUPPORTED, "kv4_prompt_kernel: built with %d registers", at.numRegs);
    if (int rc = check_cuda(cudaFuncSetAttribute(kv4_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kPSmem<HD>),
                            "cudaFuncSetAttribute(kv4_prompt)"))
      return rc;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  return launch_pdl(kv4_prompt_kernel<HD>, dim3(static_cast<unsigned>(sm_count())), dim3(kPThreads), kPSmem<HD>, st,
                    "kv4_prompt_kernel", a);
}

}  // namespace

size_t kv4_prompt_ticket_bytes() { return (static_cast<size_t>(sm_count()) * 8 * sizeof(int) + 255) & ~static_cast<size_t>(255); }
size_t kv4_prompt_part_bytes(size_t head_dim) {
  return static_cast<size_t>(sm_count()) * 2 * kPRows * (head_dim + 4) * sizeof(float);
}

int kv4_prompt_run(const AttnArgs& a, int head_dim, cudaStream_t st) {
  return head_dim == 32 ? launch_prompt<32>(a, st) : head_dim == 64 ? launch_prompt<64>(a, st) : launch_prompt<128>(a, st);
}

}  // namespace gsvk
