// kv4_prompt.cu — attention over the paged 4-bit KV cache for requests with
// many new tokens (prompts, chunks of prompts): 128-row tiles on tcgen05.
//
// An item is 256 query rows (two blocks of 128) of one (request, kv head), its
// unit of work a tile of 128 of the keys they see (head_dim 128: 64).  One
// persistent CTA per SM takes an equal run of the line of units (kv4_attn.cuh),
// so no SM waits for the longest item, and the loads and the unpacking of an
// item overlap the end of the last.  A run's first and last item may be shared with
// other CTAs: the warp that finishes its 32 rows last joins the pieces.  Roles:
//   warps 0-3, 4-7    softmax of the first and the second block: a thread to a row (its TMEM lane)
//   warps 8-11, 12-15 unpack a tile's keys and values into fp16 operands
//   warp 16           copies the tile's pages into shared memory (cp.async.bulk)
//   warp 17           issues the MMAs:  S = Q K^T  and  O += W V, W from TMEM over the scores it came from
// The blocks' tiles take a ring of score tiles in TMEM in turn: three of 128
// columns (head_dim 128: four of 64) beside the sums, so that a softmax finds its
// next scores done while the other block's products run.  What is unpacked serves both.
//
// Mathematics.  k_j = a c + b (step, codes, low), so q.k_j = q.(a c) + sum(q) b.
// a c takes 15 bits: it goes in as the sum of two fp16 numbers, one product
// and one fused product for two codes, and b as one more column of K against
// sum(q), which is two columns of Q, 22 bits of it.  So a score is within
// 2^-22 |q||k| of the exact one (K as one fp16 number would move it by 2^-12).
// v_j goes in as two fp16 parts at head_dim 32 and 64.  At head_dim 128 that would double the MMAs:
//   sum_j p_j v_j = sum_j (p_j s_j) (e_j - 8) + sum_j p_j (f_j + 8 s_j)
// there, with the codes e - 8 as the operand and the last sum in the softmax.
// Either way the one rounding to fp16 beside the result's is that of the
// weights: 2^-11 of the values (centred within 8 steps at head_dim 128).
// p_j = 2^(z_j - reference).  The reference is six octaves (kPHead) below the maximum of the item's first tile, and moves
// only when a sum of weights shows that they outgrow fp16's range: so the maximum is taken once an item and the sums in
// TMEM are mostly left alone.  A weight is lost below 2^-31 of that maximum's: 60,000 keys that each weigh 2^-25 of a
// first strong one count (with the reference at the maximum they did not, 2^-9 of the values).  K and V (s) are divided by
// a power of two, that of K by tile, that of V the same for all rows.  The greatest then lies far up in fp16's range
// (kPKeyTop, kPValTop), which leaves bits to the others: none is off by more than 2^-28 (K) or 2^-32 (V) of it.  So a row's
// result does not hang on a key of 6e4 in its tile that it does not see (with the greatest at 1, 2^-20 of 6e4 were lost).
//
// What bounds it, per 256 x 128 scores at head_dim 64: 2 x (9 + 16) MMAs of 67 clocks = 3,350, and 32,768
// exponentials at 16 a clock = 2,048; a softmax warp takes 3,100 clocks for its 32 x 128 and some 7,000 between
// items.  Measured at 320 us on four prompts of 2,000 to 4,096 tokens, 16 heads of 64 (16,200 such tiles, 5,000
// clocks each); 400 us with one score tile a block, whose softmax waited for its products, and unpacking on four warps;
// 372 us with the codes as the value operand as at head_dim 128 (fewer MMAs, more work in the softmax); 385 us
// with the maximum taken of every tile.  The MMAs are issued by an elected lane of a converged warp: from
// inside a lane's own branch, where descriptors cannot stay in uniform registers, each took 122 clocks instead of 78.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4_attn.cuh"

namespace gsvk {

namespace {

constexpr int kPBlock = 128, kPRows = 2 * kPBlock;  // rows of a softmax group and of a CTA
constexpr int kPThreads = 576;  // 112 registers each
constexpr uint32_t kPTmemCols = 512;

template <int HD>
constexpr bool kPSplit = HD <= 64;  // values as two fp16 numbers (the time of either form is above)
template <int HD>
constexpr int kPTile = HD <= 64 ? 128 : 64;  // keys
template <int HD>
constexpr int kPTileShift = HD <= 64 ? 7 : 6;
template <int HD>
constexpr int kPSumTiles = kSumKeys / kPTile<HD>;  // of one item's sums; with more it counts as several items of the same rows
template <int HD>
constexpr bool kPSide = HD == 32;  // their parts side by side, in sums of their own; else both into the same sums
template <int HD>
constexpr int kPCols = kPSplit<HD> ? 2 * HD : HD;  // columns of the value operand
template <int HD>
constexpr int kPSums = kPSide<HD> ? 2 * HD : HD;  // and of the sums
template <int HD>
constexpr int kPRing = kPTile<HD> == 128 ? 3 : 4;  // tiles of scores in TMEM
// What the units of keys and values come to as operands, below 65,504 each: 128 b is a column of K, and a value may be four
// times its unit, as the sum of two parts of that size.
constexpr float kPKeyTop = 256.f, kPValTop = 4096.f;
constexpr float kPHead = 6.f;  // octaves from the reference to the greatest score that sets it
// A tile's sum of weights past which the reference follows: twice what scores that stay make at most.
template <int HD>
constexpr float kPFollow = 2.f * 64.f * kPTile<HD>;
// What the weights of a chunk of keys may sum to before the reference moves.  At head_dim 128 they go in times the values'
// step in their unit, which reaches four (unpack, below): either way no product passes 2^15, and fp16 holds it.
template <int HD>
constexpr float kPHigh = kPSplit<HD> ? 32768.f : 8192.f;
constexpr int kPPar = 3;  // tiles of parameters: no more than of scores, so that no group lags by a round

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
                       kPPar * static_cast<int>(sizeof(TileParams<HD>));

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
// One lane of the warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Waits for two phases, asked for at once: what each takes when it is there is a latency, some 100 clocks beside the
// other warps.
__device__ __forceinline__ bool wait_for(uint64_t* x, uint32_t px, uint64_t* y, uint32_t py, uint32_t* status) {
  const bool there = mbar_try_wait(x, px) & mbar_try_wait(y, py);
  return there || (mbar_wait(x, px, status) && mbar_wait(y, py, status));
}
// A value that is the same in every lane, known to be so.
__device__ __forceinline__ int same(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
// CTAs that share an item at most: 100 rows over 30,000 keys, 2 heads of 64, take 65 us, with 6 97 and with 40 83.
constexpr int kPMaxPieces = 16;

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
  constexpr int kR = kPRing<HD>;
  constexpr uint32_t kO = kR * kT;  // TMEM column of the sums, block after block; below, the ring of scores
  static_assert(kO + 2 * kPSums<HD> <= kPTmemCols);
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
  __shared__ uint64_t par_full[kPPar], par_free[kPPar], most_full[2][2];
  // the scores and weights of a block's tile, which take the ring in turn,
  __shared__ uint64_t s_full[kR], p_full[kR];
  // and what belongs to a block of rows: a phase for each of its items, o_tile for each of its tiles.
  __shared__ uint64_t q_full[2], o_full[2], o_free[2], o_tile[2];
  __shared__ uint32_t raw_ok[kPRaw];
  __shared__ __align__(16) float s_most[2][2][4];
  __shared__ uint32_t tmem_slot;
  __shared__ typename L::template Runs<kPThreads> runs;
  const int tid = threadIdx.x, warp = same(tid >> 5), lane = tid & 31;

  L::template measure<kPThreads>(a, runs, static_cast<int>(gridDim.x),
                                 [](int most) { return (most + kPMaxPieces - 1) / kPMaxPieces; });
  const int me = static_cast<int>(blockIdx.x);
  const long long u0 = me * runs.share, u1 = min(runs.before[kPThreads], u0 + runs.share);
  if (u0 >= u1) {  // the whole CTA
    griddep_wait();
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kPRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_free[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_free[i], 1);
      mbar_init(&most_full[0][i], 4);
      mbar_init(&most_full[1][i], 4);
      mbar_init(&q_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 4);
      mbar_init(&o_tile[i], 1);
    }
    for (int i = 0; i < kPPar; ++i) {
      mbar_init(&par_full[i], 8);
      mbar_init(&par_free[i], 8);
    }
    for (int i = 0; i < kR; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    fence_barrier_init();
  }
  if (warp == 17) {
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
    const int block = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t sums = tmem + lanes + kO + block * kPSums<HD>;
    int mine = 0, items = 0;  // this block's tiles and items so far
    int slot = 0;  // the ring's turn of the item's first tile, its place and the parity of its round
    uint32_t round = 0;
    const auto advance = [&](int n) {
      slot += n;
      if (slot >= kR) slot -= kR, round ^= 1u;
    };
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
      const int blocks = blocks_of(at);
      const bool live_row = row < all, active = block < blocks;
      const int limit = limit_of(a, at.req, min(row, all - 1));
      const int least = __reduce_min_sync(0xffffffffu, limit);
      const int t0 = at.tile, t1 = min(min(at.tiles, t0 + run - g), t0 + kPSumTiles<HD>);
      float ref = -INFINITY, unit = 0.f, tile_sum = 0.f;
      uint64_t l2 = 0, pb2 = 0;
      for (int i = t0; i < t1; ++i, ++g) {
        const TileParams<HD>& t = par[g % kPPar];
        // Its own scores' place; a group without rows waits for the first block's: nobody may fall a round of the ring
        // behind or get one ahead, where a phase has the parity of another.
        if (active && block) advance(1);
        const int here = slot;
        ok = wait_for(&par_full[g % kPPar], static_cast<uint32_t>(g / kPPar) & 1u, &s_full[here], round, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (!active) {
          advance(1);
          if (lane == 0) mbar_arrive(&par_free[g % kPPar]);
          continue;
        }
        advance(blocks - block);
        const uint32_t scores = tmem + lanes + here * kT;
        tc_fence_after();
        const float score = t.score;
        const uint32_t page_ok = t.page_ok;
        unit = t.unit;
        // Loops of some dozen instructions: the roles share the instruction caches.
        const bool mask = i * kT + kT > least || page_ok != (1u << subs) - 1u;
        const int see = limit - i * kT;
        // 16 scores r of keys c .. c + 15 (one page's): hidden ones as minus infinity.
        const auto hide = [&](int c, uint32_t* r) {
          const int n = (page_ok >> (c >> sub_shift) & 1u) ? see - c : 0;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j >= n) r[j] = 0xff800000u;
        };
        // Scores c .. c + kChunk - 1 into r.
        constexpr int kChunk = 32;
        const auto fetch = [&](int c, uint32_t* r) {
          tmem_ld16(scores + c, r);
          tmem_ld16(scores + c + 16, r + 16);
          tmem_ld_wait();
          if (mask) {
            hide(c, r);
            hide(c + 16, r + 16);
          }
        };
        // The reference is set by the first tile's maximum.  It follows a tile late when a tile's sum has passed kPFollow, or
        // at once when that of a chunk passes kPHigh: every weight stays in fp16's range with no maximum to take of each tile.
        float rescale = t.rescale;
        bool follow = i == t0 || __any_sync(0xffffffffu, tile_sum > kPFollow<HD> || rescale != 1.f);
        float to = ref;
        if (tile_sum > kPFollow<HD>) to += static_cast<float>(static_cast<int>(__float_as_uint(tile_sum) >> 23) - 127) - kPHead;
        tile_sum = 0.f;
        int c = 0;
        bool at_once = i == t0;
        for (;;) {
          if (follow) {
            if (at_once) {  // the maximum of what is left of the tile
              float top = -INFINITY;
#pragma unroll 1
              for (int k = c; k < kT; k += kChunk) {
                uint32_t r[kChunk];
                fetch(k, r);
                float x[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < kChunk; j += 2)
                  x[(j >> 1) & 3] = fmaxf(fmaxf(x[(j >> 1) & 3], __uint_as_float(r[j]) * score),
                                          __uint_as_float(r[j + 1]) * score);
                top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
              }
              to = fmaxf(to, top - kPHead);
            }
            if (i == t0) {
              ref = to;
            } else {
              // Bring the sums to the new reference or unit, once the last tile's products are in them (those of the one
              // before are: these scores were issued after them), and this tile's weights so far: by a power of two.
              ok = mbar_wait(&o_tile[block], static_cast<uint32_t>(mine - 1) & 1u, a.status);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              tc_fence_after();
              to = to > ref ? (ref == -INFINITY ? to : ref + ceilf(to - ref)) : ref;
              const float keep = to == -INFINITY ? 1.f : ex2(ref - to);
              ref = to;
              tile_sum *= keep;
              l2 = mul2(l2, pair(keep, keep));
              pb2 = mul2(pb2, pair(keep, keep));
              const float by = keep * rescale;
#pragma unroll 1
              for (int k = 0; k < kPSums<HD>; k += 8) {
                uint32_t o[8];
                tmem_ld8(sums + k, o);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
                tmem_st8(sums + k, o);
              }
#pragma unroll 1
              for (int k = 0; k < c / 2; k += 8) {
                uint32_t w[8];
                tmem_ld8(scores + k, w);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  w[j] = f2h2(h2f(static_cast<uint16_t>(w[j])) * keep, h2f(static_cast<uint16_t>(w[j] >> 16)) * keep);
                tmem_st8(scores + k, w);
              }
              tmem_st_wait();
            }
          }
          // a row that has seen nothing yet: weights without end for all that it sees, which sets its reference
          const bool none = ref == -INFINITY;
          const float nbase = none ? 1.0e38f : -ref, high = none ? 0.f : kPHigh<HD>;
          const uint64_t nb = pair(nbase, nbase), sc = pair(score, score);
          follow = false;
#pragma unroll 1
          for (; c < kT; c += kChunk) {
            uint32_t r[kChunk], w[kChunk / 2];
            fetch(c, r);
            uint64_t even = 0, odd = 0;  // two sums: the distance between dependent additions
#pragma unroll
            for (int j = 0; j < kChunk / 2; ++j) {
              const float2 d = unpair(fma2(pair(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), sc, nb));
              const float2 e = make_float2(ex2(d.x), ex2(d.y));
              const uint64_t p = pair(e.x, e.y);
              if (j & 1) {
                odd = add2(odd, p);
              } else {
                even = add2(even, p);
              }
              if constexpr (kPSplit<HD>) {
                w[j] = f2h2(e.x, e.y);
              } else {
                const float2 x = unpair(mul2(p, *reinterpret_cast<const uint64_t*>(t.s + c + 2 * j)));
                w[j] = f2h2(x.x, x.y);
                r[2 * j] = __float_as_uint(e.x), r[2 * j + 1] = __float_as_uint(e.y);
              }
            }
            even = add2(even, odd);
            const float2 s2 = unpair(even);
            const float sum = s2.x + s2.y;
            if (__any_sync(0xffffffffu, sum > high)) {
              follow = true;
              break;
            }
            tile_sum += sum;
            if constexpr (!kPSplit<HD>) {
#pragma unroll
              for (int j = 0; j < kChunk / 2; ++j)
                pb2 = fma2(pair(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])),
                           *reinterpret_cast<const uint64_t*>(t.f + c + 2 * j), pb2);
            }
            tmem_st8(scores + c / 2, w);
            tmem_st8(scores + c / 2 + 8, w + 8);
          }
          if (!follow) break;
          rescale = 1.f;
          to = ref;
          at_once = true;
        }
        l2 = add2(l2, pair(tile_sum, 0.f));
        if (!ok) break;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&p_full[here]);
          mbar_arrive(&par_free[g % kPPar]);
        }
        ++mine;
      }
      if (!ok) break;
      // the next item's queries, over those that the last scores have used, while the last sums are made; or more of this
      // item's keys
      const typename L::Cursor done = at;
      const bool more = t1 < done.tiles && g < run;
      if (more) {
        at.tile = t1;
        if (active && lane == 0) mbar_arrive(&q_full[block]);
      } else if (g < run) {
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
      if (!more) item_start += done.tiles;
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
      // in which it has the item's earlier keys already, where there are more than kSumKeys
      const bool earlier = t0 > max(0, -start);
      float by = 1.f, by0 = 0.f, all_l = l;
      if (earlier) {
        const float2 before = *reinterpret_cast<const float2*>(record);
        const float top = fmaxf(ref, before.x), base = top == -INFINITY ? 0.f : top;
        by = ex2(ref - base);
        by0 = ex2(before.x - base);
        ref = top;
        all_l = fmaf(l, by, before.y * by0);
      }
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t o[16];
        tmem_ld16(sums + c, o);
        if constexpr (kPSide<HD>) {
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
            float4* r0 = record + (1 + c / 4 + 2 * u) * kPRows;
            float4* r1 = r0 + kPRows;
            if (earlier) {
              const float4 x = *r0, y = *r1;
              v[0] = fmaf(v[0], by, x.x * by0);
              v[1] = fmaf(v[1], by, x.y * by0);
              v[2] = fmaf(v[2], by, x.z * by0);
              v[3] = fmaf(v[3], by, x.w * by0);
              v[4] = fmaf(v[4], by, y.x * by0);
              v[5] = fmaf(v[5], by, y.y * by0);
              v[6] = fmaf(v[6], by, y.z * by0);
              v[7] = fmaf(v[7], by, y.w * by0);
            }
            *r0 = make_float4(v[0], v[1], v[2], v[3]);
            *r1 = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[block]);
      if (!whole) {
        *record = make_float4(ref, all_l, 0.f, 0.f);
        if (more) continue;
        __threadfence();
        __syncwarp();
        // of these 32 rows; none of an item of this CTA alone, whose place is the last item's
        int* ticket = a.long_tickets + first * 8 + warp;
        int n = 0;
        if (lane == 0 && first != last) n = atomicAdd(ticket, 1);
        n = __shfl_sync(0xffffffffu, n, 0);
        if (n == last - first) {  // the others' pieces are there: join them in the order of their keys
          __threadfence();
          if (lane == 0 && first != last) *ticket = 0;
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
  } else if (warp < 16) {
    // ----------------------------------------------------------------- unpack: warps 8-11 the keys, 12-15 the values
    constexpr int kPer = 128 / kT;         // threads to a key
    constexpr int kWords = HD / 8 / kPer;  // words of codes of a thread
    const int v = warp >= 12;              // 1: the values
    const int me_key = (tid - 256) & 127, key = me_key / kPer, part = me_key % kPer;
    const int sub_bytes = kv4_head_bytes(sub_shift, HD), sub_mask = (1 << sub_shift) - 1;
    const int at_sub = (key >> sub_shift) * sub_bytes, at_key = key & sub_mask;
    const int at_codes = at_sub + (v ? kv4_v_codes(sub_shift, HD) : 0) + at_key * (HD / 2) + part * (kWords * 4);
    bool ok = true;
    while (g < run && ok) {
      float unit = 0.f, per_unit = 0.f;
      const int keys = at.keys, t1 = min(at.tiles, at.tile + run - g);
      for (int i = at.tile; i < t1; ++i, ++g) {
        const int rs = g % kPRaw, buf = g & 1;
        const uint32_t ph = static_cast<uint32_t>(g >> 1) & 1u;
        ok = wait_for(&raw_full[rs], static_cast<uint32_t>(g / kPRaw) & 1u, &par_free[g % kPPar],
                      (static_cast<uint32_t>(g / kPPar) & 1u) ^ 1u, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t page_ok = raw_ok[rs];
        const uint8_t* sub = sRaw + rs * kPRawBytes<HD> + at_sub;
        const uint32_t kp = *reinterpret_cast<const uint32_t*>(sub + kv4_k_par(sub_shift, HD) + at_key * 4);
        const uint32_t vp = *reinterpret_cast<const uint32_t*>(sub + kv4_v_par(sub_shift, HD) + at_key * 4);
        const uint8_t* codes = sRaw + rs * kPRawBytes<HD> + at_codes;
        // What lies past every row's limit or in a page that is not there counts as zero.  Keys or values that are
        // not numbers reach the rows that see them by their scores, which a row that does not see the key replaces.
        const bool seen = i * kT + key < keys && (page_ok >> (key >> sub_shift) & 1u);
        const bool number = (kp & 0x7c00u) != 0x7c00u && (kp & 0x7c000000u) != 0x7c000000u && (vp & 0x7c00u) != 0x7c00u &&
                            (vp & 0x7c000000u) != 0x7c000000u;
        const uint32_t mine = !seen || !number ? 0u : v ? vp : kp;
        const float step = h2f(static_cast<uint16_t>(mine)), low = h2f(static_cast<uint16_t>(mine >> 16));
        // the unit: the greatest key or value (or 16 steps; of values at head_dim 128 the greatest step) of the tile
        {
          const float m = warp_max(v && !kPSplit<HD> ? step : fmaxf(fabsf(low), 16.f * step));
          if (lane == 0) {
            s_most[v][buf][warp & 3] = m;
            mbar_arrive(&most_full[v][buf]);
          }
          ok = mbar_wait(&most_full[v][buf], ph, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        const float4 m4 = *reinterpret_cast<const float4*>(&s_most[v][buf][0]);
        const float most = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
        TileParams<HD>& t = par[g % kPPar];
        if (!v) {
          const float key_unit = unit_above(most, &per_unit) * (1.f / kPKeyTop);
          per_unit *= kPKeyTop;
          if (me_key == 0) {
            t.score = fmaxf(fabsf(a.scale_log2) * key_unit, 1e-30f);  // not 0, which a hidden score could not be scaled by
            t.page_ok = page_ok;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&par_full[g % kPPar]);
          ok = mbar_wait(&k_free[buf], ph ^ 1u, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* dst = sK + buf * kPKeyBytes<HD>;
          const __half2 s2 = __float2half2_rn(step * per_unit);
#pragma unroll 1
          for (int u = 0; u < kWords; ++u) {
            uint4 first, second;
            two_parts(*reinterpret_cast<const uint32_t*>(codes + 4 * u), s2, &first, &second);
            const uint32_t to = unit_at<HD>(key, part * kWords + u, kT);
            *reinterpret_cast<uint4*>(dst + to) = first;
            *reinterpret_cast<uint4*>(dst + kPHalfBytes<HD> + to) = second;
          }
          if (part == 0) {
            const float b = seen && !number ? __int_as_float(0x7fffffff) : low * per_unit;
            put_two(dst + 2 * kPHalfBytes<HD>, key, b * 128.f, b * 0.0625f);
          }
        } else {
          float rescale = 1.f;  // the values' unit holds until something passes four times it
          if (most > 4.f * unit) {
            const float before = unit;
            unit = unit_above(most, &per_unit);
            rescale = before * per_unit;
          }
          if constexpr (!kPSplit<HD>) {
            if (part == 0) {
              t.s[key] = step * per_unit;
              t.f[key] = fmaf(8.f, step, low);
            }
          }
          if (me_key == 0) {
            t.unit = kPSplit<HD> ? unit * (1.f / kPValTop) : unit;
            t.rescale = rescale;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&par_full[g % kPPar]);
          ok = mbar_wait(&v_free[buf], ph ^ 1u, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* dst = sV + buf * kPValBytes<HD>;
          const float up = per_unit * kPValTop;
          const __half2 s2 = __float2half2_rn(step * up), low2 = __float2half2_rn(low * up);
#pragma unroll 1
          for (int u = 0; u < kWords; ++u) {
            const int to = part * kWords + u;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + 4 * u);
            uint4 first, second;
            if constexpr (kPSplit<HD>) {
              two_parts(w, s2, low2, &first, &second);
              *reinterpret_cast<uint4*>(dst + unit_at<kPCols<HD>>(key, HD / 8 + to, kT)) = second;
            } else {
              uint32_t y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t c = (w >> (4 * j) & 0x000f000fu) | 0x64006400u;
                const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&c),
                                          __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));  // code - 8
                y[j] = *reinterpret_cast<const uint32_t*>(&h);
              }
              first = make_uint4(y[0], y[1], y[2], y[3]);
            }
            *reinterpret_cast<uint4*>(dst + unit_at<kPCols<HD>>(key, to, kT)) = first;
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(v ? &v_full[buf] : &k_full[buf]);
          mbar_arrive(&raw_free[rs]);
        }
      }
      if (ok && g < run) at.next_item(a);
    }
  } else {
    if (warp == 16) {
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
    } else if (warp == 17) {
      // ------------------------------------------------------------------- MMA
      constexpr uint32_t sw = HD == 32 ? 4 : 2, sbo = HD == 32 ? 512 : 1024;  // value rows: 128 bytes
      constexpr uint32_t idesc_s = idesc_f16_f32(kPBlock, kT);
      constexpr uint32_t idesc_o = idesc_f16_f32(kPBlock, kPSums<HD>) | 1u << 16;  // B contiguous along N
      // operand descriptors of the first buffers; others lie at offsets in 16 bytes, which no field overflows on
      // The whole warp runs this role and one elected lane issues: so addresses and descriptors stay in uniform registers,
      // which the MMAs take them from.
      const uint32_t tm = static_cast<uint32_t>(same(static_cast<int>(tmem)));
      const uint32_t base = static_cast<uint32_t>(same(static_cast<int>(smem_u32(smem))));
      constexpr uint32_t oS = kPQBytes<HD>, oK = oS + kPRows * 32, oV = oK + 2 * kPKeyBytes<HD>;
      // operand descriptors of the first buffers; others lie at offsets in 16 bytes, which no field overflows on
      const uint64_t q0 = operand_desc(base, 16, sbo, sw), k0 = operand_desc(base + oK, 16, sbo, sw);
      const uint64_t qs0 = operand_desc(base + oS, 16, 256, 6);
      const uint64_t ks0 = operand_desc(base + oK + 2 * kPHalfBytes<HD>, 16, 256, 6);
      const uint64_t v0 = operand_desc(base + oV, kT * 128, 1024, 2);
      // scores of block b and K buffer `buf` into a place of the ring
      const auto scores = [&](int place, int buf, int b, bool last) {
        const uint32_t at_key = static_cast<uint32_t>(buf * (kPKeyBytes<HD> / 16));
        const uint64_t q = q0 + static_cast<uint32_t>(b * (kPQBytes<HD> / 32)), k = k0 + at_key;
        const uint64_t qs = qs0 + static_cast<uint32_t>(b * (kPBlock * 2)), ks = ks0 + at_key;
        const uint32_t to = tm + place * kT;
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < HD / 16; ++j)  // 16 values are 32 bytes
              tc_mma_f16(to, q + (j >> 2) * (kPBlock * 8) + (j & 3) * 2,
                         k + h * (kPHalfBytes<HD> / 16) + (j >> 2) * (kT * 8) + (j & 3) * 2, idesc_s, (h | j) ? 1u : 0u);
          tc_mma_f16(to, qs, ks, idesc_s, 1u);
          tc_commit(&s_full[place]);
          if (last) tc_commit(&k_free[buf]);
        }
        __syncwarp();
      };
      // a step's weights times 16 keys j of its values
      const auto product = [&](uint32_t sums, uint32_t weights, uint64_t v, int j, uint32_t accumulate) {
        tc_mma_f16_ts(sums, weights + j * 8, v + j * 128, idesc_o, accumulate);
        if constexpr (kPSplit<HD> && !kPSide<HD>) tc_mma_f16_ts(sums, weights + j * 8, v + kT * 8 + j * 128, idesc_o, 1u);
      };
      const auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.status)) != 0;
      };
      int item = 0, item1 = 0;  // so far: all, and those of two blocks
      int place = 0;  // the ring's turn of the item's next step, and the parity of its round
      uint32_t round = 0;
      bool ok = true;
      g = 0;
      const int n_run = same(run);
      while (g < n_run && ok) {
        const int blocks = same(blocks_of(at));
        const int end = same(g + min(min(at.tiles - at.tile, n_run - g), kPSumTiles<HD>));
        // Steps: the first block's tile, the second's, the next tile ...  The scores run ahead of the sums by the
        // ring, one block's by two tiles (there are two buffers of K): a softmax group finds its next scores done.
        const int lead = blocks == 2 ? kR : 2;
        int next = g, next_b = 0, next_place = place;  // of the scores
        const auto issue = [&]() {
          if (next == end) return true;
          if (next_b == 0 && !wait(&k_full[next & 1], static_cast<uint32_t>(next >> 1) & 1u)) return false;
          if (next == g && !wait(&q_full[next_b], static_cast<uint32_t>(next_b ? item1 : item) & 1u)) return false;
          tc_fence_after();
          scores(next_place, next & 1, next_b, next_b == blocks - 1);
          if (++next_place == kR) next_place = 0;
          if (++next_b == blocks) next_b = 0, ++next;
          return true;
        };
#pragma unroll 1
        for (int k = 0; k < lead && ok; ++k) ok = issue();
#pragma unroll 1
        for (int i = g, b = 0; i < end && ok;) {
          const uint64_t v = v0 + static_cast<uint32_t>((i & 1) * (kPValBytes<HD> / 16));
          const uint32_t weights = tm + place * kT, sums = tm + kO + b * kPSums<HD>;
          const uint32_t more = i > g;
          // for an item's first tile the sums' columns; the values and the weights
          ok = (more || wait(&o_free[b], (static_cast<uint32_t>(b ? item1 : item) & 1u) ^ 1u)) &&
               __all_sync(0xffffffffu, wait_for(&v_full[i & 1], static_cast<uint32_t>(i >> 1) & 1u, &p_full[place], round,
                                                a.status));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kT / 16; ++j) product(sums, weights, v, j, j ? 1u : more);
            tc_commit(&o_tile[b]);
            if (i + 1 == end) tc_commit(&o_full[b]);
            if (b == blocks - 1) tc_commit(&v_free[i & 1]);
          }
          __syncwarp();
          if (++place == kR) place = 0, round ^= 1u;
          ok = issue();  // over weights that have been read: MMAs run in order
          if (++b == blocks) b = 0, ++i;
        }
        ++item;
        if (blocks == 2) ++item1;
        at.tile += end - g;
        g = end;
        if (ok && g < n_run && at.tile == at.tiles) at.next_item(a);
      }
    }
  }
  __syncthreads();
  if (warp == 17) {
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
