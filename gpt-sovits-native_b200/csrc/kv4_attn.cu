// kv4_attn.cu — attention over the paged 4-bit KV cache (gsvk_kv4_attention):
// the kernel for requests with few new tokens (decoding, drafts) and the entry
// points.  Long runs of new tokens are kv4_prompt.cu's.
#include <algorithm>

#include "gsvk_internal.hpp"
#include "kv4_attn.cuh"

namespace gsvk {

namespace {

// ------------------------------------------------------------ few query rows
// Work.  The line of units (kv4_attn.cuh) in tiles of 64 keys is cut into one
// run per warp of the grid, so ragged lengths leave no warp idle and a single
// long request fills the GPU.  Every CTA works the line out for itself from
// the lengths.  An item cut between warps is joined by the warp that
// arrives last, in the order of the runs, so results do not depend on timing.
//
// Data.  A tile is one contiguous block per page and head; a lane per page
// copies it with cp.async.bulk into its warp's own ring of shared memory,
// several tiles ahead.  Warps never wait for one another.
//
// Mathematics.  With k_j = a_j c_j + b_j (step, codes, low) the score is
//   q.k_j = a_j (q.c_j) + b_j sum(q),
// and sum_j p_j v_j = sum_j (p_j a_j) c_j + sum_j p_j b_j, so both products run
// on the tensor cores (m16n8k16, fp32 sums) over the codes alone.  A nibble
// pair masked out of a word, (w >> s) & 0x000f000f, is a pair of fp16
// subnormals worth c 2^-24, which the tensor cores multiply exactly; the
// nibbles at bits 4 and 20 are worth 16 c 2^-24 and have sums of their own.
// So a code costs 5/8 of an instruction to unpack for the scores, and 5/4 for
// the values, where two tokens' words are first interleaved by prmt and the codes are
// taken less 8 (low then stands for code 8): the tensor cores' sums are cut off, not
// rounded, and over 60,000 keys sums of positive codes moved the result by 1.6e-3 of
// its size, at 135 us for 8 rows of 32 heads of 128 over as many keys each (2.1e-4 and
// 156 us so, the rounding of the result; a sum of its own for each tile, 4e-4 and 151 us).
// The weights p_j a_j, scaled by a power of two so that the greatest step seen
// comes to less than 2^15 (kTop), go in as two fp16 parts.  Their sum holds 22
// bits of every weight down to 2^-17 of that bound, and all of them to
// within 2^-40 of it: so 60,000 keys that each weigh 2^-25 of a first strong one
// count in full (with weights up to 1 they were lost, 2^-9 of the values).  Up to
// 8 rows, the second part takes the unused rows 8..15 of the same MMA.
//
// Between the products the scores pass through shared memory to a layout with
// two keys to a lane, so that the softmax costs what the rows there are cost
// (not the 8 or 16 of an MMA), a key's parameters are converted once, and a
// maximum is one redux.
constexpr int kTile = 64;          // keys of a unit
constexpr int kSplitWarps = 4;     // warps of a CTA
// Units that a warp takes at least of an item of `most`: with p pieces the warps take most / p units each and the join
// p pieces, so the best p goes with the root; a unit takes about eight times a piece's part of the join of up to
// four rows, four times that of sixteen.  One request of 4,000 keys, 8 heads of 64: 12 us (1 row), 16 (4 rows) and 39
// (16); with up to 64 pieces whatever the length 14, 39 and 138, of 60,000 keys 39, 77 and 223 against 38, 48 and 110.
template <int ROWS>
__device__ __forceinline__ int least_share(int most) {
  return static_cast<int>(sqrtf(static_cast<float>(most) * (ROWS >= 8 ? 0.25f : 0.125f)) + 0.5f);
}

constexpr float kTop = 32768.f;  // what the weights' unit comes to as an operand: fp16's range ends at 65,504

// As many CTAs as registers and shared memory take; with one less an SM the long caches' 156 us were 40 % longer.
template <int HD, int ROWS>
constexpr int kCtasPerSm = HD == 128 ? 2 : (HD == 64 ? 3 : 4) - (ROWS == 16);
template <int HD, int ROWS>
constexpr int kStages = HD == 32 ? 4 : 3;
template <int HD>
constexpr int kTileBytes = kTile * (HD + 8);
template <int HD>
constexpr int kRecord = HD + 4;  // floats of a joined row: maximum, sum, (pad), values
constexpr int kRecords = 3;      // of a warp
// Scores (two keys each, 64 bits) or weights (two fp16 each, first and second part) of a row between
// the products: 32 pairs, and 32 bytes that keep eight rows off each other's banks.
constexpr int kRowBytes = 32 * 8 + 32;
template <int HD, int ROWS>
constexpr int kWarpBytes = kStages<HD, ROWS> * kTileBytes<HD> + (ROWS * kRowBytes + 127) / 128 * 128;

__device__ __forceinline__ void mma_16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same without a sum to add to.
__device__ __forceinline__ void mma_16816_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The nibbles at bits SHIFT and SHIFT + 16, less 8, as fp16 numbers (of bits 4 and 20: 16 times that).
template <int SHIFT>
__device__ __forceinline__ uint32_t centred(uint32_t w) {
  const uint32_t c = (w & (0x000f000fu << SHIFT)) | 0x64006400u;  // 1024 + code
  const __half2 less = __halves2half2(__ushort_as_half(SHIFT ? 0x6480 : 0x6408), __ushort_as_half(SHIFT ? 0x6480 : 0x6408));
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&c), less);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The state of ROWS query rows over the tiles seen so far.  As an MMA operand
// lane (g, t) = (lane / 4, lane % 4) has row g (ROWS = 16: and row g + 8); its
// part of the sums o is head_dim / 4 dimensions from t head_dim / 4 on (up to 8 rows: in two
// parts).  m is the same in every lane; l and pb are a lane's parts of sum p and sum p b.
template <int HD, int ROWS>
struct RowState {
  static constexpr int kR = ROWS == 16 ? 2 : 1;
  uint32_t q[HD / 32][2][2 * kR];  // [word][even, odd nibbles][A registers]
  float o[HD / 8][4];
  float m[ROWS], l[ROWS], pb[ROWS], qsum[ROWS];
  float unit;  // the weights' power of two
};

template <int HD, int ROWS>
__device__ __forceinline__ void load_rows(const AttnArgs& a, const Request& rq, int head, int block, int lane,
                                          RowState<HD, ROWS>& s) {
  constexpr int kR = RowState<HD, ROWS>::kR;
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int k = 0; k < kR; ++k) {
    const int row = block * ROWS + 8 * k + g;
    const bool ok = 8 * k + g < ROWS && row < rq.n * a.group;
    const int r = !ok || rq.n == 1 ? 0 : row / a.group;
    const uint16_t* src = a.q + static_cast<size_t>(rq.q0 + r) * a.q_stride +
                          static_cast<size_t>(head * a.group + (row - r * a.group)) * HD + t * (HD / 4);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < HD / 32; ++w) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (ok) x = *reinterpret_cast<const uint4*>(src + 8 * w);
      float f[8];
      unpack8(x, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += f[i];
      s.q[w][0][k] = __byte_perm(x.x, x.z, 0x5410);
      s.q[w][0][kR + k] = __byte_perm(x.y, x.w, 0x5410);
      s.q[w][1][k] = __byte_perm(x.x, x.z, 0x7632);
      s.q[w][1][kR + k] = __byte_perm(x.y, x.w, 0x7632);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    sum *= a.scale_log2;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * k + i < ROWS) s.qsum[8 * k + i] = __shfl_sync(0xffffffffu, sum, 4 * i);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    s.m[r] = -INFINITY;
    s.l[r] = 0.f;
    s.pb[r] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) s.o[i][c] = 0.f;
  s.unit = 0.f;
}

// One tile.  rows: rows of the block; limit: in lane r, the keys of the tile that row r sees; page_ok: a bit for each of
// the tile's pages that is there.
template <int HD, int ROWS>
__device__ __forceinline__ void add_tile(const uint8_t* tile, uint8_t* mid, int sub_shift, float scale_log2, int rows,
                                         int limit, unsigned page_ok, int lane, RowState<HD, ROWS>& s) {
  constexpr int kR = RowState<HD, ROWS>::kR;
  const int g = lane >> 2, t = lane & 3;
  const int sub_bytes = kv4_head_bytes(sub_shift, HD), sub_mask = (1 << sub_shift) - 1;
  // ------------------------------------------------------------------ scores
  // Column g of a score MMA over keys 8 i .. 8 i + 7 is key 8 i + g / 2 + 4 (g % 2), so lane (g, t) gets keys
  // 8 i + t and 8 i + 4 + t, the pair that the value MMA wants of it; pair (i, t) lies at place
  // 8 (i / 2) + 2 t + i % 2 of a row.
  constexpr int kSide = HD / 32;  // MMAs of several eights of keys side by side: each waits for its own last one only
#pragma unroll
  for (int i0 = 0; i0 < kTile / 8; i0 += kSide) {
    uint32_t w[kSide][HD / 32];
    float even[kSide][4], odd[kSide][4];
#pragma unroll
    for (int i = 0; i < kSide; ++i) {
      const int j = 8 * (i0 + i) + (g >> 1) + 4 * (g & 1);
      const uint8_t* src = tile + (j >> sub_shift) * sub_bytes + (j & sub_mask) * (HD / 2) + t * (HD / 8);
      if constexpr (HD == 32) {
        w[i][0] = *reinterpret_cast<const uint32_t*>(src);
      } else if constexpr (HD == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        w[i][0] = v.x, w[i][1] = v.y;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
      }
    }
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
      const uint32_t *q0 = s.q[u][0], *q1 = s.q[u][1];
      const uint32_t e1 = kR == 2 ? q0[1] : 0u, e2 = q0[kR], e3 = kR == 2 ? q0[3 % (2 * kR)] : 0u;
      const uint32_t o1 = kR == 2 ? q1[1] : 0u, o2 = q1[kR], o3 = kR == 2 ? q1[3 % (2 * kR)] : 0u;
#pragma unroll
      for (int i = 0; i < kSide; ++i) {
        const uint32_t x = w[i][u], y = x >> 8;
        if (u == 0) {
          mma_16816_first(even[i], q0[0], e1, e2, e3, x & 0x000f000fu, y & 0x000f000fu);
          mma_16816_first(odd[i], q1[0], o1, o2, o3, x & 0x00f000f0u, y & 0x00f000f0u);
        } else {
          mma_16816(even[i], q0[0], e1, e2, e3, x & 0x000f000fu, y & 0x000f000fu);
          mma_16816(odd[i], q1[0], o1, o2, o3, x & 0x00f000f0u, y & 0x00f000f0u);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kSide; ++i) {
      const int place = 8 * ((i0 + i) >> 1) + 2 * t + ((i0 + i) & 1);
#pragma unroll
      for (int k = 0; k < kR; ++k)
        if (ROWS >= 8 || g < ROWS)
          *reinterpret_cast<float2*>(mid + (8 * k + g) * kRowBytes + place * 8) =
              make_float2(fmaf(odd[i][2 * k], 0.0625f, even[i][2 * k]),
                          fmaf(odd[i][2 * k + 1], 0.0625f, even[i][2 * k + 1]));
    }
  }
  // ----------------------------------------------------------------- softmax
  // This lane's keys: pair (i, t) = (lane / 4, lane % 4), the lane's place in a row likewise.
  const int j0 = 8 * g + t, sub0 = j0 >> sub_shift;  // the second key, 4 on, has the same page
  const uint8_t* par = tile + sub0 * sub_bytes + (j0 & sub_mask) * 4;
  const bool here = page_ok >> sub0 & 1u;
  const uint32_t kp0 = *reinterpret_cast<const uint32_t*>(par + kv4_k_par(sub_shift, HD));
  const uint32_t kp1 = *reinterpret_cast<const uint32_t*>(par + kv4_k_par(sub_shift, HD) + 16);
  const uint32_t vp0 = *reinterpret_cast<const uint32_t*>(par + kv4_v_par(sub_shift, HD));
  const uint32_t vp1 = *reinterpret_cast<const uint32_t*>(par + kv4_v_par(sub_shift, HD) + 16);
  int any = __shfl_sync(0xffffffffu, limit, rows - 1);
  if (!here) any = 0;
  // the greatest step among the values that any row sees sets the unit of the weights
  uint32_t most = 0;
  if (j0 < any && (vp0 & 0xffffu) < 0x7c00u) most = vp0 & 0xffffu;
  if (j0 + 4 < any && (vp1 & 0xffffu) < 0x7c00u) most = max(most, vp1 & 0xffffu);
  most = __reduce_max_sync(0xffffffffu, most);
  // the power of two above it: its fp32 exponent, plus one
  const float step_unit =
      __uint_as_float((__float_as_uint(h2f(static_cast<uint16_t>(most))) & 0x7f800000u) + 0x00800000u);
  const float unit = most ? fmaxf(s.unit, step_unit) : s.unit;
  const float per_unit = unit > 0.f ? __uint_as_float(0x7f000000u - __float_as_uint(unit)) : 0.f;  // 1 / unit
  const float rescale = s.unit * per_unit;
  s.unit = unit;
  const float scale_up = per_unit * kTop;
  const float a0 = h2f(static_cast<uint16_t>(kp0)) * (scale_log2 * 16777216.f), b0 = h2f(static_cast<uint16_t>(kp0 >> 16));
  const float a1 = h2f(static_cast<uint16_t>(kp1)) * (scale_log2 * 16777216.f), b1 = h2f(static_cast<uint16_t>(kp1 >> 16));
  const float step0 = h2f(static_cast<uint16_t>(vp0)), step1 = h2f(static_cast<uint16_t>(vp1));
  const float st0 = step0 * scale_up, low0 = fmaf(8.f, step0, h2f(static_cast<uint16_t>(vp0 >> 16)));  // of code 8
  const float st1 = step1 * scale_up, low1 = fmaf(8.f, step1, h2f(static_cast<uint16_t>(vp1 >> 16)));
  const int place = 8 * (g >> 1) + 2 * t + (g & 1);
  __syncwarp();
  float fix[kR];
  bool changed = rescale != 1.f;
#pragma unroll
  for (int k = 0; k < kR; ++k) fix[k] = rescale;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (r % 4 == 0 && r >= rows) break;  // four rows at a time, for the distance between dependent steps
    uint8_t* at = mid + r * kRowBytes + place * 8;
    const float2 z = *reinterpret_cast<const float2*>(at);
    const int lim = __shfl_sync(0xffffffffu, limit, r);
    const bool see0 = here && j0 < lim, see1 = here && j0 + 4 < lim;
    const float z0 = see0 ? fmaf(z.x, a0, b0 * s.qsum[r]) : -INFINITY;
    const float z1 = see1 ? fmaf(z.y, a1, b1 * s.qsum[r]) : -INFINITY;
    const float top = fmaxf(s.m[r], warp_max(fmaxf(z0, z1)));
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = ex2(s.m[r] - base);
    s.m[r] = top;
    const float p0 = ex2(z0 - base), p1 = ex2(z1 - base);
    s.l[r] = fmaf(s.l[r], keep, p0 + p1);
    // a key that is not seen has p = 0, whatever its parameters
    s.pb[r] = fmaf(s.pb[r], keep, (see0 ? p0 * low0 : 0.f) + (see1 ? p1 * low1 : 0.f));
    const float w0 = see0 ? p0 * st0 : 0.f, w1 = see1 ? p1 * st1 : 0.f;
    const __half2 h = __floats2half2_rn(w0, w1);
    const float2 f = __half22float2(h);
    *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&h), f2h2(w0 - f.x, w1 - f.y));
    changed |= keep != 1.f;
    if (r < 8) {
      if (g == r) fix[0] = keep * rescale;
    } else {
      if (g == r - 8) fix[kR - 1] = keep * rescale;
    }
  }
  __syncwarp();
  if (changed) {  // the same in every lane
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      s.o[i][0] *= fix[0];
      s.o[i][1] *= fix[0];
      s.o[i][2] *= fix[kR - 1];
      s.o[i][3] *= fix[kR - 1];
    }
  }
  // ------------------------------------------------------------------ values
#pragma unroll
  for (int i = 0; i < kTile / 16; ++i) {
    // [row][key pair 16 i + t + {0, 4}, 16 i + 8 + t + {0, 4}]: first part, second part of each
    uint4 w[kR];
#pragma unroll
    for (int k = 0; k < kR; ++k) {
      w[k] = make_uint4(0, 0, 0, 0);
      if (8 * k + g < rows) w[k] = *reinterpret_cast<const uint4*>(mid + (8 * k + g) * kRowBytes + (8 * i + 2 * t) * 8);
    }
    const auto add = [&](int n, uint32_t x, uint32_t y) {
      if constexpr (kR == 1) {
        mma_16816(s.o[n], w[0].x, w[0].y, w[0].z, w[0].w, x, y);
      } else {
        mma_16816(s.o[n], w[0].x, w[kR - 1].x, w[0].z, w[kR - 1].z, x, y);
        mma_16816(s.o[n], w[0].y, w[kR - 1].y, w[0].w, w[kR - 1].w, x, y);
      }
    };
    const auto four = [&](int n, uint32_t x, uint32_t y) {  // four nibbles of two pairs of tokens
      add(n, centred<0>(x), centred<0>(y));
      add(n + 1, centred<4>(x), centred<4>(y));
      x >>= 8, y >>= 8;
      add(n + 2, centred<0>(x), centred<0>(y));
      add(n + 3, centred<4>(x), centred<4>(y));
    };
    const int j = 16 * i + t;
    const uint8_t* src = tile + (j >> sub_shift) * sub_bytes + kv4_v_codes(sub_shift, HD) + (j & sub_mask) * (HD / 2);
    if constexpr (HD == 32) {
      uint32_t x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const uint32_t*>(src + 4 * c * (HD / 2) + (g >> 1) * 4);
      const uint32_t pick = (g & 1) ? 0x7632u : 0x5410u;
      four(0, __byte_perm(x[0], x[1], pick), __byte_perm(x[2], x[3], pick));
    } else if constexpr (HD == 64) {
      uint32_t x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const uint32_t*>(src + 4 * c * (HD / 2) + g * 4);
      four(0, __byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410));
      four(4, __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
    } else {
      uint2 x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const uint2*>(src + 4 * c * (HD / 2) + g * 8);
      four(0, __byte_perm(x[0].x, x[1].x, 0x5410), __byte_perm(x[2].x, x[3].x, 0x5410));
      four(4, __byte_perm(x[0].x, x[1].x, 0x7632), __byte_perm(x[2].x, x[3].x, 0x7632));
      four(8, __byte_perm(x[0].y, x[1].y, 0x5410), __byte_perm(x[2].y, x[3].y, 0x5410));
      four(12, __byte_perm(x[0].y, x[1].y, 0x7632), __byte_perm(x[2].y, x[3].y, 0x7632));
    }
  }
}

// A warp's records, ROWS rows each: of its first item, if that began in another warp; of its last one, if that goes on in
// the next, or of one of more than kSumKeys keys; and of the latest of such an item's keys.
template <int HD, int ROWS>
__device__ __forceinline__ float* record_of(const AttnArgs& a, int warp, int i) {
  return a.parts + (static_cast<size_t>(warp) * kRecords + i) * ROWS * kRecord<HD>;
}
// Adds a record's rows to another's: a lane to head_dim / 32 dimensions.
template <int HD>
__device__ __forceinline__ void add_record(float* to, const float* from, int rows, int lane) {
#pragma unroll 1
  for (int row = 0; row < rows; ++row, to += kRecord<HD>, from += kRecord<HD>) {
    const float2 x = *reinterpret_cast<const float2*>(to), y = *reinterpret_cast<const float2*>(from);
    __syncwarp();
    const float top = fmaxf(x.x, y.x), base = top == -INFINITY ? 0.f : top;
    const float by = ex2(x.x - base), by1 = ex2(y.x - base);
    if (lane == 0) *reinterpret_cast<float2*>(to) = make_float2(top, fmaf(x.y, by, y.y * by1));
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) {
      float* v = to + 4 + lane + 32 * d;
      *v = fmaf(*v, by, from[4 + lane + 32 * d] * by1);
    }
  }
  __syncwarp();
}

// Joins the pieces of an item (records of warps first .. last) in their order: a lane to head_dim / 32 dimensions.  The
// loads of up to four rows and four pieces are in flight together; row by row and two pieces at a time the join was most
// of a short call's time (64 requests of 1,000 to 2,000 keys, 16 rows on 8 heads of 32: 58 us, 76 so).
template <int HD, int ROWS>
__device__ __forceinline__ void join_pieces(const AttnArgs& a, const Request& rq, int head, int block, int first, int last,
                                            int lane) {
  constexpr int kD = HD / 32, kSide = ROWS < 4 ? ROWS : 4, kAhead = kSide > 1 && HD == 128 ? 2 : 4;
  const int rows = min(ROWS, rq.n * a.group - block * ROWS), n = last - first + 1;
  const size_t stride = static_cast<size_t>(kRecords) * ROWS * kRecord<HD>;  // from a warp's records to the next's
#pragma unroll 1
  for (int row0 = 0; row0 < rows; row0 += kSide) {
    // the first warp's piece is its last one (second record), the others' their first; rows past the last hold
    // numbers of no meaning and are not written
    const float* r0 = record_of<HD, ROWS>(a, first, 1) + row0 * kRecord<HD>;
    const float* r1 = record_of<HD, ROWS>(a, first, 0) + row0 * kRecord<HD>;
    float base[kSide], sum[kSide], acc[kSide][kD];
#pragma unroll
    for (int k = 0; k < kSide; ++k) base[k] = -INFINITY;
#pragma unroll 1
    for (int i = lane; i < n; i += 32) {
      const float* r = i ? r1 + i * stride : r0;
#pragma unroll
      for (int k = 0; k < kSide; ++k) base[k] = fmaxf(base[k], r[k * kRecord<HD>]);
    }
#pragma unroll
    for (int k = 0; k < kSide; ++k) {
      base[k] = warp_max(base[k]);
      if (base[k] == -INFINITY) base[k] = 0.f;
      sum[k] = 0.f;
#pragma unroll
      for (int d = 0; d < kD; ++d) acc[k][d] = 0.f;
    }
#pragma unroll(kAhead)
    for (int i = 0; i < n; ++i) {
      const float* r = i ? r1 + i * stride : r0;
#pragma unroll
      for (int k = 0; k < kSide; ++k, r += kRecord<HD>) {
        const float w = ex2(r[0] - base[k]);
        sum[k] = fmaf(w, r[1], sum[k]);
#pragma unroll
        for (int d = 0; d < kD; ++d) acc[k][d] = fmaf(w, r[4 + lane + 32 * d], acc[k][d]);
      }
    }
#pragma unroll
    for (int k = 0; k < kSide; ++k) {
      if (row0 + k >= rows) break;
      uint16_t* o = out_row(a, rq, head, block * ROWS + row0 + k, HD);
#pragma unroll
      for (int d = 0; d < kD; ++d) o[lane + 32 * d] = f2h(sum[k] == 0.f ? 0.f : acc[k][d] / sum[k]);
    }
  }
}

template <int HD, int ROWS>
__global__ void __launch_bounds__(kSplitWarps * 32, kCtasPerSm<HD, ROWS>) kv4_attn_split_kernel(const AttnArgs a) {
  constexpr int kR = RowState<HD, ROWS>::kR;
  constexpr int kS = kStages<HD, ROWS>;
  constexpr int kThreads = kSplitWarps * 32;
  extern __shared__ __align__(128) uint8_t split_smem[];
  __shared__ uint64_t bars[kSplitWarps][kS];
  using L = Line<ROWS, kTile, false>;
  __shared__ typename L::template Runs<kThreads> runs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = split_smem + warp * kWarpBytes<HD, ROWS>;
  uint8_t* mid = ring + kS * kTileBytes<HD>;
  const int warps = static_cast<int>(gridDim.x) * kSplitWarps;

  griddep_launch_dependents();  // the kernel for longer requests may start beside this one

  if (lane < kS) mbar_init(&bars[warp][lane], 1);
  fence_barrier_init();
  L::template measure<kThreads>(a, runs, warps, [](int most) { return least_share<ROWS>(most); });
  const long long total = runs.before[kThreads];
  const int me = static_cast<int>(blockIdx.x) * kSplitWarps + warp;
  const long long u0 = me * runs.share, u1 = min(total, u0 + runs.share);
  if (u0 >= u1) return;
  // from here on units count from u0: a run has fewer than 2^31
  const int share = static_cast<int>(runs.share);
  const int run = static_cast<int>(u1 - u0);
  typename L::Cursor at = L::template place<kThreads>(a, runs, u0);
  int item_start = -at.tile;  // the item's tile 0, counted from u0

  const int sub_shift = min(a.shift, 6), subs = kTile >> sub_shift;  // pages of a tile, or parts of one
  // The copies run kS tiles ahead of the sums; the page of the next copy is
  // read one tile earlier still, so that nothing waits for it.
  typename L::Cursor ahead = at;
  int to_load = run;
  int page = -1;
  unsigned ok_bits = 0;  // 8 bits for each stage: pages that are there
  const auto fetch_page = [&]() {
    const int j = ahead.tile * kTile + (lane << sub_shift);
    page = lane < subs && j < ahead.keys ? a.table[static_cast<size_t>(ahead.seq) * a.max_blocks + (j >> a.shift)] : -1;
  };
  const auto issue = [&](int stage) {
    const bool ok = page >= 0 && page < a.n_pages;
    const unsigned mask = __ballot_sync(0xffffffffu, ok);
    const int bytes = kv4_head_bytes(sub_shift, HD);
    uint64_t* bar = &bars[warp][stage];
    if (lane == 0) mbar_arrive_expect_tx(bar, __popc(mask) * bytes);
    __syncwarp();
    if (ok) {
      const uint8_t* src = a.pages + static_cast<size_t>(page) * a.page_bytes +
                           static_cast<size_t>(ahead.head) * kv4_head_bytes(a.shift, HD);
      uint8_t* dst = ring + stage * kTileBytes<HD> + lane * bytes;
      if (a.shift <= 6) {
        bulk_load(dst, src, bytes, bar);
      } else {  // half of a page of 128: its four parts
        const int half = ahead.tile & 1;
        const int codes = kv4_v_codes(6, HD);
        bulk_load(dst, src + half * codes, codes, bar);
        bulk_load(dst + codes, src + kv4_v_codes(7, HD) + half * codes, codes, bar);
        bulk_load(dst + kv4_k_par(6, HD), src + kv4_k_par(7, HD) + half * 256, 256, bar);
        bulk_load(dst + kv4_v_par(6, HD), src + kv4_v_par(7, HD) + half * 256, 256, bar);
      }
    }
    ok_bits = (ok_bits & ~(0xffu << (8 * stage))) | mask << (8 * stage);
    if (--to_load > 0) {
      if (++ahead.tile == ahead.tiles) ahead.next_item(a);
      fetch_page();
    }
  };
  fetch_page();
#pragma unroll 1
  for (int st = 0; st < kS; ++st)
    if (to_load > 0) issue(st);

  RowState<HD, ROWS> s;
  int stage = 0;
  uint32_t parity = 0;
  int u = 0;
  bool alive = true;
#pragma unroll 1
  while (u < run) {
    const int t1 = min(min(at.tiles, at.tile + (run - u)), at.tile + kSumKeys / kTile);
    load_rows<HD, ROWS>(a, at.req, at.head, at.block, lane, s);
    const int all = at.req.n * a.group, rows = min(ROWS, all - at.block * ROWS);
    const int limit = limit_of(a, at.req, min(at.block * ROWS + lane, all - 1));  // of row `lane`
#pragma unroll 1
    for (int tile = at.tile; tile < t1; ++tile, ++u) {
      if (alive) alive = mbar_wait(&bars[warp][stage], parity, a.status);
      if (!__all_sync(0xffffffffu, alive)) {
        alive = false;
        break;
      }
      add_tile<HD, ROWS>(ring + stage * kTileBytes<HD>, mid, sub_shift, a.scale_log2, rows, limit - tile * kTile,
                         ok_bits >> (8 * stage), lane, s);
      __syncwarp();  // every lane has read the tile
      if (to_load > 0) issue(stage);
      if (++stage == kS) {
        stage = 0;
        parity ^= 1u;
      }
    }
    if (!alive) break;
    // the item's rows so far: sums over the lanes of a row, and the codes' unit
    const bool whole = at.tile == 0 && t1 == at.tiles;
    // keys of this run that are in the item's record already: these go into the third one, and from there to them
    const bool earlier = at.tile > max(0, -item_start);
    // the warps that share the item
    const int first = me - (item_start < 0 ? (share - 1 - item_start) / share : 0);
    const int last = me + (item_start + at.tiles - 1) / share;
    const float up = s.unit * (1.f / kTop);
#pragma unroll
    for (int k = 0; k < kR; ++k) {
      float l = 0.f, pb = 0.f, m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (8 * k + i < ROWS && 8 * k + i < rows) {
          const float sum = warp_sum(s.l[(8 * k + i) % ROWS]), low = warp_sum(s.pb[(8 * k + i) % ROWS]);
          if ((lane >> 2) == i) l = sum, pb = low, m = s.m[(8 * k + i) % ROWS];
        }
      }
      const int in_block = 8 * k + (lane >> 2), row = at.block * ROWS + in_block;
      if (in_block < rows) {
        float v[HD / 4];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float sum = kR == 1 ? s.o[i][c] + s.o[i][2 + c] : s.o[i][2 * k + c];
            v[c * (HD / 8) + i] = fmaf(sum, (i & 1) ? up * 0.0625f : up, pb);
          }
        if (whole) {
          uint16_t* o = out_row(a, at.req, at.head, row, HD) + (lane & 3) * (HD / 4);
          const float inv = 1.f / l;
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              h[j] = l == 0.f ? 0u : f2h2(v[8 * i + 2 * j] * inv, v[8 * i + 2 * j + 1] * inv);
            *reinterpret_cast<uint4*>(o + 8 * i) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        } else {
          float* r = record_of<HD, ROWS>(a, me, earlier ? 2 : me == first ? 1 : 0) + in_block * kRecord<HD>;
          if ((lane & 3) == 0) *reinterpret_cast<float2*>(r) = make_float2(m, l);
#pragma unroll
          for (int i = 0; i < HD / 16; ++i)
            *reinterpret_cast<float4*>(r + 4 + (lane & 3) * (HD / 4) + 4 * i) =
                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
      }
    }
    if (!whole) {
      if (earlier) {
        __syncwarp();
        add_record<HD>(record_of<HD, ROWS>(a, me, me == first ? 1 : 0), record_of<HD, ROWS>(a, me, 2), rows, lane);
      }
      if (t1 < at.tiles && u < run) {  // more of the item in this run
        at.tile = t1;
        continue;
      }
      __threadfence();
      __syncwarp();
      int n = 0;
      // an item of this warp alone takes no ticket: that place is the last item's, which others may have drawn from
      if (lane == 0 && first != last) n = atomicAdd(a.tickets + first, 1);
      n = __shfl_sync(0xffffffffu, n, 0);
      if (n == last - first) {
        __threadfence();
        join_pieces<HD, ROWS>(a, at.req, at.head, at.block, first, last, lane);
        if (lane == 0 && first != last) a.tickets[first] = 0;
      }
    }
    item_start += at.tiles;
    if (u < run) at.next_item(a);
  }
  if (!alive) {  // a copy never came: leave once those in flight have landed, as far as waits go
    for (int st = 0; st < kS; ++st) mbar_wait(&bars[warp][st], parity ^ (st < stage ? 1u : 0u), a.status);
  }
}

template <int HD, int ROWS>
int launch_split(const AttnArgs& a, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(kSplitWarps) * kWarpBytes<HD, ROWS>;
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kv4_attn_split_kernel<HD, ROWS>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)),
                            "cudaFuncSetAttribute(kv4_attn_split)"))
      return rc;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  kv4_attn_split_kernel<HD, ROWS>
      <<<static_cast<unsigned>(sm_count() * kCtasPerSm<HD, ROWS>), kSplitWarps * 32, smem, st>>>(a);
  return check_launch("kv4_attn_split_kernel");
}

// Query rows of a request to a kv head past which 128-row tiles are used.  8 requests of 1,000 to 2,000 keys on 8 heads of
// 32: 24 to 64 rows take 58 us here and 32 there, 64 requests 115 to 176 and 106; 16 rows 35 and 30, but 64 requests 58
// and 102.
constexpr int kMostSplitRows = 16;

// The workspace: tickets of both kernels (zero between calls), then their records.  The tickets' places are those of the
// most warps whatever the head_dim, so that calls of every head_dim can share a workspace: no record lies on a ticket.
size_t split_warps(size_t hd) {
  return static_cast<size_t>(sm_count()) * kSplitWarps *
         (hd == 128 ? kCtasPerSm<128, 1> : hd == 64 ? kCtasPerSm<64, 1> : kCtasPerSm<32, 1>);
}
static_assert(kCtasPerSm<32, 1> >= kCtasPerSm<64, 1> && kCtasPerSm<32, 1> >= kCtasPerSm<128, 1>);
size_t tickets_bytes() { return (split_warps(32) * sizeof(int) + 255) & ~static_cast<size_t>(255); }
// Offset of the records: after both kernels' tickets.
size_t attention_parts() { return tickets_bytes() + kv4_prompt_ticket_bytes(); }
// Whether some request of n_tokens rows may have enough for the kernel for longer requests.
bool may_be_long(size_t n_tokens, size_t group) { return n_tokens * group > kMostSplitRows; }

}  // namespace
}  // namespace gsvk

using namespace gsvk;

extern "C" {

size_t gsvk_kv4_attention_workspace(size_t n_seq, size_t n_tokens, size_t heads, size_t kv_heads,
                                    size_t head_dim) {
  if (n_seq == 0 || n_seq > 16384 || kv_heads == 0 || kv_heads > 1024 || heads % kv_heads ||
      heads == 0 || heads > 65536 || n_tokens > 0x7fffffff / (heads / kv_heads) ||
      (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return 0;
  return attention_parts() + split_warps(head_dim) * kRecords * 16 * (head_dim + 4) * sizeof(float) +
         (may_be_long(n_tokens, heads / kv_heads) ? kv4_prompt_part_bytes(head_dim) : 0);
}

int gsvk_kv4_attention(const gsvk_kv4_attention_args* g, gsvk_stream_t stream) {
  if (!g) return fail(GSVK_ERR_INVALID, "kv4_attention: null arguments");
  if (int rc = kv4_check(&g->cache, "kv4_attention")) return rc;
  if (g->n_tokens == 0) return GSVK_OK;
  if (!g->q || !g->out || !g->q_start || !g->kv_len || !g->block_table || !g->workspace)
    return fail(GSVK_ERR_INVALID, "kv4_attention: null pointer");
  if (g->heads == 0 || g->n_seq == 0 || g->max_blocks == 0)
    return fail(GSVK_ERR_INVALID, "kv4_attention: zero size");
  if (g->heads % g->cache.kv_heads)
    return fail(GSVK_ERR_INVALID, "kv4_attention: %zu query heads over %d kv heads", g->heads,
                g->cache.kv_heads);
  const int shift = kv4_page_shift(g->cache.page_size), hd = g->cache.head_dim;
  const size_t need = gsvk_kv4_attention_workspace(g->n_seq, g->n_tokens, g->heads,
                                                   g->cache.kv_heads, hd);
  if (need == 0 || g->max_blocks > (0x7fffff00u >> shift))
    return fail(GSVK_ERR_UNSUPPORTED, "kv4_attention: too many requests, rows, heads or blocks");
  if (g->workspace_bytes < need)
    return fail(GSVK_ERR_INVALID, "kv4_attention: workspace of %zu bytes, %zu needed",
                g->workspace_bytes, need);
  const size_t width = g->heads * hd;
  if (g->n_tokens > 1 && (g->q_stride < width || g->out_stride < width))
    return fail(GSVK_ERR_INVALID, "kv4_attention: row stride below %zu", width);
  if (!aligned16(g->q) || !aligned16(g->out) || g->q_stride % 8 || g->out_stride % 8 ||
      (reinterpret_cast<uintptr_t>(g->workspace) & 255u))
    return fail(GSVK_ERR_ALIGN, "kv4_attention: rows not in whole 16 bytes or workspace not 256-byte aligned");
  AttnArgs a{};
  a.pages = g->cache.pages;
  a.page_bytes = gsvk_kv4_page_bytes(g->cache.page_size, g->cache.kv_heads, hd);
  a.n_pages = static_cast<int>(g->cache.n_pages);
  a.shift = shift;
  a.kv_heads = g->cache.kv_heads;
  a.q = g->q;
  a.q_stride = g->q_stride;
  a.out = g->out;
  a.out_stride = g->out_stride;
  a.heads = static_cast<int>(g->heads);
  a.group = a.heads / a.kv_heads;
  a.n_tokens = static_cast<int>(g->n_tokens);
  a.n_seq = static_cast<int>(g->n_seq);
  a.max_blocks = static_cast<int>(g->max_blocks);
  a.q_start = g->q_start;
  a.kv_len = g->kv_len;
  a.prefix = g->prefix;
  a.table = g->block_table;
  a.scale_log2 = g->scale * 1.4426950408889634f;
  a.tickets = static_cast<int*>(g->workspace);
  uint8_t* ws = static_cast<uint8_t*>(g->workspace);
  a.long_tickets = reinterpret_cast<int*>(ws + tickets_bytes());
  a.parts = reinterpret_cast<float*>(ws + attention_parts());
  a.long_parts = reinterpret_cast<float*>(ws + attention_parts() + split_warps(hd) * kRecords * 16 * (hd + 4) * sizeof(float));
  a.status = device_status();
  cudaStream_t st = as_cuda(stream);
  // Requests with more rows than this take the kernel with 128-row tiles.
  const size_t rows = g->max_q * a.group;
  const bool prompts = rows > kMostSplitRows && may_be_long(g->n_tokens, a.group);
  a.most_rows = prompts ? kMostSplitRows : 0x7fffffff;
  // as few MMA and softmax rows as the requests' tokens need
  const auto split = [&](auto launch32, auto launch64, auto launch128) {
    return hd == 32 ? launch32(a, st) : hd == 64 ? launch64(a, st) : launch128(a, st);
  };
  int rc;
  if (rows <= 1)
    rc = split(launch_split<32, 1>, launch_split<64, 1>, launch_split<128, 1>);
  else if (rows <= 4)
    rc = split(launch_split<32, 4>, launch_split<64, 4>, launch_split<128, 4>);
  else if (rows <= 8)
    rc = split(launch_split<32, 8>, launch_split<64, 8>, launch_split<128, 8>);
  else
    rc = split(launch_split<32, 16>, launch_split<64, 16>, launch_split<128, 16>);
  return rc || !prompts ? rc : kv4_prompt_run(a, hd, st);
}

}  // extern "C"
