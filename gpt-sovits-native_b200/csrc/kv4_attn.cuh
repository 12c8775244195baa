// kv4_attn.cuh — what the kernels of the 4-bit cache's attention share.
#pragma once

#include "kv4.cuh"
#include "tma.cuh"

namespace gsvk {

struct AttnArgs {
  const uint8_t* pages;
  size_t page_bytes;
  int n_pages, shift, kv_heads;
  const uint16_t* q;
  size_t q_stride;
  uint16_t* out;
  size_t out_stride;
  int heads, group, n_tokens, n_seq, max_blocks;
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* prefix;
  const int32_t* table;
  float scale_log2;  // scale * log2(e)
  int* tickets;      // of the items that several warps share
  float* parts;      // their records
  int* long_tickets;  // the same for the kernel for longer requests
  float* long_parts;
  uint32_t* status;
  int most_rows;     // rows of a request (to a kv head) that the few-row kernel takes
};

// Keys of one sum on the tensor cores.  They cut each step of 16 keys off at 24 bits, so that a sum whose terms do not
// cancel shrinks by up to 2^-24 a step: 2^-14 over these keys in two parts, 3.5e-4 over 60,000.  What a worker has of an
// item past these keys is put into its record, rounded, and summed anew.
constexpr int kSumKeys = 8192;

// One request's rows and the keys they see.
struct Request {
  int q0, n, len, prefix;
};
__device__ __forceinline__ Request request_of(const AttnArgs& a, int s) {
  Request r;
  r.q0 = a.q_start[s];
  r.n = min(a.q_start[s + 1], a.n_tokens) - r.q0;
  if (r.q0 < 0) r.n = 0;
  r.len = a.kv_len[s];
  r.prefix = a.prefix ? a.prefix[s] : 0;
  return r;
}
// Keys that query row `row` of a request's kv head sees (64-bit on the way: lengths are the caller's).
__device__ __forceinline__ int limit_of(const AttnArgs& a, const Request& q, int row) {
  const int r = q.n == 1 || a.group == 1 ? (q.n == 1 ? 0 : row) : row / a.group;
  const long long causal = static_cast<long long>(q.len) - q.n + r + 1;
  const long long see = max(causal, static_cast<long long>(q.prefix));
  const long long have = min(q.len, a.max_blocks << a.shift);
  return static_cast<int>(max(0LL, min(see, have)));
}
// The line of units.  An item is (request, kv head, block of up to ROWS query
// rows), a row being one (new token, query head of the group); its unit of work
// is a tile of TILE keys.  The units of all items lie on one line (request, head, block,
// tile), which is cut into equal runs for the workers of the grid.  LONG: the
// requests with more than most_rows rows to a kv head, else the others.
template <int ROWS, int TILE, bool LONG>
struct Line {
  __device__ static __forceinline__ int blocks(const AttnArgs& a, const Request& q) {
    const int rows = q.n * a.group;
    return rows <= 0 || (rows > a.most_rows) != LONG ? 0 : (rows + ROWS - 1) / ROWS;
  }
  // Keys that any row of a block sees, and their tiles (one where there are none: its rows are zeros).
  __device__ static __forceinline__ int keys(const AttnArgs& a, const Request& q, int block) {
    return limit_of(a, q, min((block + 1) * ROWS, q.n * a.group) - 1);
  }
  __device__ static __forceinline__ int tiles(int keys) { return max(1, (keys + TILE - 1) / TILE); }
  // Units of one kv head of a request; *most keeps the longest item.
  __device__ static __forceinline__ long long head_units(const AttnArgs& a, const Request& q, int* most) {
    long long u = 0;
    const int nb = blocks(a, q);
#pragma unroll 1
    for (int b = 0; b < nb; ++b) {
      const int t = tiles(keys(a, q, b));
      u += t;
      *most = max(*most, t);
    }
    return u;
  }

  // A place on the line.
  struct Cursor {
    Request req;
    int seq, head, block, blocks, tile, tiles, keys;

    __device__ __forceinline__ void set_block(const AttnArgs& a, int b) {
      block = b;
      keys = Line::keys(a, req, b);
      tiles = Line::tiles(keys);
    }
    __device__ __forceinline__ void enter(const AttnArgs& a, int s) {
      seq = s;
      req = request_of(a, s);
      blocks = Line::blocks(a, req);
    }
    __device__ __forceinline__ void next_item(const AttnArgs& a) {
      tile = 0;
      if (++block == blocks) {
        block = 0;
        if (++head == a.kv_heads) {
          head = 0;
          do {
            if (seq + 1 >= a.n_seq) return;  // the end of the line
            enter(a, seq + 1);
          } while (blocks == 0);
        } else if (blocks == 1) {
          return;
        }
      }
      set_block(a, block);
    }
  };

  // What a CTA of THREADS threads knows of the line.
  template <int THREADS>
  struct Runs {
    long long before[THREADS + 1];  // units before each thread's requests
    long long share;                // units of a run
    int most;                       // units of the longest item
  };
  // Measures the line: an equal share for each worker, and no less than least(units of the longest item).
  template <int THREADS, class Least>
  __device__ static __forceinline__ void measure(const AttnArgs& a, Runs<THREADS>& r, int workers, const Least& least) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = (a.n_seq + THREADS - 1) / THREADS;
    if (tid == 0) r.most = 0;
    long long inc = 0;
    int most = 0;
    for (int s = tid * per; s < min((tid + 1) * per, a.n_seq); ++s) inc += a.kv_heads * head_units(a, request_of(a, s), &most);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();  // r.most is there
    if (lane == 0) atomicMax(&r.most, most);
    r.before[tid + 1] = inc;
    __syncthreads();
    for (int w = 0; w < warp; ++w) inc += r.before[32 * (w + 1)];
    __syncthreads();
    r.before[tid + 1] = inc;
    if (tid == 0) r.before[0] = 0;
    if (tid == THREADS - 1)
      r.share = max((inc + workers - 1) / workers, static_cast<long long>(least(r.most)));
    __syncthreads();
  }
  // The place of unit u0 < the line's length (a whole warp).
  template <int THREADS>
  __device__ static __forceinline__ Cursor place(const AttnArgs& a, const Runs<THREADS>& r, long long u0) {
    const int lane = threadIdx.x & 31, per = (a.n_seq + THREADS - 1) / THREADS;
    int lo = 0, hi = THREADS;  // the last run of requests that starts at or before u0
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (r.before[m] <= u0) {
        lo = m;
      } else {
        hi = m;
      }
    }
    long long left = u0 - r.before[lo], u = 1;
    int s = lo * per, most = 0;
#pragma unroll 1
    for (;; s += 32) {  // a lane to a request of the run
      const long long mine = s + lane < a.n_seq ? head_units(a, request_of(a, s + lane), &most) : 0;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const unsigned found = __ballot_sync(0xffffffffu, left < sum * a.kv_heads);
      if (found || s + 32 >= a.n_seq) {  // found: u0 lies on the line
        const int i = max(__ffs(static_cast<int>(found)) - 1, 0);
        s += i;
        u = max(1LL, __shfl_sync(0xffffffffu, mine, i));
        left -= __shfl_sync(0xffffffffu, sum - mine, i) * a.kv_heads;
        break;
      }
      left -= __shfl_sync(0xffffffffu, sum, 31) * a.kv_heads;
    }
    // left < kv_heads units of the request
    Cursor at;
    at.head = (u >> 31) == 0 && (left >> 31) == 0 ? static_cast<int>(left) / static_cast<int>(u) : static_cast<int>(left / u);
    left -= at.head * u;
    at.enter(a, s);
    at.set_block(a, 0);
    while (left >= at.tiles && at.block + 1 < at.blocks) {
      left -= at.tiles;
      at.set_block(a, at.block + 1);
    }
    at.tile = static_cast<int>(left);
    return at;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Where query row `row` of a request's kv head goes.
__device__ __forceinline__ uint16_t* out_row(const AttnArgs& a, const Request& rq, int head, int row, int hd) {
  const int r = rq.n == 1 ? 0 : row / a.group;
  return a.out + static_cast<size_t>(rq.q0 + r) * a.out_stride +
         static_cast<size_t>(head * a.group + row - r * a.group) * hd;
}

// Attention of the requests with more than a.most_rows rows to a kv head (kv4_prompt.cu), and the bytes of its
// tickets (zero between calls) and records.
int kv4_prompt_run(const AttnArgs& a, int head_dim, cudaStream_t st);
size_t kv4_prompt_ticket_bytes();
size_t kv4_prompt_part_bytes(size_t head_dim);

}  // namespace gsvk
