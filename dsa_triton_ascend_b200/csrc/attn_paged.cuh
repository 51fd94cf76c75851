// What the kernels of attn_paged.cu share: arguments, and the division of the work.
#pragma once

#include <cuda_runtime.h>

#include "dsa_b200.h"
#include "sm100.cuh"

namespace dsa {
namespace attn_paged {

constexpr int kRope = 64;
constexpr int kSmemLimit = 232448;
constexpr float kRescale = 8.0f;    // log2 units a score may pass the reference

struct Maps {
  CUtensorMap q, qr, k, kr;
};

struct Args {
  const int32_t* act_q;
  const int32_t* act_k;
  const int32_t* block_table;
  void* out;
  float* softmax_max;
  float* softmax_sum;
  int* error_flag;
  int32_t* ws_prefix;   // [rows + 1] units of the rows before each
  float* ws_o;          // [slots][NH][D], slots: two of each CTA, then one of each row (diag > 0)
  float4* ws_s;         // [slots][NH]: reference and running maximum (log2 units), sum, raw
                        // running maximum
  int32_t rows, s1, n1;
  // Several new tokens of a batch as one row of s1 * heads heads (s1 is 1 then): the kernels take
  // the keys that all of them see; the last `diag` ones, which only the later tokens see, are
  // taken in by the join.
  int32_t diag, heads;
  const void *q, *qr, *k, *kr;   // for the join's own products; strides in elements
  int64_t q_batch, q_head, qr_batch, qr_head, k_page, k_row, kr_page, kr_row;
  int32_t page_size, max_blocks, num_pages, mode;
  // keys of a box of rotary parts or (pair kernel) of values, 8 or 16, and the groups of 8 of a
  // tile at which one begins
  int32_t box_rows;
  uint32_t box_mask;
  float scale;
};

// Keys that query row `row` sees.
__device__ __forceinline__ int token_keys(const Args& a, int row) {
  const int b = row / a.s1, s = row - b * a.s1;
  const int ak = a.act_k[b], aq = a.act_q ? a.act_q[b] : a.s1;
  int64_t n = min((int64_t)ak, (int64_t)a.max_blocks * a.page_size);
  if (a.mode == 3) n = min(n, (int64_t)ak - aq + s + 1 - a.diag);
  if (s >= aq || n < 0) n = 0;
  return (int)n;
}
__device__ __forceinline__ int row_keys(const Args& a, int row) { return token_keys(a, row); }

// Where rows share keys (attn_shared.cu), a call is two launches, whose pieces take the place of the rows
// above: prefixes, for runs of neighbouring tokens each, and the rest, rows (or the tokens of a batch,
// packed) over the other keys of theirs.
struct Item {
  int32_t keys;     // 0: nothing to do
  int32_t first;    // position of its first key, at the start of a page
  int32_t table;    // row of the block table
  int32_t head0;    // its first row of all batch * s1 * n1 rows of queries, and how many
  int32_t heads;
  int32_t part;     // whether its result is a part in any case
  int32_t place;    // of its heads' results, behind the shares' slots, where one CTA takes all of it
  int32_t unused;
};
struct ItemArgs : Args {
  const Item* items;      // [rows]
};

__device__ __forceinline__ int row_keys(const ItemArgs& a, int row) { return a.items[row].keys; }
// Row of the block table, position of the first key, heads, where a row's results go among all
// rows * n1, whether they are a part in any case.
__device__ __forceinline__ int row_table(const Args& a, int row) { return row / a.s1; }
__device__ __forceinline__ int row_table(const ItemArgs& a, int row) { return a.items[row].table; }
__device__ __forceinline__ int row_first(const Args&, int) { return 0; }
__device__ __forceinline__ int row_first(const ItemArgs& a, int row) { return a.items[row].first; }
__device__ __forceinline__ int row_heads(const Args& a, int) { return a.n1; }
__device__ __forceinline__ int row_heads(const ItemArgs& a, int row) { return a.items[row].heads; }
__device__ __forceinline__ int64_t row_result(const Args&, int row, int heads) { return (int64_t)row * heads; }
__device__ __forceinline__ int64_t row_result(const ItemArgs& a, int row, int) { return a.items[row].head0; }
__device__ __forceinline__ bool row_is_part(const Args& a, int) { return a.diag > 0; }
__device__ __forceinline__ bool row_is_part(const ItemArgs& a, int row) { return a.items[row].part; }
// Coordinates of a row's queries in their tensor map.
struct QueryAt {
  int head, s, b;
};
__device__ __forceinline__ QueryAt row_query(const Args& a, int row) {
  const int b = row / a.s1;
  return {0, row - b * a.s1, b};
}
__device__ __forceinline__ QueryAt row_query(const ItemArgs& a, int row) { return {a.items[row].head0, 0, 0}; }
// First of the workspace's places (of a head each) for a row that one CTA takes all of, behind the
// two slots of each share.
template <int NH>
__device__ __forceinline__ int64_t own_place(const Args&, int shares, int row) { return ((int64_t)2 * shares + row) * NH; }
template <int NH>
__device__ __forceinline__ int64_t own_place(const ItemArgs& a, int shares, int row) {
  return (int64_t)2 * shares * NH + a.items[row].place;
}
template <int kTile, int kCost, typename A>
__device__ __forceinline__ int row_units(const A& a, int row) {
  const int tiles = (row_keys(a, row) + kTile - 1) / kTile;
  return tiles > 0 ? tiles + kCost : 0;
}

// Work is divided by units: a row of T tiles (with all of its heads) has T + kCost of them, the
// first kCost standing for what a CTA spends on starting a row (queries, filling the pipeline,
// the result).  CTA c of n takes units [U c / n, U (c + 1) / n) of all U.

// CTAs (pairs of them in the pair kernel) that share `units`; each takes kMinUnits at least, as
// fewer cost more in joining than they save.
constexpr int kMinUnits = 2;
__device__ __forceinline__ int64_t ctas_used(int64_t units, int grid) {
  const int64_t c = (units + kMinUnits - 1) / kMinUnits;
  return c < 1 ? 1 : c < grid ? c : grid;
}

// Exclusive prefix of v over the block (kThreads threads) and its total.
template <int kThreads>
__device__ __forceinline__ int block_scan(int v, int* tmp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += tmp[w];
    sum += tmp[w];
  }
  *total = sum;
  return before + x - v;
}

// One CTA's share: `left` units from unit `unit` of a row on.
struct Work {
  int row, unit, left;
};
// A run of tiles of one row.
struct Segment {
  int row, first, count, keys, tiles;
};
// The next run of `w` (false when the share is done); `w` moves past it.
template <int kTile, int kCost, typename A>
__device__ __forceinline__ bool next_segment(const A& a, Work& w, Segment& s) {
  while (w.left > 0 && w.row < a.rows) {
    s.row = w.row++;
    s.keys = row_keys(a, s.row);
    s.tiles = (s.keys + kTile - 1) / kTile;
    if (s.tiles == 0) continue;
    const int end = min(s.tiles + kCost, w.unit + w.left);
    s.first = max(0, w.unit - kCost);
    s.count = max(0, end - kCost) - s.first;
    w.left -= end - w.unit;
    w.unit = 0;
    if (s.count > 0) return true;
  }
  return false;
}

// units * c / ctas, by 32-bit numbers where they hold it (a 64-bit division takes as long as a
// trip to L2).
__device__ __forceinline__ int64_t share_begin(int64_t units, int64_t c, int64_t ctas) {
  if (units * ctas < (1LL << 32)) return (uint32_t)(units * c) / (uint32_t)ctas;
  return units * c / ctas;
}

// The share of CTA (or pair) `cta` of `ctas_max`.  All threads of the block call it.  The first CTA
// also writes the rows' prefix for the join.
template <int kTile, int kCost, int kThreads, typename A>
__device__ __forceinline__ Work share_of(const A& a, int cta, int ctas_max, bool first_cta, int* tmp,
                                         int32_t* start) {
  Work work{0, 0, 0};
  if (a.rows <= 32) {
    // each warp for itself, without a barrier
    const int lane = threadIdx.x & 31;
    const int mine = lane < a.rows ? row_units<kTile, kCost>(a, lane) : 0;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int total = __shfl_sync(0xffffffffu, x, 31);
    if (first_cta && threadIdx.x < 32) {
      if (lane < a.rows) a.ws_prefix[lane] = x - mine;
      if (lane == 0) a.ws_prefix[a.rows] = total;
    }
    const int64_t units = total, ctas = ctas_used(units, ctas_max);
    if (cta >= ctas) return work;
    const int64_t from = share_begin(units, cta, ctas);
    work.left = (int)(share_begin(units, cta + 1, ctas) - from);
    const int first = x - mine;
    const uint32_t here = __ballot_sync(0xffffffffu, mine > 0 && first <= from && from < (int64_t)first + mine);
    if (here == 0) {   // no unit at all
      work.left = 0;
      return work;
    }
    work.row = __ffs(here) - 1;
    work.unit = (int)(from - __shfl_sync(0xffffffffu, first, work.row));
    return work;
  }
  int64_t total = 0;
  int mine = 0, before = 0;   // the units of the thread's last row and of the rows before it
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    int sum;
    mine = r < a.rows ? row_units<kTile, kCost>(a, r) : 0;
    before = block_scan<kThreads>(mine, tmp, &sum);
    if (first_cta && r < a.rows) a.ws_prefix[r] = (int)total + before;
    total += sum;
  }
  if (first_cta && threadIdx.x == 0) a.ws_prefix[a.rows] = (int)total;
  const int64_t units = total, ctas = ctas_used(units, ctas_max);
  if (units == 0 || cta >= ctas) return work;
  const int64_t from = share_begin(units, cta, ctas);
  work.left = (int)(share_begin(units, cta + 1, ctas) - from);
  int64_t seen = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    int sum = (int)total;
    if (a.rows > kThreads) {
      mine = r < a.rows ? row_units<kTile, kCost>(a, r) : 0;
      before = block_scan<kThreads>(mine, tmp, &sum);
    }
    const int64_t first = seen + before;
    if (mine > 0 && first <= from && from < first + mine) {
      start[0] = r;
      start[1] = (int)(from - first);
    }
    seen += sum;
    if (seen > from) break;   // the same for every thread
  }
  __syncthreads();
  work.row = start[0];
  work.unit = start[1];
  return work;
}

// The next kernel may start: a join before the barrier at which this CTA has its tensor memory (behind it
// 46.5 us a call become 48.5: 8 rows x 2 tokens of 64 heads, D = 256), a kernel that may take some itself before it
// waits behind it.
template <bool kBehind>
__device__ __forceinline__ void release_next(const Args&) {
  if (!kBehind) griddep_launch_dependents();
}
template <bool kBehind>
__device__ __forceinline__ void release_next(const ItemArgs&) {
  if (kBehind) griddep_launch_dependents();
}

// The statistics of one (row, head): raw maximum `top`, sum over the exponents' reference `ref`,
// whose running maximum is `run` (log2 units).  A sum that is NaN (a NaN or infinite score) makes
// both NaN.
__device__ __forceinline__ void put_stats(const Args& a, int64_t at, float top, float ref, float run, float sum) {
  const bool any = run != -INFINITY, bad = sum != sum;
  a.softmax_max[at] = bad ? sum : any ? top * fabsf(a.scale) : 0.0f;
  a.softmax_sum[at] = bad ? sum : any ? sum * exp2f(ref - run) : 0.0f;
}

// 2^x, 2^-126 and below flushed to 0
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace attn_paged
}  // namespace dsa
