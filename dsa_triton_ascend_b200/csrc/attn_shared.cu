// Attention of new tokens over a paged cache for a batch whose rows share their first pages.
//
// A row's keys are its group's prefix, which lies in pages that all rows of the group hold, and the
// rest.  With the softmax's parts over any split of the keys,
//   m_i = max z,  l_i = sum exp(z - m_i),  o_i = sum exp(z - m_i) v,
// the result is sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i, M = max_i m_i.  So the prefix is taken
// by pieces of several tokens of the group (their heads side by side, as many as the kernel holds),
// which read its keys once, the rest by rows of their own, and the join puts a row's parts of both
// together, in a fixed order.
//
// Four launches: shared_plan_kernel makes the pieces from the lengths, in one block, so that a captured call
// follows them; a kernel of attn_paged.cu takes the prefixes' pieces, 64 or 128 heads each, bound by
// products; another one, of the size that a row's own heads need, the rests, bound by memory.  Each
// waits for the one before it, as only that is promised to show it what that one and the plan wrote: the
// second does not run beside the first.  A group shares the whole pages of its prefix, at most as
// many as all of its rows see, where that costs less than its rows by themselves.
//
// Measured (against attn_paged.cu alone): 64 rows of 16 heads, D = 512, with 32811 shared and 17 to 2048 own
// keys, 118.5 us against 309; 84 rows of 20 heads in five groups, 9 of them alone, 82 against 98; 64 rows x 5 tokens
// of 16 heads, D = 512, with 32768 shared keys, 389 against 511; 24 rows x 2 tokens of 32 heads, D = 256, in two groups
// save too little and go to attn_paged.cu (52).  Of the 118.5: plan 5, pieces 80, rests 24, join 10.  The pair kernel's
// tile of 128 keys and 128 heads takes 3,645 cycles, 2,176 of them products.  (Beside one another, the second launch
// reading the plan before a wait of its own, the two took 108 in all; 72 in the five groups, 47 for the drafted tokens.)
#include <cuda_runtime.h>

#include <type_traits>

#include "attn_paged.cuh"
#include "attn_paged_heads.cuh"
#include "attn_paged_join.cuh"
#include "attn_paged_pair.cuh"
#include "attn_paged_wide.cuh"
#include "dsa_b200.h"
#include "rotary.cuh"
#include "sm100.cuh"

namespace dsa {
namespace attn_paged {

constexpr int kPlanThreads = 512;
constexpr int kPlanRows = 1984;     // batch rows and groups whose lists fit into shared memory
constexpr int kPlanGroups = 1024;
constexpr int64_t kMaxGroups = 1 << 30;

// What a launch of either kind is made of: keys of a tile (1 << shift), units of starting a piece,
// multiprocessors of a share; and in cycles what a tile takes, and a piece's start and end.
struct Kind {
  int32_t shift, start, sms, cost, piece;
};

struct PlanArgs {
  Args a;            // of the rest
  Item* pieces;      // [most]
  Item* rest;        // [rows]
  // [batch]: shared keys (0: none), first token of the row's group, and what to add to the number of a
  // window of the group for its piece, and to that number times a piece's units for the piece's first one
  int4* by_row;
  int4* by_group;    // [groups]: shared keys, pieces, first row with keys, first piece
  int32_t* by_units; // [groups]: first unit
  const int32_t* starts;
  const int32_t* prefixes;
  int32_t groups, batch, s1, packed;   // packed: tokens of a row of the rest
  int32_t most, per_item, nh;          // pieces at most; tokens and places of each
  rotary::FastDiv item;                // by per_item
  Kind prefix, own;
  int64_t least_saving;
};

// Of the s1 tokens of a batch row with `ak` keys and `aq` queries those that see a key are
// first .. first + tokens - 1; the first of them sees `keys` (0: no token sees one).
struct Seen {
  int first, tokens, keys;
};
__device__ __forceinline__ Seen seen_of(const PlanArgs& p, int ak, int aq) {
  const int cap = p.a.max_blocks * p.a.page_size;   // (below 2^31, as the host has seen to)
  int64_t first = 0, n = ak;
  if (p.a.mode == 3) {
    first = max((int64_t)aq - ak, (int64_t)0);      // (with more queries than keys)
    n = max((int64_t)ak - aq + 1, (int64_t)1);
  }
  const int64_t tokens = min(p.s1, aq) - first;
  if (ak <= 0 || tokens <= 0) return {0, 0, 0};
  return {(int)first, (int)tokens, (int)(n < cap ? n : cap)};
}

// A group's pieces are windows of per_item of its tokens, in the order of the tokens; those without a
// token that sees a key (of idle rows, or padding) are left out.  Of a batch row: the windows that are
// in no row of the group before it, first .. first + count - 1, which are the pieces `index` and on, and
// what a window's number and its piece's differ by.
struct Windows {
  int first, count, index, shift;
};
struct Counter {
  int last, pieces;   // the last window so far (-1), how many there are
};
__device__ __forceinline__ int windows_up_to(const PlanArgs& p, int tokens) { return (int)p.item.div((uint32_t)tokens + p.per_item - 1); }
// By a warp, row b of the group each; moves `c` on.
__device__ __forceinline__ Windows windows_of(const PlanArgs& p, const Seen& seen, int b, Counter& c) {
  const int lane = threadIdx.x & 31, token = b * p.s1 + seen.first;
  const bool some = seen.tokens > 0;
  const int w0 = some ? (int)p.item.div((uint32_t)token) : 0, w1 = some ? (int)p.item.div((uint32_t)(token + seen.tokens - 1)) : -1;
  int last = max(w1, c.last);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, last, o);
    if (lane >= o) last = max(last, y);
  }
  int before = __shfl_up_sync(0xffffffffu, last, 1);
  if (lane == 0) before = c.last;
  Windows w;
  w.first = max(w0, before + 1);
  w.count = some ? w1 + 1 - w.first : 0;
  int sum = w.count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  w.index = c.pieces + sum - w.count;
  w.shift = w.index - w.first;   // (a window that the row before has, too, is the piece before)
  c.last = __shfl_sync(0xffffffffu, last, 31);
  c.pieces += __shfl_sync(0xffffffffu, sum, 31);
  return w;
}

__device__ __forceinline__ int tiles_of(const Kind& k, int keys) {
  return (int)(((uint32_t)keys + (1u << k.shift) - 1) >> k.shift);
}
__device__ __forceinline__ int units_of(const Kind& k, int keys) { return keys > 0 ? tiles_of(k, keys) + k.start : 0; }

// One block: what the inputs hold is fetched at once and held in shared memory where it fits, since each
// trip to memory, each barrier and each line of code takes its time here, and nothing else does.
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const __grid_constant__ PlanArgs p) {
  __shared__ int4 group_room[kPlanGroups];
  __shared__ int unit_room[kPlanGroups], start_room[kPlanGroups + 1];
  __shared__ int2 length_room[kPlanRows];   // keys and queries
  __shared__ int shared_room[kPlanRows];
  __shared__ unsigned long long saved;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kPlanThreads / 32;
  griddep_wait();
  griddep_launch_dependents();
  const bool groups_here = p.groups <= kPlanGroups, rows_here = p.batch <= kPlanRows;
  int4* by_group = groups_here ? group_room : p.by_group;
  int* by_units = groups_here ? unit_room : p.by_units;
  const int32_t* starts = groups_here ? start_room : p.starts;
  auto lengths = [&](int b) { return make_int2(p.a.act_k[b], p.a.act_q ? p.a.act_q[b] : p.s1); };
  // of row `from` + i (none behind `to`)
  auto seen_at = [&](int from, int i, int to) {
    if (from + i >= to) return Seen{0, 0, 0};
    const int2 n = rows_here ? length_room[from + i] : lengths(from + i);
    return seen_of(p, n.x, n.y);
  };
  if (tid == 0) saved = 0;
  bool bad = false;
#pragma unroll 1
  for (int g = tid; g <= p.groups; g += kPlanThreads) {
    const int from = p.starts[g], to = g < p.groups ? p.starts[g + 1] : from;
    if (groups_here) start_room[g] = from;
    bad |= from < 0 || to < from || to > p.batch;
  }
#pragma unroll 1
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    if (rows_here) {
      length_room[b] = lengths(b);
      shared_room[b] = 0;
    }
    p.by_row[b] = make_int4(0, 0, 0, 0);
  }
#pragma unroll 1
  for (int i = tid; i < p.most; i += kPlanThreads) p.pieces[i].keys = 0;
  const bool none = __syncthreads_or(bad);   // groups that are no division of the batch are not used
  if (none && tid == 0) report_error(p.a.error_flag, kErrBadIndex);
  const int groups = none ? 0 : p.groups;
  const bool any = p.least_saving < 0;   // whatever sharing costs

#pragma unroll 1
  for (int g = warp; g < groups; g += kWarps) {
    const int from = starts[g], to = starts[g + 1], prefix = p.prefixes[g];
    int least = 0x7fffffff, rows = 0, some_tokens = 0, lead = 0x7fffffff;   // those with keys
#pragma unroll 1
    for (int i = lane; i < to - from; i += 32) {
      const Seen seen = seen_at(from, i, to);
      if (seen.tokens == 0) continue;
      least = min(least, seen.keys);
      lead = min(lead, from + i);
      ++rows;
      some_tokens += seen.tokens;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    lead = __reduce_min_sync(0xffffffffu, lead);
    rows = __reduce_add_sync(0xffffffffu, rows);
    some_tokens = __reduce_add_sync(0xffffffffu, some_tokens);
    const int tokens = (to - from) * p.s1, own = p.packed > 1 ? rows : some_tokens;   // own: rows of the rest
    int items = windows_up_to(p, tokens);
    if (some_tokens < tokens) {
      Counter c{-1, 0};
#pragma unroll 1
      for (int b0 = 0; b0 < to - from; b0 += 32) windows_of(p, seen_at(from, b0 + lane, to), b0 + lane, c);
      items = c.pieces;
    }
    if (lane == 0) {
      const uint32_t some = own > 0 ? max(min(prefix, least), 0) : 0;   // (idle rows have no page to read)
      const int keys = (int)(some - some % (uint32_t)p.a.page_size);
      // shared where its pieces cost less than its keys do in its rows
      const long long less = (long long)own * tiles_of(p.own, keys) * p.own.cost * p.own.sms -
                             (long long)items * ((long long)tiles_of(p.prefix, keys) * p.prefix.cost + p.prefix.piece) * p.prefix.sms;
      by_group[g] = less > 0 || (any && keys > 0) ? make_int4(keys, items, lead, 0) : make_int4(0, 0, 0, 0);
      if (less > 0) atomicAdd(&saved, (unsigned long long)less);
    }
  }
  __syncthreads();
  const int sharing = any || (long long)saved > p.least_saving ? groups : 0;
  if (warp == 0) {
    int pieces = 0, all = 0;
#pragma unroll 1
    for (int g0 = 0; g0 < sharing; g0 += 32) {
      const int g = g0 + lane;
      const int4 group = g < groups ? by_group[g] : make_int4(0, 0, 0, 0);
      int n = group.y, u = n * units_of(p.prefix, group.x);
      const int own_n = n, own_u = u;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, n, o), y = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) n += x, u += y;
      }
      if (g < groups) {
        by_group[g].w = pieces + n - own_n;
        by_units[g] = all + u - own_u;
      }
      pieces += __shfl_sync(0xffffffffu, n, 31);
      all += __shfl_sync(0xffffffffu, u, 31);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int g = warp; g < sharing; g += kWarps) {
    const int4 group = by_group[g];
    const int from = starts[g], to = starts[g + 1];
    if (group.x == 0) continue;
    const int first = from * p.s1, tokens = (to - from) * p.s1, units = units_of(p.prefix, group.x);
    auto put_row = [&](int b, int shift) {
      p.by_row[b] = make_int4(group.x, first, group.w + shift, by_units[g] + shift * units);
      if (rows_here) shared_room[b] = group.x;
    };
    auto put_piece = [&](int at, int window) {
      const int t = window * p.per_item;
      p.pieces[at] = Item{group.x, 0, group.z, (first + t) * p.a.heads, min(p.per_item, tokens - t) * p.a.heads, 1,
                          at * p.nh, 0};
    };
    if (group.y == windows_up_to(p, tokens)) {   // each window is a piece
#pragma unroll 1
      for (int i = lane; i < group.y; i += 32) put_piece(group.w + i, i);
#pragma unroll 1
      for (int b = from + lane; b < to; b += 32) put_row(b, 0);
      continue;
    }
    Counter c{-1, 0};
#pragma unroll 1
    for (int b0 = 0; b0 < to - from; b0 += 32) {
      const int b = from + b0 + lane, done = c.pieces;
      const Windows w = windows_of(p, seen_at(from, b0 + lane, to), b0 + lane, c);
      if (b < to) put_row(b, w.shift);
      // the new pieces of these 32 rows, a lane each: the row of one is the last that begins at it or before
#pragma unroll 1
      for (int j0 = done; j0 < c.pieces; j0 += 32) {
        const int j = j0 + lane;
        int r = 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          if (__shfl_sync(0xffffffffu, w.index, r + o) <= j) r += o;
        const int shift = __shfl_sync(0xffffffffu, w.shift, r);
        if (j < c.pieces) put_piece(group.w + j, j - shift);
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int r = tid; r < p.a.rows; r += kPlanThreads) {
    const int b = r / p.a.s1, n = row_keys(p.a, r), shared = n > 0 ? rows_here ? shared_room[b] : p.by_row[b].x : 0;
    p.rest[r] = Item{n - shared, shared, b, r * p.a.n1, p.a.n1, shared > 0 || p.a.diag > 0, r * p.a.n1, 0};
  }
}

// What the join takes of the pieces' launch: its parts, and which of them are a row's.
struct SharedParts {
  const float* ws_o;
  const float4* ws_s;
  const int32_t* units;   // of all pieces
  const int4* by_row;
  int32_t shares, nh;     // shares of the launch, heads of a piece
  Kind kind;
  rotary::FastDiv n1, s1, heads, per_item;   // heads and tokens of a row, heads of a token, tokens of a piece
};

// Join a row's own parts, its group's, and the keys that only its later tokens see; zeros for a row
// without keys.  As attn_paged_combine_kernel, but the statistics of 32 parts are fetched at a time, by
// a lane each, and the first values with them.  kLanes threads take a (row, head): a block, in groups
// that take parts of their own, or one such group.
template <int D, int NH, int kCost, int kLanes, typename T>
__global__ void __launch_bounds__(kJoinThreads)
    attn_shared_join_kernel(const __grid_constant__ Args a, int grid, const __grid_constant__ SharedParts sp) {
  using E = ElemTraits<T>;
  constexpr bool kWide = kLanes == kJoinThreads;
  constexpr int kCols = D / 4;                // threads of a part, a float4 each
  constexpr int kGroups = kLanes / kCols;     // parts at a time
  // of a thread: 6 for 24 rows x 2 tokens, 32 heads, D = 256 take 47.3 us a call against 48.8 with 4 and 49.8 with 12;
  // at D = 512 6 take 1 us more than 4, as fewer blocks of more registers run at once
  constexpr int kAhead = D == 512 ? 4 : 6;
  __shared__ float4 part[kWide ? kGroups : 1][kWide ? D / 4 : 1];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t at = (int64_t)blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  if (at >= (int64_t)a.rows * a.n1) return;
  const int row = (int)sp.n1.div((uint32_t)at), head = (int)at - row * a.n1, b = (int)sp.s1.div(row);
  const int t = threadIdx.x % kLanes, grp = t / kCols, col = t % kCols, lane = threadIdx.x & 31;
  T* out = static_cast<T*>(a.out) + at * D;
  const int4 g = sp.by_row[b];
  const int piece_units = *sp.units;
  const int first = a.ws_prefix[row], count = a.ws_prefix[row + 1] - first, all = a.ws_prefix[a.rows];
  const int64_t cap = (int64_t)a.max_blocks * a.page_size, ak = a.act_k[b];
  const int tokens = (int)sp.heads.div(a.n1), s = (int)sp.heads.div(head);   // of a packed row, and the one of this head
  // keys from `common` on that this token sees beside the row's common ones; lane i looks up the i-th's page
  const int common = (int)max((int64_t)0, min(cap, ak - a.diag));
  const int late = a.diag > 0 ? (int)max((int64_t)common, min(cap, ak - a.diag + s)) - common : 0;
  int late_page = -1;
  if (lane < late) late_page = a.block_table[(int64_t)b * a.max_blocks + (common + lane) / a.page_size];
  const int64_t seen = tokens == 1 ? token_keys(a, row) : min(cap, ak - a.diag + (a.diag > 0 ? s : 0));
  // the row's own parts, then those of the piece of which it is head `head2`
  Parts p{1, 0, 0, (int64_t)2 * grid * NH + (int64_t)row * a.n1}, p2{1, 0, 0, 0};
  int head2 = 0;
  if (count > 0) find_parts(first, count, all, kCost, grid, &p);
  if (g.x > 0 && seen > 0) {
    const int token = row * tokens + s - g.y, item = (int)sp.per_item.div(token), units = units_of(sp.kind, g.x);
    head2 = (token - item * (int)sp.per_item.d) * a.heads + head - s * a.heads;
    p2.own = (int64_t)(2 * sp.shares + g.z + item) * sp.nh;
    find_parts(g.w + item * units, units, piece_units, sp.kind.start, sp.shares, &p2);
  }
  const int n1 = p.c1 - p.c0 + 1, n = n1 + p2.c1 - p2.c0 + 1;
  if (a.diag == 0 && n == 1 && n1 == 1 && p.c0 == p.c1 && g.x == 0) return;   // written whole
  if (n == 0 && late == 0) {
    if (grp == 0) *reinterpret_cast<uint2*>(out + col * 4) = make_uint2(0, 0);
    if (t == 0 && a.softmax_max) a.softmax_max[at] = a.softmax_sum[at] = 0.0f;
    return;
  }
  float ref = -INFINITY, run = -INFINITY, top = -INFINITY, sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (int k0 = 0; k0 < n; k0 += 32) {
    const int m = min(32, n - k0);
    auto place = [&](int k) { return k < n1 ? p.at(p.c0 + k, head, NH) : p2.at(p2.c0 + k - n1, head2, sp.nh); };
    auto value = [&](int k) {
      return reinterpret_cast<const float4*>((k < n1 ? a.ws_o : sp.ws_o) + place(k) * D)[col];
    };
    float4 st = make_float4(-INFINITY, -INFINITY, 0.0f, -INFINITY);
    if (lane < m) st = (k0 + lane < n1 ? a.ws_s : sp.ws_s)[place(k0 + lane)];
    float4 v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (grp + j * kGroups < m) v[j] = value(k0 + grp + j * kGroups);
    float now = st.x, all_run = st.y, all_top = st.w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
      all_run = fmaxf(all_run, __shfl_xor_sync(0xffffffffu, all_run, o));
      all_top = fmaxf(all_top, __shfl_xor_sync(0xffffffffu, all_top, o));
    }
    now = fmaxf(now, ref);
    run = fmaxf(run, all_run);
    top = fmaxf(top, all_top);
    const float f = ref == now ? 1.0f : exp2f(ref - now), w = st.x == now ? 1.0f : exp2f(st.x - now);
    ref = now;
    float more = lane < m ? w * st.z : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
    sum = sum * f + more;
    acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll 1
    for (int j0 = 0; j0 < m; j0 += kAhead * kGroups) {   // (the same turns for every lane)
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int k = j0 + grp + j * kGroups;
        const float wk = __shfl_sync(0xffffffffu, w, k & 31);
        if (k >= m) continue;
        acc.x += wk * v[j].x, acc.y += wk * v[j].y, acc.z += wk * v[j].z, acc.w += wk * v[j].w;
        if (k + kAhead * kGroups < m) v[j] = value(k0 + k + kAhead * kGroups);
      }
    }
  }
  if constexpr (kWide) {
    part[grp][col] = acc;
    __syncthreads();
    if (grp > 0) return;   // (whole warps)
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
      const float4 o = part[k][col];
      acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
    }
  }
#pragma unroll 1
  for (int i = 0; i < late; ++i) {
    const int page = __shfl_sync(0xffffffffu, late_page, i);
    if (page >= a.num_pages && lane == 0) report_error(a.error_flag, kErrBadIndex);
    if (page < 0 || page >= a.num_pages) continue;
    const T* key;
    const float dot = late_dot<D, T>(a, b, head, page, (common + i) % a.page_size, lane, &key);
    const uint2 x = *reinterpret_cast<const uint2*>(key + col * 4);
    const float raw = a.scale < 0.0f ? -dot : dot, z = dot * a.scale * 1.4426950408889634f;
    // (a score of -inf with none above it weighs nothing, as in the kernels)
    const float now = fmaxf(ref, z), f = ref == now ? 1.0f : exp2f(ref - now);
    const float w = z == -INFINITY ? 0.0f : exp2f(z - now);
    ref = now;
    run = fmaxf(run, z);
    top = fmaxf(top, raw);
    sum = sum * f + w;
    const T* e = reinterpret_cast<const T*>(&x);
    acc.x = fmaf(w, E::to_f(e[0]), acc.x * f), acc.y = fmaf(w, E::to_f(e[1]), acc.y * f);
    acc.z = fmaf(w, E::to_f(e[2]), acc.z * f), acc.w = fmaf(w, E::to_f(e[3]), acc.w * f);
  }
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
  *reinterpret_cast<uint2*>(out + col * 4) = make_uint2(E::pack2(acc.x * inv, acc.y * inv), E::pack2(acc.z * inv, acc.w * inv));
  if (t == 0 && a.softmax_max) put_stats(a, at, top, ref, run, sum);
}

// How a call is divided: heads that either launch's kernel holds, tokens of a piece of a prefix, such
// pieces at most, rows of the rest, and the workspace.
struct Layout {
  int nh, own_nh, packed;
  int64_t per_item, most, rest, shares, own_shares, places, own_places;
  int64_t lists(int64_t batch, int64_t groups) const {   // bytes of what the plan makes
    return align256((most + rest) * (int64_t)sizeof(Item)) + align256((batch + groups) * 16 + groups * 4);
  }
  int64_t bytes(int64_t d, int64_t batch, int64_t groups) const {
    return align256((places + own_places) * (d * 4 + 16) + (most + rest + 2) * 4) + lists(batch, groups);
  }
};

Layout layout_of(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t groups, bool packed) {
  Layout l;
  l.packed = packed ? (int)s1 : 1;
  // pieces of 128 heads where a group has more than 64 on the average
  const int64_t own = n1 * l.packed, mean = (batch + groups - 1) / groups * s1 * n1;
  l.nh = mean > 64 || own > 32 ? 128 : 64;
  l.own_nh = heads_of(own);
  l.per_item = l.nh / n1;
  l.rest = packed ? batch : batch * s1;
  l.most = batch * s1 / l.per_item + (groups < batch ? groups : batch);
  auto shares = [&](int nh) { return nh == 128 && d == 512 ? sm_count() / 2 : sm_count(); };
  l.shares = shares(l.nh);
  l.own_shares = shares(l.own_nh);
  l.places = (2 * l.shares + l.most) * l.nh;
  l.own_places = 2 * l.own_shares * l.own_nh + batch * s1 * n1;
  return l;
}

// Whether pieces of a prefix can hold more tokens than a row of the rest does.
bool can_share(const Layout& l) { return l.per_item > l.packed; }

// The kernel for `nh` heads, in cycles: a tile (the slope over rows of 4096 and 12288 keys, or prefixes of
// 16384 and 49152, that lie in L2), and the start and end of a piece with its parts in the join (what rows of
// 400 and 1100 keys take beyond their tiles; of 128 heads at D >= 256 what fits 400 calls of 4 to 64 rows over 1024
// to 32768 shared keys best).
Kind kind_of(int nh, int64_t d) {
  if (nh == 128 && d == 512) return {7, pair::kSegmentCost, 2, 4350, 37000};
  if (nh == 128) return {6, wide::kSegmentCost, 1, 1850, d == 256 ? 32000 : 12000};
  const int tile = d == 512 ? (nh == 64 ? 3000 : nh == 32 ? 2600 : 2400) : d == 256 ? (nh == 64 ? 1650 : 1450) : (nh == 64 ? 1600 : 1400);
  return {6, kSegmentCost, 1, tile, 12000};
}
static_assert(pair::kTile == 128 && wide::kTile == 64 && kTile == 64, "kind_of has the tiles' sizes");

// The step from one head to the next of all tokens' (a dim of size 1 has none of its own), and whether
// they lie as rows of one matrix.
int64_t row_step(const DsaAttnPagedParams* p, int64_t head, int64_t token, int64_t batch) {
  return p->n1 > 1 ? head : p->s1 > 1 ? token : p->batch > 1 ? batch : p->d;
}
bool one_matrix(const DsaAttnPagedParams* p, int64_t head, int64_t token, int64_t batch) {
  const int64_t step = row_step(p, head, token, batch);
  return (p->s1 == 1 || token == p->n1 * step) && (p->batch == 1 || batch == p->s1 * p->n1 * step);
}

// The kernel for `nh` heads over the pieces of `a`; `flat`: the queries as one matrix of rows.
template <int D, typename T>
int launch_pieces(const DsaAttnPagedParams* flat, int nh, int shares, const ItemArgs& a, cudaStream_t stream) {
  constexpr bool kBf16 = ElemTraits<T>::kIsBf16;
  Maps maps;
  auto go = [&](auto kern, int blocks, int threads, int smem, const auto&... more) -> int {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
                   launch_early(kern, blocks, threads, smem, stream, maps, more..., a)
               ? DSA_OK : DSA_ERR_CUDA;
  };
  if (!(nh == 128 && D == 512) && !make_maps<D>(&maps, flat, kBf16, nh)) return DSA_ERR_TMA_DESCRIPTOR;
  if (nh == 16) return go(attn_paged_kernel<D, 16, T, ItemArgs>, shares, kThreads, Cfg<D, 16>::kSmem);
  if (nh == 32) return go(attn_paged_kernel<D, 32, T, ItemArgs>, shares, kThreads, Cfg<D, 32>::kSmem);
  if (nh == 64) return go(attn_paged_kernel<D, 64, T, ItemArgs>, shares, kThreads, Cfg<D, 64>::kSmem);
  if constexpr (D == 512) {
    using C = pair::Cfg<D>;
    CUtensorMap map_v;
    if (!make_pair_maps<D>(&maps, &map_v, flat, kBf16, pair::kHeads)) return DSA_ERR_TMA_DESCRIPTOR;
    return go(pair::attn_paged_pair_kernel<D, T, ItemArgs>, 2 * shares, pair::kThreads, C::kSmem, map_v);
  } else {
    return go(wide::attn_paged_wide_kernel<D, T, ItemArgs>, shares, wide::kThreads, wide::Cfg<D>::kSmem);
  }
}

template <int D, typename T>
int launch_shared(const DsaAttnSharedParams* sp, const Layout& l, cudaStream_t stream) {
  const DsaAttnPagedParams* p = &sp->attn;
  // the rest, as dsa_attn_paged would take it
  DsaAttnPagedParams rest = *p;
  int diag = 0;
  if (l.packed > 1) {
    if (p->n1 == 1) rest.q_head_stride = p->q_token_stride, rest.qr_head_stride = p->qr_token_stride;
    rest.n1 = p->s1 * p->n1;
    rest.s1 = 1;
    diag = p->sparse_mode == 3 ? (int)p->s1 - 1 : 0;
  }
  DsaAttnPagedParams flat = *p;
  flat.n1 = p->batch * p->s1 * p->n1;
  flat.s1 = flat.batch = 1;
  flat.q_head_stride = flat.q_token_stride = flat.q_batch_stride =
      row_step(p, p->q_head_stride, p->q_token_stride, p->q_batch_stride);
  flat.qr_head_stride = flat.qr_token_stride = flat.qr_batch_stride =
      row_step(p, p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride);

  ItemArgs own, pre;
  static_cast<Args&>(own) = static_cast<Args&>(pre) = make_args(&rest, diag, (int)p->n1);
  own.rows = (int)l.rest;
  pre.rows = (int)l.most;
  float* o = static_cast<float*>(p->workspace);
  pre.ws_o = o, own.ws_o = o + l.places * D;
  float4* st = reinterpret_cast<float4*>(o + (l.places + l.own_places) * D);
  pre.ws_s = st, own.ws_s = st + l.places;
  pre.ws_prefix = reinterpret_cast<int32_t*>(st + l.places + l.own_places);
  own.ws_prefix = pre.ws_prefix + l.most + 1;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace) + align256((l.places + l.own_places) * (D * 4 + 16) + (l.most + l.rest + 2) * 4);
  PlanArgs plan;
  plan.pieces = reinterpret_cast<Item*>(ws);
  plan.rest = plan.pieces + l.most;
  plan.by_row = reinterpret_cast<int4*>(ws + align256((l.most + l.rest) * (int64_t)sizeof(Item)));
  plan.by_group = plan.by_row + p->batch;
  plan.by_units = reinterpret_cast<int32_t*>(plan.by_group + sp->groups);
  pre.items = plan.pieces;
  own.items = plan.rest;
  plan.a = own;
  plan.starts = sp->group_starts;
  plan.prefixes = sp->prefix_lengths;
  plan.groups = (int)sp->groups;
  plan.batch = (int)p->batch;
  plan.s1 = (int)p->s1;
  plan.packed = l.packed;
  plan.most = (int)l.most;
  plan.per_item = (int)l.per_item;
  plan.item = rotary::FastDiv((uint32_t)l.per_item);
  plan.nh = l.nh;
  plan.prefix = kind_of(l.nh, D);
  plan.own = kind_of(l.own_nh, D);
  // keys of later tokens cost this join more than the other one (64 x 5 tokens of 16 heads, D = 512: 39 us against 19)
  const bool late = diag > 0 && D == 512 && sp->least_saving > 0;
  plan.least_saving = sp->least_saving + (late ? 700 * p->batch * p->s1 * p->n1 : 0);
  if (!launch_early(shared_plan_kernel, 1, kPlanThreads, 0, stream, plan)) return DSA_ERR_CUDA;
  int rc = launch_pieces<D, T>(&flat, l.nh, (int)l.shares, pre, stream);
  if (rc == DSA_OK) rc = launch_pieces<D, T>(&flat, l.own_nh, (int)l.own_shares, own, stream);
  if (rc != DSA_OK) return rc;
  const SharedParts parts{pre.ws_o, pre.ws_s, pre.ws_prefix + l.most, plan.by_row, (int)l.shares, l.nh, plan.prefix,
                          rotary::FastDiv((uint32_t)own.n1), rotary::FastDiv((uint32_t)own.s1),
                          rotary::FastDiv((uint32_t)own.heads), rotary::FastDiv((uint32_t)l.per_item)};
  auto join = [&](auto nh, auto cost) -> int {
    constexpr int NH = decltype(nh)::value, kCost = decltype(cost)::value;
    const int64_t items = (int64_t)own.rows * own.n1;
    const bool block = items <= 2LL * sm_count();   // (few rows are split into many parts each)
    const int each = block ? kJoinThreads : D / 4;
    auto kern = block ? attn_shared_join_kernel<D, NH, kCost, kJoinThreads, T> : attn_shared_join_kernel<D, NH, kCost, D / 4, T>;
    return launch_early(kern, (items * each + kJoinThreads - 1) / kJoinThreads, kJoinThreads, 0, stream,
                        static_cast<const Args&>(own), (int)l.own_shares, parts) ? DSA_OK : DSA_ERR_CUDA;
  };
  using std::integral_constant;
  if (l.own_nh == 16) return join(integral_constant<int, 16>(), integral_constant<int, kSegmentCost>());
  if (l.own_nh == 32) return join(integral_constant<int, 32>(), integral_constant<int, kSegmentCost>());
  if (l.own_nh == 64) return join(integral_constant<int, 64>(), integral_constant<int, kSegmentCost>());
  static_assert(pair::kSegmentCost == wide::kSegmentCost, "a join for both");
  return join(integral_constant<int, 128>(), integral_constant<int, pair::kSegmentCost>());
}

template <typename T>
int launch_shared_dim(const DsaAttnSharedParams* sp, const Layout& l, cudaStream_t stream) {
  if (sp->attn.d == 512) return launch_shared<512, T>(sp, l, stream);
  if (sp->attn.d == 256) return launch_shared<256, T>(sp, l, stream);
  if (sp->attn.d == 128) return launch_shared<128, T>(sp, l, stream);
  return DSA_ERR_INVALID_ARG;
}

}  // namespace attn_paged
}  // namespace dsa

extern "C" int64_t dsa_attn_shared_workspace_size(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t groups) {
  using namespace dsa::attn_paged;
  const int64_t plain = dsa_attn_paged_workspace_size(batch, s1, n1, d);
  if (plain < 0 || groups < 0 || groups > kMaxGroups) return -1;
  int64_t most = plain;
  if (groups == 0 || batch == 0 || s1 == 0) return most;
  for (const bool packed : {false, true}) {
    if (packed && !packs(s1, n1)) continue;
    const Layout l = layout_of(batch, s1, n1, d, groups, packed);
    const int64_t bytes = l.bytes(d, batch, groups);
    if (can_share(l) && bytes > most) most = bytes;
  }
  return most;
}

extern "C" int dsa_attn_shared_looks(const DsaAttnSharedParams* sp, int counted) {
  using namespace dsa::attn_paged;
  constexpr int64_t kMax = 0x7fffffff;
  if (!sp) return 0;
  const DsaAttnPagedParams* p = &sp->attn;
  if (sp->groups < 1 || sp->groups > kMaxGroups || p->batch < 1 || p->s1 < 1 || p->n1 < 1 || p->n1 > 128 || p->batch > kMax ||
      p->s1 > kMax || p->batch * p->s1 > kMax / p->n1 || p->page_size < 1 || p->max_blocks < 1 ||
      p->max_blocks > (kMax - pair::kTile) / p->page_size)
    return 0;
  const Layout l = layout_of(p->batch, p->s1, p->n1, p->d, sp->groups, packs(p->s1, p->n1) && !counted);
  // Calls that cannot save enough are left to the other operator, by what the tables hold: with one prefix
  // of all their keys and a quarter to spare, as the plan, the pieces' launch and this join take 3 to 6 us more
  // where nothing is shared (up to 25 with later tokens' keys or 64 heads of 64 rows).
  const Kind own = kind_of(l.own_nh, p->d), pre = kind_of(l.nh, p->d);
  const int64_t cap = p->max_blocks * p->page_size;
  if (!can_share(l)) return 0;   // a token's heads fill a piece
  const int64_t pieces = (p->batch * p->s1 + l.per_item - 1) / l.per_item;
  const double most = (double)l.rest * ((cap >> own.shift) + 1) * own.cost * own.sms -
                      (double)pieces * ((double)(cap >> pre.shift) * pre.cost + pre.piece) * pre.sms;
  if (sp->least_saving > 0 && most <= 1.25 * (double)sp->least_saving) return 0;
  // (places, units and the keys of a tile of 128 are counted in 32 bits)
  const int64_t tiles = (cap + kTile - 1) / kTile + 8;
  return l.most * l.nh <= kMax && l.most + l.rest <= kMax / tiles;
}

extern "C" int dsa_attn_shared(const DsaAttnSharedParams* sp, void* stream_) {
  using namespace dsa::attn_paged;
  if (!sp || sp->attn.batch < 0 || sp->attn.s1 < 0 || sp->groups < 0) return DSA_ERR_INVALID_ARG;
  const DsaAttnPagedParams* p = &sp->attn;
  if (p->batch == 0 || p->s1 == 0) return DSA_OK;
  if (!valid_params(p, kTile) || sp->groups > kMaxGroups || (sp->groups > 0 && (!sp->group_starts || !sp->prefix_lengths)) ||
      p->workspace_bytes < dsa_attn_shared_workspace_size(p->batch, p->s1, p->n1, p->d, sp->groups))
    return DSA_ERR_INVALID_ARG;
  const int counted = p->act_q != nullptr;
  if (!dsa_attn_shared_looks(sp, counted)) return dsa_attn_paged(p, stream_);
  const Layout l = layout_of(p->batch, p->s1, p->n1, p->d, sp->groups, packs(p->s1, p->n1) && !counted);
  if (!one_matrix(p, p->q_head_stride, p->q_token_stride, p->q_batch_stride) ||
      !one_matrix(p, p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride) || l.shares < 1)
    return DSA_ERR_INVALID_ARG;
  if (p->dtype == DSA_DTYPE_BF16) return launch_shared_dim<__nv_bfloat16>(sp, l, static_cast<cudaStream_t>(stream_));
  if (p->dtype == DSA_DTYPE_FP16) return launch_shared_dim<__half>(sp, l, static_cast<cudaStream_t>(stream_));
  return DSA_ERR_INVALID_ARG;
}
