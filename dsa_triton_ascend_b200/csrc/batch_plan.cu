// A step's plan from the lengths of its requests, and the store of packed tokens by their slots.
//
// A step takes requests b = 0 .. batch - 1: slot rows[b] of a pool's state, with counts[b] new tokens
// that its length n[b] already counts.  Its tokens lie one request behind another; token i of request b
// has position n - count + i and goes to row position % page_size of page table[position / page_size].
// Neighbouring requests whose first pages are the same form a group (for attention that takes a
// shared prefix once).
//
// Two launches: plan_rows_kernel, over the whole GPU, in which some blocks write the tokens' lists (each
// finds its tokens' requests by a scan of the counts of its own, up to the last it needs), the others
// the block table's rows and how many pages each has in common with the row before it; and
// plan_groups_kernel, one block behind it: lengths and ends, then the groups.  A small step is one launch of a
// cluster of eight that does both: a CTA for the groups, one for each 1024 tokens, at least one for the rows, whose
// warps have two turns each at most (32 requests with tables of up to 256 blocks and a token each take 64 of 96 turns).  Bound by latency, of a chain of
// dependent loads (slot, length, page), and the host: 32 requests, tables of 64 blocks, 7.6 us a call against 9.5
// with two launches (the kernel 4.2, replayed one behind another 6.2 against 6.4); 509 requests, tables of
// 512 blocks, 9.6 a call (10.4 replayed).
#include <cuda_runtime.h>

#include "dsa_b200.h"
#include "rotary.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace dsa {
namespace plan {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTokens = 4 * kThreads;   // of a block
constexpr int kRows = 1024;             // requests scanned at a time
constexpr int kSpan = 256;              // table entries of a warp's turn
constexpr int kGroupThreads = 512;
constexpr int kCluster = 8;             // CTAs that plan a small step

struct Args {
  DsaBatchPlanParams p;
  int32_t* common;   // [batch] pages shared with the row before
  int32_t token_blocks, spans;
};

struct Request {
  int32_t slot, tokens, count;   // one that asks for what cannot be: 0, 0, and places for its tokens
};
__device__ __forceinline__ Request request_of(const DsaBatchPlanParams& p, int64_t b, bool* bad) {
  Request r{p.rows[b], 0, 0};
  const bool there = r.slot >= 0 && r.slot < p.slots;
  const int64_t n = there ? p.seq_lengths[r.slot] : 0, c = p.counts[b];
  if (!there || c < 0 || c > n || n > p.max_blocks * p.page_size) {
    *bad = true;
    return Request{0, 0, c > 0 ? (int32_t)c : 0};
  }
  r.tokens = (int32_t)n;
  r.count = (int32_t)c;
  return r;
}

// Inclusive prefix of v over the block; `tmp` has a place for each warp.
template <int kBlock>
__device__ __forceinline__ int64_t block_prefix(int64_t v, int64_t* tmp, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = v;
  __syncthreads();
  int64_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kBlock / 32; ++w) {
    if (w < warp) before += tmp[w];
    sum += tmp[w];
  }
  *total = sum;
  return v + before;
}

__device__ __forceinline__ void plan_tokens(const Args& a, int64_t block) {
  const DsaBatchPlanParams& p = a.p;
  __shared__ int64_t tmp[kWarps];
  __shared__ int64_t ends[kRows];
  __shared__ int32_t slot[kRows], tokens[kRows];
  constexpr int kPer = kRows / kThreads;
  const int64_t t0 = block * kTokens, t1 = min(t0 + kTokens, p.num_tokens);
  int64_t before = 0;   // tokens of the requests before these
  bool bad = false;
  for (int64_t b0 = 0; b0 < p.batch && before < t1; b0 += kRows) {
    int64_t mine = 0, sums[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = (int)threadIdx.x * kPer + i;
      Request q{0, 0, 0};
      if (b0 + r < p.batch) q = request_of(p, b0 + r, &bad);
      slot[r] = q.slot;
      tokens[r] = q.tokens;
      sums[i] = mine += q.count;
    }
    int64_t total;
    const int64_t first = before + block_prefix<kThreads>(mine, tmp, &total) - mine;
#pragma unroll
    for (int i = 0; i < kPer; ++i) ends[threadIdx.x * kPer + i] = first + sums[i];
    __syncthreads();
    const int rows = (int)min((int64_t)kRows, p.batch - b0);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += kThreads) {
      if (t < before || t >= before + total) continue;
      int lo = 0, hi = rows - 1;   // the first request that ends behind t
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (ends[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int64_t at = tokens[lo] - (ends[lo] - t);   // below 0: of a request that cannot be
      const uint32_t pos = (uint32_t)max(at, (int64_t)0), size = (uint32_t)p.page_size, block = pos / size;
      const int32_t page = at < 0 ? -1 : p.block_table[(int64_t)slot[lo] * p.max_blocks + block];
      bad |= page < 0;
      p.token_rows[t] = at < 0 ? -1 : (int32_t)(b0 + lo);
      p.positions[t] = (int32_t)pos;
      p.slot_map[t] = page < 0 ? -1 : page * p.page_size + (pos - block * size);
    }
    before += total;
    __syncthreads();   // the lists are read
  }
  for (int64_t t = t0 + threadIdx.x; t < t1; t += kThreads)
    if (t >= before) {   // behind the last request
      p.token_rows[t] = -1;
      p.positions[t] = 0;
      p.slot_map[t] = -1;
    }
  if (bad) report_error(p.error_flag, kErrBadIndex);
}

// The block table's rows and the comparisons, those of warp `warp` of `warps`.
__device__ __forceinline__ void plan_rows(const Args& a, int64_t warp, int64_t warps) {
  const DsaBatchPlanParams& p = a.p;
  const int lane = threadIdx.x & 31;
  bool bad = false;   // (told by plan_groups)
  for (int64_t job = warp; job < p.batch * (a.spans + 1); job += warps) {
    // the comparisons, which are the longest, first
    const int64_t b = job < p.batch ? job : (job - p.batch) / a.spans;
    const Request q = request_of(p, b, &bad);
    const int32_t* row = p.block_table + (int64_t)q.slot * p.max_blocks;
    if (job >= p.batch) {
      const int64_t j0 = (job - p.batch - b * a.spans) * kSpan;
      const int64_t blocks = (q.tokens + p.page_size - 1) / p.page_size;
      int32_t* out = p.block_table_out + b * p.max_blocks;
      int32_t v[kSpan / 32];
#pragma unroll
      for (int i = 0; i < kSpan / 32; ++i) {
        const int64_t j = j0 + 32 * i + lane;
        v[i] = j < blocks ? row[j] : -1;
      }
#pragma unroll
      for (int i = 0; i < kSpan / 32; ++i) {
        const int64_t j = j0 + 32 * i + lane;
        if (j < p.max_blocks) out[j] = v[i];
      }
      continue;
    }
    int32_t common = 0;
    if (b > 0) {
      const Request o = request_of(p, b - 1, &bad);
      const int32_t* other = p.block_table + (int64_t)o.slot * p.max_blocks;
      // whole pages of tokens that both had before this step
      const int32_t whole = min(q.tokens - q.count, o.tokens - o.count) / (int32_t)p.page_size;
      while (common < whole) {
        uint32_t differ = 0;
        constexpr int kAhead = 8;
        int32_t x[kAhead], y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int32_t j = common + 32 * i + lane;
          x[i] = j < whole ? row[j] : -1;
          y[i] = j < whole ? other[j] : -1;
        }
        int32_t same = 0;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const uint32_t m = __ballot_sync(0xffffffffu, x[i] < 0 || x[i] != y[i]);
          if (differ == 0) same += m ? __ffs(m) - 1 : 32;
          differ |= m;
        }
        common += same;
        if (differ) break;
      }
    }
    if (lane == 0) a.common[b] = common;
  }
}

__global__ void __launch_bounds__(kThreads) plan_rows_kernel(const __grid_constant__ Args a) {
  griddep_wait();
  griddep_launch_dependents();
  if ((int)blockIdx.x < a.token_blocks) {
    plan_tokens(a, blockIdx.x);
    return;
  }
  plan_rows(a, (int64_t)(blockIdx.x - a.token_blocks) * kWarps + (threadIdx.x >> 5),
            (int64_t)(gridDim.x - a.token_blocks) * kWarps);
}

// Lengths, ends and groups, by one block of kBlock threads.  `wait` returns when the comparisons are made.
template <int kBlock, typename Wait>
__device__ __forceinline__ void plan_groups(const Args& a, Wait wait) {
  const DsaBatchPlanParams& p = a.p;
  __shared__ int64_t tmp[kBlock / 32];
  __shared__ int32_t least_room[kBlock];
  const int tid = threadIdx.x;
  constexpr int32_t kNone = 0x7fffffff;
  const int64_t least = p.min_prefix > p.page_size ? p.min_prefix : p.page_size;
  // smallest prefix of each group, in shared memory where all requests are looked at together
  const bool together = p.batch <= kBlock;
  int32_t* smallest = together ? least_room : p.prefix_lengths;
  const int64_t listed = together ? kBlock : p.max_groups;
  int64_t tokens = 0, groups = 0, total;
  bool bad = false;
#pragma unroll 1
  for (int64_t b0 = 0; b0 < p.batch; b0 += kBlock) {
    const int64_t b = b0 + tid;
    Request q{0, 0, 0};
    if (b < p.batch) q = request_of(p, b, &bad);
    const int64_t end = tokens + block_prefix<kBlock>(q.count, tmp, &total);
    if (b < p.batch) {
      p.key_lengths[b] = q.tokens;
      p.query_ends[b] = (int32_t)min(end, (int64_t)0x7fffffff);
    }
    tokens += total;
  }
#pragma unroll 1
  for (int64_t g = tid; g < listed; g += kBlock) smallest[g] = kNone;
  if (tokens > p.num_tokens) bad = true;   // the last ones are not listed
  if (bad) report_error(p.error_flag, kErrBadIndex);
  wait();
#pragma unroll 1
  for (int64_t b0 = 0; b0 < p.batch; b0 += kBlock) {
    const int64_t b = b0 + tid, common = b < p.batch ? a.common[b] * p.page_size : 0;
    const bool first = b < p.batch && (b == 0 || common < least);
    const int64_t group = groups + block_prefix<kBlock>(first, tmp, &total) - 1;
    groups += total;
    if (first && group <= p.max_groups) p.group_starts[group] = (int32_t)b;
    if (b < p.batch && !first && group < listed) atomicMin(smallest + group, (int32_t)common);
  }
#pragma unroll 1
  for (int64_t g = groups + tid; g <= p.max_groups; g += kBlock) p.group_starts[g] = (int32_t)p.batch;
  __syncthreads();
#pragma unroll 1
  for (int64_t g = tid; g < p.max_groups; g += kBlock) {
    const int32_t v = g < listed ? *const_cast<volatile int32_t*>(smallest + g) : kNone;
    p.prefix_lengths[g] = v == kNone ? 0 : v;
  }
}

// (Nothing is read before the wait: what the kernel above has waited for is not yet this one's to see.)
__global__ void __launch_bounds__(kGroupThreads) plan_groups_kernel(const __grid_constant__ Args a) {
  griddep_wait();
  plan_groups<kGroupThreads>(a, [] {});
}

// All of a small step by one cluster: the groups by its first CTA, tokens by the last ones.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) plan_step_kernel(const __grid_constant__ Args a) {
  griddep_wait();
  griddep_launch_dependents();
  const int rows = kCluster - 1 - a.token_blocks;   // CTAs
  if (blockIdx.x == 0) {
    plan_groups<kThreads>(a, [] { cluster_sync(); });
    return;
  }
  if ((int)blockIdx.x <= rows) plan_rows(a, ((int)blockIdx.x - 1) * kWarps + (threadIdx.x >> 5), rows * kWarps);
  else plan_tokens(a, blockIdx.x - 1 - rows);
  cluster_sync();
}

// ---------------------------------------------------------------------------------------
// store
// ---------------------------------------------------------------------------------------
constexpr int kStoreThreads = 128;
constexpr int kInFlight = 4;   // 16-byte pieces of a lane that are loaded before any is stored

struct StoreArgs {
  DsaCacheRows e[DSA_APPEND_MAX_ENTRIES];
  uint32_t first[DSA_APPEND_MAX_ENTRIES];   // first piece of each entry
  const int64_t* slots;
  int* error_flag;
  int64_t tokens, num_slots;
  rotary::FastDiv page;
  uint32_t pieces;
  int32_t entries;
};

// A copy, bound by memory: a warp per token, whose pieces are read while its slot is (the plan's slots and the
// tokens are read at once, then the slot's row is written).  14,460 tokens of 1408 bytes, cold: 9.2 us,
// 4.4 TB/s of 40.7 MB; 32 tokens 2.2 us.
__global__ void __launch_bounds__(kStoreThreads) store_kernel(const __grid_constant__ StoreArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5);
  griddep_wait();
  griddep_launch_dependents();
  if (token >= a.tokens) return;
  const int64_t slot = a.slots[token];
  bool known = false;
  int64_t page = 0, row = 0;
  for (uint32_t u0 = lane; u0 < a.pieces; u0 += 32 * kInFlight) {
    uint4 v[kInFlight];
    int at[kInFlight], entry[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const uint32_t u = u0 + 32 * k;
      if (u >= a.pieces) break;
      int i = 0;
      while (i + 1 < a.entries && u >= a.first[i + 1]) ++i;
      entry[k] = i;
      at[k] = (int)(u - a.first[i]) * 16;
      v[k] = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.e[i].src) + token * a.e[i].src_token_stride + at[k]);
    }
    if (u0 == (uint32_t)lane) {   // first looked at with loads in flight
      known = slot >= 0 && slot < a.num_slots;
      if (slot >= a.num_slots && lane == 0) report_error(a.error_flag, kErrBadIndex);
      if (slot < (1LL << 31)) page = a.page.div((uint32_t)slot);
      else page = slot / a.page.d;
      row = slot - page * a.page.d;
    }
    if (!known) return;
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (u0 + 32 * k >= a.pieces) break;
      const DsaCacheRows& e = a.e[entry[k]];
      *reinterpret_cast<uint4*>(static_cast<char*>(e.cache) + page * e.page_stride + row * e.row_stride + at[k]) = v[k];
    }
  }
}

// A launch that may begin before the stream's kernel before it has ended; the kernels here wait for it.
cudaLaunchConfig_t early_launch(cudaLaunchAttribute* attr, int threads, cudaStream_t stream) {
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace plan
}  // namespace dsa

extern "C" int64_t dsa_batch_plan_workspace_size(int64_t batch) { return batch < 0 || batch > 0x7fffffff ? -1 : 4 * batch; }

extern "C" int dsa_batch_plan(const DsaBatchPlanParams* p, void* stream_) {
  using namespace dsa::plan;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  constexpr int64_t kMax = 0x7fffffff;
  if (!p || p->batch < 0 || p->batch > kMax || p->slots < 1 || p->slots > kMax || p->page_size < 1 ||
      p->page_size > kMax || p->max_blocks < 1 || p->max_blocks > kMax / p->page_size || p->num_tokens < 0 ||
      p->num_tokens > kMax || p->max_groups < 0 || p->max_groups > kMax || p->min_prefix < 0 || !p->block_table ||
      !p->seq_lengths || !p->group_starts || (p->max_groups > 0 && !p->prefix_lengths) ||
      (p->num_tokens > 0 && (!p->token_rows || !p->positions || !p->slot_map)) ||
      (p->batch > 0 && (!p->rows || !p->counts || !p->block_table_out || !p->key_lengths || !p->query_ends ||
                        !p->workspace || p->workspace_bytes < dsa_batch_plan_workspace_size(p->batch))))
    return DSA_ERR_INVALID_ARG;
  Args a;
  a.p = *p;
  a.common = static_cast<int32_t*>(p->workspace);
  a.token_blocks = (int)((p->num_tokens + kTokens - 1) / kTokens);
  a.spans = (int)((p->max_blocks + kSpan - 1) / kSpan);
  const int sms = dsa::sm_count();
  if (sms < 1) return DSA_ERR_CUDA;
  cudaLaunchAttribute early[1];
  cudaLaunchConfig_t cfg = early_launch(early, kThreads, stream);
  const int64_t warps = p->batch * (a.spans + 1), jobs = (warps + kWarps - 1) / kWarps, most = 8LL * sms;
  // up to two turns of a warp: one launch
  if (a.token_blocks < kCluster - 1 && warps <= 2 * (kCluster - 1 - a.token_blocks) * kWarps) {
    cfg.gridDim = dim3(kCluster);
    return cudaLaunchKernelEx(&cfg, plan_step_kernel, a) == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
  }
  cfg.gridDim = dim3((unsigned)(a.token_blocks + (jobs < most ? jobs : most)));
  if (cudaLaunchKernelEx(&cfg, plan_rows_kernel, a) != cudaSuccess) return DSA_ERR_CUDA;
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kGroupThreads);
  return cudaLaunchKernelEx(&cfg, plan_groups_kernel, a) == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
}

extern "C" int dsa_cache_store(const DsaCacheStoreParams* p, void* stream_) {
  using namespace dsa::plan;
  constexpr int64_t kMax = 0x7fffffff;
  if (!p || p->tokens < 0) return DSA_ERR_INVALID_ARG;
  if (p->tokens == 0) return DSA_OK;
  if (p->entries < 1 || p->entries > DSA_APPEND_MAX_ENTRIES || !p->slots || p->page_size < 1 || p->page_size > kMax ||
      p->num_pages < 1 || p->num_pages > kMax || p->tokens > kMax)
    return DSA_ERR_INVALID_ARG;
  StoreArgs a = {};
  for (int i = 0; i < p->entries; ++i) {
    const DsaCacheRows& e = p->rows[i];
    if (!e.src || !e.cache || e.width_bytes < 16 || e.width_bytes > (1 << 24) || e.width_bytes % 16 ||
        !aligned16(e.src) || !aligned16(e.cache) || e.src_token_stride % 16 || e.page_stride % 16 ||
        e.row_stride % 16 || e.rotary != DSA_ROTARY_NONE)
      return DSA_ERR_INVALID_ARG;
    a.e[i] = e;
    a.first[i] = a.pieces;
    a.pieces += (uint32_t)(e.width_bytes / 16);
  }
  a.entries = p->entries;
  a.slots = p->slots;
  a.error_flag = p->error_flag;
  a.tokens = p->tokens;
  a.num_slots = p->num_pages * p->page_size;
  a.page = dsa::rotary::FastDiv((uint32_t)p->page_size);
  const int64_t blocks = (a.tokens + kStoreThreads / 32 - 1) / (kStoreThreads / 32);
  cudaLaunchAttribute early[1];
  cudaLaunchConfig_t cfg = early_launch(early, kStoreThreads, static_cast<cudaStream_t>(stream_));
  cfg.gridDim = dim3((unsigned)blocks);
  return cudaLaunchKernelEx(&cfg, store_kernel, a) == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
}
