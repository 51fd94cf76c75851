// Attention of new tokens over a paged cache for a batch whose rows share their first pages.
//
// A row's keys are its group's prefix, which lies in pages that all rows of the group hold, and the
// rest.  With the softmax's parts over any split of the keys,
//   m_i = max z,  l_i = sum exp(z - m_i),  o_i = sum exp(z - m_i) v,
// the result is sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i, M = max_i m_i.  So the prefix is taken
// by pieces of several tokens of the group (their heads side by side, as many as the kernel holds),
// which read its keys once, the rest by rows of their own; the join of attn_paged.cu, which puts a
// row's parts together in a fixed order, takes the prefix's parts among them.
//
// The pieces are made on the device, from the lengths, by one block (shared_plan_kernel), so that a
// captured call follows the lengths; then the kernels of attn_paged.cu take prefixes and rests in one
// launch, by equal shares.  A group shares the whole pages of its prefix, at most as many as all of
// its rows see.
#include <cuda_runtime.h>

#include "attn_paged.cuh"
#include "attn_paged_heads.cuh"
#include "attn_paged_join.cuh"
#include "attn_paged_pair.cuh"
#include "attn_paged_wide.cuh"
#include "dsa_b200.h"
#include "sm100.cuh"

namespace dsa {
namespace attn_paged {

constexpr int kPlanThreads = 1024;

struct PlanArgs {
  ItemArgs a;
  Item* items;
  int4* by_row;      // [batch], what ItemArgs::groups points to
  int4* by_group;    // [groups]: shared keys, items, first row with keys, first item
  const int32_t* starts;
  const int32_t* prefixes;
  int32_t groups, batch, s1, packed;   // packed: tokens of a row of the rest
};

// Keys that the first token of batch row b with any sees (0: no token of the row sees one).
__device__ __forceinline__ int least_seen(const PlanArgs& p, int b) {
  const int64_t ak = p.a.act_k[b], aq = p.a.act_q ? p.a.act_q[b] : p.s1;
  const int64_t cap = (int64_t)p.a.max_blocks * p.a.page_size;
  if (ak <= 0 || aq <= 0) return 0;
  int64_t n = ak;
  if (p.a.mode == 3) {
    n = ak - aq + 1 > 1 ? ak - aq + 1 : 1;
    if (ak - aq + min((int64_t)p.s1, aq) < 1) return 0;   // (more queries counted than there are)
  }
  return (int)(n < cap ? n : cap);
}

__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const __grid_constant__ PlanArgs p) {
  __shared__ int tmp[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kPlanThreads / 32;
  griddep_wait();
  griddep_launch_dependents();
  bool bad = false;
  for (int g = tid; g < p.groups; g += kPlanThreads) {
    const int from = p.starts[g], to = p.starts[g + 1];
    bad |= from < 0 || to < from || to > p.batch;
  }
  for (int b = tid; b < p.batch; b += kPlanThreads) p.by_row[b] = make_int4(0, 0, 0, 0);
  for (int i = tid; i < p.a.shared_items; i += kPlanThreads) p.items[i] = Item{};
  const bool none = __syncthreads_or(bad);   // groups that are no division of the batch are not used
  if (none && tid == 0) report_error(p.a.error_flag, kErrBadIndex);
  const int groups = none ? 0 : p.groups;
  for (int g = warp; g < groups; g += kWarps) {
    const int from = p.starts[g], to = p.starts[g + 1];
    int least = 0x7fffffff, rows = 0, lead = 0x7fffffff;
    for (int b = from + lane; b < to; b += 32) {
      const int n = least_seen(p, b);
      if (n == 0) continue;
      least = min(least, n);
      lead = min(lead, b);
      ++rows;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    lead = __reduce_min_sync(0xffffffffu, lead);
    rows = __reduce_add_sync(0xffffffffu, rows);
    if (lane == 0) {
      int keys = min(p.prefixes[g], least);
      keys -= keys % p.a.page_size;
      const int64_t tokens = (int64_t)(to - from) * p.s1;
      const int items = (int)((tokens + p.a.per_item - 1) / p.a.per_item);
      // (a row of the rest holds `packed` tokens; without fewer pieces than rows nothing is saved)
      const bool shares = keys > 0 && rows > 1 && items < (int64_t)rows * (p.s1 / p.packed);
      p.by_group[g] = shares ? make_int4(keys, items, lead, 0) : make_int4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  int before = 0;
  for (int g0 = 0; g0 < groups; g0 += kPlanThreads) {
    const int g = g0 + tid, items = g < groups ? p.by_group[g].y : 0;
    int sum;
    const int at = before + block_scan<kPlanThreads>(items, tmp, &sum);
    if (g < groups) p.by_group[g].w = at;
    before += sum;
    __syncthreads();
  }
  for (int g = warp; g < groups; g += kWarps) {
    const int4 group = p.by_group[g];
    const int from = p.starts[g], to = p.starts[g + 1];
    if (group.x == 0 || group.w + group.y > p.a.shared_items) continue;
    const int first = from * p.s1, tokens = (to - from) * p.s1;
    for (int i = lane; i < group.y; i += 32) {
      const int t = i * p.a.per_item;
      p.items[group.w + i] = Item{group.x, 0, group.z, (first + t) * p.a.heads, min(p.a.per_item, tokens - t) * p.a.heads, 1};
    }
    for (int b = from + lane; b < to; b += 32) p.by_row[b] = make_int4(group.x, group.w, first, 0);
  }
  __syncthreads();
  for (int r = tid; r < p.a.rows - p.a.shared_items; r += kPlanThreads) {
    const int b = r / p.a.s1, n = token_keys(p.a, r), shared = n > 0 ? p.by_row[b].x : 0;
    p.items[p.a.shared_items + r] = Item{n - shared, shared, b, r * p.a.n1, p.a.n1, shared > 0 || p.a.diag > 0};
  }
}

// How a call is divided: heads that the kernel holds, tokens of a piece of a prefix, such pieces at
// most, rows of the rest, and the workspace.
struct Layout {
  int nh, packed;
  int64_t per_item, shared_items, rest, shares, places;
  int64_t bytes(int64_t d, int64_t batch, int64_t groups) const {
    return align256(places * (d * 4 + 16) + (shared_items + rest + 1) * 4) +
           align256((shared_items + rest) * (int64_t)sizeof(Item)) + align256((batch + groups) * 16);
  }
};

Layout layout_of(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t groups, bool packed) {
  Layout l;
  l.packed = packed ? (int)s1 : 1;
  // as many heads as a group has on the average: 64 of them, or 128
  const int64_t own = n1 * l.packed, mean = (batch + groups - 1) / groups * s1 * n1;
  l.nh = heads_of(mean > 128 ? 128 : mean > own ? mean : own);
  l.per_item = l.nh / n1;
  l.rest = packed ? batch : batch * s1;
  l.shared_items = batch * s1 / l.per_item + (groups < batch / 2 ? groups : batch / 2);
  l.shares = l.nh == 128 && d == 512 ? sm_count() / 2 : sm_count();
  l.places = (2 * l.shares + l.shared_items) * l.nh + batch * s1 * n1;
  return l;
}

// Whether pieces of a prefix can hold more tokens than a row of the rest does.
bool can_share(const Layout& l) { return l.per_item > l.packed; }

// The step from one head to the next of all tokens' (a dim of size 1 has none of its own), and whether
// they lie as rows of one matrix.
int64_t row_step(const DsaAttnPagedParams* p, int64_t head, int64_t token, int64_t batch) {
  return p->n1 > 1 ? head : p->s1 > 1 ? token : p->batch > 1 ? batch : p->d;
}
bool one_matrix(const DsaAttnPagedParams* p, int64_t head, int64_t token, int64_t batch) {
  const int64_t step = row_step(p, head, token, batch);
  return (p->s1 == 1 || token == p->n1 * step) && (p->batch == 1 || batch == p->s1 * p->n1 * step);
}

template <int D, typename T>
int launch_items(const DsaAttnPagedParams* p, const Layout& l, const ItemArgs& a, const DsaAttnPagedParams* rest,
                 cudaStream_t stream) {
  constexpr bool kBf16 = ElemTraits<T>::kIsBf16;
  // every token's heads as one matrix of rows
  DsaAttnPagedParams flat = *p;
  flat.n1 = p->batch * p->s1 * p->n1;
  flat.s1 = flat.batch = 1;
  flat.q_head_stride = flat.q_token_stride = flat.q_batch_stride =
      row_step(p, p->q_head_stride, p->q_token_stride, p->q_batch_stride);
  flat.qr_head_stride = flat.qr_token_stride = flat.qr_batch_stride =
      row_step(p, p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride);
  Maps maps;
  auto go = [&](auto kern, int blocks, int threads, int smem, const auto&... more) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
           launch_early(kern, blocks, threads, smem, stream, maps, more..., a);
  };
  auto small = [&](auto nh) {
    constexpr int NH = decltype(nh)::value;
    if (!make_maps<D>(&maps, &flat, kBf16, NH)) return DSA_ERR_TMA_DESCRIPTOR;
    if (!go(attn_paged_kernel<D, NH, T, ItemArgs>, (int)l.shares, kThreads, Cfg<D, NH>::kSmem)) return DSA_ERR_CUDA;
    return launch_join<D, NH, kSegmentCost, T>(rest, a, (int)l.shares, stream);
  };
  if (l.nh == 16) return small(std::integral_constant<int, 16>());
  if (l.nh == 32) return small(std::integral_constant<int, 32>());
  if (l.nh == 64) return small(std::integral_constant<int, 64>());
  if constexpr (D == 512) {
    using C = pair::Cfg<D>;
    CUtensorMap map_v;
    if (!make_maps<D>(&maps, &flat, kBf16, pair::kHeads) || !make_value_map<D>(&map_v, p, kBf16, C::kVChunks))
      return DSA_ERR_TMA_DESCRIPTOR;
    if (!go(pair::attn_paged_pair_kernel<D, T, ItemArgs>, 2 * (int)l.shares, pair::kThreads, C::kSmem, map_v))
      return DSA_ERR_CUDA;
    return launch_join<D, 2 * pair::kHeads, pair::kSegmentCost, T>(rest, a, (int)l.shares, stream);
  } else {
    if (!make_maps<D>(&maps, &flat, kBf16, wide::kHeads)) return DSA_ERR_TMA_DESCRIPTOR;
    if (!go(wide::attn_paged_wide_kernel<D, T, ItemArgs>, (int)l.shares, wide::kThreads, wide::Cfg<D>::kSmem))
      return DSA_ERR_CUDA;
    return launch_join<D, wide::kHeads, wide::kSegmentCost, T>(rest, a, (int)l.shares, stream);
  }
}

template <typename T>
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
  PlanArgs plan;
  static_cast<Args&>(plan.a) = make_args(&rest, diag, (int)p->n1);
  ItemArgs& a = plan.a;
  a.shared_items = (int)l.shared_items;
  a.per_item = (int)l.per_item;
  a.rows = (int)(l.shared_items + l.rest);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.ws_o = reinterpret_cast<float*>(ws);
  a.ws_s = reinterpret_cast<float4*>(ws + l.places * p->d * 4);
  a.ws_prefix = reinterpret_cast<int32_t*>(ws + l.places * (p->d * 4 + 16));
  ws += align256(l.places * (p->d * 4 + 16) + (l.shared_items + l.rest + 1) * 4);
  plan.items = reinterpret_cast<Item*>(ws);
  a.items = plan.items;
  ws += align256((l.shared_items + l.rest) * (int64_t)sizeof(Item));
  plan.by_row = reinterpret_cast<int4*>(ws);
  a.groups = plan.by_row;
  plan.by_group = plan.by_row + p->batch;
  plan.starts = sp->group_starts;
  plan.prefixes = sp->prefix_lengths;
  plan.groups = (int)sp->groups;
  plan.batch = (int)p->batch;
  plan.s1 = (int)p->s1;
  plan.packed = l.packed;
  if (!launch_early(shared_plan_kernel, 1, kPlanThreads, 0, stream, plan)) return DSA_ERR_CUDA;
  if (p->d == 512) return launch_items<512, T>(p, l, a, &rest, stream);
  if (p->d == 256) return launch_items<256, T>(p, l, a, &rest, stream);
  if (p->d == 128) return launch_items<128, T>(p, l, a, &rest, stream);
  return DSA_ERR_INVALID_ARG;
}

}  // namespace attn_paged
}  // namespace dsa

extern "C" int64_t dsa_attn_shared_workspace_size(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t groups) {
  using namespace dsa::attn_paged;
  constexpr int64_t kMax = 0x7fffffff;
  const int64_t plain = dsa_attn_paged_workspace_size(batch, s1, n1, d);
  if (plain < 0 || groups < 0 || groups > kMax) return -1;
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

extern "C" int dsa_attn_shared(const DsaAttnSharedParams* sp, void* stream_) {
  using namespace dsa::attn_paged;
  if (!sp || sp->attn.batch < 0 || sp->attn.s1 < 0 || sp->groups < 0) return DSA_ERR_INVALID_ARG;
  const DsaAttnPagedParams* p = &sp->attn;
  if (p->batch == 0 || p->s1 == 0) return DSA_OK;
  constexpr int64_t kMax = 0x7fffffff;
  if (!valid_params(p, kTile) || sp->groups > kMax || (sp->groups > 0 && (!sp->group_starts || !sp->prefix_lengths)) ||
      p->workspace_bytes < dsa_attn_shared_workspace_size(p->batch, p->s1, p->n1, p->d, sp->groups))
    return DSA_ERR_INVALID_ARG;
  if (sp->groups > 0) {
    const Layout l = layout_of(p->batch, p->s1, p->n1, p->d, sp->groups, packs(p->s1, p->n1) && !p->act_q);
    if (can_share(l)) {
      const int64_t tiles = (p->max_blocks * p->page_size + kTile - 1) / kTile + 8;
      if (!one_matrix(p, p->q_head_stride, p->q_token_stride, p->q_batch_stride) ||
          !one_matrix(p, p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride) ||
          l.shared_items + l.rest > kMax / tiles || l.shares < 1)
        return DSA_ERR_INVALID_ARG;
      if (p->dtype == DSA_DTYPE_BF16) return launch_shared<__nv_bfloat16>(sp, l, static_cast<cudaStream_t>(stream_));
      if (p->dtype == DSA_DTYPE_FP16) return launch_shared<__half>(sp, l, static_cast<cudaStream_t>(stream_));
      return DSA_ERR_INVALID_ARG;
    }
  }
  return dsa_attn_paged(p, stream_);   // a token's heads fill a piece, or there is no group: nothing to share
}
