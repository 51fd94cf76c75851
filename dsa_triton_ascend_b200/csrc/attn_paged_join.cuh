// The join of the parts that a row's CTAs left, and what the launches of attn_paged.cu share.
#pragma once

#include <cmath>

#include "attn_paged.cuh"
#include "dsa_b200.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace dsa {
namespace attn_paged {

// Where the parts of one (row, head) are: CTAs c0 .. c1, whose slot of a part is 2 c, but 2 c0 + 1
// where the row begins inside the share of c0; or the row's own place (c0 == c1).
struct Parts {
  int c0, c1, skip;
  int64_t own;
  __device__ __forceinline__ int64_t at(int c, int h, int nh) const {
    return (c0 == c1 ? own : (int64_t)(2 * c + (c == c0 ? skip : 0)) * nh) + h;
  }
};

// Of a row with `count` units behind the first `first` of all `total`, `cost` of them for its start.
__device__ __forceinline__ void find_parts(int first, int count, int64_t total, int cost, int grid, Parts* p) {
  const int64_t units = total, ctas = ctas_used(units, grid), x0 = first;
  const int64_t lo = (x0 + cost + 1) * ctas - 1, hi = (x0 + count) * ctas - 1;
  if (units * ctas < (1LL << 32)) {
    const uint32_t u = (uint32_t)units;
    p->c0 = (int)((uint32_t)lo / u);
    p->c1 = (int)((uint32_t)hi / u);
  } else {
    p->c0 = (int)(lo / units);
    p->c1 = (int)(hi / units);
  }
  p->skip = share_begin(units, p->c0, ctas) < x0 ? 1 : 0;
}

// False for a row without a part (c1 < c0).
template <int NH, int kCost>
__device__ __forceinline__ bool parts_of(const Args& a, int grid, int row, Parts* p) {
  const int first = a.ws_prefix[row], next = a.ws_prefix[row + 1], all = a.ws_prefix[a.rows];
  const int count = next - first;   // units
  p->own = own_place<NH>(a, grid, row);
  p->skip = 0;
  p->c0 = 1;
  p->c1 = 0;
  if (count == 0) return false;
  find_parts(first, count, all, kCost, grid, p);
  return true;
}

// q . k + qr . kr of packed head `head` of batch `b` and the key in row `row` of page `page`, by a warp.
template <int D, typename T>
__device__ __forceinline__ float late_dot(const Args& a, int b, int head, int page, int row, int lane, const T** key) {
  const T* k = static_cast<const T*>(a.k) + page * a.k_page + row * a.k_row;
  const T* kr = static_cast<const T*>(a.kr) + page * a.kr_page + row * a.kr_row;
  const T* q = static_cast<const T*>(a.q) + b * a.q_batch + head * a.q_head;
  const T* qr = static_cast<const T*>(a.qr) + b * a.qr_batch + head * a.qr_head;
  float sum = 0.0f;
  for (int i = lane; i < (D + kRope) / 8; i += 32) {
    const bool rope = i >= D / 8;
    const uint4 x = *reinterpret_cast<const uint4*>(rope ? qr + (i - D / 8) * 8 : q + i * 8);
    const uint4 y = *reinterpret_cast<const uint4*>(rope ? kr + (i - D / 8) * 8 : k + i * 8);
    const T *xe = reinterpret_cast<const T*>(&x), *ye = reinterpret_cast<const T*>(&y);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sum = fmaf(ElemTraits<T>::to_f(xe[e]), ElemTraits<T>::to_f(ye[e]), sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  *key = k;
  return sum;
}

// The same of the key at position `pos`; false if there is no such page.
template <int D, typename T>
__device__ __forceinline__ bool warp_dot(const Args& a, int b, int head, int pos, int lane, float* dot,
                                         const T** key) {
  const int page = a.block_table[(int64_t)b * a.max_blocks + pos / a.page_size], row = pos % a.page_size;
  if (page >= a.num_pages && lane == 0) report_error(a.error_flag, kErrBadIndex);
  if (page < 0 || page >= a.num_pages) return false;
  *dot = late_dot<D, T>(a, b, head, page, row, lane, key);
  return true;
}

constexpr int kMaxDiag = 7;

// Join the parts that a row's CTAs left, and the keys that only its later tokens see; zeros for a
// row without keys.  kLanes threads go through the parts of one (row, head), D / 4 of them taking
// a part's float4s side by side: a whole block where there are few rows (and so many parts of
// each), else a warp.
constexpr int kJoinThreads = 256;

template <int D, int NH, int kCost, int kLanes, typename T>
__global__ void __launch_bounds__(kJoinThreads) attn_paged_combine_kernel(const Args a, int grid) {
  using E = ElemTraits<T>;
  constexpr bool kWide = kLanes == kJoinThreads;
  constexpr int kCols = kLanes < D / 4 ? kLanes : D / 4;   // threads of a part
  constexpr int kPer = D / 4 / kCols;                      // float4s of each
  constexpr int kGroups = kLanes / kCols;                  // parts at a time
  __shared__ float4 part[kWide ? kGroups : 1][kWide ? D / 4 : 1];
  __shared__ float psum[kGroups];
  __shared__ float late_dot[kWide ? 8 : 1];
  __shared__ const T* late_key[kWide ? 8 : 1];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t at = (int64_t)blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  if (at >= (int64_t)a.rows * a.n1) return;
  const int row = (int)(at / a.n1), head = (int)(at - (int64_t)row * a.n1);
  const int t = threadIdx.x % kLanes, grp = t / kCols, col = t % kCols, lane = threadIdx.x & 31;
  T* out = static_cast<T*>(a.out) + at * D;
  Parts p;
  const bool some = parts_of<NH, kCost>(a, grid, row, &p);
  // keys from `common` on that this token sees beside the row's common ones
  int late = 0, common = 0;
  if (a.diag > 0) {
    const int64_t cap = (int64_t)a.max_blocks * a.page_size, ak = a.act_k[row];
    common = (int)max((int64_t)0, min(cap, ak - a.diag));
    late = (int)(max((int64_t)common, min(cap, ak - a.diag + head / a.heads)) - common);
  } else if (some && p.c0 == p.c1) {
    return;   // written whole
  }
  if (!some && late == 0) {
    if (grp == 0)
#pragma unroll
      for (int i = 0; i < kPer; ++i) *reinterpret_cast<uint2*>(out + (i * kCols + col) * 4) = make_uint2(0, 0);
    if (t == 0 && a.softmax_max) a.softmax_max[at] = a.softmax_sum[at] = 0.0f;
    return;
  }
  if (kWide && (threadIdx.x >> 5) < late) {   // a warp per late key
    float dot = 0.0f;
    const T* key = nullptr;
    if (!warp_dot<D, T>(a, row, head, common + (threadIdx.x >> 5), lane, &dot, &key)) key = nullptr;
    late_dot[threadIdx.x >> 5] = dot;
    late_key[threadIdx.x >> 5] = key;
  }
  float ref = -INFINITY, run = -INFINITY, top = -INFINITY;
  for (int c = p.c0 + lane; c <= p.c1; c += 32) {
    const float4 s = a.ws_s[p.at(c, head, NH)];
    ref = fmaxf(ref, s.x);
    run = fmaxf(run, s.y);
    top = fmaxf(top, s.w);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    run = fmaxf(run, __shfl_xor_sync(0xffffffffu, run, o));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  float4 acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
#pragma unroll 4
  for (int c = p.c0 + grp; c <= p.c1; c += kGroups) {
    const float4 s = a.ws_s[p.at(c, head, NH)];
    const float4* o = reinterpret_cast<const float4*>(a.ws_o + p.at(c, head, NH) * D) + col;
    const float w = s.x == ref ? 1.0f : exp2f(s.x - ref);
    sum += w * s.z;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float4 x = o[i * kCols];
      acc[i].x += w * x.x, acc[i].y += w * x.y, acc[i].z += w * x.z, acc[i].w += w * x.w;
    }
  }
  if constexpr (kWide) {
    part[grp][col] = acc[0];
    if (col == 0) psum[grp] = sum;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
      const float4 o = part[k][col];
      sum += psum[k];
      acc[0].x += o.x, acc[0].y += o.y, acc[0].z += o.z, acc[0].w += o.w;
    }
  }
  for (int i = 0; i < late; ++i) {
    float dot = 0.0f;
    const T* key = nullptr;
    if constexpr (kWide) {
      dot = late_dot[i];
      key = late_key[i];
    } else {
      if (!warp_dot<D, T>(a, row, head, common + i, lane, &dot, &key)) key = nullptr;
    }
    if (!key) continue;
    const float raw = a.scale < 0.0f ? -dot : dot, z = dot * a.scale * 1.4426950408889634f;
    // (a score of -inf with none above it weighs nothing, as in the kernels)
    const float now = fmaxf(ref, z), f = ref == now ? 1.0f : exp2f(ref - now);
    const float w = z == -INFINITY ? 0.0f : exp2f(z - now);
    ref = now;
    run = fmaxf(run, z);
    top = fmaxf(top, raw);
    sum = sum * f + w;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint2 v = *reinterpret_cast<const uint2*>(key + (k * kCols + col) * 4);
      const T* e = reinterpret_cast<const T*>(&v);
      acc[k].x = fmaf(w, E::to_f(e[0]), acc[k].x * f), acc[k].y = fmaf(w, E::to_f(e[1]), acc[k].y * f);
      acc[k].z = fmaf(w, E::to_f(e[2]), acc[k].z * f), acc[k].w = fmaf(w, E::to_f(e[3]), acc[k].w * f);
    }
  }
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    *reinterpret_cast<uint2*>(out + (i * kCols + col) * 4) =
        make_uint2(E::pack2(acc[i].x * inv, acc[i].y * inv), E::pack2(acc[i].z * inv, acc[i].w * inv));
  if (t == 0 && a.softmax_max) put_stats(a, at, top, ref, run, sum);
}

// Heads of a row as the kernels hold them: the smallest size that they fit.  Past 64 they are
// taken whole: at D = 512 by the pair kernel (32 rows of 8192 .. 65536 keys, 128 heads, in a burst:
// 356 us against 502 for two items of 64), below by the wide one (the same rows at D = 256: 185 us
// against 266; a pair there took 314).
inline int heads_of(int64_t n1) { return n1 <= 16 ? 16 : n1 <= 32 ? 32 : n1 <= 64 ? 64 : 128; }

inline int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// What the kernels take, but for the workspace's parts.
inline Args make_args(const DsaAttnPagedParams* p, int diag, int heads) {
  Args a;
  a.act_q = p->act_q;
  a.act_k = p->act_k;
  a.block_table = p->block_table;
  a.out = p->out;
  a.softmax_max = p->softmax_max;
  a.softmax_sum = p->softmax_sum;
  a.error_flag = p->error_flag;
  a.rows = (int)(p->batch * p->s1);
  a.s1 = (int)p->s1;
  a.n1 = (int)p->n1;
  a.page_size = (int)p->page_size;
  a.max_blocks = (int)p->max_blocks;
  a.num_pages = (int)p->num_pages;
  a.mode = p->sparse_mode;
  a.scale = p->scale;
  a.box_rows = p->page_size % 16 ? 8 : 16;
  a.box_mask = p->page_size % 16 ? 0xffffu : 0x5555u;
  a.diag = diag;
  a.heads = heads;
  a.q = p->query, a.qr = p->query_rope, a.k = p->key_cache, a.kr = p->key_rope_cache;
  a.q_batch = p->q_batch_stride, a.q_head = p->q_head_stride;
  a.qr_batch = p->qr_batch_stride, a.qr_head = p->qr_head_stride;
  a.k_page = p->k_page_stride, a.k_row = p->k_row_stride;
  a.kr_page = p->kr_page_stride, a.kr_row = p->kr_row_stride;
  return a;
}

// Tensor maps of the queries (boxes of `nh` heads) and keys (boxes of 8 keys; of their rotary
// parts 16 where the page size allows).
template <int D>
bool make_maps(Maps* maps, const DsaAttnPagedParams* p, bool bf16, uint32_t nh) {
  const uint64_t n1 = p->n1, s1 = p->s1, b = p->batch, page = p->page_size, pages = p->num_pages;
  const uint64_t dims[5] = {64, n1, D / 64, s1, b};
  const uint64_t st[4] = {(uint64_t)p->q_head_stride * 2, 128, (uint64_t)p->q_token_stride * 2,
                          (uint64_t)p->q_batch_stride * 2};
  const uint32_t box[5] = {64, nh, D / 64, 1, 1};
  const uint64_t rdims[5] = {64, n1, 1, s1, b};
  const uint64_t rst[4] = {(uint64_t)p->qr_head_stride * 2, 128, (uint64_t)p->qr_token_stride * 2,
                           (uint64_t)p->qr_batch_stride * 2};
  const uint32_t rbox[5] = {64, nh, 1, 1, 1};
  const uint64_t kdims[4] = {64, page, D / 64, pages};
  const uint64_t kst[3] = {(uint64_t)p->k_row_stride * 2, 128, (uint64_t)p->k_page_stride * 2};
  const uint32_t kbox[4] = {64, 8, D / 64, 1};
  const uint64_t krdims[4] = {64, page, 1, pages};
  const uint64_t krst[3] = {(uint64_t)p->kr_row_stride * 2, 128, (uint64_t)p->kr_page_stride * 2};
  const uint32_t krbox[4] = {64, page % 16 ? 8u : 16u, 1, 1};
  return make_tmap_16b(&maps->q, p->query, bf16, 5, dims, st, box) &&
         make_tmap_16b(&maps->qr, p->query_rope, bf16, 5, rdims, rst, rbox) &&
         make_tmap_16b(&maps->k, p->key_cache, bf16, 4, kdims, kst, kbox) &&
         make_tmap_16b(&maps->kr, p->key_rope_cache, bf16, 4, krdims, krst, krbox);
}

// Tensor maps of the pair kernel: the others', and one of values, boxes of 8 or 16 keys, a CTA's half of the dims.
template <int D>
bool make_pair_maps(Maps* maps, CUtensorMap* values, const DsaAttnPagedParams* p, bool bf16, uint32_t nh) {
  const uint64_t dims[4] = {64, (uint64_t)p->page_size, D / 64, (uint64_t)p->num_pages};
  const uint64_t st[3] = {(uint64_t)p->k_row_stride * 2, 128, (uint64_t)p->k_page_stride * 2};
  const uint32_t box[4] = {64, p->page_size % 16 ? 8u : 16u, D / 128, 1};
  return make_maps<D>(maps, p, bf16, nh) && make_tmap_16b(values, p->key_cache, bf16, 4, dims, st, box);
}

// A launch that may begin before the stream's kernel before it has ended: the kernels here wait
// for that one's results (griddep_wait) once they are set up.
template <typename... P, typename... A>
bool launch_early(void (*kern)(P...), int64_t blocks, int threads, int smem, cudaStream_t stream, const A&... args) {
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess;
}

template <int D, int NH, int kCost, typename T>
int launch_join(const Args& a, int shares, cudaStream_t stream) {
  const int64_t items = (int64_t)a.rows * a.n1;
  // a block each up to eight a multiprocessor (what runs at once), else a warp each
  const bool wide = items <= 8LL * sm_count();
  const int64_t blocks = wide ? items : (items + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
  auto kern = wide ? attn_paged_combine_kernel<D, NH, kCost, kJoinThreads, T>
                   : attn_paged_combine_kernel<D, NH, kCost, 32, T>;
  return launch_early(kern, blocks, kJoinThreads, 0, stream, a, shares) ? DSA_OK : DSA_ERR_CUDA;
}

// Whether several new tokens of a batch can be taken as one row of s1 * n1 heads, so that their
// keys are read once: up to 8 tokens, all of them valid (with act_q each is a row of its own), with
// 128 heads in all at most (4 x 8 tokens, 16 heads, D = 256, up to 65536 keys: 53 us against 115
// token by token; short rows lose, 8 x 2 tokens of 64 heads over 500 .. 4000 keys 31 against 28).
inline bool packs(int64_t s1, int64_t n1) {
  return s1 > 1 && s1 <= kMaxDiag + 1 && s1 * n1 <= 128;
}

inline bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether the kernels can take a call with rows (all but its workspace's size); `tile`: the least keys of a step.
inline bool valid_params(const DsaAttnPagedParams* p, int tile) {
  if (p->n1 < 1 || p->n1 > 128 || p->page_size < 8 || p->page_size % 8 || p->max_blocks < 1 ||
      p->num_pages < 1 || (p->sparse_mode != 0 && p->sparse_mode != 3) || !std::isfinite(p->scale) || !p->query ||
      !p->query_rope || !p->key_cache || !p->key_rope_cache || !p->act_k || !p->block_table ||
      !p->out || !p->workspace)
    return false;
  // sizes the kernels index with 32 bits: rows * n1 blocks, tiles, pages
  constexpr int64_t kMax = 0x7fffffff;
  // (units are counted in 32 bits: a row's tiles and its start)
  if (p->batch > kMax || p->s1 > kMax || p->batch * p->s1 > kMax / p->n1 || p->num_pages > kMax ||
      p->page_size > (1 << 20) || p->max_blocks > (kMax - tile) / p->page_size ||
      p->batch * p->s1 > kMax / ((p->max_blocks * p->page_size + tile - 1) / tile + 8))
    return false;
  if ((p->softmax_max == nullptr) != (p->softmax_sum == nullptr)) return false;
  const int64_t strides[10] = {p->q_head_stride,  p->q_token_stride,  p->q_batch_stride,
                               p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride,
                               p->k_row_stride,   p->k_page_stride,   p->kr_row_stride,
                               p->kr_page_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return false;
  if (!aligned(p->query, 16) || !aligned(p->query_rope, 16) || !aligned(p->key_cache, 16) ||
      !aligned(p->key_rope_cache, 16) || !aligned(p->workspace, 32) || !aligned(p->out, 32))
    return false;
  return true;
}

}  // namespace attn_paged
}  // namespace dsa
