// Attention of new tokens over the whole paged latent cache (MLA-absorb, one key head).
//
// For a query row r (one token) with n visible keys, head h and t < n:
//   z[h][t] = scale * (q[h] . k[t] + qr[h] . kr[t]),  m = max_t z,  p = exp(z - m),
//   l = sum_t p,  out[h] = (sum_t p k[t][0:D]) / l.
// Scores, maxima, sums, the products' results and the join are fp32.  p alone is rounded to the
// key type, as the operand of the second product that the tensor core takes (by up to 2^-8 of p in
// bf16, 2^-11 in fp16; l is the sum of the unrounded ones).  In bf16 the result's relative error is
// 2.0e-3 on 1021 keys, where fp32 probabilities with one rounding of the result leave 1.7e-3, and
// 1.7e-3 for both on 8192 .. 65536 keys.
//
// attn_paged_kernel: a persistent CTA per SM takes an equal share of all rows' tiles of 64 keys,
// so a long row is split over several CTAs and short rows share one.  The
// products are formed with the keys on the M side of the tensor core:
//   S^T [64 keys x NH heads]  = K [64 x (D + 64)] Q^T       (M = 64)
//   O^T [D x NH heads]       += V^T [D x 64] P^T            (M = 128, D / 128 blocks)
// One copy of a key tile in shared memory serves both: K-major rows for S^T, and the same
// bytes as the MN-major operand V^T.  The pool is read once, by TMA boxes of 8 keys (which
// never straddle a page, as page_size is a multiple of 8).
//
// More than 64 heads: attn_paged_pair.cuh (D = 512) and attn_paged_wide.cuh.
//
// attn_paged_combine_kernel joins the parts of rows that were split and writes zeros for rows
// that see no key.
#include <cuda_runtime.h>

#include <cmath>

#include "attn_paged.cuh"
#include "attn_paged_heads.cuh"
#include "attn_paged_join.cuh"
#include "attn_paged_pair.cuh"
#include "attn_paged_wide.cuh"
#include "dsa_b200.h"
#include "sm100.cuh"

namespace dsa {
namespace attn_paged {

// The same with the workspace divided; `nh` heads a row, `shares` of the work.
Args make_args(const DsaAttnPagedParams* p, int nh, int shares, int diag, int heads) {
  Args a = make_args(p, diag, heads);
  const int64_t slots = (int64_t)2 * shares + (diag > 0 ? a.rows : 0);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.ws_o = reinterpret_cast<float*>(ws);
  ws += slots * nh * p->d * 4;
  a.ws_s = reinterpret_cast<float4*>(ws);
  ws += slots * nh * 16;
  a.ws_prefix = reinterpret_cast<int32_t*>(ws);
  return a;
}

template <int D, int NH, typename T>
int launch(const DsaAttnPagedParams* p, int diag, int heads, cudaStream_t stream) {
  using C = Cfg<D, NH>;
  const int grid = sm_count();
  if (grid < 1) return DSA_ERR_CUDA;
  Maps maps;
  if (!make_maps<D>(&maps, p, ElemTraits<T>::kIsBf16, NH)) return DSA_ERR_TMA_DESCRIPTOR;
  const Args a = make_args(p, NH, grid, diag, heads);
  auto kern = attn_paged_kernel<D, NH, T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
      cudaSuccess)
    return DSA_ERR_CUDA;
  if (!launch_early(kern, grid, kThreads, C::kSmem, stream, maps, a)) return DSA_ERR_CUDA;
  return launch_join<D, NH, kSegmentCost, T>(a, grid, stream);
}

template <typename T>
int launch_pair(const DsaAttnPagedParams* p, int diag, int heads, cudaStream_t stream) {
  constexpr int D = 512;
  using C = pair::Cfg<D>;
  constexpr bool kBf16 = ElemTraits<T>::kIsBf16;
  const int pairs = sm_count() / 2;
  if (pairs < 1) return DSA_ERR_CUDA;
  Maps maps;
  CUtensorMap map_v;
  if (!make_pair_maps<D>(&maps, &map_v, p, kBf16, pair::kHeads))
    return DSA_ERR_TMA_DESCRIPTOR;
  const Args a = make_args(p, 2 * pair::kHeads, pairs, diag, heads);
  auto kern = pair::attn_paged_pair_kernel<D, T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
      cudaSuccess)
    return DSA_ERR_CUDA;
  if (!launch_early(kern, 2 * pairs, pair::kThreads, C::kSmem, stream, maps, map_v, a)) return DSA_ERR_CUDA;
  return launch_join<D, 2 * pair::kHeads, pair::kSegmentCost, T>(a, pairs, stream);
}

template <int D, typename T>
int launch_wide(const DsaAttnPagedParams* p, int diag, int heads, cudaStream_t stream) {
  using C = wide::Cfg<D>;
  const int grid = sm_count();
  if (grid < 1) return DSA_ERR_CUDA;
  Maps maps;
  if (!make_maps<D>(&maps, p, ElemTraits<T>::kIsBf16, wide::kHeads)) return DSA_ERR_TMA_DESCRIPTOR;
  const Args a = make_args(p, wide::kHeads, grid, diag, heads);
  auto kern = wide::attn_paged_wide_kernel<D, T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
      cudaSuccess)
    return DSA_ERR_CUDA;
  if (!launch_early(kern, grid, wide::kThreads, C::kSmem, stream, maps, a)) return DSA_ERR_CUDA;
  return launch_join<D, wide::kHeads, wide::kSegmentCost, T>(a, grid, stream);
}

template <int D, typename T>
int launch_heads(const DsaAttnPagedParams* p, int diag, int heads, cudaStream_t stream) {
  switch (heads_of(p->n1)) {
    case 16: return launch<D, 16, T>(p, diag, heads, stream);
    case 32: return launch<D, 32, T>(p, diag, heads, stream);
    case 64: return launch<D, 64, T>(p, diag, heads, stream);
    default:
      if constexpr (D == 512) return launch_pair<T>(p, diag, heads, stream);
      else return launch_wide<D, T>(p, diag, heads, stream);
  }
}

template <typename T>
int launch_dim(const DsaAttnPagedParams* p, cudaStream_t stream) {
  DsaAttnPagedParams q = *p;
  int diag = 0;
  // (the heads of a token and the next token's have to be one step apart)
  if (packs(p->s1, p->n1) && !p->act_q &&
      (p->n1 == 1 || (p->q_token_stride == p->n1 * p->q_head_stride &&
                      p->qr_token_stride == p->n1 * p->qr_head_stride))) {
    if (p->n1 == 1) q.q_head_stride = p->q_token_stride, q.qr_head_stride = p->qr_token_stride;
    q.n1 = p->s1 * p->n1;
    q.s1 = 1;
    diag = p->sparse_mode == 3 ? (int)p->s1 - 1 : 0;
  }
  const int heads = (int)p->n1;
  if (p->d == 512) return launch_heads<512, T>(&q, diag, heads, stream);
  if (p->d == 256) return launch_heads<256, T>(&q, diag, heads, stream);
  if (p->d == 128) return launch_heads<128, T>(&q, diag, heads, stream);
  return DSA_ERR_INVALID_ARG;
}

}  // namespace attn_paged
}  // namespace dsa

extern "C" int dsa_attn_paged_shares_keys(int64_t s1, int64_t n1) {
  return s1 >= 1 && n1 >= 1 && n1 <= 128 && dsa::attn_paged::packs(s1, n1);
}

extern "C" int64_t dsa_attn_paged_workspace_size(int64_t batch, int64_t s1, int64_t n1, int64_t d) {
  using namespace dsa::attn_paged;
  constexpr int64_t kMax = 0x7fffffff;   // of rows * n1, as in dsa_attn_paged
  if (batch < 0 || s1 < 0 || n1 < 1 || n1 > 128 || d < 1 || d > 512 || batch > kMax || s1 > kMax ||
      batch * s1 > kMax / n1)
    return -1;
  const int64_t sms = dsa::sm_count();
  if (sms < 1) return -1;
  auto size = [&](int64_t rows, int64_t heads, int64_t own) {
    const int64_t nh = heads_of(heads), shares = nh == 128 && d == 512 ? sms / 2 : sms;
    return align256((2 * shares + own) * nh * (d * 4 + 16) + (rows + 1) * 4);
  };
  const int64_t plain = size(batch * s1, n1, 0), packed = packs(s1, n1) ? size(batch, s1 * n1, batch) : 0;
  return plain > packed ? plain : packed;
}

extern "C" int dsa_attn_paged(const DsaAttnPagedParams* p, void* stream_) {
  using namespace dsa::attn_paged;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!p || p->batch < 0 || p->s1 < 0) return DSA_ERR_INVALID_ARG;
  if (p->batch == 0 || p->s1 == 0) return DSA_OK;
  if (!valid_params(p, kTile)) return DSA_ERR_INVALID_ARG;
  if (p->workspace_bytes < dsa_attn_paged_workspace_size(p->batch, p->s1, p->n1, p->d))
    return DSA_ERR_INVALID_ARG;
  if (p->dtype == DSA_DTYPE_BF16) return launch_dim<__nv_bfloat16>(p, stream);
  if (p->dtype == DSA_DTYPE_FP16) return launch_dim<__half>(p, stream);
  return DSA_ERR_INVALID_ARG;
}
