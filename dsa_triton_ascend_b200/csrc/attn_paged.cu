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
#include "attn_paged_pair.cuh"
#include "attn_paged_wide.cuh"
#include "dsa_b200.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace dsa {
namespace attn_paged {

constexpr int kTile = 64;       // keys of a step
constexpr int kSegmentCost = 2; // of starting a row, in tiles
constexpr int kSoftmaxThreads = 128;   // of a warpgroup; there are two (warps 0-3, 4-7), each with
                                       // half of the heads
constexpr int kLoadWarp = 8;           // warps 8-11: loads (one warp issues a box in 160 cycles,
                                       // so 16 boxes a tile from one warp took 2,600 of them)
constexpr int kQkWarp = 12;
constexpr int kPvWarp = 13;
constexpr int kQueryWarp = 14;
constexpr int kThreads = 480;
constexpr int kMaxStages = 8;

template <int D, int NH>
struct Cfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kBlocks = D / 128;
  static constexpr int kGroupBytes = kChunks * 1024;   // 8 keys: [chunk][8][128 B]
  static constexpr int kKeyBytes = 8 * kGroupBytes;
  static constexpr int kRopeBytes = 64 * 128;
  static constexpr int kStageBytes = kKeyBytes + kRopeBytes;
  static constexpr int kQBytes = NH * (D + kRope) * 2;
  static constexpr int kHeads = NH / 2;   // of a softmax warpgroup
  static constexpr int kPBytes = kTile * NH * 2;
  // per warp row maxima and sums, then factors, barriers and the rest
  static constexpr int kSmallBytes = 2 * 4 * NH * 4 + NH * 4 + 512;
  static constexpr int kRoom = (kSmemLimit - kQBytes - kPBytes - kSmallBytes) / kStageBytes;
  static constexpr int kStages = kRoom < kMaxStages ? kRoom : kMaxStages;
  // the next segment's queries are loaded while this one's are in use, where they fit
  static constexpr int kQBufs =
      kStages * kStageBytes + 2 * kQBytes + kPBytes + kSmallBytes <= kSmemLimit ? 2 : 1;
  static constexpr int kSmem = kStages * kStageBytes + kQBufs * kQBytes + kPBytes + kSmallBytes;
  static constexpr uint32_t kCols = (4 + kBlocks) * NH;   // S of two tiles in two parts each, O
  static constexpr uint32_t kTmem = kCols <= 32 ? 32 : kCols <= 64 ? 64 : kCols <= 128 ? 128
                                    : kCols <= 256 ? 256 : 512;
  static_assert(kStages >= 2, "two key tiles have to fit");
};

// P^T as the MN-major operand: a key's NH heads are one row of NH * 2 bytes, with the swizzle
// of that width (128, 64 or 32 bytes).  Byte offset of 16-byte chunk `c` of key row `key`.
template <int NH>
__device__ __forceinline__ uint32_t p_offset(uint32_t key, uint32_t c) {
  if constexpr (NH == 64) return key * 128u + ((c ^ (key & 7u)) << 4);
  if constexpr (NH == 32) return key * 64u + ((c ^ ((key >> 1) & 3u)) << 4);
  return key * 32u + ((c ^ ((key >> 2) & 1u)) << 4);
}
template <int NH>
__device__ __forceinline__ uint64_t p_desc(uint32_t saddr) {
  constexpr uint64_t kSwizzle = NH == 64 ? 2 : NH == 32 ? 4 : 6;
  constexpr uint32_t kAtom = 8 * NH * 2;
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(kAtom >> 4) << 32 |
         (uint64_t)1 << 46 | kSwizzle << 61;
}

// 16 lanes x 256 bits, repeated over N columns: lane l holds rows l / 4 and l / 4 + 8, and of
// every 8 columns the pair 2 (l % 4).  r[4 i + {0, 1}] is the first row, {2, 3} the second.
template <int N>
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[N / 2]) {
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr));
  else if constexpr (N == 16)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// The four warps of softmax warpgroup `wg` meet.
__device__ __forceinline__ void softmax_bar(int wg) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + wg), "n"(kSoftmaxThreads) : "memory");
}

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st16(taddr, r); }
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int D, int NH, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    attn_paged_kernel(const __grid_constant__ Maps maps, const Args a) {
  using C = Cfg<D, NH>;
  using E = ElemTraits<T>;
  constexpr bool kBf16 = E::kIsBf16;
  // half has few exponents below 1: its probabilities are held 2^6 higher (at most 2^14 with
  // the lazy reference), and the sums with them
  constexpr float kShift = kBf16 ? 0.0f : 6.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t s_q = base + C::kStages * C::kStageBytes;
  const uint32_t s_p = s_q + C::kQBufs * C::kQBytes;
  uint8_t* small = smem + C::kStages * C::kStageBytes + C::kQBufs * C::kQBytes + C::kPBytes;
  float* wmax = reinterpret_cast<float*>(small);          // [4][NH], then the sums, [4][NH]
  float* factor = wmax + 2 * 4 * NH;                      // [NH]
  uint64_t* bars = reinterpret_cast<uint64_t*>(factor + NH);
  int32_t* tmask = reinterpret_cast<int32_t*>(bars + 32);  // [kMaxStages][4]
  int32_t* tmp = tmask + 4 * kMaxStages;                   // [16]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmp + 16);
  int32_t* start = reinterpret_cast<int32_t*>(tmem_ptr + 1);   // [2]

  const uint32_t b0 = smem_u32(bars);
  auto full = [&](int s) { return b0 + 8u * s; };
  auto empty = [&](int s) { return b0 + 8u * (kMaxStages + s); };
  auto s_full = [&](int s) { return b0 + 8u * (2 * kMaxStages + s); };
  const uint32_t p_full = b0 + 8u * (2 * kMaxStages + 2), p_empty = b0 + 8u * (2 * kMaxStages + 3);
  auto q_full = [&](int s) { return b0 + 8u * (2 * kMaxStages + 4 + s); };
  auto q_empty = [&](int s) { return b0 + 8u * (2 * kMaxStages + 6 + s); };
  const uint32_t o_empty = b0 + 8u * (2 * kMaxStages + 8);
  auto s_empty = [&](int s) { return b0 + 8u * (2 * kMaxStages + 9 + s); };
  auto drained = [&](int s) { return b0 + 8u * (2 * kMaxStages + 11 + s); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {
    if (threadIdx.x == 0) report_error(a.error_flag, kErrMisaligned);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 4);
      mbar_init(empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full(s), 1);
      mbar_init(q_full(s), 1);
      mbar_init(q_empty(s), 1);
      mbar_init(s_empty(s), 8);
      mbar_init(drained(s), 1);
    }
    mbar_init(p_full, 8);
    mbar_init(p_empty, 1);
    mbar_init(o_empty, 8);
    fence_mbarrier_init();
  }
  if (warp == kQkWarp) tmem_alloc<1>(smem_u32(tmem_ptr), C::kTmem);
  griddep_wait();   // what the stream's kernels before this one wrote may be read from here on

  if (threadIdx.x == kLoadWarp * 32) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.kr);
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.qr);
  }
  Work work = share_of<kTile, kSegmentCost, kThreads>(a, blockIdx.x, gridDim.x, blockIdx.x == 0, tmp, start);
  griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const uint32_t t_o = tmem + 4 * NH;
  bool failed = false;

  if (warp >= kLoadWarp && warp < kQkWarp) {
    // -------------------------------------------------------------------- loads
    const int w = warp - kLoadWarp;
    // this warp loads groups 2 w and 2 w + 1 (of 8 keys) of every tile: lanes 0 and 1 their
    // latent rows, lanes 2 and 3 the rotary ones (lane 2 both, in boxes of 16).  (Bringing tiles
    // into L2 ahead of their load gained 1.6 % at 64 rows of up to 16411 keys and lost 3 % at
    // D = 256 with 64 heads.)
    const int grp = 2 * w + (lane & 1);
    const bool is_rope = lane & 2, loads = !is_rope || (a.box_mask >> grp & 1u);
    Segment sg;
    int g = 0;
    while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
      const int b = sg.row / a.s1;
      const int32_t* table = a.block_table + (int64_t)b * a.max_blocks;
      auto page_of = [&](int tile) {   // -1: no such page
        const int pos = tile * kTile + grp * 8;
        if (lane >= 4 || pos >= sg.keys) return -1;
        const int id = table[pos / a.page_size];
        if (id >= a.num_pages && !is_rope) report_error(a.error_flag, kErrBadIndex);
        return id < a.num_pages ? id : -1;
      };
      int page = page_of(sg.first);
      for (int i = 0; i < sg.count; ++i, ++g) {
        const int st = g % C::kStages, tile = sg.first + i;
        const int now = page;
        if (i + 1 < sg.count) page = page_of(tile + 1);
        if (g >= C::kStages) mbar_wait_hot(empty(st), (g / C::kStages - 1) & 1, a.error_flag, &failed);
        failed = __any_sync(0xffffffffu, failed);
        if (failed) break;
        const uint32_t mask = __ballot_sync(0xffffffffu, now >= 0) & 3u;
        const uint32_t dst = base + st * C::kStageBytes;
        if (lane == 0) {
          tmask[4 * st + w] = (int)mask;
          const uint32_t bytes = __popc(mask) * C::kGroupBytes + __popc(mask & a.box_mask) * (a.box_rows * 128);
          if (bytes) mbar_arrive_expect_tx(full(st), bytes);
          else mbar_arrive(full(st));
        }
        __syncwarp();
        if (now >= 0 && loads)
          tma_load_4d(dst + (is_rope ? C::kKeyBytes + grp * 1024 : grp * C::kGroupBytes),
                      is_rope ? &maps.kr : &maps.k, full(st), 0, (tile * kTile + grp * 8) % a.page_size, 0, now);
      }
    }
    if (failed) {   // the copies in flight land before the CTA ends
      bool gave_up = false;
      for (int t = max(0, g - C::kStages); t < g; ++t)
        mbar_wait(full(t % C::kStages), (t / C::kStages) & 1, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp == kQueryWarp) {
    // -------------------------------------------------------------------- queries
    Segment sg;
    int nseg = 0;
    while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
      const int b = sg.row / a.s1, s = sg.row - b * a.s1;
      const int buf = nseg % C::kQBufs, use = nseg / C::kQBufs;
      if (use > 0) mbar_wait_hot(q_empty(buf), (use - 1) & 1, a.error_flag, &failed);
      failed = __any_sync(0xffffffffu, failed);
      if (failed) break;
      if (lane == 0) {
        const uint32_t dst = s_q + buf * C::kQBytes;
        mbar_arrive_expect_tx(q_full(buf), C::kQBytes);
        tma_load_5d(dst, &maps.q, q_full(buf), 0, 0, 0, s, b);
        tma_load_5d(dst + NH * D * 2, &maps.qr, q_full(buf), 0, 0, 0, s, b);
      }
      __syncwarp();
      ++nseg;
    }
    if (failed) {
      bool gave_up = false;
      for (int t = max(0, nseg - C::kQBufs); t < nseg; ++t)
        mbar_wait(q_full(t % C::kQBufs), (t / C::kQBufs) & 1, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp == kQkWarp || warp == kPvWarp) {
    // -------------------------------------------------------------------- MMA
    // S and O are made by a warp each: an issuing warp is held up while the tensor core is busy,
    // and a look at a barrier takes some 100 cycles beside the core's operand reads, so one warp
    // for both left gaps between them.
    Segment sg;
    int g = 0, nseg = 0;
    if (warp == kQkWarp) {
      constexpr uint32_t kIdQk = idesc_f16(64, NH, kBf16, false, false);
      while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
        const int buf = nseg % C::kQBufs;
        mbar_wait_hot(q_full(buf), (nseg / C::kQBufs) & 1, a.error_flag, &failed);
        for (int i = 0; i < sg.count; ++i, ++g) {
          const int st = g % C::kStages;
          if (g >= 2) mbar_wait_hot(s_empty(g & 1), ((g >> 1) - 1) & 1, a.error_flag, &failed);
          mbar_wait_hot(full(st), (g / C::kStages) & 1, a.error_flag, &failed);
          failed = __any_sync(0xffffffffu, failed);
          if (failed) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ka = smem_desc_sw128(base + st * C::kStageBytes, 16, C::kGroupBytes);
            const uint64_t ra = smem_desc_sw128(base + st * C::kStageBytes + C::kKeyBytes, 16, 1024);
            const uint64_t qb = smem_desc_sw128(s_q + buf * C::kQBytes, 16, 1024);
            // in two sums over half of the k-steps each, added by the softmax warps: the core cuts
            // off what a sum's fp32 does not hold, and half as many, half as large cuts leave half
            // the error (softmax_max 1.8e-6 too low in one sum)
            const uint32_t d = tmem + (g & 1) * 2 * NH;
            constexpr int kSteps = 4 * C::kChunks + 4;
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
              const int c = u / 4, k = u % 4;
              umma_f16<1>(d + (u < kSteps / 2 ? 0 : NH),
                          c < C::kChunks ? ka + ((c * 1024 + k * 32) >> 4) : ra + ((k * 32) >> 4),
                          qb + ((c * NH * 128 + k * 32) >> 4), kIdQk, u % (kSteps / 2) > 0);
            }
            umma_commit(s_full(g & 1));
            if (i == sg.count - 1) umma_commit(q_empty(buf));
          }
          __syncwarp();
        }
        ++nseg;
      }
    } else {
      constexpr uint32_t kIdPv = idesc_f16(128, NH, kBf16, true, true);
      while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
        for (int i = 0; i < sg.count; ++i, ++g) {
          const int st = g % C::kStages;
          if (i == 0 && nseg > 0) mbar_wait_hot(o_empty, (nseg - 1) & 1, a.error_flag, &failed);
          mbar_wait_hot(p_full, g & 1, a.error_flag, &failed);
          failed = __any_sync(0xffffffffu, failed);
          if (failed) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t va = smem_desc_sw128(base + st * C::kStageBytes, 1024, C::kGroupBytes);
            const uint64_t pb = p_desc<NH>(s_p);
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
#pragma unroll
              for (int m = 0; m < C::kBlocks; ++m)
                umma_f16<1>(t_o + m * NH, va + ((k * 2 * C::kGroupBytes + m * 2048) >> 4),
                            pb + ((k * 16 * NH * 2) >> 4), kIdPv, (i > 0) | (k > 0));
            umma_commit(empty(st));
            umma_commit(p_empty);
          }
          __syncwarp();
        }
        ++nseg;
      }
    }
    if (failed) {   // the products in flight end before the tensor memory is given back
      bool gave_up = false;
      const uint32_t bar = drained(warp == kQkWarp ? 0 : 1);
      if (elect_one()) umma_commit(bar);
      __syncwarp();
      mbar_wait(bar, 0, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp < kLoadWarp) {
    // -------------------------------------------------------------------- softmax
    constexpr int HW = C::kHeads;    // heads of this warpgroup, from `head0` on
    constexpr int kPairs = HW / 8;   // column pairs of a thread
    constexpr int kCols = HW < 16 ? 8 : 16;
    const int wg = warp >> 2, quarter = warp & 3, head0 = wg * HW;
    // scores in log2 units are raw * c2; a negative scale turns the raw scores over
    const bool flip = a.scale < 0.0f;
    // (a scale of 0 leaves masked keys, whose raw score is -inf, at -inf)
    const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-38f);
    const uint32_t lane_base = (uint32_t)quarter * 32u << 16;
    // a failed wait is not a way out of this loop: the four warps meet at their barrier as often
    // as there are tiles, and only the waits are passed over
    const int key0 = quarter * 16 + (lane >> 2);   // and key0 + 8
    const int col = head0 + 2 * (lane & 3);     // heads 8 i + col, 8 i + col + 1
    // per column: the reference of the exponents in log2 units (one for all four warps), the raw
    // score above which it has to be raised, this thread's running maximum (raw) and sum
    float ref[2 * kPairs], lim[2 * kPairs], run[2 * kPairs], sum[2 * kPairs];
    Segment sg;
    int g = 0, nseg = 0;
    while (next_segment<kTile, kSegmentCost>(a, work, sg)) {
#pragma unroll
      for (int j = 0; j < 2 * kPairs; ++j) {
        ref[j] = run[j] = lim[j] = -INFINITY;
        sum[j] = 0.0f;
      }
      for (int i = 0; i < sg.count; ++i, ++g) {
        const int st = g % C::kStages;
        mbar_wait_hot(full(st), (g / C::kStages) & 1, a.error_flag, &failed);
        const uint32_t mask = (uint32_t)tmask[4 * st + quarter];   // of this warp's 16 keys
        const int valid = sg.keys - (sg.first + i) * kTile;        // keys of this tile, >= 1
        const bool whole_tile = valid >= kTile && mask == 3u;
        mbar_wait_hot(s_full(g & 1), (g >> 1) & 1, a.error_flag, &failed);
        tc_fence_after();
        uint32_t raw[HW / 2], more[HW / 2];
        tmem_ld_frag<HW>(tmem + (g & 1) * 2 * NH + head0 + lane_base, raw);
        tmem_ld_frag<HW>(tmem + (g & 1) * 2 * NH + NH + head0 + lane_base, more);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty(g & 1));

        float z[HW / 2];
#pragma unroll
        for (int j = 0; j < HW / 2; ++j) z[j] = __uint_as_float(raw[j]) + __uint_as_float(more[j]);
        if (flip)
#pragma unroll
          for (int j = 0; j < HW / 2; ++j) z[j] = -z[j];
        if (!whole_tile) {
          const bool ok0 = (mask & 1u) && key0 < valid, ok1 = (mask & 2u) && key0 + 8 < valid;
#pragma unroll
          for (int j = 0; j < kPairs; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (!ok0) z[4 * j + e] = -INFINITY;
              if (!ok1) z[4 * j + 2 + e] = -INFINITY;
            }
        }
        bool raise = i == 0;
#pragma unroll
        for (int j = 0; j < 2 * kPairs; ++j) {
          const float m = fmaxf(z[4 * (j >> 1) + (j & 1)], z[4 * (j >> 1) + 2 + (j & 1)]);
          raise |= m > lim[j];
          run[j] = fmaxf(run[j], m);
        }
        // The maxima of the columns are joined over the warpgroup only where the reference has
        // to move: at the first tile, and when a score passes it by 2^8, which keeps the
        // probabilities within range.  Otherwise one barrier per tile tells that nobody asks.
        if (named_bar_or(1 + wg, kSoftmaxThreads, raise)) {
          float top[2 * kPairs];
#pragma unroll
          for (int j = 0; j < 2 * kPairs; ++j) top[j] = run[j];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
#pragma unroll
            for (int j = 0; j < 2 * kPairs; ++j)
              top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
          if (lane < 4)
#pragma unroll
            for (int j = 0; j < kPairs; ++j)
              *reinterpret_cast<float2*>(wmax + quarter * NH + 8 * j + col) =
                  make_float2(top[2 * j], top[2 * j + 1]);
          softmax_bar(wg);
          float f[2 * kPairs];
#pragma unroll
          for (int j = 0; j < 2 * kPairs; ++j) {
            const int h = 8 * (j >> 1) + col + (j & 1);
            const float m = fmaxf(fmaxf(wmax[h], wmax[NH + h]), fmaxf(wmax[2 * NH + h], wmax[3 * NH + h]));
            const float now = m == -INFINITY ? -INFINITY : m * c2;   // no key so far: stays -inf
            f[j] = ref[j] == now ? 1.0f : exp2f(ref[j] - now);
            sum[j] *= f[j];
            ref[j] = now;
            lim[j] = (now + kRescale) / c2;
          }
          if (quarter == 0 && lane < 4)
#pragma unroll
            for (int j = 0; j < 2 * kPairs; ++j) factor[8 * (j >> 1) + col + (j & 1)] = f[j];
          softmax_bar(wg);   // the factors are there, the maxima read
          if (i > 0) {
            mbar_wait_hot(p_empty, (g - 1) & 1, a.error_flag, &failed);
            tc_fence_after();
#pragma unroll 1
            for (int m = 0; m < C::kBlocks; ++m)
#pragma unroll 1
              for (int h0 = head0; h0 < head0 + HW; h0 += kCols) {
                uint32_t o[kCols];
                tmem_ld_cols(t_o + m * NH + h0 + lane_base, o);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < kCols; ++j)
                  o[j] = __float_as_uint(__uint_as_float(o[j]) * factor[h0 + j]);
                tmem_st_cols(t_o + m * NH + h0 + lane_base, o);
              }
            tmem_st_wait();
          }
          softmax_bar(wg);   // the factors are read: the next tile may write its own
        }
        const bool p_free = g == 0 || mbar_test_wait(p_empty, (g - 1) & 1);   // used below
        // probabilities, summed in fp32 and rounded for the product; a column without any key so
        // far has reference -inf and stays zero
        uint32_t packed[HW / 4];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float r = ref[2 * j + e] == -INFINITY ? 0.0f : kShift - ref[2 * j + e];
            p[e] = exp2_approx(fmaf(z[4 * j + e], c2, r));
            p[2 + e] = exp2_approx(fmaf(z[4 * j + 2 + e], c2, r));
            sum[2 * j + e] += p[e] + p[2 + e];
          }
          packed[2 * j] = E::pack2(p[0], p[1]);
          packed[2 * j + 1] = E::pack2(p[2], p[3]);
        }
        if (!p_free) mbar_wait_hot(p_empty, (g - 1) & 1, a.error_flag, &failed);
        uint8_t* ps = smem + (s_p - base);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          *reinterpret_cast<uint32_t*>(ps + p_offset<NH>(key0, head0 / 8 + j) + 4 * (lane & 3)) = packed[2 * j];
          *reinterpret_cast<uint32_t*>(ps + p_offset<NH>(key0 + 8, head0 / 8 + j) + 4 * (lane & 3)) = packed[2 * j + 1];
        }
        if (valid < kTile || mask != 3u) {
          // rows of this tile that no key stands in hold what was there before (or a page's
          // stale tail): cleared, so that 0 x NaN cannot enter the product
          const int key = quarter * 16 + (lane >> 1);
          if (key >= valid || !(mask >> (key >> 3 & 1) & 1u)) {
            uint8_t* row = smem + st * C::kStageBytes + (key >> 3) * C::kGroupBytes + (key & 7) * 128;
            for (int c = 2 * wg + (lane & 1); c < C::kChunks; c += 4)
#pragma unroll
              for (int x = 0; x < 8; ++x)
                *reinterpret_cast<uint4*>(row + c * 1024 + x * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }

      // ---- the segment's result: maxima and sums over the warpgroup ----
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 2 * kPairs; ++j) {
          sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
          run[j] = fmaxf(run[j], __shfl_xor_sync(0xffffffffu, run[j], o));
        }
      float* wsum = wmax + 4 * NH;
      if (lane < 4)
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          *reinterpret_cast<float2*>(wsum + quarter * NH + 8 * j + col) =
              make_float2(sum[2 * j], sum[2 * j + 1]);
          *reinterpret_cast<float2*>(wmax + quarter * NH + 8 * j + col) =
              make_float2(run[2 * j], run[2 * j + 1]);
        }
      softmax_bar(wg);
      // opaque, so that what hangs on it (a test per head) is not made before the loop and held in
      // registers through it: 28 bytes of spills at 64 heads, 140 us against 138 at D = 256
      int n1 = a.n1;
      asm volatile("" : "+r"(n1));
      const bool all = sg.count == sg.tiles, whole = all && a.diag == 0;
      const int64_t slot = all ? (int64_t)2 * gridDim.x + sg.row : 2 * blockIdx.x + (nseg == 0 ? 0 : 1);
      if (quarter == 0 && lane < 4)
#pragma unroll
        for (int j = 0; j < 2 * kPairs; ++j) {
          const int h = 8 * (j >> 1) + col + (j & 1);
          const float l = wsum[h] + wsum[NH + h] + wsum[2 * NH + h] + wsum[3 * NH + h];
          const float m = fmaxf(fmaxf(wmax[h], wmax[NH + h]), fmaxf(wmax[2 * NH + h], wmax[3 * NH + h]));
          const bool any = m != -INFINITY;
          const float most = any ? m * c2 : -INFINITY;
          factor[h] = !whole ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
          if (h >= n1) continue;
          if (!whole) {
            a.ws_s[slot * NH + h] = make_float4(ref[j] - kShift, most, l, m);
          } else if (a.softmax_max) {
            put_stats(a, (int64_t)sg.row * n1 + h, m, ref[j] - kShift, most, l);
          }
        }
      softmax_bar(wg);
      mbar_wait_hot(p_empty, (g - 1) & 1, a.error_flag, &failed);
      tc_fence_after();
      const int heads = min(head0 + HW, n1);
      const int dim = quarter * 32 + lane;
#pragma unroll 1
      for (int m = 0; m < C::kBlocks; ++m)
#pragma unroll 1
        for (int h0 = head0; h0 < heads; h0 += kCols) {
          uint32_t o[kCols];
          tmem_ld_cols(t_o + m * NH + h0 + lane_base, o);
          tmem_ld_wait();
          if (whole) {
            T* out = static_cast<T*>(a.out) +
                     ((int64_t)sg.row * n1 + h0) * D + m * 128 + dim;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
              if (h0 + j < heads) out[j * D] = E::from_f(__uint_as_float(o[j]) * factor[h0 + j]);
          } else {
            float* out = a.ws_o + (slot * NH + h0) * D + m * 128 + dim;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
              if (h0 + j < heads) out[j * D] = __uint_as_float(o[j]);
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty);
      ++nseg;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kQkWarp) {
    tmem_relinquish<1>();
    tmem_dealloc<1>(tmem, C::kTmem);
  }
}

// Where the parts of one (row, head) are: CTAs c0 .. c1, whose slot of a part is 2 c, but 2 c0 + 1
// where the row begins inside the share of c0; or the row's own slot (c0 == c1).
struct Parts {
  int c0, c1, skip, own;
  template <int NH>
  __device__ __forceinline__ int64_t at(int c, int h) const {
    return (int64_t)(c0 == c1 ? own : 2 * c + (c == c0 ? skip : 0)) * NH + h;
  }
};

// False for a row without a part (c1 < c0).
template <int kCost>
__device__ __forceinline__ bool parts_of(const Args& a, int grid, int row, Parts* p) {
  const int first = a.ws_prefix[row], next = a.ws_prefix[row + 1], all = a.ws_prefix[a.rows];
  const int count = next - first;   // units
  p->own = 2 * grid + row;
  p->skip = 0;
  p->c0 = 1;
  p->c1 = 0;
  if (count == 0) return false;
  const int64_t units = all, ctas = ctas_used(units, grid), x0 = first;
  const int64_t lo = (x0 + kCost + 1) * ctas - 1, hi = (x0 + count) * ctas - 1;
  if (units * ctas < (1LL << 32)) {
    const uint32_t u = (uint32_t)units;
    p->c0 = (int)((uint32_t)lo / u);
    p->c1 = (int)((uint32_t)hi / u);
  } else {
    p->c0 = (int)(lo / units);
    p->c1 = (int)(hi / units);
  }
  p->skip = share_begin(units, p->c0, ctas) < x0 ? 1 : 0;
  return true;
}

// q . k + qr . kr of packed head `head` of batch `b` and the key at position `pos`, by a warp; false
// if there is no such page.
template <int D, typename T>
__device__ __forceinline__ bool warp_dot(const Args& a, int b, int head, int pos, int lane, float* dot,
                                         const T** key) {
  const int page = a.block_table[(int64_t)b * a.max_blocks + pos / a.page_size], row = pos % a.page_size;
  if (page >= a.num_pages && lane == 0) report_error(a.error_flag, kErrBadIndex);
  if (page < 0 || page >= a.num_pages) return false;
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
  *dot = sum;
  *key = k;
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
  const bool some = parts_of<kCost>(a, grid, row, &p);
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
    const float4 s = a.ws_s[p.at<NH>(c, head)];
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
    const float4 s = a.ws_s[p.at<NH>(c, head)];
    const float4* o = reinterpret_cast<const float4*>(a.ws_o + p.at<NH>(c, head) * D) + col;
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
int heads_of(int64_t n1) { return n1 <= 16 ? 16 : n1 <= 32 ? 32 : n1 <= 64 ? 64 : 128; }

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// What the kernels take; `nh` heads a row, `shares` of the work.
Args make_args(const DsaAttnPagedParams* p, int nh, int shares, int diag, int heads) {
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
  const int64_t slots = (int64_t)2 * shares + (diag > 0 ? a.rows : 0);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.ws_o = reinterpret_cast<float*>(ws);
  ws += slots * nh * p->d * 4;
  a.ws_s = reinterpret_cast<float4*>(ws);
  ws += slots * nh * 16;
  a.ws_prefix = reinterpret_cast<int32_t*>(ws);
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
int launch_join(const DsaAttnPagedParams* p, const Args& a, int shares, cudaStream_t stream) {
  const int64_t items = p->batch * p->s1 * p->n1;
  // a block each up to eight a multiprocessor (what runs at once), else a warp each
  const bool wide = items <= 8LL * sm_count();
  const int64_t blocks = wide ? items : (items + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
  auto kern = wide ? attn_paged_combine_kernel<D, NH, kCost, kJoinThreads, T>
                   : attn_paged_combine_kernel<D, NH, kCost, 32, T>;
  return launch_early(kern, blocks, kJoinThreads, 0, stream, a, shares) ? DSA_OK : DSA_ERR_CUDA;
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
  return launch_join<D, NH, kSegmentCost, T>(p, a, grid, stream);
}

template <typename T>
int launch_pair(const DsaAttnPagedParams* p, int diag, int heads, cudaStream_t stream) {
  constexpr int D = 512;
  using C = pair::Cfg<D>;
  constexpr bool kBf16 = ElemTraits<T>::kIsBf16;
  const int pairs = sm_count() / 2;
  if (pairs < 1) return DSA_ERR_CUDA;
  Maps maps;
  CUtensorMap map_v;   // boxes of 8 or 16 keys, a CTA's half of the dims
  const uint64_t dims[4] = {64, (uint64_t)p->page_size, D / 64, (uint64_t)p->num_pages};
  const uint64_t st[3] = {(uint64_t)p->k_row_stride * 2, 128, (uint64_t)p->k_page_stride * 2};
  const uint32_t box[4] = {64, p->page_size % 16 ? 8u : 16u, C::kVChunks, 1};
  if (!make_maps<D>(&maps, p, kBf16, pair::kHeads) ||
      !make_tmap_16b(&map_v, p->key_cache, kBf16, 4, dims, st, box))
    return DSA_ERR_TMA_DESCRIPTOR;
  const Args a = make_args(p, 2 * pair::kHeads, pairs, diag, heads);
  auto kern = pair::attn_paged_pair_kernel<D, T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
      cudaSuccess)
    return DSA_ERR_CUDA;
  if (!launch_early(kern, 2 * pairs, pair::kThreads, C::kSmem, stream, maps, map_v, a)) return DSA_ERR_CUDA;
  return launch_join<D, 2 * pair::kHeads, pair::kSegmentCost, T>(p, a, pairs, stream);
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
  return launch_join<D, wide::kHeads, wide::kSegmentCost, T>(p, a, grid, stream);
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

// Whether several new tokens of a batch can be taken as one row of s1 * n1 heads, so that their
// keys are read once: up to 8 tokens, all of them valid (with act_q each is a row of its own), with
// 128 heads in all at most (4 x 8 tokens, 16 heads, D = 256, up to 65536 keys: 53 us against 115
// token by token; short rows lose, 8 x 2 tokens of 64 heads over 500 .. 4000 keys 31 against 28).
bool packs(int64_t s1, int64_t n1) {
  return s1 > 1 && s1 <= kMaxDiag + 1 && s1 * n1 <= 128;
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

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

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
  if (p->n1 < 1 || p->n1 > 128 || p->page_size < 8 || p->page_size % 8 || p->max_blocks < 1 ||
      p->num_pages < 1 || (p->sparse_mode != 0 && p->sparse_mode != 3) || !std::isfinite(p->scale) || !p->query ||
      !p->query_rope || !p->key_cache || !p->key_rope_cache || !p->act_k || !p->block_table ||
      !p->out || !p->workspace)
    return DSA_ERR_INVALID_ARG;
  // sizes the kernels index with 32 bits: rows * n1 blocks, tiles, pages
  constexpr int64_t kMax = 0x7fffffff;
  // (units are counted in 32 bits: a row's tiles and its start)
  if (p->batch > kMax || p->s1 > kMax || p->batch * p->s1 > kMax / p->n1 || p->num_pages > kMax ||
      p->page_size > (1 << 20) || p->max_blocks > (kMax - kTile) / p->page_size ||
      p->batch * p->s1 > kMax / ((p->max_blocks * p->page_size + kTile - 1) / kTile + 8))
    return DSA_ERR_INVALID_ARG;
  if ((p->softmax_max == nullptr) != (p->softmax_sum == nullptr)) return DSA_ERR_INVALID_ARG;
  const int64_t strides[10] = {p->q_head_stride,  p->q_token_stride,  p->q_batch_stride,
                               p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride,
                               p->k_row_stride,   p->k_page_stride,   p->kr_row_stride,
                               p->kr_page_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return DSA_ERR_INVALID_ARG;
  if (!aligned(p->query, 16) || !aligned(p->query_rope, 16) || !aligned(p->key_cache, 16) ||
      !aligned(p->key_rope_cache, 16) || !aligned(p->workspace, 32) || !aligned(p->out, 32))
    return DSA_ERR_INVALID_ARG;
  if (p->workspace_bytes < dsa_attn_paged_workspace_size(p->batch, p->s1, p->n1, p->d))
    return DSA_ERR_INVALID_ARG;
  if (p->dtype == DSA_DTYPE_BF16) return launch_dim<__nv_bfloat16>(p, stream);
  if (p->dtype == DSA_DTYPE_FP16) return launch_dim<__half>(p, stream);
  return DSA_ERR_INVALID_ARG;
}
