// Attention over the paged cache for up to 64 heads: a CTA per SM, keys on the M side of the tensor
// core.  attn_paged.cu has the mathematics.
#pragma once

#include "attn_paged.cuh"
#include "sm100.cuh"

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

template <int D, int NH, typename T, typename A = Args>
__global__ void __launch_bounds__(kThreads, 1)
    attn_paged_kernel(const __grid_constant__ Maps maps, const A a) {
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
    griddep_wait();   // (this kernel's end stands for the one's before it)
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
  release_next<false>(a);
  tc_fence_before();
  __syncthreads();
  release_next<true>(a);
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
      const int32_t* table = a.block_table + (int64_t)row_table(a, sg.row) * a.max_blocks;
      const int key0 = row_first(a, sg.row);
      auto page_of = [&](int tile) {   // -1: no such page
        const int pos = tile * kTile + grp * 8;
        if (lane >= 4 || pos >= sg.keys) return -1;
        const int id = table[(key0 + pos) / a.page_size];
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
                      is_rope ? &maps.kr : &maps.k, full(st), 0, (key0 + tile * kTile + grp * 8) % a.page_size, 0, now);
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
      const QueryAt at = row_query(a, sg.row);
      const int buf = nseg % C::kQBufs, use = nseg / C::kQBufs;
      if (use > 0) mbar_wait_hot(q_empty(buf), (use - 1) & 1, a.error_flag, &failed);
      failed = __any_sync(0xffffffffu, failed);
      if (failed) break;
      if (lane == 0) {
        const uint32_t dst = s_q + buf * C::kQBytes;
        mbar_arrive_expect_tx(q_full(buf), C::kQBytes);
        tma_load_5d(dst, &maps.q, q_full(buf), 0, at.head, 0, at.s, at.b);
        tma_load_5d(dst + NH * D * 2, &maps.qr, q_full(buf), 0, at.head, 0, at.s, at.b);
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
      int n1 = row_heads(a, sg.row);
      asm volatile("" : "+r"(n1));
      const bool all = sg.count == sg.tiles, whole = all && !row_is_part(a, sg.row);
      const int64_t place = all ? own_place<NH>(a, gridDim.x, sg.row) : (int64_t)(2 * blockIdx.x + (nseg == 0 ? 0 : 1)) * NH;
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
            a.ws_s[place + h] = make_float4(ref[j] - kShift, most, l, m);
          } else if (a.softmax_max) {
            put_stats(a, row_result(a, sg.row, n1) + h, m, ref[j] - kShift, most, l);
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
            T* out = static_cast<T*>(a.out) + (row_result(a, sg.row, n1) + h0) * D + m * 128 + dim;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
              if (h0 + j < heads) out[j * D] = E::from_f(__uint_as_float(o[j]) * factor[h0 + j]);
          } else {
            float* out = a.ws_o + (place + h0) * D + m * 128 + dim;
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

}  // namespace attn_paged
}  // namespace dsa
