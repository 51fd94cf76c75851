// Attention over the paged cache for more than 64 heads at D = 512: a pair of CTAs per row.
//
// The product of 128 heads x 512 dims fills the tensor memory of one SM, so a pair shares it
// (cta_group::2, M = 128: 64 heads in each CTA), as it shares the operands:
//   S [128 heads x 128 keys] = Q K^T: each CTA holds its 64 heads' queries and 64 of the keys
//   O [128 heads x D]       += P V:   each CTA holds its 64 heads' P and D / 2 of the dims of
//                                     all 128 keys
// so a CTA loads its keys whole (K-major) and its half of every key's value part (MN-major): the
// pool is read once from HBM, 1.9 times from L2.  Against two CTAs that each take 64 heads and
// all keys (the other kernel, twice) the tensor core's operand reads from shared memory fall
// from 555 KB to 260 KB per 128 keys and CTA, which is what bounded that form.
//
// A tile of 128 keys and the queries leave room for one buffer each of K and V at D = 512.  V is
// held in halves of 64 keys with barriers of their own, so that the next tile's first half is on
// its way while the second is in work.  32 rows of 8192 .. 65536 keys and 128 heads take
// 342 to 355 us in a burst (1,965 MHz) and 385 to 425 under the power cap, by the card (400 at
// 985 W and 1,470 to 1,530 MHz).  (Not kept, as slower at those rows: K in three
// parts of 192 dims, refilled one by one, 369 us against 347, since the loads then meet QK's
// operand reads, and shared memory, at 400 KB a tile and CTA, is what bounds this kernel; P in
// halves, 366 against 351; tiles brought into L2 ahead of their load, 364 against 356.)
#pragma once

#include "attn_paged.cuh"
#include "sm100.cuh"

namespace dsa {
namespace attn_paged {
namespace pair {

constexpr int kTile = 128;
constexpr int kSegmentCost = 4;    // of starting a row, in tiles
constexpr int kHeads = 64;          // of a CTA
constexpr int kSoftmaxThreads = 256;
constexpr int kKeyWarp = 8;         // warps 8-11 load K
constexpr int kValueWarp = 12;      // warps 12, 13 load V, warp 12 the queries too
constexpr int kMmaWarp = 14;
constexpr int kThreads = 480;

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kGroupBytes = kChunks * 1024;           // 8 keys of K: [chunk][8][128 B]
  static constexpr int kKeyBytes = 8 * kGroupBytes;            // this CTA's 64 keys
  static constexpr int kKBytes = kKeyBytes + 64 * 128;         // and their rotary parts
  static constexpr int kVChunks = D / 128;                     // this CTA's dims
  static constexpr int kHalfBytes = kVChunks * 64 * 128;       // of V: 64 keys
  static constexpr int kQBytes = kHeads * (D + kRope) * 2;
  static constexpr int kPBytes = kHeads * kTile * 2;
  static constexpr int kSmallBytes = 2 * 4 * kHeads * 4 + 384;
  static constexpr int kOffK = kQBytes;
  static constexpr int kOffV = kOffK + kKBytes;
  static constexpr int kOffP = kOffV + 2 * kHalfBytes;
  static constexpr int kOffSmall = kOffP + kPBytes;
  static constexpr int kSmem = kOffSmall + kSmallBytes;
  static constexpr int kPvN = 256;                             // dims of one PV instruction
  static constexpr int kPvs = D / kPvN;
  static constexpr uint32_t kColsO = 256;                      // after S of two tiles in two parts each
  static constexpr uint32_t kTmem = 512;
  static_assert(D == 512 && kSmem <= kSmemLimit, "one buffer of each operand has to fit");
};

// The tiles of a share one by one.
struct Tiles {
  Work w;
  Segment s;
  int i, seg;
  __device__ __forceinline__ bool next(const Args& a) {
    if (seg >= 0 && i + 1 < s.count) {
      ++i;
      return true;
    }
    i = 0;
    ++seg;
    return next_segment<kTile, kSegmentCost>(a, w, s);
  }
};

template <int D, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_paged_pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ CUtensorMap map_v,
                           const Args a) {
  using C = Cfg<D>;
  using E = ElemTraits<T>;
  constexpr bool kBf16 = E::kIsBf16;
  constexpr float kShift = kBf16 ? 0.0f : 6.0f;   // half's probabilities are held 2^6 higher
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  float* wmax = reinterpret_cast<float*>(smem + C::kOffSmall);   // [4][kHeads]
  float* wsum = wmax + 4 * kHeads;                               // [4][kHeads]
  uint64_t* bars = reinterpret_cast<uint64_t*>(wsum + 4 * kHeads);
  int32_t* tmp = reinterpret_cast<int32_t*>(bars + 16);          // [16]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmp + 16);
  int32_t* start = reinterpret_cast<int32_t*>(tmem_ptr + 1);     // [2]

  const uint32_t b0 = smem_u32(bars);
  const uint32_t k_full = b0, k_empty = b0 + 8;                // the leader's; each CTA's
  auto v_full = [&](int s) { return b0 + 16u + 8u * s; };      // leader's
  auto v_empty = [&](int s) { return b0 + 32u + 8u * s; };
  auto v_tail = [&](int s) { return b0 + 48u + 8u * s; };
  auto s_full = [&](int s) { return b0 + 64u + 8u * s; };
  const uint32_t q_full = b0 + 80, q_empty = b0 + 88;          // leader's; each CTA's
  const uint32_t p_full = b0 + 96, p_empty = b0 + 104;         // leader's; each CTA's
  const uint32_t o_empty = b0 + 112, drained = b0 + 120;       // leader's

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {   // the same in both CTAs
    if (threadIdx.x == 0) report_error(a.error_flag, kErrMisaligned);
    return;
  }
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    mbar_init(k_full, 4);
    mbar_init(k_empty, 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(v_full(s), 2);
      mbar_init(v_empty(s), 1);
      mbar_init(v_tail(s), 2);
      mbar_init(s_full(s), 1);
    }
    mbar_init(p_full, 16);
    mbar_init(drained, 1);
    mbar_init(p_empty, 1);
    mbar_init(o_empty, 16);
    fence_mbarrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc<2>(smem_u32(tmem_ptr), C::kTmem);
  griddep_wait();
  if (threadIdx.x == kKeyWarp * 32) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.kr);
    tma_prefetch_desc(&map_v);
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.qr);
  }
  Work work = share_of<kTile, kSegmentCost, kThreads>(a, blockIdx.x >> 1, gridDim.x >> 1, blockIdx.x == 0, tmp, start);
  griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  bool failed = false;

  // Lane l < 16 looks up the page of keys 8 l .. 8 l + 7 of a tile.  -1: no such page.  (Every
  // role that has to know which keys are there looks for itself, one tile ahead, so that nobody
  // waits for a message.)
  auto page_of = [&](const Segment& sg, const int32_t* table, int tile, bool tell) {
    const int pos = tile * kTile + lane * 8;
    if (lane >= 16 || pos >= sg.keys) return -1;
    const int id = table[pos / a.page_size];
    if (tell && id >= a.num_pages) report_error(a.error_flag, kErrBadIndex);
    return id < a.num_pages ? id : -1;
  };
  auto table_of = [&](const Segment& sg) { return a.block_table + (int64_t)(sg.row / a.s1) * a.max_blocks; };

  if (warp >= kKeyWarp && warp < kValueWarp) {
    // -------------------------------------------------------------------- K
    // This warp loads groups 2 w and 2 w + 1 (of 8 keys) of this CTA's 64 keys of every tile.
    // The leader's barrier counts the bytes of both CTAs.
    const int w = warp - kKeyWarp, g0 = 8 * (int)rank + 2 * w;
    const int grp = lane - 8 * (int)rank;
    Tiles t{work, {}, 0, -1};
    int g = 0, page = -1;
    for (; t.next(a); ++g) {
      const int32_t* table = table_of(t.s);
      const int tile = t.s.first + t.i;
      const int now = t.i == 0 ? page_of(t.s, table, tile, rank == 0 && w == 0) : page;
      if (t.i + 1 < t.s.count) page = page_of(t.s, table, tile + 1, rank == 0 && w == 0);
      const uint32_t mask = __ballot_sync(0xffffffffu, now >= 0);
      const int in_page = (tile * kTile + lane * 8) % a.page_size;
      if (g > 0) mbar_wait_hot(k_empty, (g - 1) & 1, a.error_flag, &failed);
      failed = __any_sync(0xffffffffu, failed);
      if (failed) break;
      if (rank == 0 && lane == 0) {
        // (of a rotary box of 16 keys the first half has to be there)
        const uint32_t both = mask & (3u << (2 * w) | 3u << (8 + 2 * w));
        const uint32_t bytes = __popc(both) * C::kGroupBytes + __popc(both & a.box_mask) * (a.box_rows * 128);
        if (bytes) mbar_arrive_expect_tx(k_full, bytes);
        else mbar_arrive(k_full);
      }
      __syncwarp();
      if (now >= 0 && (lane == g0 || lane == g0 + 1)) {
        const uint32_t bar = mapa_shared(k_full, 0), dst = base + C::kOffK;
        tma_load_4d_pair(dst + grp * C::kGroupBytes, &maps.k, bar, 0, in_page, 0, now);
        if (a.box_mask >> lane & 1u)
          tma_load_4d_pair(dst + C::kKeyBytes + grp * 1024, &maps.kr, bar, 0, in_page, 0, now);
      }
      __syncwarp();
    }
    if (failed && rank == 0) {   // the copies in flight, of both CTAs, land before the pair ends
      bool gave_up = false;
      if (g > 0) mbar_wait(k_full, (g - 1) & 1, a.error_flag, &gave_up, true);
    }
    __syncwarp();
  } else if (warp >= kValueWarp && warp < kMmaWarp) {
    // -------------------------------------------------------------------- V, queries
    // This warp loads half of each half of the tile, this CTA's dims of it, in boxes of box_rows keys,
    // [box][chunk][box_rows][128 B]; 16 where the page size allows, as a box takes a warp 160 cycles.
    // A tile with keys that are not there completes on barriers of the CTA's own, since its
    // softmax warps clear those rows before the product; their P then tells the leader.
    const int w = warp - kValueWarp;
    Tiles t{work, {}, 0, -1};
    int g = 0, page = -1;
    int sent = 0, tails = 0, queries = 0;   // halves, halves on the CTA's own barriers, segments' queries
    for (; t.next(a); ++g) {
      const int32_t* table = table_of(t.s);
      const int tile = t.s.first + t.i;
      const int now = t.i == 0 ? page_of(t.s, table, tile, false) : page;
      if (t.i + 1 < t.s.count) page = page_of(t.s, table, tile + 1, false);
      const uint32_t mask = __ballot_sync(0xffffffffu, now >= 0) & 0xffffu;
      const bool tail = mask != 0xffffu || t.s.keys - tile * kTile < kTile;
      const int in_page = (tile * kTile + lane * 8) % a.page_size;
      if (w == 0 && t.i == 0) {
        const int b = t.s.row / a.s1, s = t.s.row - b * a.s1;
        if (t.seg > 0) mbar_wait_hot(q_empty, (t.seg - 1) & 1, a.error_flag, &failed);
        failed = __any_sync(0xffffffffu, failed);
        if (failed) break;
        if (lane == 0) {
          const uint32_t bar = mapa_shared(q_full, 0);
          if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * C::kQBytes);
          tma_load_5d_pair(base, &maps.q, bar, 0, kHeads * (int)rank, 0, s, b);
          tma_load_5d_pair(base + kHeads * D * 2, &maps.qr, bar, 0, kHeads * (int)rank, 0, s, b);
        }
        ++queries;
        __syncwarp();
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if (g > 0) mbar_wait_hot(v_empty(hf), (g - 1) & 1, a.error_flag, &failed);
        failed = __any_sync(0xffffffffu, failed);
        if (failed) break;
        if (lane == 0) {
          const uint32_t bytes = __popc(mask & a.box_mask & (0xfu << (8 * hf + 4 * w))) * (a.box_rows * C::kVChunks * 128);
          if (tail) {
            if (bytes) mbar_arrive_expect_tx(v_tail(hf), bytes);
            else mbar_arrive(v_tail(hf));
          }
          if (rank == 0) {
            if (tail) mbar_arrive(v_full(hf));
            else mbar_arrive_expect_tx(v_full(hf), 2 * bytes);
          }
        }
        __syncwarp();
        if (now >= 0 && lane < 16 && (lane >> 2) == 2 * hf + w && (a.box_mask >> lane & 1u)) {
          const uint32_t dst = base + C::kOffV + lane * (C::kVChunks * 1024);
          if (tail)
            tma_load_4d(dst, &map_v, v_tail(hf), 0, in_page, C::kVChunks * (int)rank, now);
          else
            tma_load_4d_pair(dst, &map_v, mapa_shared(v_full(hf), 0), 0, in_page, C::kVChunks * (int)rank, now);
        }
        ++sent;
        tails += tail;
        __syncwarp();
      }
      if (failed) break;
    }
    if (failed) {   // half x is the x / 2-th use of its barrier
      bool gave_up = false;
      for (int x = max(0, tails - 2); x < tails; ++x)
        mbar_wait(v_tail(x & 1), (x >> 1) & 1, a.error_flag, &gave_up);
      for (int x = max(0, sent - 2); x < sent && rank == 0; ++x)
        mbar_wait(v_full(x & 1), (x >> 1) & 1, a.error_flag, &gave_up, true);
      if (queries > 0 && rank == 0) mbar_wait(q_full, (queries - 1) & 1, a.error_flag, &gave_up, true);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // -------------------------------------------------------------------- MMA (leader)
    if (rank == 0) {
      constexpr uint32_t kIdQk = idesc_f16(128, kTile, kBf16, false, false);
      constexpr uint32_t kIdPv = idesc_f16(128, C::kPvN, kBf16, false, true);
      // Whichever product has its operands goes next: QK(na) at most two tiles ahead of PV(nb),
      // which goes half by half, as there are two buffers of scores and PV(na - 2) waited for the
      // probabilities made of S(na - 2).  One warp issues both whole: with a warp for each (as in
      // the other kernel) their instructions alternate, and the same rows took 395 us for 349.
      // bytes between V's groups of 8 keys, and between its 128 dims of one instruction and the next
      const uint32_t v_group = a.box_rows == 16 ? 1024 : C::kVChunks * 1024;
      const uint32_t v_next = (2 * a.box_rows * 128) >> 4;
      Tiles q{work, {}, 0, -1}, v{work, {}, 0, -1};
      bool more_q = q.next(a), more_v = v.next(a);
      int na = 0, nb = 0, pb = 0;
      uint64_t t0 = 0;
      auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
      for (uint32_t idle = 0; more_v && !failed;) {
        if (more_q && na - nb < 2 &&
            all((q.i > 0 || mbar_test_wait_cluster(q_full, q.seg & 1)) && mbar_test_wait_cluster(k_full, na & 1))) {
          tc_fence_after();
          if (elect_one()) {
            const uint64_t qa = smem_desc_sw128(base, 16, 1024);
            const uint32_t ks = base + C::kOffK;
            const uint64_t kb = smem_desc_sw128(ks, 16, C::kGroupBytes);
            const uint64_t rb = smem_desc_sw128(ks + C::kKeyBytes, 16, 1024);
            // in two sums over half of the k-steps each, as in the other kernel
            const uint32_t d = tmem + 128 * (na & 1);
            constexpr int kSteps = 4 * C::kChunks + 4;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
              const int c = i / 4, u = i % 4;
              umma_f16<2>(d + (i < kSteps / 2 ? 0 : 64), qa + ((c * kHeads * 128 + u * 32) >> 4),
                          c < C::kChunks ? kb + ((c * 1024 + u * 32) >> 4) : rb + ((u * 32) >> 4), kIdQk,
                          i % (kSteps / 2) > 0);
            }
            umma_commit_pair(s_full(na & 1), 3);
            umma_commit_pair(k_empty, 3);
            if (q.i == q.s.count - 1) umma_commit_pair(q_empty, 3);
          }
          __syncwarp();
          more_q = q.next(a);
          ++na;
          idle = 0;
          continue;
        }
        if (nb < na && all((pb > 0 || mbar_test_wait_cluster(p_full, nb & 1)) &&
                           mbar_test_wait_cluster(v_full(pb), nb & 1) &&
                           (v.i + pb > 0 || v.seg == 0 || mbar_test_wait_cluster(o_empty, (v.seg - 1) & 1)))) {
          tc_fence_after();
          if (elect_one()) {
            const uint64_t pd = smem_desc_sw128(base + C::kOffP + pb * (kHeads * 128), 16, 1024);
            const uint64_t vb = smem_desc_sw128(base + C::kOffV + pb * C::kHalfBytes, a.box_rows * 128, v_group);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int n = 0; n < C::kPvs; ++n)
                umma_f16<2>(tmem + C::kColsO + n * (C::kPvN / 2), pd + ((k * 32) >> 4),
                            vb + ((k * 16 * C::kVChunks * 128) >> 4) + n * v_next, kIdPv, (v.i + pb > 0) | (k > 0));
            umma_commit_pair(v_empty(pb), 3);
            if (pb == 1) umma_commit_pair(p_empty, 3);
          }
          __syncwarp();
          if (pb == 1) {
            more_v = v.next(a);
            ++nb;
          }
          pb ^= 1;
          idle = 0;
          continue;
        }
        if ((++idle & 1023u) == 0) {   // nothing for long: a bounded wait
          const uint64_t now = globaltimer();
          if (idle == 1024u) t0 = now;
          else if (now - t0 > kWaitLimitNs) failed = true;
          failed = __any_sync(0xffffffffu, failed);
          if (failed && lane == 0) report_error(a.error_flag, kErrTimeout);
        }
      }
    }
    if (failed) {   // the products in flight end before the tensor memory is given back
      bool gave_up = false;
      if (elect_one()) umma_commit_pair(drained, 1);
      __syncwarp();
      mbar_wait(drained, 0, a.error_flag, &gave_up);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------------- softmax
    // Lanes 0-63 of the tensor memory hold this CTA's heads with the first half of the columns
    // (keys, or dims of O), lanes 64-127 the same heads with the second half; warpgroup wg
    // takes the wg-th half of those columns.  So four threads share a head.  No wait's failure is
    // a way out of this loop: the warps meet at their barrier as often as there are tiles.
    const int wg = warp >> 2, q = warp & 3, half = q >> 1;
    const int h = 32 * (q & 1) + lane, part = 2 * half + wg;
    const uint32_t lane_addr = (uint32_t)(32 * q) << 16;
    const bool flip = a.scale < 0.0f;   // a negative scale turns the raw scores over
    const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-38f);
    const uint32_t lead_p = mapa_shared(p_full, 0), lead_o = mapa_shared(o_empty, 0);
    uint8_t* prow = smem + C::kOffP + half * (kHeads * 128) + h * 128;
    constexpr int kDims = D / 4;   // of O, of one thread
    Work w = work;
    Segment sg;
    int g = 0, nseg = 0;
    int tails = 0;   // tiles with keys that are not there
    while (next_segment<kTile, kSegmentCost>(a, w, sg)) {
      const int32_t* table = table_of(sg);
      float ref = -INFINITY, lim = -INFINITY, run = -INFINITY, sum = 0.0f;
      int page = page_of(sg, table, sg.first, false);
      for (int i = 0; i < sg.count; ++i, ++g) {
        const int tile = sg.first + i;
        const uint32_t mask = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
        if (i + 1 < sg.count) page = page_of(sg, table, tile + 1, false);
        const int valid = sg.keys - tile * kTile;
        const bool tail = mask != 0xffffu || valid < kTile;
        mbar_wait_hot(s_full(g & 1), (g >> 1) & 1, a.error_flag, &failed);
        tc_fence_after();
        uint32_t r[32], more[32];
        const uint32_t s_at = tmem + 128 * (g & 1) + 32 * wg + lane_addr;
        tmem_ld32(s_at, r);
        tmem_ld32(s_at + 64, more);
        tmem_ld_wait_regs(r);
        tmem_ld_wait_regs(more);
        float z[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = __uint_as_float(r[j]) + __uint_as_float(more[j]);
        tc_fence_before();
        if (flip)
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = -z[j];
        if (tail) {
          const int k0 = 64 * half + 32 * wg;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (k0 + j >= valid || !(mask >> ((k0 + j) >> 3) & 1u)) z[j] = -INFINITY;
        }
        float top = z[0];
#pragma unroll
        for (int j = 1; j < 32; ++j) top = fmaxf(top, z[j]);
        run = fmaxf(run, top);
        // the reference moves at the first tile, and when a score passes it by 2^8
        if (named_bar_or(1, kSoftmaxThreads, i == 0 || top > lim)) {
          wmax[part * kHeads + h] = run;
          asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
          const float m = fmaxf(fmaxf(wmax[h], wmax[kHeads + h]), fmaxf(wmax[2 * kHeads + h], wmax[3 * kHeads + h]));
          const float now = m == -INFINITY ? -INFINITY : m * c2;
          const float f = ref == now ? 1.0f : exp2f(ref - now);
          sum *= f;
          ref = now;
          lim = (now + kRescale) / c2;
          if (i > 0) {
            mbar_wait_hot(p_empty, (g - 1) & 1, a.error_flag, &failed);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kDims; c += 16) {
              uint32_t o[16];
              tmem_ld16(tmem + C::kColsO + wg * kDims + c + lane_addr, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(tmem + C::kColsO + wg * kDims + c + lane_addr, o);
            }
            tmem_st_wait();
          }
          asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");   // the maxima are read
        }
        const bool p_free = g == 0 || mbar_test_wait(p_empty, (g - 1) & 1);
        // probabilities, summed in fp32 and rounded for the product (see attn_paged.cu); a head
        // without any key so far has reference -inf and stays zero
        const float off = ref == -INFINITY ? 0.0f : kShift - ref;
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float p0 = exp2_approx(fmaf(z[2 * j], c2, off));
          const float p1 = exp2_approx(fmaf(z[2 * j + 1], c2, off));
          sum += p0 + p1;
          pk[j] = E::pack2(p0, p1);
        }
        if (!p_free) mbar_wait_hot(p_empty, (g - 1) & 1, a.error_flag, &failed);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(prow + (((4 * wg + j) ^ (h & 7)) << 4)) =
              make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
        if (tail) {
          // rows of this tile that no key stands in hold what was there before (or a page's
          // stale tail): cleared, so that 0 x NaN cannot enter the product
          const int key = threadIdx.x >> 1;
          mbar_wait_hot(v_tail(key >> 6), tails & 1, a.error_flag, &failed);
          ++tails;
          if (key >= valid || !(mask >> (key >> 3) & 1u)) {
            const int box = key / a.box_rows;
            uint8_t* row = smem + C::kOffV + box * (a.box_rows * C::kVChunks * 128) + (key - box * a.box_rows) * 128;
            for (int c = threadIdx.x & 1; c < C::kVChunks; c += 2)
#pragma unroll
              for (int x = 0; x < 8; ++x)
                *reinterpret_cast<uint4*>(row + c * (a.box_rows * 128) + x * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) mbar_arrive(p_full);
          else mbar_arrive_cluster(lead_p);
        }
      }

      // ---- the segment's result ----
      wsum[part * kHeads + h] = sum;
      wmax[part * kHeads + h] = run;
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
      const float l = wsum[h] + wsum[kHeads + h] + wsum[2 * kHeads + h] + wsum[3 * kHeads + h];
      const float m = fmaxf(fmaxf(wmax[h], wmax[kHeads + h]), fmaxf(wmax[2 * kHeads + h], wmax[3 * kHeads + h]));
      const bool any = m != -INFINITY;
      const float most = any ? m * c2 : -INFINITY;
      const bool all = sg.count == sg.tiles, whole = all && a.diag == 0;
      const int64_t slot = all ? (int64_t)gridDim.x + sg.row : 2 * (blockIdx.x >> 1) + (nseg == 0 ? 0 : 1);
      const int head = kHeads * (int)rank + h;
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      if (part == 0 && head < a.n1) {
        if (!whole) {
          a.ws_s[slot * (2 * kHeads) + head] = make_float4(ref - kShift, most, l, m);
        } else if (a.softmax_max) {
          const int64_t at = (int64_t)sg.row * a.n1 + head;
          put_stats(a, at, m, ref - kShift, most, l);
        }
      }
      mbar_wait_hot(p_empty, (g - 1) & 1, a.error_flag, &failed);
      tc_fence_after();
      const int dim = half * (D / 2) + wg * kDims;
#pragma unroll 1
      for (int c = 0; c < kDims; c += 32) {
        uint32_t o[32];
        tmem_ld32(tmem + C::kColsO + wg * kDims + c + lane_addr, o);
        tmem_ld_wait_regs(o);
        if (head >= a.n1) {
          // a padded head: nothing to write
        } else if (whole) {   // whole 32-byte sectors, as a lane's neighbours write other rows
          T* out = static_cast<T*>(a.out) + ((int64_t)sg.row * a.n1 + head) * D + dim + c;
#pragma unroll
          for (int j = 0; j < 32; j += 16) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[k] = E::pack2(__uint_as_float(o[j + 2 * k]) * inv, __uint_as_float(o[j + 2 * k + 1]) * inv);
            st_global_v8(out + j, v);
          }
        } else {
          float* out = a.ws_o + (slot * (2 * kHeads) + head) * D + dim + c;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            const uint32_t v[8] = {o[j], o[j + 1], o[j + 2], o[j + 3], o[j + 4], o[j + 5], o[j + 6], o[j + 7]};
            st_global_v8(out + j, v);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) mbar_arrive(o_empty);
        else mbar_arrive_cluster(lead_o);
      }
      ++nseg;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == kMmaWarp) {
    tmem_relinquish<2>();
    tmem_dealloc<2>(tmem, C::kTmem);
  }
}

}  // namespace pair
}  // namespace attn_paged
}  // namespace dsa
