// Attention over the paged cache for more than 64 heads at D <= 256: a CTA per row, as in the
// kernel for fewer heads, but with the heads on the M side of the tensor core:
//   S [128 heads x 64 keys] = Q K^T     (M = 128, N = 64)
//   O [128 heads x D]      += P V       (M = 128, N = D)
// One copy of a key tile is the K-major operand K and, as the same bytes, the MN-major operand V.
// An instruction takes 32 B x (rows of A + rows of B) / 128 B cycles, so at D = 256 a tile costs
// 20 x 48 + 4 x 128 = 1,472 of them, where two items of 64 heads with the keys on the M side
// cost 2 x (20 x 32 + 8 x 48) = 2,048 and load every key twice.  The result and scores of two
// tiles (three at D = 128; in two sums each) fill the tensor memory; the probabilities take the place of their
// scores, as the operand A from tensor memory, which leaves shared memory for a fourth tile.
//
// A lane of tensor memory is a head, so the two warps that share 32 heads (one for each half of
// a tile's keys, and of the dims) need only each other: their barrier has 64 threads.
//
// 32 rows of 8192 .. 65536 keys, 128 heads: 185 us at D = 256 and 147 at D = 128, against 266 and
// 243 as two items of 64 heads.  A tile takes 2,200 and 1,850 cycles there: with two (three)
// buffers the way from S over the softmax (1,250) to the end of PV is what is waited for.
// (Probabilities through shared memory, and so three tiles at D = 256, took 191 and 156 us; the
// softmax warps' own look at the page table for the loads' barrier, 163 at D = 128.)
#pragma once

#include "attn_paged.cuh"
#include "sm100.cuh"

namespace dsa {
namespace attn_paged {
namespace wide {

constexpr int kTile = 64;
constexpr int kSegmentCost = 4;    // of starting a row, in tiles (8 rows of 4000 .. 32768 keys: 45 us
                                   // against 47 with 2)
constexpr int kHeads = 128;
constexpr int kLoadWarp = 8;       // warps 0-7: softmax; 8-11: loads
constexpr int kQkWarp = 12;
constexpr int kPvWarp = 13;
constexpr int kQueryWarp = 14;
constexpr int kThreads = 480;
constexpr int kMaxStages = 8;

constexpr int imin(int a, int b) { return a < b ? a : b; }

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kGroupBytes = kChunks * 1024;   // 8 keys: [chunk][8][128 B]
  static constexpr int kKeyBytes = 8 * kGroupBytes;
  static constexpr int kRopeBytes = kTile * 128;
  static constexpr int kQBytes = kHeads * (D + kRope) * 2;
  static constexpr int kSmallBytes = 2 * 2 * kHeads * 4 + 576;
  // latent and rotary parts in rings of their own, as the rotary ones are free after S
  static constexpr int kRoom = kSmemLimit - kQBytes - kSmallBytes;
  static constexpr int kStages = imin((kRoom - 2 * kRopeBytes) / kKeyBytes, kMaxStages);
  static constexpr int kRopes = imin((kRoom - kStages * kKeyBytes) / kRopeBytes, kStages);
  static constexpr int kOffRope = kStages * kKeyBytes;
  static constexpr int kOffQ = kOffRope + kRopes * kRopeBytes;
  static constexpr int kOffSmall = kOffQ + kQBytes;
  static constexpr int kSmem = kOffSmall + kSmallBytes;
  static constexpr int kBufs = (512 - D) / (2 * kTile);   // of S (in two sums) and P: 2 or 3
  static constexpr uint32_t kColsO = kBufs * 2 * kTile;
  static constexpr uint32_t kTmem = 512;
  static_assert(D <= 256 && kStages >= 4 && kRopes >= 2 && kSmem <= kSmemLimit, "a result of 128 heads has to leave room for the scores");
};

template <int D, typename T, typename A = Args>
__global__ void __launch_bounds__(kThreads, 1)
    attn_paged_wide_kernel(const __grid_constant__ Maps maps, const A a) {
  using C = Cfg<D>;
  using E = ElemTraits<T>;
  constexpr bool kBf16 = E::kIsBf16;
  constexpr float kShift = kBf16 ? 0.0f : 6.0f;   // half's probabilities are held 2^6 higher
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t s_q = base + C::kOffQ;
  float* wmax = reinterpret_cast<float*>(smem + C::kOffSmall);   // [2][kHeads]
  float* wsum = wmax + 2 * kHeads;                               // [2][kHeads]
  uint64_t* bars = reinterpret_cast<uint64_t*>(wsum + 2 * kHeads);
  int32_t* tmask = reinterpret_cast<int32_t*>(bars + 46);        // [kMaxStages][4]
  int32_t* tmp = tmask + 4 * kMaxStages;                         // [16]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmp + 16);
  int32_t* start = reinterpret_cast<int32_t*>(tmem_ptr + 1);     // [2]

  const uint32_t b0 = smem_u32(bars);
  auto full = [&](int s) { return b0 + 8u * s; };
  auto empty = [&](int s) { return b0 + 8u * (kMaxStages + s); };
  auto r_full = [&](int s) { return b0 + 8u * (2 * kMaxStages + s); };
  auto r_empty = [&](int s) { return b0 + 8u * (3 * kMaxStages + s); };
  auto s_full = [&](int s) { return b0 + 8u * (4 * kMaxStages + s); };
  auto p_full = [&](int s) { return b0 + 8u * (4 * kMaxStages + 3 + s); };
  auto p_empty = [&](int s) { return b0 + 8u * (4 * kMaxStages + 6 + s); };
  auto drained = [&](int s) { return b0 + 8u * (4 * kMaxStages + 9 + s); };
  const uint32_t q_full = b0 + 8u * (4 * kMaxStages + 11), q_empty = b0 + 8u * (4 * kMaxStages + 12);
  const uint32_t o_empty = b0 + 8u * (4 * kMaxStages + 13);
  constexpr int kBufs = C::kBufs;

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
    for (int s = 0; s < C::kRopes; ++s) {
      mbar_init(r_full(s), 4);
      mbar_init(r_empty(s), 1);
    }
    for (int s = 0; s < kBufs; ++s) {
      mbar_init(s_full(s), 1);
      mbar_init(p_full(s), 8);
      mbar_init(p_empty(s), 1);
    }
    mbar_init(drained(0), 1);
    mbar_init(drained(1), 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_empty, 8);
    fence_mbarrier_init();
  }
  if (warp == kQkWarp) tmem_alloc<1>(smem_u32(tmem_ptr), C::kTmem);
  griddep_wait();
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
  bool failed = false;
  Segment sg;
  int g = 0, nseg = 0;

  if (warp >= kLoadWarp && warp < kQkWarp) {
    // -------------------------------------------------------------------- loads
    // As in the kernel for fewer heads: this warp loads groups 2 w and 2 w + 1 (of 8 keys) of
    // every tile, lanes 0 and 1 their latent rows, lanes 2 and 3 the rotary ones.
    const int w = warp - kLoadWarp;
    const int grp = 2 * w + (lane & 1);
    const bool is_rope = lane & 2;
    int sent = 0;   // tiles of latent rows
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
        const int st = g % C::kStages, rs = g % C::kRopes, tile = sg.first + i;
        const int now = page, in_page = (key0 + tile * kTile + grp * 8) % a.page_size;
        if (i + 1 < sg.count) page = page_of(tile + 1);
        const uint32_t mask = __ballot_sync(0xffffffffu, now >= 0) & 3u;
        if (g >= C::kStages) mbar_wait_hot(empty(st), (g / C::kStages - 1) & 1, a.error_flag, &failed);
        failed = __any_sync(0xffffffffu, failed);
        if (failed) break;
        if (lane == 0) {
          tmask[4 * st + w] = (int)mask;
          const uint32_t bytes = __popc(mask) * C::kGroupBytes;
          if (bytes) mbar_arrive_expect_tx(full(st), bytes);
          else mbar_arrive(full(st));
        }
        __syncwarp();
        if (now >= 0 && !is_rope)
          tma_load_4d(base + st * C::kKeyBytes + grp * C::kGroupBytes, &maps.k, full(st), 0, in_page, 0, now);
        ++sent;
        if (g >= C::kRopes) mbar_wait_hot(r_empty(rs), (g / C::kRopes - 1) & 1, a.error_flag, &failed);
        failed = __any_sync(0xffffffffu, failed);
        if (failed) break;
        if (lane == 0) {
          const uint32_t bytes = __popc(mask & a.box_mask) * (a.box_rows * 128);
          if (bytes) mbar_arrive_expect_tx(r_full(rs), bytes);
          else mbar_arrive(r_full(rs));
        }
        __syncwarp();
        if (now >= 0 && is_rope && (a.box_mask >> grp & 1u))
          tma_load_4d(base + C::kOffRope + rs * C::kRopeBytes + grp * 1024, &maps.kr, r_full(rs), 0, in_page, 0, now);
      }
    }
    if (failed) {   // the copies in flight land before the CTA ends
      bool gave_up = false;
      for (int t = max(0, sent - C::kStages); t < sent; ++t)
        mbar_wait(full(t % C::kStages), (t / C::kStages) & 1, a.error_flag, &gave_up);
      for (int t = max(0, g - C::kRopes); t < g; ++t)
        mbar_wait(r_full(t % C::kRopes), (t / C::kRopes) & 1, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp == kQueryWarp) {
    // -------------------------------------------------------------------- queries
    while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
      const QueryAt at = row_query(a, sg.row);
      if (nseg > 0) mbar_wait_hot(q_empty, (nseg - 1) & 1, a.error_flag, &failed);
      failed = __any_sync(0xffffffffu, failed);
      if (failed) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, C::kQBytes);
        tma_load_5d(s_q, &maps.q, q_full, 0, at.head, 0, at.s, at.b);
        tma_load_5d(s_q + kHeads * D * 2, &maps.qr, q_full, 0, at.head, 0, at.s, at.b);
      }
      __syncwarp();
      ++nseg;
    }
    if (failed) {
      bool gave_up = false;
      if (nseg > 0) mbar_wait(q_full, (nseg - 1) & 1, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp == kQkWarp || warp == kPvWarp) {
    // -------------------------------------------------------------------- MMA, a warp for each product
    if (warp == kQkWarp) {
      constexpr uint32_t kIdQk = idesc_f16(kHeads, kTile, kBf16, false, false);
      const uint64_t qa = smem_desc_sw128(s_q, 16, 1024);
      while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
        mbar_wait_hot(q_full, nseg & 1, a.error_flag, &failed);
        for (int i = 0; i < sg.count; ++i, ++g) {
          const int st = g % C::kStages, rs = g % C::kRopes;
          mbar_wait_hot(full(st), (g / C::kStages) & 1, a.error_flag, &failed);
          mbar_wait_hot(r_full(rs), (g / C::kRopes) & 1, a.error_flag, &failed);
          // last what comes last: the probabilities stand in the scores' place until their product
          // is done (and a look at a barrier takes 200 cycles here)
          if (g >= kBufs) mbar_wait_hot(p_empty(g % kBufs), (g / kBufs - 1) & 1, a.error_flag, &failed);
          failed = __any_sync(0xffffffffu, failed);
          if (failed) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t kb = smem_desc_sw128(base + st * C::kKeyBytes, 16, C::kGroupBytes);
            const uint64_t rb = smem_desc_sw128(base + C::kOffRope + rs * C::kRopeBytes, 16, 1024);
            // in two sums over half of the k-steps each, as in the kernel for fewer heads
            const uint32_t d = tmem + (g % kBufs) * 2 * kTile;
            constexpr int kSteps = 4 * C::kChunks + 4;
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
              const int c = u / 4, k = u % 4;
              umma_f16<1>(d + (u < kSteps / 2 ? 0 : kTile), qa + ((c * kHeads * 128 + k * 32) >> 4),
                          c < C::kChunks ? kb + ((c * 1024 + k * 32) >> 4) : rb + ((k * 32) >> 4), kIdQk,
                          u % (kSteps / 2) > 0);
            }
            umma_commit(s_full(g % kBufs));
            umma_commit(r_empty(rs));
            if (i == sg.count - 1) umma_commit(q_empty);
          }
          __syncwarp();
        }
        ++nseg;
      }
    } else {
      constexpr uint32_t kIdPv = idesc_f16(kHeads, D, kBf16, false, true);
      while (!failed && next_segment<kTile, kSegmentCost>(a, work, sg)) {
        for (int i = 0; i < sg.count; ++i, ++g) {
          const int st = g % C::kStages;
          if (i == 0 && nseg > 0) mbar_wait_hot(o_empty, (nseg - 1) & 1, a.error_flag, &failed);
          mbar_wait_hot(p_full(g % kBufs), (g / kBufs) & 1, a.error_flag, &failed);
          failed = __any_sync(0xffffffffu, failed);
          if (failed) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vb = smem_desc_sw128(base + st * C::kKeyBytes, 1024, C::kGroupBytes);
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)   // 16 keys of P are 8 columns
              umma_f16_ts(tmem + C::kColsO, tmem + (g % kBufs) * 2 * kTile + 8 * k, vb + ((k * 2 * C::kGroupBytes) >> 4),
                          kIdPv, (i > 0) | (k > 0));
            umma_commit(empty(st));
            umma_commit(p_empty(g % kBufs));
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
    // Warps q and q + 4 hold heads 32 q .. 32 q + 31, a thread each, with half wg of the tile's keys
    // and of the dims.  No wait's failure is a way out of this loop: the two meet at their barrier
    // as often as there are tiles.
    const int wg = warp >> 2, q = warp & 3, h = 32 * q + lane;
    const uint32_t lane_addr = (uint32_t)(32 * q) << 16;
    const bool flip = a.scale < 0.0f;   // a negative scale turns the raw scores over
    const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-38f);
    constexpr int kDims = D / 2;   // of O, of one thread
    const uint32_t o_at = tmem + C::kColsO + wg * kDims + lane_addr;
    auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory"); };
    while (next_segment<kTile, kSegmentCost>(a, work, sg)) {
      float ref = -INFINITY, lim = -INFINITY, run = -INFINITY, sum = 0.0f;
      for (int i = 0; i < sg.count; ++i, ++g) {
        const int st = g % C::kStages;
        mbar_wait_hot(full(st), (g / C::kStages) & 1, a.error_flag, &failed);
        const int4 m4 = *reinterpret_cast<const int4*>(tmask + 4 * st);
        const uint32_t mask = m4.x | m4.y << 2 | m4.z << 4 | m4.w << 6;   // a bit per 8 keys
        const int valid = sg.keys - (sg.first + i) * kTile;               // keys of this tile, >= 1
        const bool tail = mask != 0xffu || valid < kTile;
        mbar_wait_hot(s_full(g % kBufs), (g / kBufs) & 1, a.error_flag, &failed);
        tc_fence_after();
        uint32_t r[32], more[32];
        const uint32_t s_at = tmem + (g % kBufs) * 2 * kTile + 32 * wg + lane_addr;
        tmem_ld32(s_at, r);
        tmem_ld32(s_at + kTile, more);
        tmem_ld_wait_regs(r);
        tmem_ld_wait_regs(more);
        tc_fence_before();
        float z[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = __uint_as_float(r[j]) + __uint_as_float(more[j]);
        if (flip)
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = -z[j];
        if (tail)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (32 * wg + j >= valid || !(mask >> (4 * wg + (j >> 3)) & 1u)) z[j] = -INFINITY;
        float top = z[0];
#pragma unroll
        for (int j = 1; j < 32; ++j) top = fmaxf(top, z[j]);
        run = fmaxf(run, top);
        // the reference moves at the first tile, and when a score passes it by 2^8
        if (named_bar_or(1 + q, 64, i == 0 || top > lim)) {
          wmax[wg * kHeads + h] = run;
          meet();
          const float m = fmaxf(wmax[h], wmax[kHeads + h]);
          const float now = m == -INFINITY ? -INFINITY : m * c2;
          const float f = ref == now ? 1.0f : exp2f(ref - now);
          sum *= f;
          ref = now;
          lim = (now + kRescale) / c2;
          if (i > 0) {
            mbar_wait_hot(p_empty((g - 1) % kBufs), (g - 1) / kBufs & 1, a.error_flag, &failed);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kDims; c += 16) {
              uint32_t o[16];
              tmem_ld16(o_at + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(o_at + c, o);
            }
            tmem_st_wait();
          }
          meet();   // the maxima are read
        }
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
        // in the place of the scores, which both warps have read before they met
        tc_fence_after();
        tmem_st16(tmem + (g % kBufs) * 2 * kTile + 16 * wg + lane_addr, pk);
        if (tail) {
          // rows of this tile that no key stands in hold what was there before (or a page's
          // stale tail): cleared, so that 0 x NaN cannot enter the product; 8 keys a warp
          const int key = 8 * warp + (lane >> 2);
          if (key >= valid || !(mask >> warp & 1u)) {
            uint8_t* row = smem + st * C::kKeyBytes + warp * C::kGroupBytes + (lane >> 2) * 128;
            for (int c = lane & 3; c < C::kChunks; c += 4)
#pragma unroll
              for (int x = 0; x < 8; ++x)
                *reinterpret_cast<uint4*>(row + c * 1024 + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(g % kBufs));
      }

      // ---- the segment's result ----
      wsum[wg * kHeads + h] = sum;
      wmax[wg * kHeads + h] = run;
      meet();
      const float l = wsum[h] + wsum[kHeads + h], m = fmaxf(wmax[h], wmax[kHeads + h]);
      meet();   // both are read: the next segment may write its own
      const float most = m != -INFINITY ? m * c2 : -INFINITY;
      const bool all = sg.count == sg.tiles, whole = all && !row_is_part(a, sg.row);
      const int64_t place = all ? own_place<kHeads>(a, gridDim.x, sg.row) : (int64_t)(2 * blockIdx.x + (nseg == 0 ? 0 : 1)) * kHeads;
      const int heads = row_heads(a, sg.row);
      const int64_t result = row_result(a, sg.row, heads);
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      if (wg == 0 && h < heads) {
        if (!whole)
          a.ws_s[place + h] = make_float4(ref - kShift, most, l, m);
        else if (a.softmax_max)
          put_stats(a, result + h, m, ref - kShift, most, l);
      }
      mbar_wait_hot(p_empty((g - 1) % kBufs), (g - 1) / kBufs & 1, a.error_flag, &failed);
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < kDims; c += 32) {
        uint32_t o[32];
        tmem_ld32(o_at + c, o);
        tmem_ld_wait_regs(o);
        if (h >= heads) {
          // a padded head: nothing to write
        } else if (whole) {   // whole 32-byte sectors, as a lane's neighbours write other rows
          T* out = static_cast<T*>(a.out) + (result + h) * D + wg * kDims + c;
#pragma unroll
          for (int j = 0; j < 32; j += 16) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[k] = E::pack2(__uint_as_float(o[j + 2 * k]) * inv, __uint_as_float(o[j + 2 * k + 1]) * inv);
            st_global_v8(out + j, v);
          }
        } else {
          float* out = a.ws_o + (place + h) * D + wg * kDims + c;
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

}  // namespace wide
}  // namespace attn_paged
}  // namespace dsa
