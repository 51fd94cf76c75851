// Attention of new tokens over the whole paged latent cache (MLA-absorb, one key head).
//
// For a query row r (one token) with n visible keys, head h and t < n:
//   z[h][t] = scale * (q[h] . k[t] + qr[h] . kr[t]),  m = max_t z,  p = exp(z - m),
//   l = sum_t p,  out[h] = (sum_t p k[t][0:D]) / l.
//
// attn_paged_kernel: a persistent CTA per SM takes an equal share of all (row, head group)
// tiles of 64 keys, so a long row is split over several CTAs and short rows share one.  The
// products are formed with the keys on the M side of the tensor core:
//   S^T [64 keys x NH heads]  = K [64 x (D + 64)] Q^T       (M = 64)
//   O^T [D x NH heads]       += V^T [D x 64] P^T            (M = 128, D / 128 blocks)
// One copy of a key tile in shared memory serves both: K-major rows for S^T, and the same
// bytes as the MN-major operand V^T.  The pool is read once, by TMA boxes of 8 keys (which
// never straddle a page, as page_size is a multiple of 8).
//
// attn_paged_combine_kernel joins the parts of rows that were split and writes zeros for rows
// that see no key.
#include <cuda_runtime.h>

#include "dsa_b200.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace dsa {
namespace attn_paged {

constexpr int kTile = 64;       // keys of a step
constexpr int kRope = 64;
constexpr int kSmemLimit = 232448;
constexpr int kSoftmaxThreads = 128;   // warps 0-3
constexpr int kThreads = 192;          // warp 4: loads, warp 5: MMA
constexpr int kMaxStages = 8;
constexpr int kMinTiles = 2;    // tiles a CTA takes at least: fewer cost more in joining than they save
constexpr float kRescale = 8.0f;       // log2 units the running max may pass the reference

template <int D, int NH>
struct Cfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kBlocks = D / 128;
  static constexpr int kGroupBytes = kChunks * 1024;   // 8 keys: [chunk][8][128 B]
  static constexpr int kKeyBytes = 8 * kGroupBytes;
  static constexpr int kRopeBytes = 64 * 128;
  static constexpr int kStageBytes = kKeyBytes + kRopeBytes;
  static constexpr int kQBytes = NH * (D + kRope) * 2;
  static constexpr int kPBytes = kTile * NH * 2;
  // row maxima of two tiles per warp, factors, barriers and the rest
  static constexpr int kSmallBytes = 2 * 4 * NH * 4 + NH * 4 + 512;
  static constexpr int kRoom = (kSmemLimit - kQBytes - kPBytes - kSmallBytes) / kStageBytes;
  static constexpr int kStages = kRoom < kMaxStages ? kRoom : kMaxStages;
  static constexpr int kSmem = kStages * kStageBytes + kQBytes + kPBytes + kSmallBytes;
  static constexpr uint32_t kCols = (2 + kBlocks) * NH;
  static constexpr uint32_t kTmem = kCols <= 32 ? 32 : kCols <= 64 ? 64 : kCols <= 128 ? 128
                                    : kCols <= 256 ? 256 : 512;
  static_assert(kStages >= 2, "two key tiles have to fit");
};

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
  int32_t* ws_prefix;   // [rows + 1] first tile of each row
  float* ws_o;          // [2 * CTAs][NH][D]
  float4* ws_s;         // [2 * CTAs][NH]: reference, running max, sum
  int32_t rows, s1, n1, groups;
  int32_t page_size, max_blocks, num_pages, mode;
  float scale;
};

// Keys that query row `row` sees.
__device__ __forceinline__ int row_keys(const Args& a, int row) {
  const int b = row / a.s1, s = row - b * a.s1;
  const int ak = a.act_k[b], aq = a.act_q ? a.act_q[b] : a.s1;
  int64_t n = min((int64_t)ak, (int64_t)a.max_blocks * a.page_size);
  if (a.mode == 3) n = min(n, (int64_t)ak - aq + s + 1);
  if (s >= aq || n < 0) n = 0;
  return (int)n;
}
__device__ __forceinline__ int row_tiles(const Args& a, int row) {
  return (row_keys(a, row) + kTile - 1) / kTile;
}

// CTAs that share `tiles` tiles.
__device__ __forceinline__ int64_t ctas_used(int64_t tiles, int grid) {
  const int64_t c = (tiles + kMinTiles - 1) / kMinTiles;
  return c < 1 ? 1 : c < grid ? c : grid;
}

// Exclusive prefix of v over the block (kThreads threads) and its total.
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

// One CTA's share: tiles from (row, head group, tile) on, `left` of them.
struct Work {
  int row, group, tile, left;
};
// A run of tiles of one (row, head group).
struct Segment {
  int row, group, first, count, keys, tiles;
};
// The next run of `w` (false when the share is done); `w` moves past it.
__device__ __forceinline__ bool next_segment(const Args& a, Work& w, Segment& s) {
  while (w.left > 0 && w.row < a.rows) {
    s.keys = row_keys(a, w.row);
    s.tiles = (s.keys + kTile - 1) / kTile;
    if (s.tiles == 0) {
      ++w.row;
      continue;
    }
    s.row = w.row;
    s.group = w.group;
    s.first = w.tile;
    s.count = min(s.tiles - w.tile, w.left);
    w.left -= s.count;
    w.tile = 0;
    if (++w.group == a.groups) {
      w.group = 0;
      ++w.row;
    }
    return true;
  }
  return false;
}

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
  if constexpr (N == 16)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  else if constexpr (N == 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
        "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

__device__ __forceinline__ void softmax_bar() {
  asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
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
  const uint32_t s_p = s_q + C::kQBytes;
  uint8_t* small = smem + C::kStages * C::kStageBytes + C::kQBytes + C::kPBytes;
  float* wmax = reinterpret_cast<float*>(small);          // [2][4][NH]
  float* factor = wmax + 2 * 4 * NH;                      // [NH]
  uint64_t* bars = reinterpret_cast<uint64_t*>(factor + NH);
  int32_t* tmask = reinterpret_cast<int32_t*>(bars + 32);  // [kMaxStages]
  int32_t* tmp = tmask + kMaxStages;                       // [16]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmp + 16);
  int32_t* start = reinterpret_cast<int32_t*>(tmem_ptr + 1);   // [3]

  const uint32_t b0 = smem_u32(bars);
  auto full = [&](int s) { return b0 + 8u * s; };
  auto empty = [&](int s) { return b0 + 8u * (kMaxStages + s); };
  auto s_full = [&](int s) { return b0 + 8u * (2 * kMaxStages + s); };
  auto s_empty = [&](int s) { return b0 + 8u * (2 * kMaxStages + 2 + s); };
  const uint32_t p_full = b0 + 8u * (2 * kMaxStages + 4), p_empty = b0 + 8u * (2 * kMaxStages + 5);
  const uint32_t q_full = b0 + 8u * (2 * kMaxStages + 6), q_empty = b0 + 8u * (2 * kMaxStages + 7);
  const uint32_t o_empty = b0 + 8u * (2 * kMaxStages + 8);
  const uint32_t drained = b0 + 8u * (2 * kMaxStages + 9);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {
    if (threadIdx.x == 0) report_error(a.error_flag, kErrMisaligned);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full(s), 1);
      mbar_init(s_empty(s), 4);
    }
    mbar_init(p_full, 4);
    mbar_init(p_empty, 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_empty, 4);
    mbar_init(drained, 1);
    fence_mbarrier_init();
  }
  if (warp == 5) tmem_alloc<1>(smem_u32(tmem_ptr), C::kTmem);

  // ---- this CTA's share of the tiles ----
  int64_t total = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    int sum;
    const int v = r < a.rows ? row_tiles(a, r) : 0;
    const int before = block_scan(v, tmp, &sum);
    if (blockIdx.x == 0 && r < a.rows) a.ws_prefix[r] = (int)total + before;
    total += sum;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ws_prefix[a.rows] = (int)total;
  griddep_launch_dependents();
  const int64_t tiles = total * a.groups;
  const int64_t ctas = ctas_used(tiles, gridDim.x);
  Work work{0, 0, 0, 0};
  int64_t from = 0;
  if (blockIdx.x < ctas) {
    from = tiles * blockIdx.x / ctas;
    work.left = (int)(tiles * (blockIdx.x + 1) / ctas - from);
  }
  {
    int64_t seen = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
      const int r = r0 + threadIdx.x;
      int sum;
      const int v = r < a.rows ? row_tiles(a, r) : 0;
      const int64_t first = (seen + block_scan(v, tmp, &sum)) * a.groups;
      if (v > 0 && first <= from && from < first + (int64_t)v * a.groups) {
        const int in = (int)(from - first);
        start[0] = r;
        start[1] = in / v;
        start[2] = in - (in / v) * v;
      }
      seen += sum;
      if (seen * a.groups > from) break;   // the same for every thread
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const uint32_t t_o = tmem + 2 * NH;
  if (work.left > 0) {
    work.row = start[0];
    work.group = start[1];
    work.tile = start[2];
  }
  bool failed = false;

  if (warp == 4) {
    // -------------------------------------------------------------------- loads
    if (lane == 0) {
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.qr);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.kr);
    }
    Segment sg;
    int g = 0, nseg = 0;
    while (!failed && next_segment(a, work, sg)) {
      const int b = sg.row / a.s1, s = sg.row - b * a.s1;
      const int32_t* table = a.block_table + (int64_t)b * a.max_blocks;
      // lane l < 8 takes keys 8 l .. 8 l + 7 of a tile; -1: no such page
      auto page_of = [&](int tile) {
        const int pos = tile * kTile + lane * 8;
        if (lane >= 8 || pos >= sg.keys) return -1;
        const int id = table[pos / a.page_size];
        if (id >= a.num_pages) report_error(a.error_flag, kErrBadIndex);
        return id < a.num_pages ? id : -1;
      };
      int page = page_of(sg.first);
      if (nseg > 0) mbar_wait(q_empty, (nseg - 1) & 1, a.error_flag, &failed);
      if ((failed = __any_sync(0xffffffffu, failed))) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, C::kQBytes);
        tma_load_5d(s_q, &maps.q, q_full, 0, sg.group * NH, 0, s, b);
        tma_load_5d(s_q + NH * D * 2, &maps.qr, q_full, 0, sg.group * NH, 0, s, b);
      }
      for (int i = 0; i < sg.count; ++i, ++g) {
        const int st = g % C::kStages, tile = sg.first + i;
        const int now = page;
        if (i + 1 < sg.count) page = page_of(tile + 1);
        if (g >= C::kStages) mbar_wait(empty(st), (g / C::kStages - 1) & 1, a.error_flag, &failed);
        if ((failed = __any_sync(0xffffffffu, failed))) break;
        const uint32_t mask = __ballot_sync(0xffffffffu, now >= 0);
        const uint32_t dst = base + st * C::kStageBytes;
        if (lane == 0) {
          tmask[st] = (int)mask;
          const uint32_t bytes = __popc(mask) * (C::kGroupBytes + 1024);
          if (bytes) mbar_arrive_expect_tx(full(st), bytes);
          else mbar_arrive(full(st));
        }
        __syncwarp();
        if (now >= 0) {
          const int in_page = (tile * kTile + lane * 8) % a.page_size;
          tma_load_4d(dst + lane * C::kGroupBytes, &maps.k, full(st), 0, in_page, 0, now);
          tma_load_4d(dst + C::kKeyBytes + lane * 1024, &maps.kr, full(st), 0, in_page, 0, now);
        }
      }
      ++nseg;
    }
    if (failed) {   // the copies in flight land before the CTA ends
      bool gave_up = false;
      if (nseg > 0) mbar_wait(q_full, (nseg - 1) & 1, a.error_flag, &gave_up);
      for (int t = max(0, g - C::kStages); t < g; ++t)
        mbar_wait(full(t % C::kStages), (t / C::kStages) & 1, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp == 5) {
    // -------------------------------------------------------------------- MMA
    constexpr uint32_t kIdQk = idesc_f16(64, NH, kBf16, false, false);
    constexpr uint32_t kIdPv = idesc_f16(128, NH, kBf16, true, true);
    bool pv_due = false, pv_first = false;
    int pv_tile = 0, pv_seg = 0;
    auto issue_pv = [&]() {
      if (pv_first && pv_seg > 0)
        mbar_wait_spin(o_empty, (pv_seg - 1) & 1, a.error_flag, &failed);
      mbar_wait_spin(p_full, pv_tile & 1, a.error_flag, &failed);
      pv_due = false;
      if ((failed = __any_sync(0xffffffffu, failed))) return;
      tc_fence_after();
      const int st = pv_tile % C::kStages;
      if (elect_one()) {
        const uint64_t va = smem_desc_sw128(base + st * C::kStageBytes, 1024, C::kGroupBytes);
        const uint64_t pb = p_desc<NH>(s_p);
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
#pragma unroll
          for (int m = 0; m < C::kBlocks; ++m)
            umma_f16<1>(t_o + m * NH, va + ((k * 2 * C::kGroupBytes + m * 2048) >> 4),
                        pb + ((k * 16 * NH * 2) >> 4), kIdPv, !(pv_first && k == 0));
        umma_commit(empty(st));
        umma_commit(p_empty);
      }
      __syncwarp();
    };
    Segment sg;
    int g = 0, nseg = 0;
    while (!failed && next_segment(a, work, sg)) {
      for (int i = 0; i < sg.count && !failed; ++i, ++g) {
        const int st = g % C::kStages;
        // while this tile's keys (or the segment's queries) are on their way, the product
        // of the tile before goes first
        if (pv_due) {
          const bool here = (i > 0 || mbar_try_wait(q_full, nseg & 1)) &&
                            mbar_try_wait(full(st), (g / C::kStages) & 1);
          if (!__all_sync(0xffffffffu, here)) issue_pv();
        }
        if (i == 0) mbar_wait_spin(q_full, nseg & 1, a.error_flag, &failed);
        mbar_wait_spin(full(st), (g / C::kStages) & 1, a.error_flag, &failed);
        if (g >= 2) mbar_wait_spin(s_empty(g & 1), ((g >> 1) - 1) & 1, a.error_flag, &failed);
        if ((failed = __any_sync(0xffffffffu, failed))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t ka = smem_desc_sw128(base + st * C::kStageBytes, 16, C::kGroupBytes);
          const uint64_t ra =
              smem_desc_sw128(base + st * C::kStageBytes + C::kKeyBytes, 16, 1024);
          const uint64_t qb = smem_desc_sw128(s_q, 16, 1024);
          const uint32_t d = tmem + (g & 1) * NH;
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16<1>(d, ka + ((c * 1024 + k * 32) >> 4), qb + ((c * NH * 128 + k * 32) >> 4),
                          kIdQk, c + k > 0);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16<1>(d, ra + ((k * 32) >> 4), qb + ((C::kChunks * NH * 128 + k * 32) >> 4),
                        kIdQk, 1);
          umma_commit(s_full(g & 1));
          if (i == sg.count - 1) umma_commit(q_empty);
        }
        __syncwarp();
        if (pv_due) issue_pv();
        pv_due = true;
        pv_first = i == 0;
        pv_tile = g;
        pv_seg = nseg;
      }
      ++nseg;
    }
    if (pv_due && !failed) issue_pv();
    if (failed) {   // the products in flight end before the tensor memory is given back
      bool gave_up = false;
      if (elect_one()) umma_commit(drained);
      __syncwarp();
      mbar_wait(drained, 0, a.error_flag, &gave_up);
      __syncwarp();
    }
  } else if (warp < 4) {
    // -------------------------------------------------------------------- softmax
    constexpr int kPairs = NH / 8;   // column pairs of a thread
    const float c2 = a.scale * 1.4426950408889634f;
    const uint32_t lane_base = (uint32_t)warp * 32u << 16;
    // a failed wait is not a way out of this loop: the four warps meet at their barrier as often
    // as there are tiles, and only the waits are passed over
    const int key0 = warp * 16 + (lane >> 2);   // and key0 + 8
    const int col = 2 * (lane & 3);             // heads 8 i + col, 8 i + col + 1
    float ref[2 * kPairs], run[2 * kPairs], sum[2 * kPairs];
    Segment sg;
    int g = 0, nseg = 0;
    while (next_segment(a, work, sg)) {
#pragma unroll
      for (int j = 0; j < 2 * kPairs; ++j) {
        ref[j] = run[j] = -INFINITY;
        sum[j] = 0.0f;
      }
      for (int i = 0; i < sg.count; ++i, ++g) {
        const int st = g % C::kStages;
        mbar_wait_spin(s_full(g & 1), (g >> 1) & 1, a.error_flag, &failed);
        mbar_wait_spin(full(st), (g / C::kStages) & 1, a.error_flag, &failed);
        tc_fence_after();
        uint32_t raw[NH / 2];
        tmem_ld_frag<NH>(tmem + (g & 1) * NH + lane_base, raw);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty(g & 1));

        const uint32_t mask = (uint32_t)tmask[st];
        const int valid = sg.keys - (sg.first + i) * kTile;   // keys of this tile, >= 1
        const bool ok0 = (mask >> (2 * warp) & 1u) && key0 < valid;
        const bool ok1 = (mask >> (2 * warp + 1) & 1u) && key0 + 8 < valid;
        float z[NH / 2], top[2 * kPairs];
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            z[4 * j + e] = ok0 ? __uint_as_float(raw[4 * j + e]) * c2 : -INFINITY;
            z[4 * j + 2 + e] = ok1 ? __uint_as_float(raw[4 * j + 2 + e]) * c2 : -INFINITY;
            top[2 * j + e] = fmaxf(z[4 * j + e], z[4 * j + 2 + e]);
          }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
          for (int j = 0; j < 2 * kPairs; ++j)
            top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
        float* wm = wmax + (g & 1) * 4 * NH;
        if (lane < 4)
#pragma unroll
          for (int j = 0; j < kPairs; ++j)
            *reinterpret_cast<float2*>(wm + warp * NH + 8 * j + col) =
                make_float2(top[2 * j], top[2 * j + 1]);
        softmax_bar();
        bool raise = false;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          float2 m = *reinterpret_cast<float2*>(wm + 8 * j + col);
#pragma unroll
          for (int w = 1; w < 4; ++w) {
            const float2 y = *reinterpret_cast<float2*>(wm + w * NH + 8 * j + col);
            m.x = fmaxf(m.x, y.x);
            m.y = fmaxf(m.y, y.y);
          }
          run[2 * j] = fmaxf(run[2 * j], m.x);
          run[2 * j + 1] = fmaxf(run[2 * j + 1], m.y);
          raise |= run[2 * j] > ref[2 * j] + kRescale || run[2 * j + 1] > ref[2 * j + 1] + kRescale;
        }
        if (i == 0) {
#pragma unroll
          for (int j = 0; j < 2 * kPairs; ++j) ref[j] = run[j];
        } else if (__any_sync(0xffffffffu, raise)) {
          // every warp sees the same maxima, so all four come here together
          if (g > 0) mbar_wait_spin(p_empty, (g - 1) & 1, a.error_flag, &failed);
            tc_fence_after();
#pragma unroll
          for (int j = 0; j < 2 * kPairs; ++j) {
            const float f = ref[j] == run[j] ? 1.0f : exp2f(ref[j] - run[j]);
            sum[j] *= f;
            ref[j] = run[j];
            if (warp == 0 && lane < 4) factor[8 * (j >> 1) + col + (j & 1)] = f;
          }
          softmax_bar();
#pragma unroll 1
          for (int cc = 0; cc < C::kBlocks * NH; cc += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + cc + lane_base, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              o[j] = __float_as_uint(__uint_as_float(o[j]) * factor[(cc + j) % NH]);
            tmem_st16(t_o + cc + lane_base, o);
          }
          tmem_st_wait();
        }
        // probabilities; a column without any key so far has reference -inf and stays zero
        uint32_t packed[NH / 4];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float r = ref[2 * j + e] == -INFINITY ? 0.0f : ref[2 * j + e] - kShift;
            p[e] = exp2f(z[4 * j + e] - r);
            p[2 + e] = exp2f(z[4 * j + 2 + e] - r);
            sum[2 * j + e] += p[e] + p[2 + e];
          }
          packed[2 * j] = E::pack2(p[0], p[1]);
          packed[2 * j + 1] = E::pack2(p[2], p[3]);
        }
        if (g > 0) mbar_wait_spin(p_empty, (g - 1) & 1, a.error_flag, &failed);
        uint8_t* ps = smem + (s_p - base);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          *reinterpret_cast<uint32_t*>(ps + p_offset<NH>(key0, j) + 2 * col) = packed[2 * j];
          *reinterpret_cast<uint32_t*>(ps + p_offset<NH>(key0 + 8, j) + 2 * col) = packed[2 * j + 1];
        }
        if (valid < kTile || mask != 0xffu) {
          // rows of this tile that no key stands in hold what was there before (or a page's
          // stale tail): cleared, so that 0 x NaN cannot enter the product
          const int key = threadIdx.x >> 1;
          if (key >= valid || !(mask >> (key >> 3) & 1u)) {
            uint8_t* row = smem + st * C::kStageBytes + (key >> 3) * C::kGroupBytes + (key & 7) * 128 +
                           (threadIdx.x & 1) * (C::kChunks / 2) * 1024;
            for (int c = 0; c < C::kChunks / 2; ++c)
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

      // ---- the segment's result ----
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 2 * kPairs; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
      float* ws = wmax + (g & 1) * 4 * NH;   // the maxima of the tile after this one come later
      if (lane < 4)
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
          *reinterpret_cast<float2*>(ws + warp * NH + 8 * j + col) =
              make_float2(sum[2 * j], sum[2 * j + 1]);
      softmax_bar();
      const bool whole = sg.count == sg.tiles;
      const int slot = 2 * blockIdx.x + (nseg == 0 ? 0 : 1);
      if (warp == 0 && lane < 4)
#pragma unroll
        for (int j = 0; j < 2 * kPairs; ++j) {
          const int h = 8 * (j >> 1) + col + (j & 1), head = sg.group * NH + h;
          const float l = ws[h] + ws[NH + h] + ws[2 * NH + h] + ws[3 * NH + h];
          factor[h] = !whole ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
          if (head >= a.n1) continue;
          if (!whole) {
            a.ws_s[(int64_t)slot * NH + h] = make_float4(ref[j] - kShift, run[j], l, 0.0f);
          } else if (a.softmax_max) {
            const int64_t at = (int64_t)sg.row * a.n1 + head;
            const bool any = run[j] != -INFINITY;
            a.softmax_max[at] = any ? run[j] * 0.6931471805599453f : 0.0f;
            a.softmax_sum[at] = any ? l * exp2f(ref[j] - kShift - run[j]) : 0.0f;
          }
        }
      softmax_bar();
      mbar_wait_spin(p_empty, (g - 1) & 1, a.error_flag, &failed);
      tc_fence_after();
      const int heads = min(NH, a.n1 - sg.group * NH);
      const int dim = warp * 32 + lane;
#pragma unroll 1
      for (int m = 0; m < C::kBlocks; ++m)
#pragma unroll 1
        for (int h0 = 0; h0 < heads; h0 += 16) {
          uint32_t o[16];
          tmem_ld16(t_o + m * NH + h0 + lane_base, o);
          tmem_ld_wait();
          if (whole) {
            T* out = static_cast<T*>(a.out) +
                     ((int64_t)sg.row * a.n1 + sg.group * NH + h0) * D + m * 128 + dim;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (h0 + j < heads) out[j * D] = E::from_f(__uint_as_float(o[j]) * factor[h0 + j]);
          } else {
            float* out = a.ws_o + ((int64_t)slot * NH + h0) * D + m * 128 + dim;
#pragma unroll
            for (int j = 0; j < 16; ++j)
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
  if (warp == 5) {
    tmem_relinquish<1>();
    tmem_dealloc<1>(tmem, C::kTmem);
  }
}

// One block per (row, head): join the parts that the row's CTAs left.
template <int D, int NH, typename T>
__global__ void __launch_bounds__(128) attn_paged_combine_kernel(const Args a, int grid) {
  using E = ElemTraits<T>;
  constexpr int kPer = D / 128;
  griddep_wait();
  const int row = blockIdx.x / a.n1, head = blockIdx.x - row * a.n1;
  const int64_t at = blockIdx.x;
  const int first = a.ws_prefix[row], count = a.ws_prefix[row + 1] - first;
  T* out = static_cast<T*>(a.out) + at * D + threadIdx.x * kPer;
  if (count == 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) out[j] = E::from_f(0.0f);
    if (threadIdx.x == 0 && a.softmax_max) a.softmax_max[at] = a.softmax_sum[at] = 0.0f;
    return;
  }
  const int64_t tiles = (int64_t)a.ws_prefix[a.rows] * a.groups;
  const int64_t ctas = ctas_used(tiles, grid);
  const int group = head / NH, h = head - group * NH;
  const int64_t x0 = (int64_t)first * a.groups + (int64_t)group * count, x1 = x0 + count;
  const int c0 = (int)(((x0 + 1) * ctas - 1) / tiles), c1 = (int)((x1 * ctas - 1) / tiles);
  if (c0 == c1) return;   // written whole
  // the part of CTA c is its first one unless the row begins inside its share
  auto slot = [&](int c) { return 2 * c + (tiles * c / ctas < x0 ? 1 : 0); };
  float ref = -INFINITY, run = -INFINITY;
  for (int c = c0; c <= c1; ++c) {
    const float4 s = a.ws_s[(int64_t)slot(c) * NH + h];
    ref = fmaxf(ref, s.x);
    run = fmaxf(run, s.y);
  }
  float acc[kPer] = {}, sum = 0.0f;
  if (ref != -INFINITY) {
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const int64_t sl = (int64_t)slot(c) * NH + h;
      const float4 s = a.ws_s[sl];
      const float w = s.x == ref ? 1.0f : exp2f(s.x - ref);
      sum += w * s.z;
      const float* o = a.ws_o + sl * D + threadIdx.x * kPer;
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] += w * o[j];
    }
  }
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) out[j] = E::from_f(acc[j] * inv);
  if (threadIdx.x == 0 && a.softmax_max) {
    const bool any = run != -INFINITY;
    a.softmax_max[at] = any ? run * 0.6931471805599453f : 0.0f;
    a.softmax_sum[at] = any ? sum * exp2f(ref - run) : 0.0f;
  }
}

int heads_of(int64_t n1) { return n1 <= 16 ? 16 : n1 <= 32 ? 32 : 64; }

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

template <int D, int NH, typename T>
int launch(const DsaAttnPagedParams* p, cudaStream_t stream) {
  using C = Cfg<D, NH>;
  constexpr bool kBf16 = ElemTraits<T>::kIsBf16;
  const int64_t b = p->batch, s1 = p->s1, n1 = p->n1;
  const int grid = sm_count();
  if (grid < 1) return DSA_ERR_CUDA;
  Maps maps;
  {
    const uint64_t dims[5] = {64, (uint64_t)n1, D / 64, (uint64_t)s1, (uint64_t)b};
    const uint64_t st[4] = {(uint64_t)p->q_head_stride * 2, 128, (uint64_t)p->q_token_stride * 2,
                            (uint64_t)p->q_batch_stride * 2};
    const uint32_t box[5] = {64, NH, D / 64, 1, 1};
    const uint64_t rdims[5] = {64, (uint64_t)n1, 1, (uint64_t)s1, (uint64_t)b};
    const uint64_t rst[4] = {(uint64_t)p->qr_head_stride * 2, 128, (uint64_t)p->qr_token_stride * 2,
                             (uint64_t)p->qr_batch_stride * 2};
    const uint32_t rbox[5] = {64, NH, 1, 1, 1};
    const uint64_t kdims[4] = {64, (uint64_t)p->page_size, D / 64, (uint64_t)p->num_pages};
    const uint64_t kst[3] = {(uint64_t)p->k_row_stride * 2, 128, (uint64_t)p->k_page_stride * 2};
    const uint32_t kbox[4] = {64, 8, D / 64, 1};
    const uint64_t krdims[4] = {64, (uint64_t)p->page_size, 1, (uint64_t)p->num_pages};
    const uint64_t krst[3] = {(uint64_t)p->kr_row_stride * 2, 128, (uint64_t)p->kr_page_stride * 2};
    const uint32_t krbox[4] = {64, 8, 1, 1};
    if (!make_tmap_16b(&maps.q, p->query, kBf16, 5, dims, st, box) ||
        !make_tmap_16b(&maps.qr, p->query_rope, kBf16, 5, rdims, rst, rbox) ||
        !make_tmap_16b(&maps.k, p->key_cache, kBf16, 4, kdims, kst, kbox) ||
        !make_tmap_16b(&maps.kr, p->key_rope_cache, kBf16, 4, krdims, krst, krbox))
      return DSA_ERR_TMA_DESCRIPTOR;
  }
  Args a;
  a.act_q = p->act_q;
  a.act_k = p->act_k;
  a.block_table = p->block_table;
  a.out = p->out;
  a.softmax_max = p->softmax_max;
  a.softmax_sum = p->softmax_sum;
  a.error_flag = p->error_flag;
  a.rows = (int)(b * s1);
  a.s1 = (int)s1;
  a.n1 = (int)n1;
  a.groups = (int)((n1 + NH - 1) / NH);
  a.page_size = (int)p->page_size;
  a.max_blocks = (int)p->max_blocks;
  a.num_pages = (int)p->num_pages;
  a.mode = p->sparse_mode;
  a.scale = p->scale;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.ws_o = reinterpret_cast<float*>(ws);
  ws += (int64_t)2 * grid * NH * D * 4;
  a.ws_s = reinterpret_cast<float4*>(ws);
  ws += (int64_t)2 * grid * NH * 16;
  a.ws_prefix = reinterpret_cast<int32_t*>(ws);

  auto kern = attn_paged_kernel<D, NH, T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
      cudaSuccess)
    return DSA_ERR_CUDA;
  kern<<<grid, kThreads, C::kSmem, stream>>>(maps, a);
  if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(b * s1 * n1));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, attn_paged_combine_kernel<D, NH, T>, a, grid) != cudaSuccess)
    return DSA_ERR_CUDA;
  return DSA_OK;
}

template <int D, typename T>
int launch_heads(const DsaAttnPagedParams* p, cudaStream_t stream) {
  switch (heads_of(p->n1)) {
    case 16: return launch<D, 16, T>(p, stream);
    case 32: return launch<D, 32, T>(p, stream);
    default: return launch<D, 64, T>(p, stream);
  }
}

template <typename T>
int launch_dim(const DsaAttnPagedParams* p, cudaStream_t stream) {
  if (p->d == 512) return launch_heads<512, T>(p, stream);
  if (p->d == 256) return launch_heads<256, T>(p, stream);
  if (p->d == 128) return launch_heads<128, T>(p, stream);
  return DSA_ERR_INVALID_ARG;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace attn_paged
}  // namespace dsa

extern "C" int64_t dsa_attn_paged_workspace_size(int64_t batch, int64_t s1, int64_t n1, int64_t d) {
  using namespace dsa::attn_paged;
  if (batch < 0 || s1 < 0 || n1 < 1 || n1 > 128 || d < 1) return -1;
  const int64_t nh = heads_of(n1), grid = sm_count();
  if (grid < 1) return -1;
  return align256(2 * grid * nh * (d * 4 + 16) + (batch * s1 + 1) * 4);
}

extern "C" int dsa_attn_paged(const DsaAttnPagedParams* p, void* stream_) {
  using namespace dsa::attn_paged;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!p || p->batch < 0 || p->s1 < 0) return DSA_ERR_INVALID_ARG;
  if (p->batch == 0 || p->s1 == 0) return DSA_OK;
  if (p->n1 < 1 || p->n1 > 128 || p->page_size < 8 || p->page_size % 8 || p->max_blocks < 1 ||
      p->num_pages < 1 || (p->sparse_mode != 0 && p->sparse_mode != 3) || !p->query ||
      !p->query_rope || !p->key_cache || !p->key_rope_cache || !p->act_k || !p->block_table ||
      !p->out || !p->workspace)
    return DSA_ERR_INVALID_ARG;
  // sizes the kernels index with 32 bits: rows * n1 blocks, tiles, pages
  constexpr int64_t kMax = 0x7fffffff;
  if (p->batch > kMax || p->s1 > kMax || p->batch * p->s1 > kMax / p->n1 || p->num_pages > kMax ||
      p->page_size > (1 << 20) || p->max_blocks > (kMax - kTile) / p->page_size ||
      p->batch * p->s1 > kMax / ((p->max_blocks * p->page_size + kTile - 1) / kTile))
    return DSA_ERR_INVALID_ARG;
  if ((p->softmax_max == nullptr) != (p->softmax_sum == nullptr)) return DSA_ERR_INVALID_ARG;
  const int64_t strides[10] = {p->q_head_stride,  p->q_token_stride,  p->q_batch_stride,
                               p->qr_head_stride, p->qr_token_stride, p->qr_batch_stride,
                               p->k_row_stride,   p->k_page_stride,   p->kr_row_stride,
                               p->kr_page_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return DSA_ERR_INVALID_ARG;
  if (!aligned16(p->query) || !aligned16(p->query_rope) || !aligned16(p->key_cache) ||
      !aligned16(p->key_rope_cache) || !aligned16(p->workspace))
    return DSA_ERR_INVALID_ARG;
  if (p->workspace_bytes < dsa_attn_paged_workspace_size(p->batch, p->s1, p->n1, p->d))
    return DSA_ERR_INVALID_ARG;
  if (p->dtype == DSA_DTYPE_BF16) return launch_dim<__nv_bfloat16>(p, stream);
  if (p->dtype == DSA_DTYPE_FP16) return launch_dim<__half>(p, stream);
  return DSA_ERR_INVALID_ARG;
}
