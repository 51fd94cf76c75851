// The pages of a cache: appending new tokens, and copying, forking, growing, compacting and
// freeing pages.
//
// A pool of num_pages pages is described by int32 state on the device: block_table
// [slots][max_blocks] (page of each block of a sequence, -1 where there is none), seq_lengths
// [slots], ref_counts [num_pages] (sequences that hold a page; 0: free).  One table serves
// every cache of the pool (layers; latent, rotary and index keys).  The bookkeeping calls read
// that state and write a new one, so nothing waits for the host and a call can be captured;
// the page data is moved in place.  Pages are handed out lowest id first.
//
// A call is two launches: page_plan_kernel finds the pages, page_apply_kernel writes the new table
// and moves the data, both over the whole GPU.  What the plan needs in order (which free page is
// the k-th) is one block's work: it makes a bit per page of ref_counts (read once, eight loads a
// thread in flight) and ranks the pages by prefix sums over the bits' counts; the other blocks
// copy the counts meanwhile.
#include <cuda_runtime.h>

#include "dsa_b200.h"
#include "rotary.cuh"
#include "tma_host.h"

namespace dsa {
namespace pages {

// ---------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------
constexpr int kAppendThreads = 128;
constexpr int kInFlight = 4;   // copied pieces of a lane that are loaded before any is stored

struct AppendArgs {
  DsaCacheRows e[DSA_APPEND_MAX_ENTRIES];       // copied rows first, then the rotated ones
  uint32_t first[DSA_APPEND_MAX_ENTRIES + 1];   // first piece of each entry, of its kind
  const int32_t* block_table;
  const int32_t* starts;
  const int32_t* counts;
  const float* table;
  int* error_flag;
  int64_t tokens;
  rotary::FastDiv page;
  uint32_t copied, turned;   // pieces
  int32_t plain, entries, s, max_blocks, num_pages, max_positions, dim;
};

// A piece of a rotated row: an interleaved one, a pair of the half layout, or one that is copied.
template <typename T>
struct Piece {
  static constexpr int kN = rotary::Vec<T>::kN;
  uint4 v, w;
  int entry, at;   // byte offset in the row
  bool pair, turned;
  __device__ __forceinline__ void load(const AppendArgs& a, uint32_t u, int64_t b, int s) {
    int i = a.plain;
    while (i + 1 < a.entries && u >= a.first[i + 1]) ++i;
    const DsaCacheRows& e = a.e[i];
    entry = i;
    const int half = a.dim / 2, piece = (int)(u - a.first[i]) * kN;
    int in = piece;   // value in the row
    pair = e.rotary == DSA_ROTARY_HALF && piece < half;
    if (pair) {
      in = (int)e.offset + piece;
    } else if (e.rotary == DSA_ROTARY_HALF) {   // the copied ones, around the rotated part
      in = piece - half;
      if (in >= e.offset) in += a.dim;
    }
    turned = pair || (e.rotary == DSA_ROTARY_INTERLEAVED && in >= e.offset && in < e.offset + a.dim);
    at = in * (int)sizeof(T);
    const char* src = static_cast<const char*>(e.src) + b * e.src_batch_stride + s * e.src_token_stride + at;
    v = *reinterpret_cast<const uint4*>(src);
    if (pair) w = *reinterpret_cast<const uint4*>(src + half * sizeof(T));
  }
  __device__ __forceinline__ void store(const AppendArgs& a, int64_t pos, int32_t page, uint32_t row) {
    const DsaCacheRows& e = a.e[entry];
    char* dst = static_cast<char*>(e.cache) + page * e.page_stride + row * e.row_stride + at;
    const float* angles = a.table + pos * a.dim;
    const int half = a.dim / 2, in = at / (int)sizeof(T) - (int)e.offset;
    if (pair) {
      float cs[kN], sn[kN];
      rotary::load_angles<kN>(angles, half, in, 1.0f, cs, sn);
      rotary::turn_half<T>(v, w, cs, sn);
      *reinterpret_cast<uint4*>(dst + half * sizeof(T)) = w;
    } else if (turned) {
      float cs[kN / 2], sn[kN / 2];
      rotary::load_angles<kN / 2>(angles, half, in / 2, 1.0f, cs, sn);
      v = rotary::turn_interleaved<T>(v, cs, sn);
    }
    *reinterpret_cast<uint4*>(dst) = v;
  }
};

// A warp per token: its rows are read while its page is looked up.  Rotated rows hold values of T.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  const int64_t b = token / a.s;
  const int s = (int)(token - b * a.s);
  const int32_t start = a.starts[b];
  if (a.counts && s >= a.counts[b]) return;
  const int64_t pos = (int64_t)start + s;
  // (pages and positions are below 2^31, as the host has seen to)
  const uint32_t block = pos >= 0 && pos < (1LL << 31) - 1 ? a.page.div((uint32_t)pos) : (uint32_t)a.max_blocks;
  int32_t page = -1;
  if (block < (uint32_t)a.max_blocks) page = a.block_table[b * a.max_blocks + block];
  Piece<T> piece;
  if ((uint32_t)lane < a.turned) piece.load(a, lane, b, s);
  bool known = false;
  auto look = [&]() {   // first looked at with loads in flight
    known = page >= 0 && page < a.num_pages && !(a.table && pos >= a.max_positions);
    if (!known && lane == 0) report_error(a.error_flag, kErrBadIndex);
  };
  const uint32_t row = (uint32_t)pos - block * a.page.d;
  for (uint32_t u0 = lane; u0 < a.copied; u0 += 32 * kInFlight) {
    uint4 v[kInFlight];
    int at[kInFlight], entry[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const uint32_t u = u0 + 32 * k;
      if (u >= a.copied) break;
      int i = 0;
      while (i + 1 < a.plain && u >= a.first[i + 1]) ++i;
      const DsaCacheRows& e = a.e[i];
      entry[k] = i;
      at[k] = (int)(u - a.first[i]) * 16;
      v[k] = *reinterpret_cast<const uint4*>(static_cast<const char*>(e.src) + b * e.src_batch_stride +
                                             s * e.src_token_stride + at[k]);
    }
    if (u0 == (uint32_t)lane) look();
    if (!known) return;
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (u0 + 32 * k >= a.copied) break;
      const DsaCacheRows& e = a.e[entry[k]];
      *reinterpret_cast<uint4*>(static_cast<char*>(e.cache) + page * e.page_stride + row * e.row_stride + at[k]) = v[k];
    }
  }
  if (a.copied <= (uint32_t)lane) look();
  if (!known) return;
  for (uint32_t u = lane; u < a.turned; u += 32) {
    if (u != (uint32_t)lane) piece.load(a, u, b, s);
    piece.store(a, pos, page, row);
  }
}

// ---------------------------------------------------------------------------------------
// bookkeeping
// ---------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kApplyThreads = 256;
constexpr int kMaxCaches = 32;              // caches of one apply launch
constexpr int kSliceBytes = 16384;          // of a page, per block and turn

struct PoolArgs {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* refs;
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* refs_out;
  const int32_t* first;    // fork: parents, extend: counts, free: rows, copy: source pages
  const int32_t* second;   // fork: children, copy: destination pages
  int* error_flag;
  int32_t* header;         // [0] page copies
  int32_t* mark;           // [slots] fork: the fork that makes the row; free: 1; extend: first page
  int32_t* list_a;         // source pages (compact, fork), free pages (extend)
  int32_t* list_b;         // destination pages (compact, fork)
  int32_t* list_c;         // rows of the page that a fork copies; compact: new id of
                           // each page that moves
  uint32_t* bits;          // a bit per page, where they are too many for shared memory
  int32_t op, n, slots, max_blocks, num_pages, page_size;
};

__device__ __forceinline__ int plan_scan(int v, int* tmp, int* total) {
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
  int t = tmp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t += y;
  }
  *total = __shfl_sync(0xffffffffu, t, 31);
  const int before = __shfl_sync(0xffffffffu, t, warp) - tmp[warp];
  return before + x - v;
}

__device__ __forceinline__ int blocks_of(int64_t tokens, int page_size) {
  return (int)((tokens + page_size - 1) / page_size);
}

constexpr int kBitWords = 4096;   // pages / 32 that are held in shared memory; more in the workspace

// A bit per page: whether it is free.
__device__ __forceinline__ void free_bits(const int32_t* __restrict__ refs, int num_pages, uint32_t* bits) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int p0 = warp * 256; p0 < num_pages; p0 += kPlanWarps * 256) {
    int r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int p = p0 + 32 * k + lane;
      r[k] = p < num_pages ? __ldg(refs + p) : 1;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = __ballot_sync(0xffffffffu, r[k] <= 0);
      if (lane == 0 && p0 + 32 * k < num_pages) bits[p0 / 32 + k] = m;
    }
  }
  __syncthreads();
}

// Calls f(page, rank) for the first `limit` of the pages whose bit of word(i) is set, ranked by
// id; returns how many there are.
template <typename Word, typename F>
__device__ int rank_pages(int num_pages, int limit, int* tmp, Word word, F f) {
  const int words = (num_pages + 31) / 32;
  int before = 0;
  for (int w0 = 0; w0 < words; w0 += kPlanThreads) {
    const int w = w0 + threadIdx.x;
    uint32_t m = w < words ? word(w) : 0u;
    int sum;
    int rank = before + plan_scan(__popc(m), tmp, &sum);
    for (; m && rank < limit; ++rank, m &= m - 1) f(32 * w + __ffs(m) - 1, rank);
    before += sum;
  }
  return before;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PoolArgs a) {
  __shared__ int tmp[kPlanWarps];
  __shared__ int run_total, walk_end;
  __shared__ int walk[kPlanThreads];
  __shared__ uint32_t bit_room[kBitWords];
  const int tid = threadIdx.x;
  griddep_launch_dependents();
  if (blockIdx.x > 0) {
    // the counts go over as they are; what changes is counted in by the apply kernel
    const int stride = (gridDim.x - 1) * kPlanThreads;
    for (int p = (blockIdx.x - 1) * kPlanThreads + tid; p < a.num_pages; p += stride) a.refs_out[p] = a.refs[p];
    return;
  }
  if (tid == 0) a.header[0] = 0;
  bool bad = false, full = false;
  uint32_t* bits = a.num_pages <= 32 * kBitWords ? bit_room : a.bits;
  if (a.op != DSA_PAGES_FREE) free_bits(a.refs, a.num_pages, bits);
  auto free_word = [&](int w) { return bits[w]; };

  if (a.op == DSA_PAGES_COMPACT) {
    // live pages beyond the first n_live ids move, in order, to the free ids among those
    const int n_live = a.num_pages - rank_pages(a.num_pages, 0, tmp, free_word, [](int, int) {});
    auto below = [&](int w) {   // bits of word w whose id is below n_live
      const int n = n_live - 32 * w;
      return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
    };
    auto valid = [&](int w) {
      const int n = a.num_pages - 32 * w;
      return n >= 32 ? 0xffffffffu : (1u << n) - 1u;
    };
    const int moved = rank_pages(a.num_pages, a.num_pages, tmp,
                                 [&](int w) { return ~bits[w] & ~below(w) & valid(w); },
                                 [&](int p, int r) { a.list_a[r] = p; });
    rank_pages(a.num_pages, a.num_pages, tmp, [&](int w) { return bits[w] & below(w); },
               [&](int p, int r) { a.list_b[r] = p; });
    __syncthreads();
    for (int i = tid; i < moved; i += kPlanThreads) a.list_c[a.list_a[i]] = a.list_b[i];
    if (tid == 0) {
      a.header[0] = moved;
      a.header[1] = n_live;
    }
    return;
  }

  if (a.op == DSA_PAGES_FREE) {
    for (int r = tid; r < a.slots; r += kPlanThreads) a.mark[r] = 0;
    __syncthreads();
    for (int i = tid; i < a.n; i += kPlanThreads) {
      const int r = a.first[i];
      if (r >= 0 && r < a.slots) a.mark[r] = 1;
      else bad = true;
    }
  } else if (a.op == DSA_PAGES_EXTEND) {
    // row r grows to lens + counts tokens; the pages it needs are a run of the free ones.  Rows are
    // served in order, and one that what is left cannot serve takes nothing from those after it.
    if (tid == 0) run_total = 0;
    __syncthreads();
    const int free_pages = rank_pages(a.num_pages, a.num_pages, tmp, free_word,
                                      [&](int p, int r) { a.list_a[r] = p; });
    for (int r0 = 0; r0 < a.slots; r0 += kPlanThreads) {
      const int r = r0 + tid;
      const int before = run_total, left = free_pages - before;   // the same for every thread
      int need = 0;
      bool grows = false;
      int64_t len = 0, more = 0;
      if (r < a.slots) {
        len = a.lens[r];
        more = a.first[r];
        grows = more >= 0 && len >= 0 && len + more <= (int64_t)a.max_blocks * a.page_size;
        bad |= !grows;
        if (grows) need = blocks_of(len + more, a.page_size) - blocks_of(len, a.page_size);
      }
      bool fits = need <= left;
      int sum;
      int at = before + plan_scan(fits ? need : 0, tmp, &sum);
      int end = before + sum;
      if (sum > left) {
        // the pool runs out within these rows, so what a row gets depends on which ones before it
        // were served: one thread walks them (a call for 1,024 rows took 20.5 us with the walk; one
        // for 32 rows without it 15.5)
        walk[tid] = need;
        __syncthreads();
        if (tid == 0) {
          int next = before;
          const int rows = min(kPlanThreads, a.slots - r0);
          for (int i = 0; i < rows; ++i) {
            const int n = walk[i];
            const bool served = n <= free_pages - next;
            walk[i] = served ? next : -1;
            next += served ? n : 0;
          }
          walk_end = next;
        }
        __syncthreads();
        at = walk[tid];
        fits = at >= 0;
        end = walk_end;
      }
      if (r < a.slots) {
        full |= !fits;
        grows = grows && fits;
        a.lens_out[r] = (int)(grows ? len + more : len);
        a.mark[r] = at;
      }
      __syncthreads();
      if (tid == 0) run_total = end;
      __syncthreads();
    }
  } else {   // DSA_PAGES_FORK
    for (int r = tid; r < a.slots; r += kPlanThreads) a.mark[r] = 0x7fffffff;
    if (tid == 0) run_total = 0;
    __syncthreads();
    // the child must be an empty row; of forks into the same row the first counts
    auto valid = [&](int i) {
      const int p = a.first[i], c = a.second[i];
      if (p < 0 || p >= a.slots || c < 0 || c >= a.slots) return false;
      const int64_t len = a.lens[p];
      if (a.lens[c] != 0 || len < 0 || len > (int64_t)a.max_blocks * a.page_size) return false;
      if (len % a.page_size == 0) return true;
      const int page = a.table[(int64_t)p * a.max_blocks + len / a.page_size];
      return page >= 0 && page < a.num_pages;
    };
    for (int i = tid; i < a.n; i += kPlanThreads) {
      if (valid(i)) atomicMin(&a.mark[a.second[i]], i);
      else bad = true;
    }
    __syncthreads();
    const int free_pages = rank_pages(a.num_pages, min(a.n, a.num_pages), tmp, free_word,
                                      [&](int p, int r) { a.list_b[r] = p; });
    __syncthreads();
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
      const int i = i0 + tid;
      int rest = 0, child = -1;
      bool mine = false;
      if (i < a.n) {
        child = a.second[i];
        mine = child >= 0 && child < a.slots && a.mark[child] == i;
        bad |= !mine;
        if (mine) rest = a.lens[a.first[i]] % a.page_size;
      }
      int sum;
      const int at = run_total + plan_scan(rest > 0 ? 1 : 0, tmp, &sum);
      if (mine && rest > 0) {
        if (at < free_pages) {
          const int parent = a.first[i];
          a.list_a[at] = a.table[(int64_t)parent * a.max_blocks + a.lens[parent] / a.page_size];
          a.list_c[at] = rest;
        } else {
          full = true;
          a.mark[child] = -1;   // no page left: the child stays empty
        }
      }
      // where the apply kernel finds the child's own page
      if (mine) a.header[8 + i] = at;
      __syncthreads();
      if (tid == 0) {
        run_total += sum;
        a.header[0] = min(run_total, free_pages);
      }
      __syncthreads();
    }
  }
  if (bad) report_error(a.error_flag, kErrBadIndex);
  if (full) report_error(a.error_flag, kErrNoPages);
}

struct Caches {
  DsaPageCache c[kMaxCaches];
  int32_t slices[kMaxCaches];   // of kSliceBytes, rounded up, of a whole page
  int32_t count, total;
};

// Copy the first `rows` rows of page src to page dst: slice `sl` of cache `c`.
__device__ __forceinline__ void copy_slice(const DsaPageCache& c, int sl, int64_t src, int64_t dst, int rows) {
  constexpr int kPieces = kSliceBytes / 16;
  const int row_pieces = (int)(c.row_bytes / 16);
  const int64_t all = (int64_t)rows * row_pieces;
  const char* from = static_cast<const char*>(c.data) + src * c.page_stride;
  char* to = static_cast<char*>(c.data) + dst * c.page_stride;
  const bool dense = c.row_stride == c.row_bytes;
  uint4 v[kPieces / kApplyThreads];
#pragma unroll
  for (int k = 0; k < kPieces / kApplyThreads; ++k) {
    const int64_t i = (int64_t)sl * kPieces + k * kApplyThreads + threadIdx.x;
    if (i < all) {
      const int64_t at = dense ? i * 16 : i / row_pieces * c.row_stride + i % row_pieces * 16;
      v[k] = *reinterpret_cast<const uint4*>(from + at);
    }
  }
#pragma unroll
  for (int k = 0; k < kPieces / kApplyThreads; ++k) {
    const int64_t i = (int64_t)sl * kPieces + k * kApplyThreads + threadIdx.x;
    if (i < all) {
      const int64_t at = dense ? i * 16 : i / row_pieces * c.row_stride + i % row_pieces * 16;
      *reinterpret_cast<uint4*>(to + at) = v[k];
    }
  }
}

__global__ void __launch_bounds__(kApplyThreads)
    page_apply_kernel(const PoolArgs a, const __grid_constant__ Caches caches, int do_table) {
  griddep_wait();
  if (do_table && a.op != DSA_PAGES_COPY) {
    // a warp per row, or per kRowPiece entries of it
    constexpr int kRowPiece = 128;
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (kApplyThreads / 32), me = blockIdx.x * (kApplyThreads / 32) + (threadIdx.x >> 5);
    const int per_row = (a.max_blocks + kRowPiece - 1) / kRowPiece;
    const int moved = a.op == DSA_PAGES_COMPACT ? a.header[0] : 0;
    const int n_live = a.op == DSA_PAGES_COMPACT ? a.header[1] : 0;
    for (int64_t i = me * 32 + lane; i < moved; i += (int64_t)warps * 32) {
      const int from = a.list_a[i];
      a.refs_out[a.list_b[i]] = a.refs[from];
      a.refs_out[from] = 0;
    }
    for (int64_t task = me; task < (int64_t)a.slots * per_row; task += warps) {
      const int row = (int)(task / per_row), j0 = (int)(task - (int64_t)row * per_row) * kRowPiece;
      const int end = min(j0 + kRowPiece, a.max_blocks);
      const int32_t* in = a.table + (int64_t)row * a.max_blocks;
      int32_t* out = a.table_out + (int64_t)row * a.max_blocks;
      if (a.op == DSA_PAGES_COMPACT) {
#pragma unroll 4
        for (int j = j0 + lane; j < end; j += 32) {
          int v = in[j];
          if (v >= n_live && v < a.num_pages && a.refs[v] > 0) v = a.list_c[v];
          out[j] = v;
        }
      } else if (a.op == DSA_PAGES_FREE) {
        const bool gone = a.mark[row] != 0;
        if (j0 == 0 && lane == 0) a.lens_out[row] = gone ? 0 : a.lens[row];
#pragma unroll 4
        for (int j = j0 + lane; j < end; j += 32) {
          const int v = in[j];
          out[j] = gone ? -1 : v;
          if (!gone || v < 0) continue;
          // a page held more often than it is counted was free already: it stays at 0
          bool wrong = v >= a.num_pages;
          if (!wrong && atomicSub(&a.refs_out[v], 1) <= 0) {
            atomicAdd(&a.refs_out[v], 1);
            wrong = true;
          }
          if (wrong) report_error(a.error_flag, kErrBadIndex);
        }
      } else if (a.op == DSA_PAGES_EXTEND) {
        const int had = blocks_of(a.lens[row], a.page_size), has = blocks_of(a.lens_out[row], a.page_size);
        const int32_t* fresh = a.list_a + a.mark[row] - had;
#pragma unroll 4
        for (int j = j0 + lane; j < end; j += 32) {
          int v = in[j];
          if (j >= had && j < has) {
            v = fresh[j];
            a.refs_out[v] = 1;
          }
          out[j] = v;
        }
      } else {   // fork
        const int f = a.mark[row];
        const bool child = f >= 0 && f < a.n;
        const int parent = child ? a.first[f] : row, len = a.lens[parent];
        const int full = len / a.page_size;
        if (j0 == 0 && lane == 0) a.lens_out[row] = len;
        const int32_t* from = a.table + (int64_t)parent * a.max_blocks;
#pragma unroll 4
        for (int j = j0 + lane; j < end; j += 32) {
          int v = from[j];
          if (child && j < full) {
            if (v >= 0 && v < a.num_pages) {
              atomicAdd(&a.refs_out[v], 1);
            } else {   // the parent has no such page: neither has the child
              report_error(a.error_flag, kErrBadIndex);
              v = -1;
            }
          } else if (child) {
            v = -1;
            if (j == full && len % a.page_size) {
              v = a.list_b[a.header[8 + f]];
              a.refs_out[v] = 1;
            }
          }
          out[j] = v;
        }
      }
    }
  }
  if (caches.count == 0) return;
  const int copies = a.op == DSA_PAGES_COPY ? a.n
                     : a.op == DSA_PAGES_COMPACT || a.op == DSA_PAGES_FORK ? a.header[0] : 0;
  const int64_t jobs = (int64_t)copies * caches.total;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int item = (int)(job / caches.total);
    int sl = (int)(job - (int64_t)item * caches.total), c = 0;
    while (sl >= caches.slices[c]) sl -= caches.slices[c++];
    int src, dst, rows = a.page_size;
    if (a.op == DSA_PAGES_COPY) {
      src = a.first[item];
      dst = a.second[item];
      if (src < 0 || dst < 0 || src >= a.num_pages || dst >= a.num_pages) {
        // -1 skips an entry; an id past the pool is an error
        if (threadIdx.x == 0 && (src >= a.num_pages || dst >= a.num_pages))
          report_error(a.error_flag, kErrBadIndex);
        continue;
      }
    } else {
      src = a.list_a[item];
      dst = a.list_b[item];
      if (a.op == DSA_PAGES_FORK) rows = a.list_c[item];
    }
    if (src != dst) copy_slice(caches.c[c], sl, src, dst, rows);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int64_t align64(int64_t n) { return (n + 63) & ~(int64_t)63; }

}  // namespace pages
}  // namespace dsa

extern "C" int dsa_cache_append(const DsaCacheAppendParams* p, void* stream_) {
  using namespace dsa::pages;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  constexpr int64_t kMax = 0x7fffffff;
  if (!p || p->batch < 0 || p->s < 0) return DSA_ERR_INVALID_ARG;
  if (p->batch == 0 || p->s == 0) return DSA_OK;   // (empty tensors have no address)
  if (p->entries < 1 || p->entries > DSA_APPEND_MAX_ENTRIES || !p->block_table || !p->starts ||
      p->page_size < 1 || p->page_size > kMax || p->max_blocks < 1 || p->max_blocks > kMax / p->page_size ||
      p->num_pages < 1 || p->num_pages > kMax || p->batch > kMax || p->s > kMax)
    return DSA_ERR_INVALID_ARG;
  // copied rows and the rotated rows of each type, one launch for each type there is (one, as a rule)
  for (int i = 0; i < p->entries; ++i) {
    const DsaCacheRows& e = p->rows[i];
    if (!e.src || !e.cache || e.width_bytes < 16 || e.width_bytes > (1 << 24) || e.width_bytes % 16 ||
        !aligned16(e.src) || !aligned16(e.cache) || e.src_batch_stride % 16 || e.src_token_stride % 16 ||
        e.page_stride % 16 || e.row_stride % 16)
      return DSA_ERR_INVALID_ARG;
    if (e.rotary == DSA_ROTARY_NONE) continue;
    const int64_t size = e.dtype == DSA_DTYPE_FP32 ? 4 : 2, n = 16 / size;
    if ((e.dtype != DSA_DTYPE_BF16 && e.dtype != DSA_DTYPE_FP16 && e.dtype != DSA_DTYPE_FP32) ||
        (e.rotary != DSA_ROTARY_INTERLEAVED && e.rotary != DSA_ROTARY_HALF) || !p->table ||
        !aligned16(p->table) || p->dim < 8 || p->dim > 256 || p->dim % 8 || e.offset < 0 ||
        e.offset > e.width_bytes || e.offset % n || p->dim % (e.rotary == DSA_ROTARY_HALF ? 2 * n : n) ||
        (e.offset + p->dim) * size > e.width_bytes || p->max_positions < 1 || p->max_positions > kMax)
      return DSA_ERR_INVALID_ARG;
  }
  AppendArgs a = {};
  a.block_table = p->block_table;
  a.starts = p->starts;
  a.counts = p->counts;
  a.table = p->table;
  a.error_flag = p->error_flag;
  a.tokens = p->batch * p->s;
  a.page = dsa::rotary::FastDiv((uint32_t)p->page_size);
  a.s = (int)p->s;
  a.max_blocks = (int)p->max_blocks;
  a.num_pages = (int)p->num_pages;
  a.max_positions = (int)p->max_positions;
  a.dim = (int)p->dim;
  const int64_t blocks = (a.tokens + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (blocks > kMax) return DSA_ERR_INVALID_ARG;
  bool copies = true;   // not launched yet
  for (int32_t type : {DSA_DTYPE_BF16, DSA_DTYPE_FP16, DSA_DTYPE_FP32}) {
    a.entries = 0;
    a.copied = a.turned = 0;
    for (int i = 0; i < p->entries && copies; ++i)
      if (p->rows[i].rotary == DSA_ROTARY_NONE) {
        a.first[a.entries] = a.copied;
        a.e[a.entries++] = p->rows[i];
        a.copied += (uint32_t)(p->rows[i].width_bytes / 16);
      }
    a.plain = a.entries;
    for (int i = 0; i < p->entries; ++i) {
      const DsaCacheRows& e = p->rows[i];
      if (e.rotary == DSA_ROTARY_NONE || e.dtype != type) continue;
      a.first[a.entries] = a.turned;
      a.e[a.entries++] = e;
      const int64_t pairs = e.rotary == DSA_ROTARY_HALF ? p->dim / 2 * (type == DSA_DTYPE_FP32 ? 4 : 2) / 16 : 0;
      a.turned += (uint32_t)(e.width_bytes / 16 - pairs);
    }
    // (copied rows go with the first rotated type; alone if there is none)
    if (a.turned == 0 && (type != DSA_DTYPE_FP32 || a.copied == 0)) continue;
    copies = false;
    if (type == DSA_DTYPE_BF16) append_kernel<__nv_bfloat16><<<(unsigned)blocks, kAppendThreads, 0, stream>>>(a);
    else if (type == DSA_DTYPE_FP16) append_kernel<__half><<<(unsigned)blocks, kAppendThreads, 0, stream>>>(a);
    else append_kernel<float><<<(unsigned)blocks, kAppendThreads, 0, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  }
  return DSA_OK;
}

extern "C" int64_t dsa_pages_workspace_size(int32_t op, int64_t n, int64_t slots, int64_t num_pages) {
  using namespace dsa::pages;
  constexpr int64_t kMax = 0x7fffffff;
  if (n < 0 || slots < 0 || num_pages < 0 || n > kMax || slots > kMax || num_pages > kMax) return -1;
  if (op == DSA_PAGES_COPY) return 0;
  return 4 * (align64(8 + (op == DSA_PAGES_FORK ? n : 0)) + align64(slots) + 3 * align64(num_pages) +
              align64(num_pages / 32 + 1));
}

extern "C" int dsa_pages(const DsaPagesParams* p, void* stream_) {
  using namespace dsa::pages;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  constexpr int64_t kMax = 0x7fffffff;
  if (!p || p->op < DSA_PAGES_COPY || p->op > DSA_PAGES_COMPACT) return DSA_ERR_INVALID_ARG;
  const bool copy = p->op == DSA_PAGES_COPY;
  if (p->n < 0 || p->n > kMax || p->num_pages < 1 || p->num_pages > kMax || p->page_size < 1 ||
      p->page_size > kMax || p->num_caches < 0 || (p->num_caches > 0 && !p->caches))
    return DSA_ERR_INVALID_ARG;
  if (!copy && (p->slots < 1 || p->slots > kMax || p->max_blocks < 1 ||
                p->max_blocks > kMax / p->page_size || p->slots > kMax / p->max_blocks || !p->block_table || !p->block_table_out ||
                !p->ref_counts || !p->ref_counts_out || !p->workspace ||
                p->workspace_bytes < dsa_pages_workspace_size(p->op, p->n, p->slots, p->num_pages)))
    return DSA_ERR_INVALID_ARG;
  if (!copy && p->op != DSA_PAGES_COMPACT && (!p->seq_lengths || !p->seq_lengths_out)) return DSA_ERR_INVALID_ARG;
  const bool two = copy || p->op == DSA_PAGES_FORK;
  if (p->op != DSA_PAGES_COMPACT && ((p->n > 0 && !p->first) || (two && p->n > 0 && !p->second)))
    return DSA_ERR_INVALID_ARG;
  if (p->op == DSA_PAGES_EXTEND && p->n != p->slots) return DSA_ERR_INVALID_ARG;
  for (int i = 0; i < p->num_caches; ++i) {
    const DsaPageCache& c = p->caches[i];
    if (!c.data || !aligned16(c.data) || c.row_bytes < 16 || c.row_bytes % 16 || c.row_stride % 16 ||
        c.page_stride % 16 || c.row_bytes > kMax / p->page_size)
      return DSA_ERR_INVALID_ARG;
  }
  if (copy && (p->n == 0 || p->num_caches == 0)) return DSA_OK;
  PoolArgs a = {};
  a.table = p->block_table, a.lens = p->seq_lengths, a.refs = p->ref_counts;
  a.table_out = p->block_table_out, a.lens_out = p->seq_lengths_out, a.refs_out = p->ref_counts_out;
  a.first = p->first, a.second = p->second;
  a.error_flag = p->error_flag;
  if (!copy) {
    int32_t* ws = static_cast<int32_t*>(p->workspace);
    a.header = ws;
    ws += align64(8 + (p->op == DSA_PAGES_FORK ? p->n : 0));
    a.mark = ws;
    ws += align64(p->slots);
    a.list_a = ws;
    a.list_b = ws + align64(p->num_pages);
    a.list_c = ws + 2 * align64(p->num_pages);
    a.bits = reinterpret_cast<uint32_t*>(ws + 3 * align64(p->num_pages));
  }
  a.op = p->op;
  a.n = (int)p->n;
  a.slots = (int)p->slots;
  a.max_blocks = (int)p->max_blocks;
  a.num_pages = (int)p->num_pages;
  a.page_size = (int)p->page_size;
  const int sms = dsa::sm_count();
  if (sms < 1) return DSA_ERR_CUDA;
  if (!copy) {
    const int64_t copy_blocks = (p->num_pages + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
    page_plan_kernel<<<1 + (unsigned)(copy_blocks < 64 ? copy_blocks : 64), kPlanThreads, 0, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  }
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  for (int i0 = 0; i0 == 0 || i0 < p->num_caches; i0 += kMaxCaches) {
    Caches c = {};
    for (int i = i0; i < p->num_caches && c.count < kMaxCaches; ++i) {
      c.c[c.count] = p->caches[i];
      c.slices[c.count] = (int)((p->caches[i].row_bytes * p->page_size + kSliceBytes - 1) / kSliceBytes);
      c.total += c.slices[c.count++];
    }
    int64_t blocks = (int64_t)sms * 8;
    if (c.count == 0) {
      const int64_t need = p->slots * ((p->max_blocks + 127) / 128) / (kApplyThreads / 32) + 1;
      if (need < blocks) blocks = need;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kApplyThreads);
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = copy || i0 > 0 ? 0 : 1;
    if (cudaLaunchKernelEx(&cfg, page_apply_kernel, a, c, i0 == 0 ? 1 : 0) != cudaSuccess) return DSA_ERR_CUDA;
  }
  return DSA_OK;
}
