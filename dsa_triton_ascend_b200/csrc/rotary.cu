// Rotary positions of queries and keys, their gradient, and the table of cosines and sines.
//
// rotary_kernel is bound by memory: it reads and writes each value once.  A thread takes one
// 16-byte piece of up to kHeads heads of one token, so that the cosines and sines are fetched
// once for those heads and several loads are in flight; neighbouring lanes take neighbouring
// pieces.  In the half layout a piece needs its partner from the other half, which a lane of the
// same warp holds where a head's pieces divide a warp; else one thread takes both pieces.
// Measured: 8192 tokens x 128 heads x 64 (bf16, interleaved) in 43.5 us, 6.2 TB/s, where a copy of
// the same tensor takes 44.6; the gradient of 2 x 4093 tokens x 64 heads x 128, half of each head
// rotated, in 45.6 us, 5.9 TB/s (49.5 with blocks of 256 threads, 51.5 with both pieces in a
// thread, 62 with two heads a thread).
#include <cuda_runtime.h>

#include "dsa_b200.h"
#include "rotary.cuh"

namespace dsa {
namespace rotary {

constexpr int kThreads = 128;
constexpr int kHeads = 4;
constexpr int kMaxPairs = 128;

struct Args {
  const void* x;
  void* out;
  const int32_t* positions;
  const float* table;
  int* error_flag;
  int64_t token0;                       // first token of this launch
  int64_t x_batch, x_token, x_head;     // strides in elements
  int64_t o_batch, o_token, o_head;
  uint32_t items;                       // threads with work
  FastDiv units, head_steps, s;         // pieces of a head; heads / kHeads, rounded up; tokens of a batch
  int32_t heads, head_dim, offset, dim, half_layout, max_positions;
  float sign;
};

enum { kInterleaved, kHalfShuffle, kHalfBoth };

template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Args a) {
  constexpr int kN = Vec<T>::kN;
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  // (the shuffle needs whole warps: lanes past the end repeat the last item and store nothing)
  const bool live = item < a.items;
  if (kMode != kHalfShuffle && !live) return;
  const uint32_t it = live ? item : a.items - 1;
  const uint32_t rest = a.units.div(it), u = it - rest * a.units.d;
  const uint32_t tok = a.head_steps.div(rest), h0 = rest - tok * a.head_steps.d;
  const int64_t token = a.token0 + tok;
  int64_t b, s;
  if (token < (1LL << 31)) {
    b = a.s.div((uint32_t)token);
    s = token - b * a.s.d;
  } else {
    b = token / a.s.d;
    s = token - b * a.s.d;
  }
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch + s * a.x_token;
  T* out = static_cast<T*>(a.out) + b * a.o_batch + s * a.o_token;
  const int32_t pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.max_positions;
  if (!known && u == 0 && h0 == 0) report_error(a.error_flag, kErrBadIndex);
  const int half = a.dim / 2;
  const float* row = a.table + (int64_t)(known ? pos : 0) * a.dim;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  auto head = [&](int j) { return (int)(h0 + j * a.head_steps.d); };

  if constexpr (kMode == kHalfBoth) {
    // the first dim / (2 kN) pieces are pairs, the others are copied
    const int pairs = half / kN;
    const bool pair = (int)u < pairs;
    int at = pair ? a.offset + (int)u * kN : ((int)u - pairs) * kN;
    if (!pair && at >= a.offset) at += a.dim;
    uint4 lo[kHeads], hi[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (head(j) >= a.heads) continue;
      lo[j] = __ldcs(reinterpret_cast<const uint4*>(x + head(j) * a.x_head + at));
      if (pair) hi[j] = __ldcs(reinterpret_cast<const uint4*>(x + head(j) * a.x_head + at + half));
    }
    float cs[kN], sn[kN];
    if (pair) load_angles<kN>(row, half, (int)u * kN, a.sign, cs, sn);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (head(j) >= a.heads) continue;
      if (pair) {
        turn_half<T>(lo[j], hi[j], cs, sn);
        __stcs(reinterpret_cast<uint4*>(out + head(j) * a.o_head + at + half), known ? hi[j] : zero);
      }
      __stcs(reinterpret_cast<uint4*>(out + head(j) * a.o_head + at), known ? lo[j] : zero);
    }
    return;
  }

  const int at = (int)u * kN, in = at - a.offset;
  const bool turned = in >= 0 && in < a.dim;
  uint4 v[kHeads];
#pragma unroll
  for (int j = 0; j < kHeads; ++j)
    if (head(j) < a.heads) v[j] = __ldcs(reinterpret_cast<const uint4*>(x + head(j) * a.x_head + at));
  if constexpr (kMode == kInterleaved) {
    float cs[kN / 2], sn[kN / 2];
    if (turned) load_angles<kN / 2>(row, half, in / 2, a.sign, cs, sn);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (head(j) >= a.heads) continue;
      if (turned) v[j] = turn_interleaved<T>(v[j], cs, sn);
      __stcs(reinterpret_cast<uint4*>(out + head(j) * a.o_head + at), known ? v[j] : zero);
    }
  } else {
    const bool second = in >= half;
    const int lane = threadIdx.x & 31, partner = turned ? (second ? lane - half / kN : lane + half / kN) : lane;
    float cs[kN], sn[kN];
    if (turned) load_angles<kN>(row, half, second ? in - half : in, second ? a.sign : -a.sign, cs, sn);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      // a warp's lanes are whole heads of up to 32 head steps, so all of a head's lanes have it
      uint4 w;
      w.x = __shfl_sync(0xffffffffu, v[j].x, partner);
      w.y = __shfl_sync(0xffffffffu, v[j].y, partner);
      w.z = __shfl_sync(0xffffffffu, v[j].z, partner);
      w.w = __shfl_sync(0xffffffffu, v[j].w, partner);
      if (!live || head(j) >= a.heads) continue;
      if (turned) v[j] = turn_half_one<T>(v[j], w, cs, sn);
      __stcs(reinterpret_cast<uint4*>(out + head(j) * a.o_head + at), known ? v[j] : zero);
    }
  }
}

// Any strides, offsets and even widths: one pair or one copied value per thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_any_kernel(const Args a) {
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  if (item >= a.items) return;
  const uint32_t rest = a.units.div(item), u = item - rest * a.units.d;
  const uint32_t tok = a.head_steps.div(rest), h = rest - tok * a.head_steps.d;
  const int64_t token = a.token0 + tok, b = token / a.s.d, s = token - b * a.s.d;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch + s * a.x_token + h * a.x_head;
  T* out = static_cast<T*>(a.out) + b * a.o_batch + s * a.o_token + h * a.o_head;
  const int32_t pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.max_positions;
  if (!known && u == 0 && h == 0) report_error(a.error_flag, kErrBadIndex);
  const int half = a.dim / 2;
  auto get = [](const T& v) {
    if constexpr (sizeof(T) == 4) return v;
    else return ElemTraits<T>::to_f(v);
  };
  auto put = [](float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return ElemTraits<T>::from_f(v);
  };
  if ((int)u < half) {
    const float* row = a.table + (int64_t)(known ? pos : 0) * a.dim;
    const int ia = a.offset + (a.half_layout ? (int)u : 2 * (int)u);
    const int ib = ia + (a.half_layout ? half : 1);
    float va = get(x[ia]), vb = get(x[ib]);
    turn(va, vb, row[u], a.sign * row[half + u]);
    out[ia] = put(known ? va : 0.0f);
    out[ib] = put(known ? vb : 0.0f);
  } else {
    int at = (int)u - half;
    if (at >= a.offset) at += a.dim;
    out[at] = known ? x[at] : put(0.0f);
  }
}

struct Frequencies {
  double f[kMaxPairs];
};

// table[p][i] = amplitude cos(p f[i]), table[p][half + i] = amplitude sin(p f[i]): the angle in
// 64 bits, since p f in 32 would be off by 2^-24 p radians (0.008 at p = 131072).
__global__ void __launch_bounds__(kThreads) rotary_table_kernel(const __grid_constant__ Frequencies fr,
                                                                float* table, int64_t n, int half,
                                                                double amplitude) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t p = i / half;
    const int j = (int)(i - p * half);
    double s, c;
    sincos((double)p * fr.f[j], &s, &c);
    table[p * 2 * half + j] = (float)(amplitude * c);
    table[p * 2 * half + half + j] = (float)(amplitude * s);
  }
}

template <typename T>
int launch(const DsaRotaryParams* p, cudaStream_t stream) {
  constexpr int kN = Vec<T>::kN;
  Args a;
  a.x = p->x;
  a.out = p->out;
  a.positions = p->positions;
  a.table = p->table;
  a.error_flag = p->error_flag;
  a.x_batch = p->x_batch_stride, a.x_token = p->x_token_stride, a.x_head = p->x_head_stride;
  a.o_batch = p->out_batch_stride, a.o_token = p->out_token_stride, a.o_head = p->out_head_stride;
  a.s = FastDiv((uint32_t)p->s);
  a.heads = (int)p->heads;
  a.head_dim = (int)p->head_dim;
  a.offset = (int)p->offset;
  a.dim = (int)p->dim;
  a.half_layout = p->half_layout;
  a.max_positions = (int)p->max_positions;
  a.sign = p->inverse ? -1.0f : 1.0f;
  bool vec = p->head_dim % kN == 0 && p->offset % kN == 0 &&
             p->dim % (p->half_layout ? 2 * kN : kN) == 0 &&
             reinterpret_cast<uintptr_t>(p->x) % 16 == 0 &&
             reinterpret_cast<uintptr_t>(p->out) % 16 == 0 &&
             reinterpret_cast<uintptr_t>(p->table) % 16 == 0 && p->dim % 8 == 0;
  for (int64_t st : {a.x_batch, a.x_token, a.x_head, a.o_batch, a.o_token, a.o_head})
    vec = vec && st % kN == 0;
  uint32_t units, steps;
  // a warp holds whole heads where a head's pieces divide it
  const bool shuffle = vec && p->half_layout && 32 % (p->head_dim / kN) == 0;
  if (vec) {
    units = (uint32_t)((p->head_dim - (p->half_layout && !shuffle ? p->dim / 2 : 0)) / kN);
    steps = (uint32_t)((p->heads + kHeads - 1) / kHeads);
  } else {
    units = (uint32_t)(p->head_dim - p->dim / 2);
    steps = (uint32_t)p->heads;
  }
  a.units = FastDiv(units);
  a.head_steps = FastDiv(steps);
  const int64_t per_token = (int64_t)units * steps, tokens = p->batch * p->s;
  if (per_token > (1LL << 30)) return DSA_ERR_INVALID_ARG;
  const int64_t chunk = (1LL << 30) / per_token;
  for (int64_t t0 = 0; t0 < tokens; t0 += chunk) {
    const int64_t n = tokens - t0 < chunk ? tokens - t0 : chunk;
    a.token0 = t0;
    a.items = (uint32_t)(n * per_token);
    const unsigned grid = (unsigned)((a.items + kThreads - 1) / kThreads);
    if (!vec) rotary_any_kernel<T><<<grid, kThreads, 0, stream>>>(a);
    else if (!p->half_layout) rotary_kernel<T, kInterleaved><<<grid, kThreads, 0, stream>>>(a);
    else if (shuffle) rotary_kernel<T, kHalfShuffle><<<grid, kThreads, 0, stream>>>(a);
    else rotary_kernel<T, kHalfBoth><<<grid, kThreads, 0, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return DSA_ERR_CUDA;
  }
  return DSA_OK;
}

}  // namespace rotary
}  // namespace dsa

extern "C" int dsa_rotary(const DsaRotaryParams* p, void* stream_) {
  using namespace dsa::rotary;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!p || p->batch < 0 || p->s < 0 || p->heads < 0) return DSA_ERR_INVALID_ARG;
  if (p->batch == 0 || p->s == 0 || p->heads == 0) return DSA_OK;
  constexpr int64_t kMax = 0x7fffffff;
  if (!p->x || !p->out || !p->positions || !p->table || p->dim < 2 || p->dim % 2 ||
      p->dim > 2 * kMaxPairs || p->offset < 0 || p->head_dim > (1 << 20) ||
      p->head_dim < p->dim || p->offset > p->head_dim - p->dim || p->max_positions < 1 || p->max_positions > kMax ||
      p->heads > (1 << 20) || p->s > kMax || p->batch > kMax)
    return DSA_ERR_INVALID_ARG;
  if (p->dtype == DSA_DTYPE_BF16) return launch<__nv_bfloat16>(p, stream);
  if (p->dtype == DSA_DTYPE_FP16) return launch<__half>(p, stream);
  if (p->dtype == DSA_DTYPE_FP32) return launch<float>(p, stream);
  return DSA_ERR_INVALID_ARG;
}

extern "C" int dsa_rotary_table(float* table, int64_t max_positions, int64_t dim,
                                const double* frequencies, double amplitude, void* stream_) {
  using namespace dsa::rotary;
  if (!table || !frequencies || max_positions < 1 || max_positions > 0x7fffffff || dim < 2 ||
      dim % 2 || dim > 2 * kMaxPairs)
    return DSA_ERR_INVALID_ARG;
  Frequencies fr = {};
  const int half = (int)dim / 2;
  for (int i = 0; i < half; ++i) fr.f[i] = frequencies[i];
  const int64_t n = max_positions * half, blocks = (n + kThreads - 1) / kThreads;
  rotary_table_kernel<<<(unsigned)(blocks < 65536 ? blocks : 65536), kThreads, 0,
                        static_cast<cudaStream_t>(stream_)>>>(fr, table, n, half, amplitude);
  return cudaGetLastError() == cudaSuccess ? DSA_OK : DSA_ERR_CUDA;
}
