// Rotary positions: the rotation shared by the stand-alone kernel and the cache append.
//
// A rotated pair (a, b) at angle t becomes (a cos t - b sin t, a sin t + b cos t); the inverse
// (the transpose, which is also the gradient) takes -sin t.  Pairs are neighbours (2 i, 2 i + 1)
// in the interleaved layout and (i, i + dim / 2) in the half layout.  The products are formed in
// fp32 and rounded once to the element type.
#pragma once

#include <stdint.h>

#include "sm100.cuh"

namespace dsa {
namespace rotary {

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994): with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (hi(m n) + n) >> l.
struct FastDiv {
  uint32_t d, m, l;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), m(0), l(0) {
    while ((1ull << l) < d) ++l;
    m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> l; }
#endif
};

template <typename T>
struct Vec {   // 16 bytes of T as fp32 values
  static constexpr int kN = 16 / sizeof(T);
  __device__ static __forceinline__ void unpack(const uint4& v, float (&f)[kN]) {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (sizeof(T) == 4) f[i] = e[i];
      else f[i] = ElemTraits<T>::to_f(e[i]);
    }
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[kN]) {
    uint4 v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (sizeof(T) == 4) e[i] = f[i];
      else e[i] = ElemTraits<T>::from_f(f[i]);
    }
    return v;
  }
};

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = fmaf(a, c, -(b * s)), y = fmaf(b, c, a * s);
  a = x;
  b = y;
}

// kN neighbouring values = kN / 2 pairs, interleaved.
template <typename T>
__device__ __forceinline__ uint4 turn_interleaved(const uint4& v, const float* cs, const float* sn) {
  float f[Vec<T>::kN];
  Vec<T>::unpack(v, f);
#pragma unroll
  for (int i = 0; i < Vec<T>::kN / 2; ++i) turn(f[2 * i], f[2 * i + 1], cs[i], sn[i]);
  return Vec<T>::pack(f);
}
// kN values of the first half and their partners of the second.
template <typename T>
__device__ __forceinline__ void turn_half(uint4& lo, uint4& hi, const float* cs, const float* sn) {
  float a[Vec<T>::kN], b[Vec<T>::kN];
  Vec<T>::unpack(lo, a);
  Vec<T>::unpack(hi, b);
#pragma unroll
  for (int i = 0; i < Vec<T>::kN; ++i) turn(a[i], b[i], cs[i], sn[i]);
  lo = Vec<T>::pack(a);
  hi = Vec<T>::pack(b);
}

// kN values of one half given their partners of the other; `sn` comes negated for the first.
template <typename T>
__device__ __forceinline__ uint4 turn_half_one(const uint4& own, const uint4& other, const float* cs,
                                               const float* sn) {
  float a[Vec<T>::kN], b[Vec<T>::kN];
  Vec<T>::unpack(own, a);
  Vec<T>::unpack(other, b);
#pragma unroll
  for (int i = 0; i < Vec<T>::kN; ++i) a[i] = fmaf(a[i], cs[i], b[i] * sn[i]);
  return Vec<T>::pack(a);
}

// `n` (2, 4 or 8) cosines and sines of a table row from pair `i` on, 4-float aligned when n >= 4.
template <int N>
__device__ __forceinline__ void load_angles(const float* row, int half, int i, float sign,
                                            float (&cs)[N], float (&sn)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 c = *reinterpret_cast<const float4*>(row + i + j);
      const float4 s = *reinterpret_cast<const float4*>(row + half + i + j);
      cs[j] = c.x, cs[j + 1] = c.y, cs[j + 2] = c.z, cs[j + 3] = c.w;
      sn[j] = sign * s.x, sn[j + 1] = sign * s.y, sn[j + 2] = sign * s.z, sn[j + 3] = sign * s.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      cs[j] = row[i + j];
      sn[j] = sign * row[half + i + j];
    }
  }
}

}  // namespace rotary
}  // namespace dsa
