// pm_rowvec.cuh -- rows of fp32 or bf16 logits read as 16-byte vectors.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "pm_device.cuh"

namespace pm {

constexpr float kNegInf = -__builtin_inff();

template <typename T> struct RowVec;
template <> struct RowVec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void unpack(uint4 r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
};
template <> struct RowVec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void unpack(uint4 r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

// Elements [i, i + n) of a row as fp32, -inf where the row has ended or the
// mask bit is clear.  Vectors without an allowed element are not read.
template <typename T>
__device__ __forceinline__ void load_vec(const T* row, int64_t i, int64_t V, bool aligned, const uint32_t* mask,
                                         float* v) {
  constexpr int n = RowVec<T>::n;
  uint32_t bits = (1u << n) - 1u;
  if (i + n > V) bits = i >= V ? 0u : (1u << (V - i)) - 1u;
  if (mask && bits) bits &= __ldg(mask + (i >> 5)) >> (i & 31);
#pragma unroll
  for (int e = 0; e < n; ++e) v[e] = kNegInf;
  if (!bits) return;
  if (aligned && i + n <= V) {
    float t[n];
    RowVec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(row + i)), t);
#pragma unroll
    for (int e = 0; e < n; ++e) v[e] = (bits >> e) & 1 ? t[e] : kNegInf;
  } else {
#pragma unroll
    for (int e = 0; e < n; ++e)
      if ((bits >> e) & 1) v[e] = RowVec<T>::get(row + i + e);
  }
}

}  // namespace pm
