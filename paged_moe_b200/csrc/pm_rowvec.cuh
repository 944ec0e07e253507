// pm_rowvec.cuh -- rows of fp32 or bf16 logits read as 16-byte vectors, and
// sums of their exponentials.
//
// Sums of e^(x / T) are kept as s 2^rho with s in 64 bits.  A thread sums a
// step's vectors in fp32 as 2^(x c - R), c = fl32(log2(e) / T) and R the
// integer nearest to the step's largest x c: x c - R is one fused
// multiply-add, R is exact, and steps of different R are added with exact
// powers of two.  So neither the order of the steps nor how a row is split
// over CTAs changes more than the last bits of a 64-bit sum: a row's
// log-sum-exp does not depend on the batch around it.  What c lacks of
// log2(e) / T is put back once per row, for the row's maximum.
//
// Where |x c| passes 2^20 it no longer has the bits for this.  Steps far below
// (masks of the type's lowest value) are left out: they add nothing to a row
// that holds anything else.  A row, or part of one, that reaches far above,
// or holds nothing but such values, is wild: it is summed once more, as
// 2^((x - m) c) with rho = m c, which 64 bits hold exactly.  Every exponent has
// the same c, so that parts of either kind join and any maximum may be taken
// off their sum: log2(e) / T here and c there would differ by m 2^-25, 0.02
// where |m c| is 2^20.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "pm_device.cuh"

namespace pm {

constexpr float kNegInf = -__builtin_inff();
constexpr double kNegInf64 = -__builtin_inf();
constexpr double kLog2e64 = 1.4426950408889634;
constexpr double kLn264 = 0.6931471805599453;
// Beyond this |x c| an integer R no longer lies within half a unit of x c.
constexpr float kWildExponent = 1048576.0f;

__device__ __forceinline__ double nan64() { return __longlong_as_double(0x7ff8000000000000ll); }

// Maxima that are NaN where an operand is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T> struct RowVec;
template <> struct RowVec<float> {
  static constexpr int n = 4;
  static constexpr uint32_t kFill = 0xff800000u;  // -inf
  static __device__ __forceinline__ void unpack(uint4 r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  // NaN if the vector holds one
  static __device__ __forceinline__ float largest(uint4 r) {
    return max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y)), __uint_as_float(r.z), __uint_as_float(r.w));
  }
  // the vector with -inf where bit e of `bits` is clear
  static __device__ __forceinline__ uint4 select(uint4 r, uint32_t bits) {
    r.x = bits & 1 ? r.x : kFill; r.y = bits & 2 ? r.y : kFill;
    r.z = bits & 4 ? r.z : kFill; r.w = bits & 8 ? r.w : kFill;
    return r;
  }
};
template <> struct RowVec<__nv_bfloat16> {
  static constexpr int n = 8;
  static constexpr uint32_t kFill = 0xff80ff80u;  // -inf twice
  static __device__ __forceinline__ void unpack(uint4 r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ float largest(uint4 r) {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(pair(r.x), pair(r.y)), __hmax2_nan(pair(r.z), pair(r.w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint32_t keep(uint32_t w, uint32_t bits) {
    // one byte per half word: 0xff where the bit is set
    const uint32_t m = ((bits & 1) ? 0xffffu : 0u) | ((bits & 2) ? 0xffff0000u : 0u);
    return (w & m) | (kFill & ~m);
  }
  static __device__ __forceinline__ uint4 select(uint4 r, uint32_t bits) {
    return make_uint4(keep(r.x, bits), keep(r.y, bits >> 2), keep(r.z, bits >> 4), keep(r.w, bits >> 6));
  }
};

// The 16 bytes that start `off` bytes (a multiple of the element size) into
// the aligned vector a, b being the one behind it.
template <typename T>
__device__ __forceinline__ uint4 shift_raw(uint4 a, uint4 b, int off) {
  uint32_t w0 = a.x, w1 = a.y, w2 = a.z, w3 = a.w, w4 = b.x, w5 = b.y, w6 = b.z, w7 = b.w;
  if (off & 8) { w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = w7; }
  if (off & 4) { w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5; }
  if (sizeof(T) == 2) {
    const int s = (off & 2) * 8;
    w0 = __funnelshift_r(w0, w1, s); w1 = __funnelshift_r(w1, w2, s);
    w2 = __funnelshift_r(w2, w3, s); w3 = __funnelshift_r(w3, w4, s);
  }
  return make_uint4(w0, w1, w2, w3);
}

// Elements [i, i + n) of a row, -inf behind its end.  A vector that lies
// across the end is read element by element.  Rows that do not start on a
// 16-byte boundary (off: bytes past one) are read as the two aligned vectors
// that hold the wanted one, each of which holds at least one of its elements.
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 load_raw(const T* row, int off, int i, int V) {
  constexpr int n = RowVec<T>::n;
  if (i + n <= V) {
    if (ALIGNED) return __ldg(reinterpret_cast<const uint4*>(row + i));
    const char* at = reinterpret_cast<const char*>(row + i) - off;
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(at));
    if (off == 0) return a;
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(at + 16));
    return shift_raw<T>(a, b, off);
  }
  constexpr uint32_t fill = RowVec<T>::kFill;
  uint4 r = make_uint4(fill, fill, fill, fill);
  if (i < V) {
    uint32_t w[4] = {fill, fill, fill, fill};
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (i + e < V) {
        if (sizeof(T) == 4) {
          w[e & 3] = __ldg(reinterpret_cast<const uint32_t*>(row) + i + e);
        } else {
          const uint32_t h = __ldg(reinterpret_cast<const uint16_t*>(row) + i + e);
          w[(e >> 1) & 3] = e & 1 ? (w[(e >> 1) & 3] & 0xffffu) | h << 16 : (w[(e >> 1) & 3] & 0xffff0000u) | h;
        }
      }
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

static __device__ __noinline__ double exp2_apart(double d) { return exp2(d); }

// 2^d for d <= 0: exact for whole numbers, which all but wild rows have.
__device__ __forceinline__ double pow2_down(double d) {
  if (d < -1000.0) return 0.0;
  const int w = (int)d;
  if ((double)w == d) return __hiloint2double((1023 + w) << 20, 0);
  return exp2_apart(d);
}

// A sum s 2^rho; rho = -inf: nothing, but s may be a NaN.
struct ExpSum {
  double s, rho;
  __device__ __forceinline__ void clear() { s = 0.0; rho = kNegInf64; }
  __device__ __forceinline__ void add(double t, double r) {
    if (r > rho) {
      s = s * pow2_down(rho - r) + t;
      rho = r;
    } else if (r == rho) {
      s += t;
    } else {
      s += r > kNegInf64 ? t * pow2_down(r - rho) : t;
    }
  }
};

// A thread's running sum, of steps with whole exponents.
struct StepSum {
  static constexpr int kNothing = -(1 << 28);
  double s;
  int rho;
  bool high, low;  // a step far above, or far below, was left out
  __device__ __forceinline__ void clear() { s = 0.0; rho = kNothing; high = low = false; }
  // whether what was left out may count in a sum of maximum m
  __device__ __forceinline__ bool wild(float m, float c) const {
    return high || (low && !(m * c > -kWildExponent + 4096.0f));
  }
  // += t 2^r for a normal t > 0: integer operations and one fused multiply-add
  __device__ __forceinline__ void add(float t, int r) {
    const uint32_t b = __float_as_uint(t);
    const double t64 = __hiloint2double((int)((b >> 3) + (896u << 20)), (int)(b << 29));
    const bool up = r > rho;
    const int apart = up ? r - rho : rho - r;
    const double shift = __hiloint2double((1023 - (apart < 1000 ? apart : 1000)) << 20, 0);
    s = dfma(up ? s : t64, shift, up ? t64 : s);
    rho = up ? r : rho;
  }
  __device__ __forceinline__ ExpSum sum() const {
    ExpSum e;
    e.s = s;
    e.rho = rho > kNothing ? (double)rho : kNegInf64;
    return e;
  }
};

// Largest of the warp's values, none of them NaN.
__device__ __forceinline__ double warp_max64(double v) {
  const long long b = __double_as_longlong(v);
  const uint64_t key = b < 0 ? ~(uint64_t)b : (uint64_t)b | 0x8000000000000000ull;
  const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(key >> 32));
  const uint32_t lo = __reduce_max_sync(kFull, hi == (uint32_t)(key >> 32) ? (uint32_t)key : 0u);
  const uint64_t most = (uint64_t)hi << 32 | lo;
  return __longlong_as_double((long long)(most >> 63 ? most & 0x7fffffffffffffffull : ~most));
}

// s 2^rho as a multiple of 2^to, to >= rho: 0 for nothing, or the NaN it holds.
__device__ __forceinline__ double scaled_to(const ExpSum& a, double to) {
  return a.rho > kNegInf64 ? a.s * pow2_down(a.rho - to) : a.s;
}

__device__ __forceinline__ float warp_max_ordered(float v) {
  return key_value((uint64_t)__reduce_max_sync(kFull, ordkey(v)) << 32);
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Whether c is a number that exponents may be multiplied by: for T below
// 4.3e-39 it is infinite (0 c is no number then), above 2e45 it is 0 (-inf c).
inline bool scale_fits(double inv_t) {
  const float c = (float)(kLog2e64 * inv_t);
  return c > 0.0f && c <= 3.402823466e38f;
}

// The constant of a row's exponentials.
struct ExpScale {
  float c;  // fl32(log2(e) / T)
  __device__ __forceinline__ explicit ExpScale(double inv_t) : c((float)(kLog2e64 * inv_t)) {}
  // m c, exact in 64 bits
  __device__ __forceinline__ double exponent(float m) const { return (double)m * (double)c; }
  // natural log of the sum of e^((x - m) / T), s 2^rho being the row's sum and m
  // its maximum: nothing as large as m itself is left in it
  __device__ __forceinline__ double log_above(const ExpSum& a, float m) const {
    return (a.rho - exponent(m)) * kLn264 + log(a.s);
  }
};

// Adds the 2^(x c) of U vectors whose largest element is tm (NaN: one of
// them holds a NaN, and so does the sum from here on).
template <typename T, int U>
__device__ __forceinline__ void add_exps(StepSum& acc, const uint4 (&raw)[U], float tm, float c) {
  constexpr int n = RowVec<T>::n;
  const float top = tm * c;
  if (fabsf(top) < kWildExponent) {
    const float magic = top + 12582912.0f;  // 1.5 2^23 + R
    const float R = magic - 12582912.0f;
    const uint64_t c2 = pk(c, c), r2 = pk(-R, -R);
    uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[n];
      RowVec<T>::unpack(raw[u], v);
#pragma unroll
      for (int e = 0; e < n; e += 4) {
        const uint64_t a = fma2(pk(v[e], v[e + 1]), c2, r2), b = fma2(pk(v[e + 2], v[e + 3]), c2, r2);
        sum0 = add2(sum0, pk(ex2_approx(lo_f(a)), ex2_approx(hi_f(a))));
        sum1 = add2(sum1, pk(ex2_approx(lo_f(b)), ex2_approx(hi_f(b))));
      }
    }
    const uint64_t sum = add2(sum0, sum1);
    acc.add(lo_f(sum) + hi_f(sum), (int)(__float_as_uint(magic) - 0x4B400000u));
  } else if (tm < 0.0f) {
    acc.low = acc.low || tm > kNegInf;
  } else {
    acc.high = true;
    if (tm != tm) acc.s = nan64();
  }
}

// A wild row's elements of one vector.
template <typename T>
__device__ __forceinline__ void add_wild(ExpSum& acc, uint4 raw, const ExpScale& k) {
  const float tm = RowVec<T>::largest(raw);
  if (tm == kNegInf) return;
  float v[RowVec<T>::n], sum = 0.0f;
  RowVec<T>::unpack(raw, v);
#pragma unroll
  for (int e = 0; e < RowVec<T>::n; ++e) sum += ex2_approx((v[e] - tm) * k.c);
  acc.add((double)sum, tm == tm ? k.exponent(tm) : kNegInf64);
}

}  // namespace pm
