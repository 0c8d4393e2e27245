// Rotation of element pairs by position-dependent angles, shared by
// rotary_embedding (rotary.hip) and the latent store (latent_store.hip).
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t) * amp,  t = pos * inv_freq[i]
//
// The angle of a far position needs more than float32: at position 10^5 a
// float32 product is off by up to 2^-25 * 10^5 = 3e-3 rad, visible in bf16.
// The product is therefore taken in float64, in quarter turns, and only its
// distance from the next whole quarter is rounded to float32 (off by 2^-26
// quarters, 2.3e-8 rad); sine and cosine of that are float32 evaluations.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pa_common.h"

namespace pa {

constexpr int kRotMaxPairs = 256;  // rotary_dim / 2

// cos and sin (times amp) of pair i at position pos.
__device__ __forceinline__ void rot_angle(double inv_freq, int32_t pos, float amp, float& c, float& s) {
  const double quarters = (double)pos * inv_freq * 0.63661977236758134;  // 2 / pi
  const double q = __builtin_rint(quarters);
  float sn, cs;
  sincospif(.5f * (float)(quarters - q), &sn, &cs);
  const int k = (int)(q - 4. * __builtin_floor(.25 * q));  // q mod 4
  if (k & 1) {
    const float x = cs;
    cs = -sn;
    sn = x;
  }
  if (k & 2) {
    cs = -cs;
    sn = -sn;
  }
  c = cs * amp;
  s = sn * amp;
}

// 16 bytes of elements as floats and back, by element type.
template <typename T>
struct RotVec;

template <>
struct RotVec<uint16_t> {  // bf16 bit patterns
  static constexpr int kN = 8;
  static __device__ __forceinline__ void load(const u32x4& v, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = bf16_lo(v[e]);
      x[2 * e + 1] = bf16_hi(v[e]);
    }
  }
  static __device__ __forceinline__ u32x4 store(const float (&x)[8]) {
    return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  }
  static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ uint16_t put(float x) { return (uint16_t)pack_bf16x2(x, 0.f); }
};

template <>
struct RotVec<_Float16> {
  static constexpr int kN = 8;
  typedef __attribute__((__vector_size__(16))) _Float16 V;
  static __device__ __forceinline__ void load(const u32x4& v, float (&x)[8]) {
    const V h = __builtin_bit_cast(V, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
  }
  static __device__ __forceinline__ u32x4 store(const float (&x)[8]) {
    V h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (_Float16)x[e];
    return __builtin_bit_cast(u32x4, h);
  }
  static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
};

template <>
struct RotVec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void load(const u32x4& v, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
  }
  static __device__ __forceinline__ u32x4 store(const float (&x)[4]) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};

// Rotates pairs inside 16 bytes (kInter: pairs 2i, 2i + 1), first pair p0.
template <typename T>
__device__ __forceinline__ u32x4 rot_inter(const u32x4& v, const float* cs, const float* sn, int p0) {
  using V = RotVec<T>;
  float x[V::kN];
  V::load(v, x);
#pragma unroll
  for (int e = 0; e < V::kN / 2; ++e) {
    const float c = cs[p0 + e], s = sn[p0 + e], a = x[2 * e], b = x[2 * e + 1];
    x[2 * e] = a * c - b * s;
    x[2 * e + 1] = a * s + b * c;
  }
  return V::store(x);
}

// Rotates 16 bytes of first halves against 16 bytes of second halves, first
// pair p0.
template <typename T>
__device__ __forceinline__ void rot_half(u32x4& va, u32x4& vb, const float* cs, const float* sn, int p0) {
  using V = RotVec<T>;
  float a[V::kN], b[V::kN];
  V::load(va, a);
  V::load(vb, b);
#pragma unroll
  for (int e = 0; e < V::kN; ++e) {
    const float c = cs[p0 + e], s = sn[p0 + e], x = a[e], y = b[e];
    a[e] = x * c - y * s;
    b[e] = x * s + y * c;
  }
  va = V::store(a);
  vb = V::store(b);
}

}  // namespace pa
