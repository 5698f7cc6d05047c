// Device-side building blocks of the 8-bit floating-point operators: element
// types, codes, power-of-two block scales.
//
// A block's scale is 2^e with e the smallest integer for which every finite
// value fits, amax <= FMAX * 2^e, and at least -127; its code is the
// round-to-nearest-even 8-bit float of x * 2^-e.  A power of two costs nothing
// against a free scale in relative precision (a float's rounding error does
// not depend on its exponent), keeps x * 2^-e and code * 2^e exact, makes the
// codes independent of how the scale is computed, and is the form the tensor
// cores multiply by themselves (ue8m0).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "f64e.h"

namespace f64e {

// ------------------------------------------------------------ scale bytes --
// FMAX = 1.75 * 2^emax in both codes: e = p - emax for a largest magnitude
// m * 2^p with m in [1, 1.75], one more above.  Subnormal magnitudes give
// exponents below -127 whatever their leading bit, so the field serves as p.
template <int CODE>
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  constexpr int emax = CODE == F64E_E4M3 ? 8 : 15;
  if (amax_bits == 0) return 0;
  const int p = (int)(amax_bits >> 23) - 127;
  const int e = p - emax + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < -127 ? -127 : e;
}
// 2^-e for e in [-127, 120]: a normal number.
__device__ __forceinline__ float inverse_scale(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }
// 2^(b - 127), b = 0 a subnormal; b = 255 stands for NaN.
__device__ __forceinline__ float scale_of_byte(uint32_t b) {
  return b == 255u ? __uint_as_float(0x7FFFFFFFu) : (b ? __uint_as_float(b << 23) : __uint_as_float(0x00400000u));
}

// ------------------------------------------------------------------ codes --
// Two codes from two scaled values, `lo` in the low byte.  Finite values are
// within FMAX by the choice of the scale; a NaN becomes a NaN code.
template <int CODE>
__device__ __forceinline__ uint32_t code2(float lo, float hi) {
  uint16_t r;
  if (CODE == F64E_E4M3)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// The code of an infinity (the conversion above would saturate it): infinity
// where the type has one, NaN in e4m3.
template <int CODE>
__device__ __forceinline__ uint32_t code_of_inf(bool negative) {
  return (CODE == F64E_E4M3 ? 0x7Fu : 0x7Cu) | (negative ? 0x80u : 0u);
}
template <int CODE>
__device__ __forceinline__ float2 values2(uint32_t codes) {
  uint32_t h;
  if (CODE == F64E_E4M3)
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  else
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// --------------------------------------------------------------- elements --
// Eight neighbouring elements of a row as 32-bit words.
template <int T>
struct Elem;
template <>
struct Elem<F64E_F32> {
  using type = float;
  static constexpr int kWords = 8;
  __device__ static float get(const uint32_t* w, int i) { return __uint_as_float(w[i]); }
  __device__ static uint32_t bits(float v) { return __float_as_uint(v); }
};
template <>
struct Elem<F64E_F16> {
  using type = __half;
  static constexpr int kWords = 4;
  __device__ static float get(const uint32_t* w, int i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i >> 1]));
    return (i & 1) ? f.y : f.x;
  }
  __device__ static uint32_t bits(float v) { return (uint32_t)__half_as_ushort(__float2half_rn(v)); }
};
template <>
struct Elem<F64E_BF16> {
  using type = __nv_bfloat16;
  static constexpr int kWords = 4;
  __device__ static float get(const uint32_t* w, int i) {
    return __uint_as_float((i & 1) ? (w[i >> 1] & 0xFFFF0000u) : (w[i >> 1] << 16));
  }
  __device__ static uint32_t bits(float v) { return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};

// Loads eight elements at p, of which the first n exist (n <= 0: none); the
// others read as zero.  vec: p is 16-byte aligned.
template <int T>
__device__ __forceinline__ void load8(const typename Elem<T>::type* p, int64_t n, bool vec, uint32_t* w) {
  if (vec && n >= 8) {
#pragma unroll
    for (int i = 0; i < Elem<T>::kWords / 4; i++) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < Elem<T>::kWords; i++) w[i] = 0;
  if (Elem<T>::kWords == 8) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) w[i] = __ldg(u + i);
  } else {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) w[i >> 1] |= (uint32_t)__ldg(u + i) << (16 * (i & 1));
  }
}

// ----------------------------------------------------------- magnitudes --
// Largest magnitude as 32-bit float bits; infinity and NaN order above every
// finite value, so "non-finite present" is amax >= kInfBits.
constexpr uint32_t kInfBits = 0x7F800000u;

template <int T>
__device__ __forceinline__ uint32_t mag(const uint32_t* w, int i) {
  return __float_as_uint(Elem<T>::get(w, i)) & 0x7FFFFFFFu;
}

// Eight codes of eight elements, all with the inverse scale r.  special: the
// block holds an infinity or a NaN.
template <int T, int CODE>
__device__ __forceinline__ uint2 codes8(const uint32_t* w, float r, bool special) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    c[i] = code2<CODE>(Elem<T>::get(w, 2 * i) * r, Elem<T>::get(w, 2 * i + 1) * r);
  if (special) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float v = Elem<T>::get(w, i);
      if ((__float_as_uint(v) & 0x7FFFFFFFu) == kInfBits)
        c[i >> 1] = (c[i >> 1] & ~(0xFFu << (8 * (i & 1)))) | (code_of_inf<CODE>(v < 0.f) << (8 * (i & 1)));
    }
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

}  // namespace f64e
