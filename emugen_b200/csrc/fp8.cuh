// Rounding to the 8-bit formats exactly as defined: code = nearest value of the format to the quotient
// x / scale (scale an f32), ties to even.
//
// A product x * (1 / scale) is within 2 units of f32's last place of the quotient, so it rounds to the
// same code unless the quotient lies that near to a border between two codes.  Those few elements
// (about one in 2^16, or all exact ties of 16-bit inputs) are decided by comparing |x| with
// border * scale, a product of at most 4 + 24 bits that f64 holds exactly.  A division for each
// element would cost twice the quantiser's instructions and still collapse near-ties into ties.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace emu {
namespace f8 {

template <int TYPE> struct Fmt;
template <> struct Fmt<EMU_FP8_E4M3> {
  static constexpr int BITS = 3;                       // stored significand bits
  static constexpr float MAX = 448.0f;
  static constexpr float MIN_NORMAL = 0x1p-6f;
  static constexpr __nv_fp8_interpretation_t KIND = __NV_E4M3;
};
template <> struct Fmt<EMU_FP8_E5M2> {
  static constexpr int BITS = 2;
  static constexpr float MAX = 57344.0f;
  static constexpr float MIN_NORMAL = 0x1p-14f;
  static constexpr __nv_fp8_interpretation_t KIND = __NV_E5M2;
};

// |x| for the group maximum: 0 for NaN and infinities, which are stored as NaN and scale nothing.
__device__ __forceinline__ float finite_magnitude(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? __uint_as_float(b) : 0.0f;
}

// The group's scale: the smallest normal f32 for groups that hold (almost) nothing, so that 1 / scale
// stays finite.
template <int TYPE>
__device__ __forceinline__ float scale_of(float amax) {
  return fmaxf(__fdiv_rn(amax, Fmt<TYPE>::MAX), 0x1p-126f);
}

// y ~ x / scale, near a border of the format?
template <int TYPE>
__device__ __forceinline__ bool near_border(float y) {
  constexpr int D = 23 - Fmt<TYPE>::BITS;              // bits of an f32 significand that the format drops
  constexpr uint32_t HALF = 1u << (D - 1);
  const float a = fabsf(y);
  // below the smallest normal the step is that of the first binade: adding its start aligns the bits
  const float t = a < Fmt<TYPE>::MIN_NORMAL ? a + Fmt<TYPE>::MIN_NORMAL : a;
  return (__float_as_uint(t) & ((1u << D) - 1u)) - (HALF - 8u) <= 16u;
}

// y near a border: the border itself if |x| / scale is exactly there, else a value clearly on its side.
template <int TYPE>
__device__ __noinline__ float settle(float x, float y, float scale) {
  constexpr int D = 23 - Fmt<TYPE>::BITS;
  const float a = fabsf(y);
  const bool sub = a < Fmt<TYPE>::MIN_NORMAL;
  const float t = sub ? a + Fmt<TYPE>::MIN_NORMAL : a;
  float mid = __uint_as_float((__float_as_uint(t) & ~((1u << D) - 1u)) | (1u << (D - 1)));
  if (sub) mid -= Fmt<TYPE>::MIN_NORMAL;
  const double q = fabs((double)x), m = __dmul_rn((double)mid, (double)scale);
  if (y != y) return y;
  const float r = q > m ? mid * (1.0f + 0x1p-10f) : q < m ? mid * (1.0f - 0x1p-10f) : mid;
  return copysignf(r, y);
}

// 8 elements -> 8 codes (byte i = element i).  inv = 1 / scale in f32.
template <int TYPE>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float scale, float inv) {
  float y[8];
  bool near_any = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = __fmaf_rn(x[i], 0.0f, __fmul_rn(x[i], inv));   // x * 0 turns an infinity into NaN and adds nothing else
    near_any |= near_border<TYPE>(y[i]);
  }
  if (near_any) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (near_border<TYPE>(y[i])) y[i] = settle<TYPE>(x[i], y[i], scale);
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, Fmt<TYPE>::KIND);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// 8 consecutive elements, `valid` of them in range (the others 0).  VEC: p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int valid, float (&x)[8]) {
  if (VEC && valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        T lo, hi;
        reinterpret_cast<uint16_t&>(lo) = (uint16_t)u[i];
        reinterpret_cast<uint16_t&>(hi) = (uint16_t)(u[i] >> 16);
        x[2 * i] = to_float<T>(lo);
        x[2 * i + 1] = to_float<T>(hi);
      }
    } else {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = i < valid ? to_float<T>(p[i]) : 0.0f;
}

// 8 codes to q (8-byte aligned), `valid` of them in range.
__device__ __forceinline__ void store8(uint8_t* q, uint2 w, int valid) {
  if (valid >= 8) {
    *reinterpret_cast<uint2*>(q) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) q[i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
}

}  // namespace f8
}  // namespace emu
