// FP4 encoding steps shared by the FP4 quantisers (quant.cu) and the quantised cache (kv_cache.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace emu {
namespace {

__device__ __forceinline__ float rcp_approx_ftz(float a) {
  float b;
  asm volatile("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(b) : "f"(a));
  return b;
}

// 8 floats -> 8 e2m1 codes in one 32-bit word (element 2i in the low nibble of byte i).
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&v)[8]) {
  uint32_t val;
  asm volatile(
      "{\n"
      ".reg .b8 byte0, byte1, byte2, byte3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 byte0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 byte1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 byte2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 byte3, %8, %7;\n"
      "mov.b32 %0, {byte0, byte1, byte2, byte3};\n"
      "}"
      : "=r"(val)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return val;
}

template <typename T> struct Vec2;
template <> struct Vec2<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 to_f2(type v) { return __half22float2(v); }
};
template <> struct Vec2<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 to_f2(type v) { return __bfloat1622float2(v); }
};

// 2^(127 - e) as f32 bits for e in [1, 255] (exact, subnormal for e >= 254).
__device__ __forceinline__ float pow2_127_minus(uint32_t e) {
  if (e >= 254u) return 0.0f;   // 2^-127 and below: subnormal, flushed as in flashinfer's build
  return __uint_as_float((254u - e) << 23);
}

// f32 subnormal -> signed zero (fast-math flush-to-zero); NaN and inf pass
__device__ __forceinline__ float ftz(float x) { return fabsf(x) < 1.17549435e-38f ? copysignf(0.0f, x) : x; }

}  // namespace
}  // namespace emu
