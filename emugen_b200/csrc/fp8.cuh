// Rounding to the 8-bit formats exactly as defined: code = nearest value of the format to the quotient
// x / scale, ties to even, where scale = fl32(amax / F), F = 7 * 2^n the type's largest value.
//
// 16-bit inputs.  F * x / amax is a quotient of short integers: against a border between two codes (an
// odd multiple of half a step, at most 5 bits) it is either equal or at least a relative 2^-16 away, since
// 7 x and border * amax have at most 14 and 16 bits.  Where it is equal, x / scale lies on the side that the
// rounding of scale decides, for the whole block alike: below the border if F * scale > amax, above it if
// F * scale < amax, on it if scale is exact.  So one product with 1 / scale, made a relative 2^-21
// smaller or larger, rounds every element right; where scale is exact, the product is rounded to 20 bits
// first, which takes its error away and leaves ties ties.
//
// f32 inputs.  x is multiplied by two numbers that enclose 1 / scale (a relative 2^-21 around it) and both
// products are converted: where the codes agree, the quotient between them has that code too.  Where they
// differ, border * scale - |x| is taken in one fused multiply-add, whose sign is exact.
//
// A division for each element would cost more than either and still turn near-ties into ties.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace emu {
namespace f8 {

template <int TYPE> struct Fmt;
template <> struct Fmt<EMU_FP8_E4M3> {
  static constexpr float MAX = 448.0f;
  static constexpr int BITS = 3;                 // stored significand bits
  static constexpr float REBIAS = 0x1p120f;      // f32's exponent bias over the type's
  static constexpr __nv_fp8_interpretation_t KIND = __NV_E4M3;
};
template <> struct Fmt<EMU_FP8_E5M2> {
  static constexpr float MAX = 57344.0f;
  static constexpr int BITS = 2;
  static constexpr float REBIAS = 0x1p112f;
  static constexpr __nv_fp8_interpretation_t KIND = __NV_E5M2;
};
constexpr uint32_t NAN_CODE = 0x7Fu;   // a NaN of both types

// 8 consecutive elements as they were read, two 16-bit elements to a word.
template <typename T> struct Raw {
  static constexpr int WORDS = 2 * sizeof(T);
  uint32_t w[WORDS];
};

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

template <typename T> __device__ __forceinline__ float element(const Raw<T>& r, int i);
template <> __device__ __forceinline__ float element(const Raw<float>& r, int i) { return __uint_as_float(r.w[i]); }
template <> __device__ __forceinline__ float element(const Raw<__nv_bfloat16>& r, int i) {
  return __uint_as_float(i & 1 ? r.w[i / 2] & 0xFFFF0000u : r.w[i / 2] << 16);
}
template <> __device__ __forceinline__ float element(const Raw<__half>& r, int i) {
  return __half2float(__ushort_as_half((unsigned short)(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2])));
}

// Magnitudes are compared as bit patterns, which order like the values, infinities and NaN above all of
// them.  Such a top tells that the block needs finite_top.
template <typename T> __device__ __forceinline__ uint32_t top_bits(const Raw<T>& r) {
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, r.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max_u16x2(m, r.w[i] & 0x7FFF7FFFu);
    return max(m & 0xFFFFu, m >> 16);
  }
}
template <typename T> __device__ __forceinline__ bool special(uint32_t bits);
template <> __device__ __forceinline__ bool special<float>(uint32_t b) { return b >= 0x7F800000u; }
template <> __device__ __forceinline__ bool special<__half>(uint32_t b) { return b >= 0x7C00u; }
template <> __device__ __forceinline__ bool special<__nv_bfloat16>(uint32_t b) { return b >= 0x7F80u; }
template <typename T> __device__ __forceinline__ float bits_to_float(uint32_t b);
template <> __device__ __forceinline__ float bits_to_float<float>(uint32_t b) { return __uint_as_float(b); }
template <> __device__ __forceinline__ float bits_to_float<__half>(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
template <> __device__ __forceinline__ float bits_to_float<__nv_bfloat16>(uint32_t b) { return __uint_as_float(b << 16); }
// one element's magnitude bits, 0 for NaN and infinities (which are stored as NaN and scale nothing)
template <typename T> __device__ __forceinline__ uint32_t finite_bits(const Raw<T>& r, int i) {
  uint32_t b;
  if constexpr (sizeof(T) == 4) b = r.w[i] & 0x7FFFFFFFu;
  else b = (i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2]) & 0x7FFFu;
  return special<T>(b) ? 0u : b;
}
template <typename T> __device__ __forceinline__ uint32_t finite_top_bits(const Raw<T>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, finite_bits(r, i));
  return m;
}

// A block's scale with what its elements are multiplied by: `lo` and `hi` around the reciprocal (f32), or `lo`
// alone (16-bit inputs; `exact`: rounded products).  The smallest normal f32 for blocks that hold (almost)
// nothing, so that 1 / scale stays finite.
// (lo and hi: the reciprocal's error, 2^-23, the product's, 2^-24, and scale's own stay within the 2^-21.)
struct Scale {
  float s, lo, hi;
  bool exact;
};
template <typename T, int TYPE> __device__ __forceinline__ Scale scale_of(float amax) {
  Scale r;
  // amax / F rounded to nearest: the product with the rounded 1 / F, corrected once by its exact remainder
  // (Markstein 1990); below 2^-126, where remainders would underflow, the result is not used
  constexpr float RCP = 1.0f / Fmt<TYPE>::MAX;
  const float d0 = __fmul_rn(amax, RCP);
  const float d = __fmaf_rn(__fmaf_rn(-d0, Fmt<TYPE>::MAX, amax), RCP, d0);
  r.s = fmaxf(d, 0x1p-126f);
  float inv;                                                   // to 1 unit of the last place
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(r.s));
  if constexpr (sizeof(T) == 4) {
    r.lo = __fmul_rn(inv, 1.0f - 0x1p-21f);
    r.hi = __fmul_rn(inv, 1.0f + 0x1p-21f);
    r.exact = false;
  } else {
    const float e = __fmaf_rn(Fmt<TYPE>::MAX, r.s, -amax);
    r.exact = e == 0.0f || d < 0x1p-126f;
    r.lo = r.exact ? inv : __fmul_rn(inv, e > 0.0f ? 1.0f - 0x1p-21f : 1.0f + 0x1p-21f);
    r.hi = r.lo;
  }
  return r;
}

template <int TYPE> __device__ __forceinline__ uint32_t cvt2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, Fmt<TYPE>::KIND);
}

// The code of x where the two products' codes differ; `lo` is the one nearer to zero.  The border above it
// is its code with half a step more, read as an f32 (subnormals included) and rebiased.
template <int TYPE> __device__ __forceinline__ uint32_t settle(float x, float scale, uint32_t lo) {
  const uint32_t m = lo & 0x7Fu;
  const float mid = __fmul_rn(__uint_as_float((2u * m + 1u) << (22 - Fmt<TYPE>::BITS)), Fmt<TYPE>::REBIAS);
  if (scale < 0x1p-60f) x *= 0x1p60f, scale *= 0x1p60f;      // the difference must not underflow
  const float d = __fmaf_rn(mid, scale, -fabsf(x));
  return (lo & 0x80u) | (m + (d < 0.0f ? 1u : d > 0.0f ? 0u : m & 1u));
}
// Out of line: few elements of f32 inputs come here, and its code eight times over would not stay in the
// instruction cache.
template <int TYPE> __device__ __noinline__ uint2 settle8(float x0, float x1, float x2, float x3, float x4, float x5,
                                                          float x6, float x7, float scale, uint2 w, uint2 h) {
  const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t& word = i < 4 ? w.x : w.y;
    const int sh = 8 * (i & 3);
    if (((word ^ (i < 4 ? h.x : h.y)) >> sh) & 0xFFu) {
      const uint32_t c = settle<TYPE>(x[i], scale, (word >> sh) & 0xFFu);
      word = (word & ~(0xFFu << sh)) | (c << sh);
    }
  }
  return w;
}

// 8 elements -> 8 codes (byte i = element i).
template <typename T, int TYPE> __device__ __forceinline__ uint2 encode8(const float (&x)[8], const Scale& s) {
  uint32_t lo[4];
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(x[i], s.lo);
  if (sizeof(T) == 2 && s.exact) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __uint_as_float((__float_as_uint(y[i]) + 8u) & ~15u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) lo[i] = cvt2<TYPE>(y[2 * i], y[2 * i + 1]);
  const uint2 w = make_uint2(__byte_perm(lo[0], lo[1], 0x5410), __byte_perm(lo[2], lo[3], 0x5410));
  if constexpr (sizeof(T) == 4) {
    uint32_t hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = cvt2<TYPE>(__fmul_rn(x[2 * i], s.hi), __fmul_rn(x[2 * i + 1], s.hi));
    const uint2 h = make_uint2(__byte_perm(hi[0], hi[1], 0x5410), __byte_perm(hi[2], hi[3], 0x5410));
    if ((w.x ^ h.x) | (w.y ^ h.y)) return settle8<TYPE>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], s.s, w, h);
  }
  return w;
}

// The same for a block that holds NaN or infinities: they become NaN.
template <typename T, int TYPE>
__device__ __noinline__ uint2 encode8_special(float x0, float x1, float x2, float x3, float x4, float x5, float x6,
                                              float x7, Scale s) {
  const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
  float y[8];
  uint2 bad = make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool b = (__float_as_uint(x[i]) & 0x7FFFFFFFu) >= 0x7F800000u;
    y[i] = b ? 0.0f : x[i];
    if (b) (i < 4 ? bad.x : bad.y) |= NAN_CODE << (8 * (i & 3));
  }
  const uint2 w = encode8<T, TYPE>(y, s);
  return make_uint2(w.x | bad.x, w.y | bad.y);
}
template <typename T, int TYPE> __device__ __forceinline__ uint2 encode8(const float (&x)[8], const Scale& s, bool specials) {
  if (specials) return encode8_special<T, TYPE>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], s);
  return encode8<T, TYPE>(x, s);
}

// 8 consecutive elements, `valid` of them in range (the others 0).  VEC: p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int valid, Raw<T>& r) {
  if (VEC && valid >= 8) {
#pragma unroll
    for (int i = 0; i < Raw<T>::WORDS / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < Raw<T>::WORDS; ++i) r.w[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= valid) continue;
    if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(p[i]);
    else r.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
  }
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
