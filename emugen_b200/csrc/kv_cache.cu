// Quantised key/value cache: rows (token, head) of D elements written to their slots in 8 or 4 bits, and
// the rows of a batch of sequences read back through a block table.
//
//   EMU_KV_FP8    E4M3 codes, one f32 scale per 128 elements of a row (the quantiser of quant_fp8.cu)
//   EMU_KV_MXFP4  e2m1 codes, one power-of-two scale byte per 32 elements (the quantiser of quant.cu)
//
// Bound: memory (one read and one write of each row); a decode step's few rows: the launch.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "fp4.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace emu {
namespace {

constexpr int MAX_TOKENS = 64;        // tokens per CTA of the write kernel
constexpr int HASH_BITS = 2048;

// `dead[i]` for each of this CTA's tokens i0 + i: a later token of the call has the same slot, so that token's
// row is the one that is kept (two rows written at once would leave a mixture).  The CTA's slots are
// hashed into a bit table; every later slot is looked up there, and only a hit is compared in full.
__device__ __forceinline__ void find_overwritten(const int64_t* __restrict__ slots, int64_t T, int64_t i0, int n,
                                                 int64_t* own, uint32_t* table, int* dead) {
  for (int i = threadIdx.x; i < HASH_BITS / 32; i += blockDim.x) table[i] = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) own[i] = slots[i0 + i], dead[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    if (own[i] < 0) continue;                                // padding: writes nothing
    const uint32_t h = (uint32_t)own[i] % HASH_BITS;
    atomicOr(&table[h >> 5], 1u << (h & 31));
  }
  __syncthreads();
  for (int64_t j = i0 + 1 + threadIdx.x; j < T; j += blockDim.x) {
    const int64_t s = slots[j];
    const uint32_t h = (uint32_t)s % HASH_BITS;
    if (s >= 0 && ((table[h >> 5] >> (h & 31)) & 1u)) {
      for (int i = 0; i < n && i0 + i < j; ++i)
        if (own[i] == s) dead[i] = 1;
    }
  }
  __syncthreads();
}

// 16 lanes take 128 elements of a row, 8 each.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvWriteArgs a, int tokens_per_cta) {
  __shared__ int64_t own[MAX_TOKENS];
  __shared__ uint32_t table[HASH_BITS / 32];
  __shared__ int dead[MAX_TOKENS];
  const int64_t i0 = (int64_t)blockIdx.x * tokens_per_cta;
  const int n = (int)min((int64_t)tokens_per_cta, a.T - i0);
  find_overwritten(a.slots, a.T, i0, n, own, table, dead);
  const int lane16 = threadIdx.x & 15;
  const int64_t G = (a.D + 127) / 128;
  const int tensors = a.x[1] ? 2 : 1;
  const int64_t per_tensor = a.H * G, per_token = per_tensor * tensors;
  const int64_t units = per_token * n, rounded = (units + 1) / 2 * 2;    // whole warps take part in the shuffles
  for (int64_t u = threadIdx.x >> 4; u < rounded; u += blockDim.x >> 4) {
    const int i = (int)(u / per_token);
    const int64_t rem = u % per_token;
    const int which = rem >= per_tensor;
    const int64_t hg = which ? rem - per_tensor : rem;
    const int64_t h = hg / G, g = hg % G;
    const int64_t d = g * 128 + lane16 * 8;
    const bool have = u < units;
    const int64_t slot = have ? own[i] : -1;
    const bool live = have && !dead[i] && slot >= 0 && slot < a.num_slots;
    const int valid = live && d < a.D ? 8 : 0;               // D is a multiple of 16
    f8::Raw<T> r;
    f8::load8<T, VEC>(static_cast<const T*>(a.x[which]) + (i0 + i) * a.token_stride[which] + h * a.head_stride[which] + d,
                      valid, r);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f8::element(r, e);
    const int64_t row = slot * a.H + h;
    if (FORMAT == EMU_KV_FP8) {
      uint32_t top = f8::top_bits(r);
#pragma unroll
      for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      const bool sp = f8::special<T>(top);
      if (__any_sync(0xFFFFFFFFu, sp)) {
        top = f8::finite_top_bits(r);
#pragma unroll
        for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      }
      const f8::Scale s = f8::scale_of<T, EMU_FP8_E4M3>(f8::bits_to_float<T>(top));
      const uint2 w = f8::encode8<T, EMU_FP8_E4M3>(v, s, sp);
      if (valid) *reinterpret_cast<uint2*>(a.q[which] + row * a.D + d) = w;
      if (live && lane16 == 0) static_cast<float*>(a.scale[which])[row * G + g] = s.s;
    } else {
      // as quant_fp4_kernel<T, 32>: the same roundings and flushes, so the same bytes
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));        // NaN is passed over
#pragma unroll
      for (int o = 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      top = ftz(ftz(top) * rcp_approx_ftz(6.0f));
      const uint8_t sf = __nv_cvt_float_to_e8m0(top, __NV_SATFINITE, cudaRoundPosInf);
      const float out_scale = top != 0.0f ? (sf == 0 ? 1.0f : pow2_127_minus(sf)) : 0.0f;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __fmul_rn(sizeof(T) == 2 && std::is_same<T, __half>::value ? v[e] : ftz(v[e]), out_scale);
      if (valid) {
        *reinterpret_cast<uint32_t*>(a.q[which] + (row * a.D + d) / 2) = f32x8_to_e2m1(y);
        if ((lane16 & 3) == 0) static_cast<uint8_t*>(a.scale[which])[row * (a.D / 32) + d / 32] = sf;
      }
    }
  }
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int READ_ROWS = 8;          // output rows per CTA of the read kernel

// 16 lanes give 128 elements of a row, 8 each.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvReadArgs a) {
  __shared__ int64_t slot_of[READ_ROWS];     // -1: a row of zeros (no such page), -2: left as it was
  const int64_t r0 = (int64_t)blockIdx.x * READ_ROWS;
  const int rows = (int)min((int64_t)READ_ROWS, a.total - r0);
  if (threadIdx.x < rows) {
    const int64_t r = r0 + threadIdx.x;
    // the last sequence that begins at or before r
    int64_t lo = 0, hi = a.B;
    while (lo < hi) {
      const int64_t m = (lo + hi) / 2;
      if ((int64_t)a.cu_lens[m + 1] > r) hi = m;
      else lo = m + 1;
    }
    int64_t slot = -2;
    if (lo < a.B && (int64_t)a.cu_lens[lo] <= r) {
      const int64_t pos = r - a.cu_lens[lo], pg = pos / a.page_size;
      const int64_t page = pg < a.table_cols ? a.table[lo * a.table_stride + pg] : -1;
      slot = page >= 0 && page < a.num_pages ? page * a.page_size + pos % a.page_size : -1;
    }
    slot_of[threadIdx.x] = slot;
  }
  __syncthreads();
  const int lane16 = threadIdx.x & 15;
  const int64_t G = (a.D + 127) / 128;
  const int tensors = a.q[1] ? 2 : 1;
  const int64_t per_tensor = a.H * G, per_row = per_tensor * tensors;
  for (int64_t u = threadIdx.x >> 4; u < per_row * rows; u += blockDim.x >> 4) {
    const int i = (int)(u / per_row);
    const int64_t rem = u % per_row;
    const int which = rem >= per_tensor;
    const int64_t hg = which ? rem - per_tensor : rem;
    const int64_t h = hg / G, g = hg % G;
    const int64_t d = g * 128 + lane16 * 8;
    const int64_t slot = slot_of[i];
    if (d >= a.D || slot == -2) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (slot >= 0) {
      const int64_t row = slot * a.H + h;
      if (FORMAT == EMU_KV_FP8) {
        const uint2 w = *reinterpret_cast<const uint2*>(a.q[which] + row * a.D + d);
        const float s = static_cast<const float*>(a.scale[which])[row * G + g];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint32_t word = e < 4 ? w.x : w.y;
          const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word >> (8 * (e & 3))), __NV_E4M3);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
          v[e] = __fmul_rn(f.x, s);
          v[e + 1] = __fmul_rn(f.y, s);
        }
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(a.q[which] + (row * a.D + d) / 2);
        const uint32_t sf = static_cast<const uint8_t*>(a.scale[which])[row * (a.D / 32) + d / 32];
        const float s = __uint_as_float(sf << 23);           // 0 -> 0, 255 -> inf, as emu_dequant_fp4
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t c = w >> (4 * e);
          const float mag = (float)e2m1_twice(c & 7u) * 0.5f;
          v[e] = __fmul_rn((c & 8u) ? -mag : mag, s);
        }
      }
    }
    T* dst = static_cast<T*>(a.out[which]) + (r0 + i) * a.token_stride[which] + h * a.D + d;
    T y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = from_float<T>(v[e]);
    if (VEC) {
#pragma unroll
      for (int e = 0; e < (int)sizeof(y) / 16; ++e) reinterpret_cast<uint4*>(dst)[e] = reinterpret_cast<const uint4*>(y)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = y[e];
    }
  }
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t stream) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int per_cta = (int)std::min<int64_t>(MAX_TOKENS, (a.T + 4 * sms - 1) / (4 * sms));
  const unsigned grid = (unsigned)((a.T + per_cta - 1) / per_cta);
  bool vec = true;
  for (int w = 0; w < 2; ++w)
    if (a.x[w]) vec = vec && ((reinterpret_cast<uintptr_t>(a.x[w]) | (uintptr_t)(a.token_stride[w] * 2) | (uintptr_t)(a.head_stride[w] * 2)) & 15) == 0;
#define EMU_KV(T, F) (vec ? kv_write_kernel<T, F, true><<<grid, 256, 0, stream>>>(a, per_cta) : kv_write_kernel<T, F, false><<<grid, 256, 0, stream>>>(a, per_cta))
  if (a.format == EMU_KV_FP8) {
    if (a.dtype == EMU_DTYPE_F16) EMU_KV(__half, EMU_KV_FP8);
    else EMU_KV(__nv_bfloat16, EMU_KV_FP8);
  } else {
    if (a.dtype == EMU_DTYPE_F16) EMU_KV(__half, EMU_KV_MXFP4);
    else EMU_KV(__nv_bfloat16, EMU_KV_MXFP4);
  }
#undef EMU_KV
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream) {
  const unsigned grid = (unsigned)((a.total + READ_ROWS - 1) / READ_ROWS);
  const int esz = a.out_dtype == EMU_DTYPE_F32 ? 4 : 2;
  bool vec = true;
  for (int w = 0; w < 2; ++w)
    if (a.out[w]) vec = vec && ((reinterpret_cast<uintptr_t>(a.out[w]) | (uintptr_t)(a.token_stride[w] * esz)) & 15) == 0;
#define EMU_KV(T, F) (vec ? kv_read_kernel<T, F, true><<<grid, 256, 0, stream>>>(a) : kv_read_kernel<T, F, false><<<grid, 256, 0, stream>>>(a))
#define EMU_KVF(F)                                               \
  if (a.out_dtype == EMU_DTYPE_F16) EMU_KV(__half, F);           \
  else if (a.out_dtype == EMU_DTYPE_BF16) EMU_KV(__nv_bfloat16, F); \
  else EMU_KV(float, F);
  if (a.format == EMU_KV_FP8) {
    EMU_KVF(EMU_KV_FP8)
  } else {
    EMU_KVF(EMU_KV_MXFP4)
  }
#undef EMU_KVF
#undef EMU_KV
  return cudaGetLastError();
}

}  // namespace emu
