// Attention of one new token for each sequence over the quantised key/value cache.
//
// With s_j = scale q . k_j over the cached rows j < len of the sequence whose page exists, k_j = code * scale as it is
// stored:  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), m = max_j s_j   (no row: o = 0, lse = -inf)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/emugen.h"
#include "kernels.h"

namespace emu {
namespace {

constexpr int MAX_D = 256, WARPS = 8;

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

// Element d of the cached row (slot, head).
template <int FORMAT> __device__ __forceinline__ float cached(const uint8_t* q, const void* scales, int64_t row, int D, int d) {
  if (FORMAT == EMU_KV_FP8) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(q[row * D + d], __NV_E4M3);
    return __fmul_rn(__half2float(*reinterpret_cast<const __half*>(&h)), static_cast<const float*>(scales)[row * ((D + 127) / 128) + d / 128]);
  }
  const uint8_t b = q[row * (D / 2) + d / 2];
  const __half_raw h = __nv_cvt_fp4_to_halfraw((__nv_fp4_storage_t)(d & 1 ? b >> 4 : b & 15), __NV_E2M1);
  const uint32_t e = static_cast<const uint8_t*>(scales)[row * (D / 32) + d / 32];
  return __fmul_rn(__half2float(*reinterpret_cast<const __half*>(&h)), __uint_as_float(e ? e << 23 : 0x00400000u));
}

template <typename T, int FORMAT> __global__ void __launch_bounds__(WARPS * 32) kv_attend_simple_kernel(const __grid_constant__ KvAttendArgs a) {
  constexpr int E = MAX_D / 32;
  __shared__ float so[WARPS][MAX_D], sm[WARPS], sl[WARPS];
  const int64_t b = blockIdx.x / a.Hq;
  const int h = (int)(blockIdx.x - b * a.Hq), kh = h / (a.Hq / a.Hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[1];
  float x[E], o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = lane + 32 * i < a.D ? widen<T>(q[lane + 32 * i]) : 0.0f, o[i] = 0.0f;
  const int64_t len = min((int64_t)a.lens[b], a.table_cols * a.page_size);
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = warp; j < len; j += WARPS) {
    const int64_t page = a.table[b * a.table_stride + j / a.page_size];
    if (page < 0 || page >= a.num_pages) continue;
    const int64_t row = (page * a.page_size + j % a.page_size) * a.Hk + kh;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (lane + 32 * i < a.D) s = __fmaf_rn(x[i], cached<FORMAT>(a.cache[0], a.scales[0], row, a.D, lane + 32 * i), s);
#pragma unroll
    for (int k = 16; k; k >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xFFFFFFFFu, s, k));
    s = __fmul_rn(s, a.scale);
    const float top = fmaxf(m, s), shift = top == -INFINITY ? 0.0f : top;
    const float old = expf(m - shift), p = expf(s - shift);
    l = __fmaf_rn(l, old, p);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (lane + 32 * i < a.D) o[i] = __fmaf_rn(p, cached<FORMAT>(a.cache[1], a.scales[1], row, a.D, lane + 32 * i), __fmul_rn(o[i], old));
    m = top;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) so[warp][lane + 32 * i] = o[i];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  float top = -INFINITY;
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm[w]);
  const float shift = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int w = 0; w < WARPS; ++w) sum = __fmaf_rn(sl[w], expf(sm[w] - shift), sum);
  const float f = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  for (int d = threadIdx.x; d < a.D; d += WARPS * 32) {
    float v = 0.0f;
    for (int w = 0; w < WARPS; ++w) v = __fmaf_rn(so[w][d], expf(sm[w] - shift), v);
    static_cast<T*>(a.out)[(b * a.Hq + h) * a.D + d] = narrow<T>(__fmul_rn(v, f));
  }
  if (threadIdx.x == 0 && a.lse) a.lse[b * a.Hq + h] = sum > 0.0f ? top + logf(sum) : sum == 0.0f ? -INFINITY : sum;
}

}  // namespace

size_t kv_attend_workspace(int64_t, int, int, int) { return 0; }

cudaError_t launch_kv_attend(const KvAttendArgs& a, cudaStream_t stream) {
  const unsigned grid = (unsigned)(a.B * a.Hq);
  const bool half = a.dtype == EMU_DTYPE_F16;
  if (a.format == EMU_KV_FP8) {
    if (half) kv_attend_simple_kernel<__half, EMU_KV_FP8><<<grid, WARPS * 32, 0, stream>>>(a);
    else kv_attend_simple_kernel<__nv_bfloat16, EMU_KV_FP8><<<grid, WARPS * 32, 0, stream>>>(a);
  } else {
    if (half) kv_attend_simple_kernel<__half, EMU_KV_MXFP4><<<grid, WARPS * 32, 0, stream>>>(a);
    else kv_attend_simple_kernel<__nv_bfloat16, EMU_KV_MXFP4><<<grid, WARPS * 32, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace emu
