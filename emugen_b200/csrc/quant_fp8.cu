// Block-scaled 8-bit quantiser (E4M3 or E5M2 codes, one f32 scale per block of 128): rows in blocks of
// 1 x 128 or tiles of 128 x 128, and the same for the transposed matrix, in one pass over the input.
//
//   scale = max(max |x| / F8_MAX rounded to f32, 2^-126) over the block's finite elements,
//   code  = nearest 8-bit value to x / scale, ties to even (fp8.cuh); NaN for NaN and infinities.
//
// Bound: memory.  Each input element is read once and kept in registers between the maximum and the
// rounding.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace emu {
namespace {

// Rows in 1 x 128 blocks.  16 lanes hold one block, 8 elements each; a CTA of 256 threads takes 4 rows
// x 4 blocks at a time (1 KB of consecutive 16-bit input per row).
template <typename T, int TYPE, bool VEC>
__global__ void __launch_bounds__(256) quant_fp8_rows_kernel(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx,
                                                             uint8_t* __restrict__ q, int64_t ldq,
                                                             float* __restrict__ scale, int64_t lds) {
  const int lane16 = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int64_t kb_count = (K + 127) / 128;
  const int64_t tiles_k = (kb_count + 3) / 4, tiles_m = (M + 3) / 4;
  for (int64_t t = blockIdx.x; t < tiles_k * tiles_m; t += gridDim.x) {
    const int64_t row = t / tiles_k * 4 + (grp >> 2);
    const int64_t kb = t % tiles_k * 4 + (grp & 3);
    const int64_t k = kb * 128 + lane16 * 8;
    const bool live = row < M && kb < kb_count;
    const int valid = live ? (int)min((int64_t)8, max((int64_t)0, K - k)) : 0;
    float v[8];
    f8::load8<T, VEC>(x + row * ldx + k, valid, v);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, f8::finite_magnitude(v[i]));
#pragma unroll
    for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const float s = f8::scale_of<TYPE>(top);
    const uint2 w = f8::encode8<TYPE>(v, s, __frcp_rn(s));
    if (!live) continue;
    f8::store8(q + row * ldq + k, w, valid);
    if (lane16 == 0) scale[kb * lds + row] = s;
  }
}

// One 128 x 128 tile per CTA of 256 threads, a thread holding 8 x 8 elements (rows 8 * (tid / 16) ..,
// columns 8 * (tid % 16) ..).  Row maxima meet in 16 lanes, column maxima in shared memory.  The
// transposed codes go through shared memory so that both outputs are written in 128-byte runs.
// TILE: one scale for the tile; otherwise one per row (q) and one per column (qt).
template <typename T, int TYPE, bool VEC, bool TILE>
__global__ void __launch_bounds__(256) quant_fp8_tile_kernel(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx,
                                                             uint8_t* __restrict__ q, int64_t ldq,
                                                             float* __restrict__ scale, int64_t lds,
                                                             uint8_t* __restrict__ qt, int64_t ldqt,
                                                             float* __restrict__ scale_t, int64_t ldst) {
  constexpr int PITCH = 136;                               // bytes per transposed row: 8-byte aligned, rows 34 banks apart
  __shared__ __align__(16) uint8_t tr[128 * PITCH];
  __shared__ float col_top[8][128];
  const int tid = threadIdx.x, cx = tid & 15, ry = tid >> 4, warp = tid >> 5;
  const int64_t tiles_k = (K + 127) / 128;
  const int64_t mb = blockIdx.x / tiles_k, kb = blockIdx.x % tiles_k;
  const int64_t r0 = mb * 128 + ry * 8, c0 = kb * 128 + cx * 8;
  const int valid_c = (int)min((int64_t)8, max((int64_t)0, K - c0));
  const int valid_r = (int)min((int64_t)8, max((int64_t)0, M - r0));
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f8::load8<T, VEC>(x + (r0 + i) * ldx + c0, i < valid_r ? valid_c : 0, v[i]);

  float row_top[8], ct[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) ct[j] = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    row_top[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = f8::finite_magnitude(v[i][j]);
      row_top[i] = fmaxf(row_top[i], a);
      ct[j] = fmaxf(ct[j], a);
    }
  }
  if (!TILE) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int o = 8; o; o >>= 1) row_top[i] = fmaxf(row_top[i], __shfl_xor_sync(0xFFFFFFFFu, row_top[i], o));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ct[j] = fmaxf(ct[j], __shfl_xor_sync(0xFFFFFFFFu, ct[j], 16));   // the warp's two row groups
      if ((tid & 16) == 0) col_top[warp][cx * 8 + j] = ct[j];
    }
  } else {
    float top = row_top[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, row_top[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if ((tid & 31) == 0) col_top[warp][0] = top;
  }
  __syncthreads();
  float tile_s = 0.0f, tile_inv = 0.0f;
  if (TILE) {
    float top = col_top[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, col_top[w][0]);
    tile_s = f8::scale_of<TYPE>(top);
    tile_inv = __frcp_rn(tile_s);
    if (tid == 0) {
      if (q) scale[mb * lds + kb] = tile_s;
      if (qt) scale_t[kb * ldst + mb] = tile_s;
    }
  }
  uint2 rows8[8];                                          // TILE: the rows' codes, shared by both outputs
  if (q || TILE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = TILE ? tile_s : f8::scale_of<TYPE>(row_top[i]);
      const float inv = TILE ? tile_inv : __frcp_rn(s);
      rows8[i] = f8::encode8<TYPE>(v[i], s, inv);
      if (q && i < valid_r) {
        f8::store8(q + (r0 + i) * ldq + c0, rows8[i], valid_c);
        if (!TILE && cx == 0) scale[kb * lds + r0 + i] = s;
      }
    }
  }
  if (!qt) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint2 w;
    if (TILE) {
      uint32_t lo = 0, hi = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo |= (((j < 4 ? rows8[i].x : rows8[i].y) >> (8 * (j & 3))) & 0xFFu) << (8 * i);
        hi |= (((j < 4 ? rows8[i + 4].x : rows8[i + 4].y) >> (8 * (j & 3))) & 0xFFu) << (8 * i);
      }
      w = make_uint2(lo, hi);
    } else {
      float top = col_top[0][cx * 8 + j];
#pragma unroll
      for (int u = 1; u < 8; ++u) top = fmaxf(top, col_top[u][cx * 8 + j]);
      const float s = f8::scale_of<TYPE>(top);
      float c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = v[i][j];
      w = f8::encode8<TYPE>(c, s, __frcp_rn(s));
      if (ry == 0 && j < valid_c) scale_t[mb * ldst + c0 + j] = s;
    }
    *reinterpret_cast<uint2*>(tr + (cx * 8 + j) * PITCH + ry * 8) = w;
  }
  __syncthreads();
  // 16 threads write one transposed row of 128 codes
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int c = u * 16 + (tid >> 4);
    const int64_t col = kb * 128 + c, r = mb * 128 + (tid & 15) * 8;
    if (col < K) f8::store8(qt + col * ldqt + r, *reinterpret_cast<const uint2*>(tr + c * PITCH + (tid & 15) * 8),
                            (int)min((int64_t)8, max((int64_t)0, M - r)));
  }
}

template <typename T, int TYPE>
cudaError_t launch_t(const T* x, int64_t M, int64_t K, int64_t ldx, int block, uint8_t* q, int64_t ldq, float* scale,
                     int64_t lds, uint8_t* qt, int64_t ldqt, float* scale_t, int64_t ldst, cudaStream_t stream) {
  // rows that start on 16 bytes are read 16 bytes at a time
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0;
  const int64_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  if (block == EMU_BLOCK_ROW && !qt) {
    const int64_t tiles = ((kb + 3) / 4) * ((M + 3) / 4);
    const unsigned grid = (unsigned)std::min<int64_t>(tiles, 0x7FFFFFFF);
    if (vec) quant_fp8_rows_kernel<T, TYPE, true><<<grid, 256, 0, stream>>>(x, M, K, ldx, q, ldq, scale, lds);
    else quant_fp8_rows_kernel<T, TYPE, false><<<grid, 256, 0, stream>>>(x, M, K, ldx, q, ldq, scale, lds);
    return cudaGetLastError();
  }
  const unsigned grid = (unsigned)(kb * mb);
#define EMU_TILE(V, TL) \
  quant_fp8_tile_kernel<T, TYPE, V, TL><<<grid, 256, 0, stream>>>(x, M, K, ldx, q, ldq, scale, lds, qt, ldqt, scale_t, ldst)
  if (block == EMU_BLOCK_TILE) {
    if (vec) EMU_TILE(true, true);
    else EMU_TILE(false, true);
  } else {
    if (vec) EMU_TILE(true, false);
    else EMU_TILE(false, false);
  }
#undef EMU_TILE
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quant_fp8(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int fp8_type, int block,
                             uint8_t* q, int64_t ldq, float* scale, int64_t lds, uint8_t* qt, int64_t ldqt,
                             float* scale_t, int64_t ldst, cudaStream_t stream) {
#define EMU_Q(T, TY) launch_t<T, TY>(static_cast<const T*>(x), M, K, ldx, block, q, ldq, scale, lds, qt, ldqt, scale_t, ldst, stream)
  if (fp8_type == EMU_FP8_E4M3) {
    if (dtype == EMU_DTYPE_F16) return EMU_Q(__half, EMU_FP8_E4M3);
    if (dtype == EMU_DTYPE_BF16) return EMU_Q(__nv_bfloat16, EMU_FP8_E4M3);
    return EMU_Q(float, EMU_FP8_E4M3);
  }
  if (dtype == EMU_DTYPE_F16) return EMU_Q(__half, EMU_FP8_E5M2);
  if (dtype == EMU_DTYPE_BF16) return EMU_Q(__nv_bfloat16, EMU_FP8_E5M2);
  return EMU_Q(float, EMU_FP8_E5M2);
#undef EMU_Q
}

}  // namespace emu
