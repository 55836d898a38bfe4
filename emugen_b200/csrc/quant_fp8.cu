// Block-scaled 8-bit quantiser (E4M3 or E5M2 codes, one f32 scale per block of 128): rows in blocks of
// 1 x 128 or tiles of 128 x 128, and the same for the transposed matrix, in one pass over the input.
//
//   scale = max(max |x| / F8_MAX rounded to f32, 2^-126) over the block's finite elements,
//   code  = nearest 8-bit value to x / scale, ties to even (fp8.cuh); NaN for NaN and infinities.
//
// Each input element is read once and kept in registers between the maximum and the rounding.  What bounds
// the kernels is their arithmetic (ALU pipe 58% busy) before the memory: 8192 x 8192 bf16 on B200, rows 45 us
// (203 MB: floor 31), rows and columns 86 us (272 MB: floor 42), tiles 35 us, tiles with the transpose 51 us; f32, two
// products and conversions an element, rows 72 us (338 MB: floor 52), rows and columns 116 us (407 MB: floor 62), tiles
// 58 us, tiles with the transpose 81 us.
// A division or a border test for each element took rows and columns to 255 us (fp8.cuh).
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace emu {
namespace {

// Rows in 1 x 128 blocks.  16 lanes hold one block, 8 elements each; a CTA of 256 threads takes 4 U rows
// x 4 blocks (1 KB of consecutive 16-bit input per row), U loads in flight per thread.
template <typename T, int TYPE, bool VEC, int U>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 0)
    quant_fp8_rows_kernel(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
                          float* __restrict__ scale, int64_t lds) {
  const int lane16 = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int64_t kb_count = (K + 127) / 128;
  const int64_t kb = (int64_t)blockIdx.x * 4 + (grp & 3), k = kb * 128 + lane16 * 8;
  const int valid_k = (int)min((int64_t)8, max((int64_t)0, K - k));
  for (int64_t m0 = (int64_t)blockIdx.y * (4 * U); m0 < M; m0 += (int64_t)gridDim.y * (4 * U)) {
    const int64_t row0 = m0 + (grp >> 2);
    f8::Raw<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + 4 * u;
      f8::load8<T, VEC>(x + row * ldx + k, row < M ? valid_k : 0, r[u]);
    }
    uint32_t top[U];
    bool sp = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      top[u] = f8::top_bits(r[u]);
      sp |= f8::special<T>(top[u]);
    }
    sp = __any_sync(0xFFFFFFFFu, sp);
    if (sp) {                                                // (rare) leave out what is not finite
#pragma unroll
      for (int u = 0; u < U; ++u) top[u] = f8::finite_top_bits(r[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (sizeof(T) == 2 && U > 1) {                         // two rows' tops to a word
        if (u & 1) continue;
        uint32_t two = top[u] | top[(u + 1) % U] << 16;
#pragma unroll
        for (int o = 8; o; o >>= 1) two = f8::max_u16x2(two, __shfl_xor_sync(0xFFFFFFFFu, two, o));
        top[u] = two & 0xFFFFu, top[(u + 1) % U] = two >> 16;
      } else {
#pragma unroll
        for (int o = 8; o; o >>= 1) top[u] = max(top[u], __shfl_xor_sync(0xFFFFFFFFu, top[u], o));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + 4 * u;
      const f8::Scale sc = f8::scale_of<T, TYPE>(f8::bits_to_float<T>(top[u]));
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = f8::element(r[u], i);
      const uint2 w = f8::encode8<T, TYPE>(v, sc, sp);
      if (row >= M || kb >= kb_count) continue;
      f8::store8(q + row * ldq + k, w, valid_k);
      if (lane16 == 0) scale[kb * lds + row] = sc.s;
    }
  }
}

// One 128 x 128 tile per CTA of 256 threads, a thread holding 8 x 8 elements (rows 8 * (tid / 16) ..,
// columns 8 * (tid % 16) ..).  Row maxima meet in 16 lanes, column maxima in shared memory.  The
// transposed codes go through shared memory so that both outputs are written in 128-byte runs.
// TILE: one scale for the tile, its codes turned as bytes; otherwise one per row (q) and one per column (qt),
// each element rounded twice (86 us at 8192 x 8192 bf16; two passes over the input would read 134 MB more).
template <typename T, int TYPE, bool VEC, bool TILE>
__global__ void __launch_bounds__(256, TILE ? 0 : sizeof(T) == 2 ? 3 : 2)
    quant_fp8_tile_kernel(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx,
                          uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale, int64_t lds,
                          uint8_t* __restrict__ qt, int64_t ldqt, float* __restrict__ scale_t, int64_t ldst) {
  constexpr int PITCH = 136;                               // bytes per transposed row: 8-byte aligned, rows 34 banks apart
  __shared__ __align__(16) uint8_t tr[128 * PITCH];
  __shared__ uint32_t col_top[8][128];
  const int tid = threadIdx.x, cx = tid & 15, ry = tid >> 4, warp = tid >> 5;
  const int tiles_k = (int)((K + 127) / 128);              // the grid holds below 2^31 tiles
  const int64_t mb = blockIdx.x / (unsigned)tiles_k, kb = blockIdx.x % (unsigned)tiles_k;
  const int64_t r0 = mb * 128 + ry * 8, c0 = kb * 128 + cx * 8;
  const int valid_c = (int)min((int64_t)8, max((int64_t)0, K - c0));
  const int valid_r = (int)min((int64_t)8, max((int64_t)0, M - r0));
  f8::Raw<T> r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f8::load8<T, VEC>(x + (r0 + i) * ldx + c0, i < valid_r ? valid_c : 0, r[i]);

  uint32_t row_top[8], ct[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) row_top[i] = f8::top_bits(r[i]);
  // specials anywhere in the tile (rare): every maximum is taken again over the finite elements
  uint32_t any = row_top[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) any = max(any, row_top[i]);
  const bool sp = __syncthreads_or(f8::special<T>(any));
  if (sp) {
#pragma unroll
    for (int i = 0; i < 8; ++i) row_top[i] = f8::finite_top_bits(r[i]);
  }
  if (!TILE) {
    if constexpr (sizeof(T) == 2) {
      uint32_t pair[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {                          // two rows' tops to a word
        pair[i] = row_top[2 * i] | (row_top[2 * i + 1] << 16);
#pragma unroll
        for (int o = 8; o; o >>= 1) pair[i] = f8::max_u16x2(pair[i], __shfl_xor_sync(0xFFFFFFFFu, pair[i], o));
        row_top[2 * i] = pair[i] & 0xFFFFu, row_top[2 * i + 1] = pair[i] >> 16;
      }
      if (qt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {                        // two columns' tops to a word
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t e = sp ? f8::finite_bits(r[i], 2 * j) | (f8::finite_bits(r[i], 2 * j + 1) << 16) : r[i].w[j] & 0x7FFF7FFFu;
            m = f8::max_u16x2(m, e);
          }
          m = f8::max_u16x2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));   // the warp's two row groups
          ct[2 * j] = m & 0xFFFFu, ct[2 * j + 1] = m >> 16;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 8; o; o >>= 1) row_top[i] = max(row_top[i], __shfl_xor_sync(0xFFFFFFFFu, row_top[i], o));
      if (qt) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ct[j] = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) ct[j] = max(ct[j], sp ? f8::finite_bits(r[i], j) : r[i].w[j] & 0x7FFFFFFFu);
          ct[j] = max(ct[j], __shfl_xor_sync(0xFFFFFFFFu, ct[j], 16));
        }
      }
    }
    if (qt && (tid & 16) == 0) {
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        *reinterpret_cast<uint4*>(&col_top[warp][cx * 8 + j]) = make_uint4(ct[j], ct[j + 1], ct[j + 2], ct[j + 3]);
    }
  } else {
    uint32_t top = row_top[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = max(top, row_top[i]);
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((tid & 31) == 0) col_top[warp][0] = top;
  }
  __syncthreads();
  f8::Scale ts{};
  if (TILE) {
    uint32_t top = col_top[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = max(top, col_top[w][0]);
    ts = f8::scale_of<T, TYPE>(f8::bits_to_float<T>(top));
    if (tid == 0) {
      if (q) scale[mb * lds + kb] = ts.s;
      if (qt) scale_t[kb * ldst + mb] = ts.s;
    }
  }
  // encoded twice over in the code, with and without the test for what is not finite
  auto encode = [&](auto specials) {
    constexpr bool SP = decltype(specials)::value;
    uint2 rows8[8];                                          // TILE: the rows' codes, shared by both outputs
    if (q || TILE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const f8::Scale s = TILE ? ts : f8::scale_of<T, TYPE>(f8::bits_to_float<T>(row_top[i]));
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = f8::element(r[i], j);
        rows8[i] = f8::encode8<T, TYPE>(v, s, SP);
        if (q && i < valid_r) {
          f8::store8(q + (r0 + i) * ldq + c0, rows8[i], valid_c);
          if (!TILE && cx == 0) scale[kb * lds + r0 + i] = s.s;
        }
      }
    }
    if (!qt) return;
    if (TILE) {
      // 8 x 8 bytes turned: column j's bytes of rows 0-3 and 4-7
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = g * 4 + u;
          uint32_t c[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = g ? rows8[i].y : rows8[i].x;
          const uint32_t sel = (uint32_t)u | (uint32_t)(u + 4) << 4;   // byte u of each of two words
          const uint32_t lo = __byte_perm(__byte_perm(c[0], c[1], sel), __byte_perm(c[2], c[3], sel), 0x5410);
          const uint32_t hi = __byte_perm(__byte_perm(c[4], c[5], sel), __byte_perm(c[6], c[7], sel), 0x5410);
          *reinterpret_cast<uint2*>(tr + (cx * 8 + j) * PITCH + ry * 8) = make_uint2(lo, hi);
        }
    } else {
      uint32_t top[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) top[j] = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const uint4 t4 = *reinterpret_cast<const uint4*>(&col_top[u][cx * 8 + j]);
          top[j] = max(top[j], t4.x), top[j + 1] = max(top[j + 1], t4.y);
          top[j + 2] = max(top[j + 2], t4.z), top[j + 3] = max(top[j + 3], t4.w);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const f8::Scale s = f8::scale_of<T, TYPE>(f8::bits_to_float<T>(top[j]));
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = f8::element(r[i], j);
        const uint2 w = f8::encode8<T, TYPE>(c, s, SP);
        if (ry == 0 && j < valid_c) scale_t[mb * ldst + c0 + j] = s.s;
        *reinterpret_cast<uint2*>(tr + (cx * 8 + j) * PITCH + ry * 8) = w;
      }
    }
  };
  if (sp) encode(std::true_type{});
  else encode(std::false_type{});
  if (!qt) return;
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
  const int sms = sm_count();
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0;
  const int64_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  if (block == EMU_BLOCK_ROW && !qt) {
    // many rows: 16 per CTA with four loads in flight per thread; few: 4 per CTA, so that more SMs work
    const int64_t tiles_k = (kb + 3) / 4;
    const bool deep = tiles_k * ((M + 15) / 16) >= 2 * sms;
#define EMU_ROWS(V, U)                                                                                             \
  quant_fp8_rows_kernel<T, TYPE, V, U>                                                                             \
      <<<dim3((unsigned)tiles_k, (unsigned)std::min<int64_t>((M + 4 * U - 1) / (4 * U), 65535)), 256, 0, stream>>>( \
          x, M, K, ldx, q, ldq, scale, lds)
    if (vec) {
      if (deep) EMU_ROWS(true, 4);
      else EMU_ROWS(true, 1);
    } else {
      EMU_ROWS(false, 1);
    }
#undef EMU_ROWS
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
