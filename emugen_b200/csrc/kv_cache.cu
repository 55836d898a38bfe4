// Quantised key/value cache: rows (token, head) of D elements written to their slots in 8 or 4 bits, and
// the rows of a batch of sequences read back through a block table.
//
//   EMU_KV_FP8    E4M3 codes, one f32 scale per 128 elements of a row (the quantiser of quant_fp8.cu)
//   EMU_KV_MXFP4  e2m1 codes, one power-of-two scale byte per 32 elements (the quantiser of quant.cu)
//
// Measured on B200 with 8 heads of 128 (bf16): reading 131072 rows back 135 us from fp8 (814 MB: 92% of the
// measured copy rate) and 118 us from MXFP4 (679 MB: 88%); writing 65536 tokens 95 us (407 MB: floor 62), where
// the quantiser's arithmetic bounds it; 32 tokens 3.6 us, where a launch is about 1.7: the rest is find_overwritten.
#include <cuda_fp4.h>
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

constexpr int MAX_TOKENS = 1024;      // tokens per CTA of the write kernel
constexpr int BUCKETS = 4096;

// A slot's bucket: the top bits of its product with 2^64 / golden ratio (Knuth), which spreads consecutive
// slots and those a power of two apart alike.
__device__ __forceinline__ int bucket_of(int64_t slot) { return (int)(((uint64_t)slot * 0x9E3779B97F4A7C15ull) >> 52); }

// A CTA's slots, hashed: chains of its tokens by bucket.
struct Slots {
  int64_t own[MAX_TOKENS];
  int16_t next[MAX_TOKENS];
  int head[BUCKETS];                  // 1 + the chain's first token, 0: none
  uint8_t dead[MAX_TOKENS];
};

// dead[i] for each of this CTA's tokens i0 + i: a later token of the call has the same slot, so that token's
// row is the one that is kept (two rows written at once would leave a mixture).  The CTA's own tokens are settled first,
// which leaves each slot in its chain once, and then every token behind them is looked up.  That is T / 2 reads of L2 per
// CTA, so a long call takes many tokens per CTA (launch_kv_write): 65536 tokens over 1024 CTAs spent 0.8 ms here.
// Padding on either side of the cache stays out of the chains (all of it in one made 131072 such tokens 9.9 ms).
__device__ __forceinline__ void find_overwritten(const int64_t* __restrict__ slots, int64_t T, int64_t num_slots, int64_t i0,
                                                 int n, Slots& s) {
  auto link = [&] {                                          // chains of the tokens that still write
    for (int i = threadIdx.x; i < BUCKETS; i += blockDim.x) s.head[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      if (s.own[i] >= 0 && !s.dead[i]) s.next[i] = (int16_t)(atomicExch(&s.head[bucket_of(s.own[i])], i + 1) - 1);
    __syncthreads();
  };
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int64_t slot = slots[i0 + i];
    s.own[i] = slot < num_slots ? slot : -1;                 // from here on a slot below 0 is one that nothing is written to
    s.dead[i] = 0;
  }
  link();                                                    // (a thread reads what it wrote itself up to the second barrier)
  if (n > 1) {
    bool any = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int64_t slot = s.own[i];
      if (slot < 0) continue;
      for (int c = s.head[bucket_of(slot)] - 1; c >= 0; c = s.next[c])
        if (c > i && s.own[c] == slot) {
          s.dead[i] = 1, any = true;
          break;
        }
    }
    if (__syncthreads_or(any)) link();
  }
  auto look_up = [&](int64_t slot) {
    if (slot < 0 || slot >= num_slots) return;
    for (int i = s.head[bucket_of(slot)] - 1; i >= 0; i = s.next[i])
      if (s.own[i] == slot) s.dead[i] = 1;
  };
  int64_t j = i0 + n + threadIdx.x;
  for (; j + 7 * (int64_t)blockDim.x < T; j += 8 * (int64_t)blockDim.x) {
    int64_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = __ldg(slots + j + u * (int64_t)blockDim.x);
#pragma unroll
    for (int u = 0; u < 8; ++u) look_up(v[u]);
  }
  for (; j < T; j += blockDim.x) look_up(slots[j]);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (s.dead[i]) s.own[i] = -1;
  __syncthreads();
}

// LPG lanes take up to 128 elements of a (token, head) row, 8 each (16 lanes; 8 or 4 where a head has at most
// 64 or 32 elements).  A lane group keeps its tensor, head and place for all of the CTA's tokens, so the
// divisions that find them are made once, and U tokens' loads are in flight together.
template <typename T, int FORMAT, bool VEC, int LPG, int NT>
__global__ void __launch_bounds__(NT) kv_write_kernel(const __grid_constant__ KvWriteArgs a, int tokens_per_cta) {
  constexpr int U = 4, GROUPS = NT / LPG;
  __shared__ Slots sl;
  const int64_t i0 = (int64_t)blockIdx.x * tokens_per_cta;
  const int n = (int)min((int64_t)tokens_per_cta, a.T - i0);
  find_overwritten(a.slots, a.T, a.num_slots, i0, n, sl);
  const int gl = threadIdx.x % LPG, group = threadIdx.x / LPG;
  const int D = (int)a.D, H = (int)a.H, G = (D + 127) / 128;
  const int64_t per_tensor = (int64_t)H * G, per_token = per_tensor * (a.x[1] ? 2 : 1);
  // few groups per token: the CTA's lane groups share out the tokens too
  const int side = per_token >= GROUPS ? 1 : GROUPS / (int)per_token;
  const int first = side == 1 ? 0 : group / (int)per_token;
  for (int64_t c = side == 1 ? group : group % (int)per_token; c < (per_token + GROUPS - 1) / GROUPS * GROUPS; c += GROUPS) {
    const bool have = c < per_token && first < side;         // whole warps stay for the shuffles
    const int which = c >= per_tensor;
    const int hg = (int)(which ? c - per_tensor : c);
    const int h = hg / G, g = hg - h * G, d = g * 128 + gl * 8;
    const int64_t stride = which ? a.token_stride[1] : a.token_stride[0];
    const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + h * (which ? a.head_stride[1] : a.head_stride[0]) + d +
                 (i0 + first) * stride;
    // (the count of rounds is the same for every lane group of a warp, whatever its `first`)
    const bool mine = have && d < D;                         // D is a multiple of 16
    // code and scale places of this lane in slot 0, and from slot to slot
    const int q_row = FORMAT == EMU_KV_FP8 ? H * D : H * (D / 2), s_row = FORMAT == EMU_KV_FP8 ? H * G : H * (D / 32);
    uint8_t* q = (which ? a.q[1] : a.q[0]) + (FORMAT == EMU_KV_FP8 ? h * D + d : (h * D + d) / 2);
    void* sc = which ? a.scale[1] : a.scale[0];
    const int s_at = FORMAT == EMU_KV_FP8 ? hg : (h * D + d) / 32;
    for (int t0 = 0; t0 < n; t0 += side * U, x += (int64_t)side * U * stride) {
      f8::Raw<T> r[U];
      int64_t slot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = t0 + first + u * side;
        slot[u] = have && i < n ? sl.own[i] : -1;
        f8::load8<T, VEC>(x + u * side * stride, mine && slot[u] >= 0 ? 8 : 0, r[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f8::element(r[u], e);
        if (FORMAT == EMU_KV_FP8) {
          uint32_t top = f8::top_bits(r[u]);
#pragma unroll
          for (int o = LPG / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
          const bool sp = __any_sync(0xFFFFFFFFu, f8::special<T>(top));
          if (sp) {
            top = f8::finite_top_bits(r[u]);
#pragma unroll
            for (int o = LPG / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
          }
          const f8::Scale s = f8::scale_of<T, EMU_FP8_E4M3>(f8::bits_to_float<T>(top));
          const uint2 w = f8::encode8<T, EMU_FP8_E4M3>(v, s, sp);
          if (slot[u] < 0) continue;
          if (mine) *reinterpret_cast<uint2*>(q + slot[u] * q_row) = w;
          if (gl == 0) static_cast<float*>(sc)[slot[u] * s_row + s_at] = s.s;
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
          for (int e = 0; e < 8; ++e) y[e] = __fmul_rn(std::is_same<T, __half>::value ? v[e] : ftz(v[e]), out_scale);
          if (slot[u] < 0 || !mine) continue;
          *reinterpret_cast<uint32_t*>(q + slot[u] * q_row) = f32x8_to_e2m1(y);
          if ((gl & 3) == 0) static_cast<uint8_t*>(sc)[slot[u] * s_row + s_at] = sf;
        }
      }
    }
  }
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int READ_ROWS = 32;         // most output rows per CTA of the read kernel

// A thread gives 8 consecutive elements (one 16-byte store of a 16-bit type, so that a warp writes whole
// lines) and keeps its tensor, head and place for all of the CTA's rows; U rows' loads are in flight together.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadArgs a, int rows_per_cta) {
  constexpr int U = 4;
  __shared__ int64_t slot_of[READ_ROWS];     // -1: a row of zeros (no such page), -2: left as it was
  const int64_t r0 = (int64_t)blockIdx.x * rows_per_cta;
  const int rows = (int)min((int64_t)rows_per_cta, a.total - r0);
  if (threadIdx.x < rows) {
    const int64_t r = r0 + threadIdx.x;
    // the sequence that ends behind r first
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
      slot = page >= 0 && page < a.num_pages ? page * a.page_size + (pos - pg * a.page_size) : -1;
    }
    slot_of[threadIdx.x] = slot;
  }
  __syncthreads();
  const int D = (int)a.D, H = (int)a.H, G = (D + 127) / 128;
  const int64_t per_tensor = (int64_t)H * (D / 8), per_row = per_tensor * (a.out[1] ? 2 : 1);
  // short rows: the CTA's threads share out the rows too
  const int side = per_row >= 256 ? 1 : 256 / (int)per_row;
  const int first = side == 1 ? 0 : threadIdx.x / (int)per_row;
  if (first >= side) return;
  for (int64_t c = side == 1 ? threadIdx.x : threadIdx.x % (int)per_row; c < per_row; c += 256) {
    const int which = c >= per_tensor;
    const int hd = (int)(which ? c - per_tensor : c) * 8;
    const int h = hd / D, d = hd - h * D;
    const int64_t stride = which ? a.token_stride[1] : a.token_stride[0];
    T* out = static_cast<T*>(which ? a.out[1] : a.out[0]) + hd + (r0 + first) * stride;
    const int q_row = FORMAT == EMU_KV_FP8 ? H * D : H * (D / 2), s_row = FORMAT == EMU_KV_FP8 ? H * G : H * (D / 32);
    const uint8_t* q = (which ? a.q[1] : a.q[0]) + (FORMAT == EMU_KV_FP8 ? hd : hd / 2);
    const void* sc = which ? a.scale[1] : a.scale[0];
    const int s_at = FORMAT == EMU_KV_FP8 ? h * G + d / 128 : hd / 32;
    for (int i0 = first; i0 < rows; i0 += side * U, out += (int64_t)side * U * stride) {
      uint2 w[U];
      float s[U];
      int64_t slot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        slot[u] = i0 + u * side < rows ? slot_of[i0 + u * side] : -2;
        w[u] = make_uint2(0, 0);                             // a row of zeros
        s[u] = 0.0f;
        if (slot[u] < 0) continue;
        if (FORMAT == EMU_KV_FP8) {
          w[u] = __ldg(reinterpret_cast<const uint2*>(q + slot[u] * q_row));
          s[u] = __ldg(static_cast<const float*>(sc) + (slot[u] * s_row + s_at));
        } else {
          w[u].x = __ldg(reinterpret_cast<const uint32_t*>(q + slot[u] * q_row));
          // 2^(byte - 127): the exponent field, but for byte 0, which is f32's subnormal 2^-127; byte 255 gives infinity
          const uint32_t e = __ldg(static_cast<const uint8_t*>(sc) + (slot[u] * s_row + s_at));
          s[u] = __uint_as_float(e ? e << 23 : 0x00400000u);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (slot[u] == -2) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          __half2_raw hr;
          if (FORMAT == EMU_KV_FP8) {
            hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((e < 4 ? w[u].x : w[u].y) >> (8 * (e & 3))), __NV_E4M3);
          } else {
            hr = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(w[u].x >> (4 * e)), __NV_E2M1);
          }
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
          v[e] = __fmul_rn(f.x, s[u]);
          v[e + 1] = __fmul_rn(f.y, s[u]);
        }
        // fp8: the product (4 + 24 bits) is rounded to f32 and then to T, so a value just beside a tie of T may go the
        // other way than in one rounding; half a step of T and of f32 bound the error.  MXFP4 products are exact.
        T* dst = out + u * side * stride;
        __align__(16) T y[8];
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
  }
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t stream) {
  const int sms = sm_count();
  // A token to a CTA of 256 threads while four CTAs per SM take them all; longer calls one CTA of 1024 threads
  // per SM, so that fewer CTAs read all later slots (8 heads of 128, fp8: 256 tokens 4.2 against 4.9 us,
  // 2048 tokens 9.0 against 6.9, 65536 tokens 136 against 95)
  const bool wide = a.T > 4 * (int64_t)sms;
  const int64_t ctas = wide ? sms : a.T;
  const int per_cta = (int)std::min<int64_t>(MAX_TOKENS, (a.T + ctas - 1) / ctas);
  const unsigned grid = (unsigned)((a.T + per_cta - 1) / per_cta);
  bool vec = true;
  for (int w = 0; w < 2; ++w)
    if (a.x[w]) vec = vec && ((reinterpret_cast<uintptr_t>(a.x[w]) | (uintptr_t)(a.token_stride[w] * 2) | (uintptr_t)(a.head_stride[w] * 2)) & 15) == 0;
#define EMU_KVN(T, F, V, L)                                                      \
  (wide ? kv_write_kernel<T, F, V, L, 1024><<<grid, 1024, 0, stream>>>(a, per_cta) \
        : kv_write_kernel<T, F, V, L, 256><<<grid, 256, 0, stream>>>(a, per_cta))
#define EMU_KVL(T, F, L) (vec ? EMU_KVN(T, F, true, L) : EMU_KVN(T, F, false, L))
#define EMU_KV(T, F) (a.D <= 32 ? EMU_KVL(T, F, 4) : a.D <= 64 ? EMU_KVL(T, F, 8) : EMU_KVL(T, F, 16))
  if (a.format == EMU_KV_FP8) {
    if (a.dtype == EMU_DTYPE_F16) EMU_KV(__half, EMU_KV_FP8);
    else EMU_KV(__nv_bfloat16, EMU_KV_FP8);
  } else {
    if (a.dtype == EMU_DTYPE_F16) EMU_KV(__half, EMU_KV_MXFP4);
    else EMU_KV(__nv_bfloat16, EMU_KV_MXFP4);
  }
#undef EMU_KV
#undef EMU_KVL
#undef EMU_KVN
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream) {
  const int sms = sm_count();
  // up to 32 rows per CTA, fewer while there are not 16 CTAs for each SM, which holds four at a time (56 to 61 registers
  // for 16-bit outputs)
  const int per_cta = (int)std::min<int64_t>(READ_ROWS, (a.total + 16 * sms - 1) / (16 * sms));
  const unsigned grid = (unsigned)((a.total + per_cta - 1) / per_cta);
  const int esz = a.out_dtype == EMU_DTYPE_F32 ? 4 : 2;
  bool vec = true;
  for (int w = 0; w < 2; ++w)
    if (a.out[w]) vec = vec && ((reinterpret_cast<uintptr_t>(a.out[w]) | (uintptr_t)(a.token_stride[w] * esz)) & 15) == 0;
#define EMU_KV(T, F) (vec ? kv_read_kernel<T, F, true><<<grid, 256, 0, stream>>>(a, per_cta) : kv_read_kernel<T, F, false><<<grid, 256, 0, stream>>>(a, per_cta))
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
