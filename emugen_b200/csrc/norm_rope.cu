// Norms of queries and keys for each head, with the position rotation in the same pass, and the gradients.
//
// For a row x of D elements (one token, one head), weights w and the angles of the token's position:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  z = n w,  y = R z
// where R turns pairs of the first 2 * half elements, (z[i], z[i + half]) or, interleaved, (z[2i], z[2i + 1]), by angle i:
//   y_a = z_a cos_i - z_b sin_i,  y_b = z_b cos_i + z_a sin_i
// Backwards, with dz = R^T dy (the same turn by -sin) and g = dz w:
//   dx = r (g - n mean(g n)),  dw = sum over rows of dz n
// All of it in f32, one rounding at the end.
//
// Bound: reading and writing the rows.  A group of 4 to 32 lanes owns a token, 8 elements a lane, and walks over that
// token's heads, so that the cosines and sines, which are four times a 16-bit row's bytes, are read once for all of them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/emugen.h"
#include "fp8.cuh"
#include "kernels.h"

namespace emu {
namespace {

constexpr int NT = 256;

// The sum over a group of LPG lanes, in every lane of it.
template <int LPG> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPG / 2; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(float v) { return v; }
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// 8 consecutive outputs; rows of the outputs start on 16 bytes (D is a multiple of 8, the outputs are contiguous).
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

// The angles of a lane's 8 elements.  y[e] = z[e] * c[e] + partner[e] * s[e], the sign of the turn being in s.
struct Turn {
  float c[8], s[8];
};
// `back`: R^T.  d: the lane's first element.  A position past the table makes NaN, which shows it.
__device__ __forceinline__ Turn load_turn(const NormRopeArgs& a, int64_t pos, int d, bool back) {
  Turn t;
  const int half = (int)a.half;
  const bool known = pos < a.table_rows;
  const float* cs = a.cos + (known ? pos : 0) * half;
  const float* sn = a.sin + (known ? pos : 0) * half;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = d + e;
    const int i = a.interleaved ? at / 2 : at < half ? at : at - half;
    const bool second = a.interleaved ? at & 1 : at >= half;
    t.c[e] = 1.0f, t.s[e] = 0.0f;
    if (at < 2 * half) {
      t.c[e] = known ? __ldg(cs + i) : __int_as_float(0x7FC00000);
      const float s = known ? __ldg(sn + i) : __int_as_float(0x7FC00000);
      t.s[e] = second != back ? s : -s;
    }
  }
  return t;
}
// z turned.  Where an element has no pair (s = 0, c = 1) it stays as it is, whatever its neighbour holds.
template <int LPG> __device__ __forceinline__ void turn(float (&z)[8], const Turn& t, const NormRopeArgs& a, int d) {
  float p[8];
  if (a.interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = z[e ^ 1];
  } else {
    // half is a multiple of 8: a lane's partners are all in one lane of its group
    const int step = (int)a.half / 8, lane = threadIdx.x & 31;
    const int src = d < a.half ? lane + step : d < 2 * a.half ? lane - step : lane;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __shfl_sync(0xFFFFFFFFu, z[e], src & 31);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d + e < 2 * a.half) z[e] = __fmaf_rn(z[e], t.c[e], __fmul_rn(p[e], t.s[e]));
}

// One unit of work: a token and up to `heads_per_unit` heads of q or of k.
struct Unit {
  int64_t token;
  int which, head0, heads;
};
__device__ __forceinline__ Unit unit_of(const NormRopeArgs& a, int64_t u) {
  Unit r;
  const int64_t per_token = a.chunks[0] + a.chunks[1];
  r.token = u / per_token;
  int c = (int)(u - r.token * per_token);
  r.which = c >= a.chunks[0];
  if (r.which) c -= a.chunks[0];
  r.head0 = c * a.heads_per_unit;
  r.heads = min(a.heads_per_unit, (int)a.heads[r.which] - r.head0);
  return r;
}

// Rows of one unit are loaded U at a time.
template <typename T, bool VEC, int LPG, bool BACK>
__global__ void __launch_bounds__(NT) norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int GROUPS = NT / LPG, U = sizeof(T) == 4 || BACK ? 2 : 4;
  const int gl = threadIdx.x % LPG, group = threadIdx.x / LPG, d = gl * 8;
  const int D = (int)a.D;
  const bool mine = d < D;
  const int64_t units = a.T * (a.chunks[0] + a.chunks[1]);
  const float inv_d = 1.0f / (float)D;
  float dw[2][8] = {};
  // every lane of a warp walks the same number of rounds, for the shuffles
  const int64_t rounds = (units + (int64_t)gridDim.x * GROUPS - 1) / ((int64_t)gridDim.x * GROUPS);
  for (int64_t round = 0; round < rounds; ++round) {
    const int64_t u = (round * gridDim.x + blockIdx.x) * GROUPS + group;
    Unit w{0, 0, 0, 0};
    int64_t pos = -1;
    if (u < units) {
      w = unit_of(a, u);
      pos = a.positions[w.token];
    }
    const bool pad = pos < 0;                                 // a row of padding: zeros
    const Turn t = load_turn(a, pad ? 0 : pos, d, false);
    float wt[8];
    {
      const T* wp = static_cast<const T*>(a.weight[w.which]);
#pragma unroll
      for (int e = 0; e < 8; ++e) wt[e] = wp && mine ? widen<T>(wp[d + e]) : 1.0f;
    }
    const T* x = static_cast<const T*>(a.x[w.which]) + w.token * a.token_stride[w.which] + d;
    const int64_t hs = a.head_stride[w.which];
    const int64_t out0 = (w.token * a.heads[w.which] + w.head0) * D + d;
    T* y = static_cast<T*>(a.y[w.which]) + out0;
    const T* dy = BACK ? static_cast<const T*>(a.dy[w.which]) + w.token * a.dy_token_stride[w.which] + d : nullptr;
    const int64_t dhs = BACK ? a.dy_head_stride[w.which] : 0;
    const int most = __reduce_max_sync(0xFFFFFFFFu, w.heads);
    for (int h0 = 0; h0 < most; h0 += U) {
      f8::Raw<T> r[U], g[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int n = mine && !pad && h0 + i < w.heads ? 8 : 0;
        f8::load8<T, VEC>(x + (w.head0 + h0 + i) * hs, n, r[i]);
        if (BACK) f8::load8<T, VEC>(dy + (w.head0 + h0 + i) * dhs, n, g[i]);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float v[8], ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = f8::element(r[i], e);
          ss = __fmaf_rn(v[e], v[e], ss);
        }
        const float inv = 1.0f / sqrtf(__fmaf_rn(group_sum<LPG>(ss), inv_d, a.eps));
        const bool write = mine && h0 + i < w.heads;
        if (!BACK) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = pad ? 0.0f : __fmul_rn(__fmul_rn(v[e], inv), wt[e]);
          turn<LPG>(v, t, a, d);
        } else {
          float z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = f8::element(g[i], e);
          Turn b = t;
#pragma unroll
          for (int e = 0; e < 8; ++e) b.s[e] = -t.s[e];
          turn<LPG>(z, b, a, d);
          float gx = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = __fmul_rn(v[e], inv);                       // n
            const float zn = write && !pad ? __fmul_rn(z[e], v[e]) : 0.0f;
            dw[0][e] = __fadd_rn(dw[0][e], w.which ? 0.0f : zn);
            dw[1][e] = __fadd_rn(dw[1][e], w.which ? zn : 0.0f);
            z[e] = __fmul_rn(z[e], wt[e]);                     // g
            gx = __fmaf_rn(z[e], v[e], gx);
          }
          const float mean = __fmul_rn(group_sum<LPG>(gx), inv_d);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = pad ? 0.0f : __fmul_rn(inv, __fmaf_rn(-v[e], mean, z[e]));
        }
        if (write) store8(y + (int64_t)(h0 + i) * D, v);
      }
    }
  }
  if constexpr (BACK) {
    // this CTA's share of the weights' gradients, its groups added up in their order
    __shared__ float part[GROUPS][LPG * 8 + 4];
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) part[group][d + e] = dw[which][e];
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += NT) {
        float s = 0.0f;
        for (int g = 0; g < GROUPS; ++g) s = __fadd_rn(s, part[g][c]);
        a.partial[((int64_t)blockIdx.x * 2 + which) * D + c] = s;
      }
    }
  }
}

// The weights' gradients from the CTAs' shares [ctas][2][D], added up in one order whatever ran first: 32 columns a CTA, 32
// rows of threads.
template <typename T> __global__ void __launch_bounds__(1024) norm_rope_weights_kernel(const float* partial, int ctas, int D, T* dwq, T* dwk) {
  __shared__ float s[32][33];
  const int which = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  T* out = which ? dwk : dwq;
  if (!out) return;
  float v = 0.0f;
  if (c < D)
    for (int i = threadIdx.y; i < ctas; i += 32) v = __fadd_rn(v, partial[((int64_t)i * 2 + which) * D + c]);
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < D) {
    if constexpr (std::is_same<T, float>::value) out[col] = v;
    else if constexpr (std::is_same<T, __half>::value) out[col] = __float2half_rn(v);
    else out[col] = __float2bfloat16_rn(v);
  }
}

int lanes_of(int64_t D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Heads of a unit and CTAs of the grid.  While the machine is not full, fewer heads to a unit.
void shape(NormRopeArgs& a, int64_t& grid, bool back, int sms) {
  const int groups = NT / lanes_of(a.D);
  a.heads_per_unit = 16;
  auto chunks = [&] {
    for (int w = 0; w < 2; ++w) a.chunks[w] = (int)((a.heads[w] + a.heads_per_unit - 1) / a.heads_per_unit);
    return a.T * (a.chunks[0] + a.chunks[1]);
  };
  while (a.heads_per_unit > 1 && chunks() < (int64_t)sms * 4 * groups) a.heads_per_unit /= 2;
  grid = (chunks() + groups - 1) / groups;
  if (back) grid = std::min<int64_t>(grid, (int64_t)sms * NORM_ROPE_CTAS);
  else grid = std::min<int64_t>(grid, 1 << 30);
}

}  // namespace

size_t norm_rope_workspace(int64_t D) { return (size_t)sm_count() * NORM_ROPE_CTAS * 2 * D * sizeof(float); }

cudaError_t launch_norm_rope(NormRopeArgs a, bool back, cudaStream_t stream) {
  int64_t grid;
  shape(a, grid, back, sm_count());
  const int esz = a.dtype == EMU_DTYPE_F32 ? 4 : 2;
  bool vec = true;
  for (int w = 0; w < 2; ++w) {
    vec = vec && ((reinterpret_cast<uintptr_t>(a.x[w]) | (uintptr_t)(a.token_stride[w] * esz) | (uintptr_t)(a.head_stride[w] * esz)) & 15) == 0;
    if (back) vec = vec && ((reinterpret_cast<uintptr_t>(a.dy[w]) | (uintptr_t)(a.dy_token_stride[w] * esz) | (uintptr_t)(a.dy_head_stride[w] * esz)) & 15) == 0;
  }
  const int lpg = lanes_of(a.D);
#define EMU_NR(T, V, L)                                                                    \
  (back ? norm_rope_kernel<T, V, L, true><<<(unsigned)grid, NT, 0, stream>>>(a)            \
        : norm_rope_kernel<T, V, L, false><<<(unsigned)grid, NT, 0, stream>>>(a))
#define EMU_NRL(T, V) (lpg == 4 ? EMU_NR(T, V, 4) : lpg == 8 ? EMU_NR(T, V, 8) : lpg == 16 ? EMU_NR(T, V, 16) : EMU_NR(T, V, 32))
#define EMU_NRT(T)                                                                                                      \
  do {                                                                                                                  \
    vec ? EMU_NRL(T, true) : EMU_NRL(T, false);                                                                         \
    if (back && (a.dw[0] || a.dw[1]))                                                                                   \
      norm_rope_weights_kernel<T><<<dim3((unsigned)((a.D + 31) / 32), 2), dim3(32, 32), 0, stream>>>(                    \
          a.partial, (int)grid, (int)a.D, static_cast<T*>(a.dw[0]), static_cast<T*>(a.dw[1]));                          \
  } while (0)
  if (a.dtype == EMU_DTYPE_F32) EMU_NRT(float);
  else if (a.dtype == EMU_DTYPE_F16) EMU_NRT(__half);
  else EMU_NRT(__nv_bfloat16);
#undef EMU_NRT
#undef EMU_NRL
#undef EMU_NR
  return cudaGetLastError();
}

}  // namespace emu
