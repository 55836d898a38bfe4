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
// Bound: reading and writing the rows.  A group of 2 to 16 lanes owns a token and walks over that token's heads, so that the
// cosines and sines are read once for all of them.  A lane has two runs of 8 elements, which hold both elements of its 8
// pairs (i .. i + 7 and i + half .. i + half + 7; interleaved, 16 neighbours): the turn needs no exchange between lanes, and
// what is done once for a row (sum, root, addresses) is spread over 16 elements.
// Measured: 16384 tokens of 32 + 8 heads of 128, bf16: 68 us (344 MB, 5.0 TB/s, 76% of a copy's rate; a group's units are whole, so that
// the longest path has 80 rows where an even share is 69).  8191 tokens of 24 + 6 heads of 96, fp16, interleaved: 30 us, gradients
// 53 + 4 (36 rows for 26, and 2 of 8 lanes have no elements at this head size).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/emugen.h"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace emu {
namespace {

constexpr int NT = 256;

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs of f32, two to an instruction.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) { return {ptx::join2(__float_as_uint(a), __float_as_uint(b))}; }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { return {ptx::mul2(a.v, b.v)}; }
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) { return {ptx::fma2(a.v, b.v, c.v)}; }
__device__ __forceinline__ F2 neg(F2 a) { return {a.v ^ 0x8000000080000000ull}; }
__device__ __forceinline__ float lo(F2 a) { return ptx::lo2(a.v); }
__device__ __forceinline__ float hi(F2 a) { return ptx::hi2(a.v); }
__device__ __forceinline__ float sum(F2 a) { return __fadd_rn(lo(a), hi(a)); }

// A lane's 16 elements as they were read: two runs of 8.
template <typename T> struct Raw {
  static constexpr int WORDS = 2 * sizeof(T);                // of a run
  uint32_t w[2][WORDS];
};
// vec: runs start on 16 bytes.  `runs`: how many of them there are (the others zeros).
template <typename T> __device__ __forceinline__ Raw<T> load(const T* p, int c0, int c1, int runs, bool vec) {
  Raw<T> r;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < Raw<T>::WORDS; ++i) r.w[k][i] = 0;
    if (k >= runs) continue;
    const T* q = p + (k ? c1 : c0);
    if (vec) {
#pragma unroll
      for (int i = 0; i < Raw<T>::WORDS; i += 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(q) + i / 4);
        r.w[k][i] = v.x, r.w[k][i + 1] = v.y, r.w[k][i + 2] = v.z, r.w[k][i + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.w[k][i] = __float_as_uint(q[i]);
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(q);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[k][i] = (uint32_t)u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
    }
  }
  return r;
}
template <typename T> __device__ __forceinline__ float element(const Raw<T>& r, int i);
template <> __device__ __forceinline__ float element(const Raw<float>& r, int i) { return __uint_as_float(r.w[i / 8][i % 8]); }
template <> __device__ __forceinline__ float element(const Raw<__nv_bfloat16>& r, int i) {
  const uint32_t w = r.w[i / 8][i % 8 / 2];
  return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
}
template <> __device__ __forceinline__ float element(const Raw<__half>& r, int i) {
  const uint32_t w = r.w[i / 8][i % 8 / 2];
  return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w)));
}
// The first and the second elements of the lane's pairs 2 j and 2 j + 1.
template <typename T, bool INTER> __device__ __forceinline__ F2 firsts(const Raw<T>& r, int j) {
  return INTER ? f2(element(r, 4 * j), element(r, 4 * j + 2)) : f2(element(r, 2 * j), element(r, 2 * j + 1));
}
template <typename T, bool INTER> __device__ __forceinline__ F2 seconds(const Raw<T>& r, int j) {
  return INTER ? f2(element(r, 4 * j + 1), element(r, 4 * j + 3)) : f2(element(r, 8 + 2 * j), element(r, 9 + 2 * j));
}
// Back to two runs (which start on 16 bytes in the outputs).
template <typename T, bool INTER> __device__ __forceinline__ void store(T* p, int c0, int c1, int runs, const F2 (&a)[4], const F2 (&b)[4]) {
  float v[16];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (INTER) v[4 * j] = lo(a[j]), v[4 * j + 1] = lo(b[j]), v[4 * j + 2] = hi(a[j]), v[4 * j + 3] = hi(b[j]);
    else v[2 * j] = lo(a[j]), v[2 * j + 1] = hi(a[j]), v[8 + 2 * j] = lo(b[j]), v[9 + 2 * j] = hi(b[j]);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k >= runs) continue;
    T* q = p + (k ? c1 : c0);
    const float* x = v + 8 * k;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(q)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(q)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(q) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
  }
}

// The sum over a group of LPG lanes, in every lane of it.
template <int LPG> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPG / 2; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
// 1 / sqrt(v): the quick one and a Newton step (0, subnormal numbers and infinity: the quick one).
__device__ __forceinline__ float root(float v) {
  const float y = rsqrtf(v);
  const float z = __fmaf_rn(__fmul_rn(0.5f, __fmaf_rn(-__fmul_rn(v, y), y, 1.0f)), y, y);
  return v > 0x1p-126f && v < INFINITY ? z : y;
}

// Angles of the lane's 8 pairs; elements that are not turned have cos 1 and sin 0.
struct Turn {
  F2 c[4], s[4];
};
// i: the lane's first pair, `turned` of them (8, or fewer at an interleaved end).  A position past the table makes NaN, which shows it.
__device__ __forceinline__ Turn load_turn(const NormRopeArgs& a, int64_t pos, int i, int turned, bool vec) {
  Turn t;
#pragma unroll
  for (int j = 0; j < 4; ++j) t.c[j] = f2(1.0f, 1.0f), t.s[j] = f2(0.0f, 0.0f);
  if (turned <= 0) return t;
  const bool known = pos < a.table_rows;
  const float* cs = a.cos + (known ? pos * a.half + i : 0);
  const float* sn = a.sin + (known ? pos * a.half + i : 0);
  if (vec && turned == 8 && known) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(cs) + j / 2), y = __ldg(reinterpret_cast<const float4*>(sn) + j / 2);
      t.c[j] = f2(x.x, x.y), t.c[j + 1] = f2(x.z, x.w), t.s[j] = f2(y.x, y.y), t.s[j + 1] = f2(y.z, y.w);
    }
    return t;
  }
  const float nan = __int_as_float(0x7FC00000);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c[2] = {1.0f, 1.0f}, s[2] = {};
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (2 * j + e < turned) c[e] = known ? __ldg(cs + 2 * j + e) : nan, s[e] = known ? __ldg(sn + 2 * j + e) : nan;
    t.c[j] = f2(c[0], c[1]), t.s[j] = f2(s[0], s[1]);
  }
  return t;
}
template <bool BACK> __device__ __forceinline__ void turn(F2 (&a)[4], F2 (&b)[4], const Turn& t, bool turned) {
  if (!turned) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const F2 bs = b[j] * t.s[j], as = a[j] * t.s[j];
    a[j] = fma(a[j], t.c[j], BACK ? bs : neg(bs));
    b[j] = fma(b[j], t.c[j], BACK ? neg(as) : as);
  }
}

// A CTA works on q (the first `a.split` CTAs) or on k, by units of a token and up to heads_per_unit of its heads; rows of a unit
// are loaded U at a time, those of the next time while the ones of this time are worked on.
template <typename T, int LPG, bool INTER, bool BACK>
__global__ void __launch_bounds__(NT, 2) norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int GROUPS = NT / LPG, U = sizeof(T) == 4 || BACK ? 1 : 2;
  const int which = (int)blockIdx.x >= a.split, cta = which ? blockIdx.x - a.split : blockIdx.x, ctas = which ? gridDim.x - a.split : a.split;
  const int gl = threadIdx.x % LPG, group = threadIdx.x / LPG;
  const int D = (int)a.D, half = (int)a.half, heads = (int)(which ? a.heads[1] : a.heads[0]), per = which ? a.heads_per_unit[1] : a.heads_per_unit[0];
  const int chunks = (heads + per - 1) / per;
  const bool vec = a.vec;
  // the lane's runs (`runs` of them exist), its first pair and how many of its 8 pairs are turned
  int c0 = gl * 16, c1 = c0 + 8, turned = max(0, min(8, half - gl * 8));
  const int pair = gl * 8;
  if (!INTER) {
    if (pair < half) c0 = pair, c1 = half + pair;
    else c0 = 2 * half + (pair - half) * 2, c1 = c0 + 8;
  }
  const int runs = c0 >= D ? 0 : c1 >= D ? 1 : 2;
  if (!runs) turned = 0;
  const int64_t units = a.T * chunks;
  const float inv_d = 1.0f / (float)D;
  const T* weight = static_cast<const T*>(which ? a.weight[1] : a.weight[0]);
  const Raw<T> wt = load<T>(weight, c0, c1, weight ? runs : 0, vec);
  const int64_t ts = which ? a.token_stride[1] : a.token_stride[0], hs = which ? a.head_stride[1] : a.head_stride[0];
  const int64_t dts = BACK ? (which ? a.dy_token_stride[1] : a.dy_token_stride[0]) : 0, dhs = BACK ? (which ? a.dy_head_stride[1] : a.dy_head_stride[0]) : 0;
  const F2 zero = f2(0.0f, 0.0f);
  F2 dw[BACK ? 8 : 1];
#pragma unroll
  for (int j = 0; j < (BACK ? 8 : 1); ++j) dw[j] = zero;
  // every lane of a warp walks the same number of rounds, for the shuffles
  const int64_t rounds = (units + (int64_t)ctas * GROUPS - 1) / ((int64_t)ctas * GROUPS);
  for (int64_t round = 0; round < rounds; ++round) {
    const int64_t u = (round * ctas + cta) * GROUPS + group;
    int64_t token = 0, pos = -1;
    int head0 = 0, n = 0;
    if (u < units) {
      token = u <= 0xFFFFFFFF ? (int64_t)((uint32_t)u / (uint32_t)chunks) : u / chunks;
      head0 = (int)(u - token * chunks) * per;
      n = min(per, heads - head0);
      pos = a.positions[token];
    }
    const bool pad = pos < 0;                                 // a row of padding: zeros
    const Turn t = load_turn(a, pos, pair, pad ? 0 : turned, a.vec_table);
    const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + token * ts + head0 * hs;
    T* y = static_cast<T*>(which ? a.y[1] : a.y[0]) + (token * heads + head0) * D;
    const T* dy = BACK ? static_cast<const T*>(which ? a.dy[1] : a.dy[0]) + token * dts + head0 * dhs : nullptr;
    const int reads = pad ? 0 : runs, most = min(per, heads);
    Raw<T> next[U], gnext[U];
    auto fetch = [&](int h0) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int any = h0 + i < n ? reads : 0;
        next[i] = load<T>(x, c0, c1, any, vec);
        x += hs;
        if (BACK) gnext[i] = load<T>(dy, c0, c1, any, vec), dy += dhs;
      }
    };
    fetch(0);
    for (int h0 = 0; h0 < most; h0 += U) {
      Raw<T> r[U], gr[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        r[i] = next[i];
        if (BACK) gr[i] = gnext[i];
      }
      if (h0 + U < most) fetch(h0 + U);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        F2 p[4], q[4], ss = zero;                             // first and second elements of the pairs
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[j] = firsts<T, INTER>(r[i], j), q[j] = seconds<T, INTER>(r[i], j);
          ss = fma(q[j], q[j], fma(p[j], p[j], ss));
        }
        // rows that are not there or padding add nothing to the weights' gradients, whatever eps is
        const float scale = root(__fmaf_rn(group_sum<LPG>(sum(ss)), inv_d, a.eps)), inv = pad || h0 + i >= n ? 0.0f : scale;
        const F2 inv2 = f2(inv, inv);
        const int writes = h0 + i < n ? runs : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = p[j] * inv2, q[j] = q[j] * inv2;       // n
        if (!BACK) {
          if (weight)
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = p[j] * firsts<T, INTER>(wt, j), q[j] = q[j] * seconds<T, INTER>(wt, j);
          turn<false>(p, q, t, turned > 0);
        } else {
          F2 gp[4], gq[4], gn = zero;
#pragma unroll
          for (int j = 0; j < 4; ++j) gp[j] = firsts<T, INTER>(gr[i], j), gq[j] = seconds<T, INTER>(gr[i], j);
          turn<true>(gp, gq, t, turned > 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            dw[BACK ? j : 0] = fma(gp[j], p[j], dw[BACK ? j : 0]), dw[BACK ? 4 + j : 0] = fma(gq[j], q[j], dw[BACK ? 4 + j : 0]);
            if (weight) gp[j] = gp[j] * firsts<T, INTER>(wt, j), gq[j] = gq[j] * seconds<T, INTER>(wt, j);
            gn = fma(gq[j], q[j], fma(gp[j], p[j], gn));
          }
          const float mean = -__fmul_rn(group_sum<LPG>(sum(gn)), inv_d);
          const F2 mean2 = f2(mean, mean);
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = inv2 * fma(p[j], mean2, gp[j]), q[j] = inv2 * fma(q[j], mean2, gq[j]);
        }
        if (pad)
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = q[j] = zero;
        store<T, INTER>(y, c0, c1, writes, p, q);
        y += D;
      }
    }
  }
  if constexpr (BACK) {
    // this CTA's share of the weights' gradients, its groups added up in their order
    __shared__ float part[GROUPS][LPG * 16 + 4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const F2 s = dw[j], v = dw[4 + j];
      if (INTER) {
        part[group][c0 + 4 * j] = lo(s), part[group][c0 + 4 * j + 1] = lo(v), part[group][c0 + 4 * j + 2] = hi(s), part[group][c0 + 4 * j + 3] = hi(v);
      } else {
        if (runs > 0) part[group][c0 + 2 * j] = lo(s), part[group][c0 + 2 * j + 1] = hi(s);
        if (runs > 1) part[group][c1 + 2 * j] = lo(v), part[group][c1 + 2 * j + 1] = hi(v);
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += NT) {
      float s = 0.0f;
#pragma unroll 8
      for (int g = 0; g < GROUPS; ++g) s = __fadd_rn(s, part[g][c]);
      a.partial[(int64_t)blockIdx.x * D + c] = s;
    }
  }
}

// The weights' gradients from the CTAs' shares [ctas][D] (q's CTAs first), added up in one order whatever ran first: 8 columns
// a CTA, 128 threads to a column.
template <typename T> __global__ void __launch_bounds__(1024) norm_rope_weights_kernel(const float* partial, int split, int ctas, int D, T* dwq, T* dwk) {
  __shared__ float s[128][9];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int which = blockIdx.y, c = blockIdx.x * 8 + threadIdx.x;
  T* out = which ? dwk : dwq;
  if (!out) return;
  float v = 0.0f;
#pragma unroll 4
  for (int i = (which ? split : 0) + threadIdx.y; i < (which ? ctas : split); i += 128) v = __fadd_rn(v, partial[(int64_t)i * D + c]);
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  const int warp = (threadIdx.y * 8 + threadIdx.x) / 32, lane = (threadIdx.y * 8 + threadIdx.x) % 32;
  if (warp >= 8) return;
  v = __fadd_rn(__fadd_rn(s[lane][warp], s[lane + 32][warp]), __fadd_rn(s[lane + 64][warp], s[lane + 96][warp]));
#pragma unroll
  for (int o = 16; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  const int col = blockIdx.x * 8 + warp;
  if (lane == 0) {
    if constexpr (std::is_same<T, float>::value) out[col] = v;
    else if constexpr (std::is_same<T, __half>::value) out[col] = __float2half_rn(v);
    else out[col] = __float2bfloat16_rn(v);
  }
}

int lanes_of(int64_t D) { return D <= 32 ? 2 : D <= 64 ? 4 : D <= 128 ? 8 : 16; }

// Heads of a unit and CTAs of the grid, q's first.  While the machine is not full, fewer heads to a unit.
int64_t shape(NormRopeArgs& a, int sms) {
  const int groups = NT / lanes_of(a.D);
  int64_t ctas[2];
  for (int most = 16; most >= 1; most /= 2) {
    for (int w = 0; w < 2; ++w) {
      const int64_t chunks = (a.heads[w] + most - 1) / most;
      a.heads_per_unit[w] = (int)((a.heads[w] + chunks - 1) / chunks);
      ctas[w] = (a.T * ((a.heads[w] + a.heads_per_unit[w] - 1) / a.heads_per_unit[w]) + groups - 1) / groups;
    }
    if (ctas[0] + ctas[1] >= 2 * sms) break;
  }
  // no more than run at once: each walks over its share of the units (and has a share of the weights' gradients)
  const int64_t most = (int64_t)sms * NORM_ROPE_CTAS, rows = a.heads[0] + a.heads[1];
  if (ctas[0] + ctas[1] > most) {
    ctas[0] = std::max<int64_t>(1, std::min<int64_t>(most - 1, (most * a.heads[0] + rows / 2) / rows));
    ctas[1] = most - ctas[0];
  }
  a.split = (int)ctas[0];
  return ctas[0] + ctas[1];
}

template <typename T, int LPG, bool INTER> cudaError_t launch(const NormRopeArgs& a, bool back, int64_t grid, cudaStream_t stream) {
  if (!back) {
    norm_rope_kernel<T, LPG, INTER, false><<<(unsigned)grid, NT, 0, stream>>>(a);
    return cudaGetLastError();
  }
  norm_rope_kernel<T, LPG, INTER, true><<<(unsigned)grid, NT, 0, stream>>>(a);
  if (!a.dw[0] && !a.dw[1]) return cudaGetLastError();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.D / 8), 2);
  cfg.blockDim = dim3(8, 128);
  cfg.stream = stream;
  cudaLaunchAttribute attr;                                  // launched early, to wait where the gradients' CTAs finish
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_rope_weights_kernel<T>, (const float*)a.partial, a.split, (int)grid, (int)a.D, static_cast<T*>(a.dw[0]), static_cast<T*>(a.dw[1]));
}
template <typename T, bool INTER> cudaError_t launch_sized(const NormRopeArgs& a, bool back, int64_t grid, cudaStream_t stream) {
  switch (lanes_of(a.D)) {
    case 2: return launch<T, 2, INTER>(a, back, grid, stream);
    case 4: return launch<T, 4, INTER>(a, back, grid, stream);
    case 8: return launch<T, 8, INTER>(a, back, grid, stream);
    default: return launch<T, 16, INTER>(a, back, grid, stream);
  }
}
template <typename T> cudaError_t launch_typed(const NormRopeArgs& a, bool back, int64_t grid, cudaStream_t stream) {
  return a.interleaved ? launch_sized<T, true>(a, back, grid, stream) : launch_sized<T, false>(a, back, grid, stream);
}

}  // namespace

size_t norm_rope_workspace(int64_t D) { return (size_t)sm_count() * NORM_ROPE_CTAS * D * sizeof(float); }

cudaError_t launch_norm_rope(NormRopeArgs a, bool back, cudaStream_t stream) {
  const int64_t grid = shape(a, sm_count());
  const int esz = a.dtype == EMU_DTYPE_F32 ? 4 : 2;
  // Runs of elements, and of cosines, that start on 16 bytes: each for itself, as halves that are no multiple of 4 (interleaved) or a
  // table off 16 bytes say nothing of the rows.  8191 tokens of 24 + 6 heads of 96, fp16, interleaved, half 18: 37 us where the
  // table alone is read by elements, 61 where the rows are too; gradients 59 against 109.
  uintptr_t rows = reinterpret_cast<uintptr_t>(a.weight[0]) | reinterpret_cast<uintptr_t>(a.weight[1]);
  for (int w = 0; w < 2; ++w) {
    rows |= reinterpret_cast<uintptr_t>(a.x[w]) | (uintptr_t)(a.token_stride[w] * esz) | (uintptr_t)(a.head_stride[w] * esz);
    if (back) rows |= reinterpret_cast<uintptr_t>(a.dy[w]) | (uintptr_t)(a.dy_token_stride[w] * esz) | (uintptr_t)(a.dy_head_stride[w] * esz);
  }
  a.vec = (rows & 15) == 0;
  a.vec_table = ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin) | (uintptr_t)(a.half * 4)) & 15) == 0;
  if (a.dtype == EMU_DTYPE_F32) return launch_typed<float>(a, back, grid, stream);
  return a.dtype == EMU_DTYPE_F16 ? launch_typed<__half>(a, back, grid, stream) : launch_typed<__nv_bfloat16>(a, back, grid, stream);
}

}  // namespace emu
