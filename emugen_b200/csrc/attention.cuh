// What the kernels of attention over packed sequences share: which keys a query sees, and the formulas row by row.
//
// Query i of a sequence with nq queries and nk keys sees keys 0 .. nk - 1, or with the causal mask those up to
// i + nk - nq (the last query stands on the last key).  With s_ij = scale q_i . k_j over the keys seen:
//   lse_i = log sum_j exp(s_ij),  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j     (no key: o = 0, lse = -inf)
// and for dO:  dp_ij = dO_i . v_j,  delta_i = dO_i . o_i,  ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij dO_i
// (dk and dv over the query heads that share the key head).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "kernels.h"

namespace emu {
namespace attn {

// Rows [begin, end) of sequence b, inside the tensor whatever the cumulative lengths say.
struct Rows {
  int64_t begin, end;
  __device__ __forceinline__ int64_t count() const { return end - begin; }
};
__device__ __forceinline__ Rows rows_of(const int32_t* cu, int64_t b, int64_t total) {
  Rows r;
  r.begin = min(max((int64_t)cu[b], (int64_t)0), total);
  r.end = min(max((int64_t)cu[b + 1], r.begin), total);
  return r;
}
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

// What rounding to T takes from v; 0 where v is infinite or NaN, or becomes it.
template <typename T> __device__ __forceinline__ float rounded_off(float v) {
  const float r = __fsub_rn(v, widen<T>(narrow<T>(v)));
  return fabsf(r) < INFINITY ? r : 0.0f;
}

// The tokens, counted from t0, of [t0, t1) with an element [d0, d1) of heads [h0, h1) that is infinite or NaN: the first and the last (none:
// INT_MAX, -1); with `stop` the search ends where the first one is known.  The whole warp; 16 lanes to a row, 8 elements each.  Rows
// start on 16 bytes, d0 and d1 are multiples of 8, d1 - d0 <= 128.
struct Span {
  int first, last;
};
template <typename T> __device__ __forceinline__ Span not_finite(const T* p, int64_t token_stride, int64_t head_stride, int64_t t0, int64_t t1, int h0, int h1, int d0, int d1, bool stop = false) {
  constexpr uint32_t EXPONENT = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  const int lane = threadIdx.x & 31, d = d0 + (lane & 15) * 8, heads = h1 - h0;
  const int tokens = heads > 0 ? (int)max((int64_t)0, t1 - t0) : 0;
  int first = 0x7FFFFFFF, last = -1, t = 0, h = lane >> 4;
  p += t0 * token_stride + h0 * head_stride + d;
  auto next = [&] {
    for (h += 2; h >= heads && t < tokens; h -= heads) ++t;
  };
  if (h >= heads) h = 0, t = 1;                              // (one head)
  while (__any_sync(0xFFFFFFFFu, t < tokens)) {
    constexpr int U = 8;                                     // rows under way
    uint4 w[U];
    int at[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      w[i] = make_uint4(0, 0, 0, 0), at[i] = t;
      if (t < tokens && d < d1) w[i] = __ldg(reinterpret_cast<const uint4*>(p + t * token_stride + h * head_stride));
      next();
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      bool bad = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u = k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w;
        bad = bad || (u & EXPONENT) == EXPONENT || (u >> 16 & EXPONENT) == EXPONENT;
      }
      if (bad) first = min(first, at[i]), last = max(last, at[i]);
    }
    if (stop && __any_sync(0xFFFFFFFFu, last >= 0)) break;
  }
  return {__reduce_min_sync(0xFFFFFFFFu, first), __reduce_max_sync(0xFFFFFFFFu, last)};
}

// Which of the lanes with `bad`, a row of sequence b that is not finite in elements [d0, d1), have to be made again: a row that sees the
// first n keys met one that it does not see only if one of keys n .. end - 1, which were multiplied too, is not finite there.  What is
// not finite by right stays as it is.  VALUES: of v, else k.  (bf16: of values past 2^118, weights of up to 2^8 can leave f32's range
// where the row's result does not; so it is made again too where none that it sees is infinite or NaN.)  low: the row of what rounding
// took from the output, or null: 0 where it is not finite, in rows that stay.  (The whole warp.)
template <typename T, bool VALUES> __device__ __noinline__ uint32_t rows_made_again(const AttnArgs& a, bool bad, int64_t b, int n, int64_t end, int kh, int d0, int d1, T* low) {
  const int64_t k0 = rows_of(a.cu_k, b, a.Tk).begin;
  const int least = __reduce_min_sync(0xFFFFFFFFu, bad ? n : 0x7FFFFFFF);
  const T* x = static_cast<const T*>(VALUES ? a.v : a.k);
  const int64_t ts = VALUES ? a.v_stride[0] : a.k_stride[0], hs = VALUES ? a.v_stride[1] : a.k_stride[1];
  const Span hidden = not_finite(x, ts, hs, k0 + least, min(k0 + end, a.Tk), kh, kh + 1, d0, d1);
  bool made = hidden.last >= 0 && n - least <= hidden.last;
  if (VALUES && std::is_same<T, __nv_bfloat16>::value) {
    const int most = __reduce_max_sync(0xFFFFFFFFu, bad ? n : 0);
    const Span seen = not_finite(x, ts, hs, k0, k0 + most, kh, kh + 1, d0, d1, true);
    made = made || seen.first >= n;
  }
  if (VALUES && low && bad && !made)
    for (int d = d0; d < d1; ++d)
      if (!(fabsf(widen<T>(low[d])) < INFINITY)) low[d] = narrow<T>(0.0f);
  return __ballot_sync(0xFFFFFFFFu, bad && made);
}

// Rows of the output or of the gradients made again from what they see alone, in f32 by one warp, 8 rows at a time: they share what is
// read of the other side, and their sums over the head share the exchanges between lanes (one row after the other: 93 ms for one infinity
// in the middle of dO of 4096 causal tokens, 32 heads on 8 of 128; so 7.5, 9.4 with two of the other side's rows at a time; without the
// infinity 0.65).  Lane l holds elements 4 l .. 4 l + 3.
//   OUT  o_i = sum_j w_ij v_j        w = exp2(c s + known.x) known.y         (known: the held shift, 1 / l)
//   DQ   dq_i = scale sum_j w_ij k_j  w = exp2(c s + known.x) (dp - known.y)  (known: the query's statistics)
//   DK   dk_j = scale sum_i w_ij q_i  the same, the statistics of query i;   DV   dv_j = sum_i w_ij dO_i,  w = exp2(c s + stats.x)
enum Again { AGAIN_OUT, AGAIN_DQ, AGAIN_DK, AGAIN_DV };

template <typename T> __device__ __forceinline__ uint2 load4(const T* p, bool any) { return any ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0); }
template <typename T> __device__ __forceinline__ void widen4(const uint2& w, float (&v)[4]) {
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = widen<T>(e[i]);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  uint2 w;
  T* e = reinterpret_cast<T*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = narrow<T>(v[i]);
  *reinterpret_cast<uint2*>(p) = w;
}
// Sums over the warp of 8 numbers of each lane: lane l gets that of number l / 4.
__device__ __forceinline__ float sum8(float (&v)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16, n = 4; o >= 4; o >>= 1, n >>= 1)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) {
        const float keep = lane & o ? v[k + n] : v[k], give = lane & o ? v[k] : v[k + n];
        v[k] = __fadd_rn(keep, __shfl_xor_sync(0xFFFFFFFFu, give, o));
      }
  float s = __fadd_rn(v[0], __shfl_xor_sync(0xFFFFFFFFu, v[0], 2));
  return __fadd_rn(s, __shfl_xor_sync(0xFFFFFFFFu, s, 1));
}

// rows: the lanes whose rows are meant; t, head: a lane's row (a query and its head, or a key and its head) in sequence b.
// Elements [d0, d1), multiples of 8, are written.  (The whole warp.)
template <typename T, Again WHAT>
__device__ __noinline__ void make_again(const AttnArgs& a, const float2* stats, uint32_t rows, int64_t b, int64_t t, int head, float2 known, int d0, int d1) {
  constexpr bool QUERIES = WHAT == AGAIN_OUT || WHAT == AGAIN_DQ, TWO = WHAT == AGAIN_DQ || WHAT == AGAIN_DK;
  constexpr bool FIRST = TWO;                                // which of the other side's two rows is added up
  constexpr int N = 8, U = 4;                                // rows at a time, rows of the other side at a time
  const int lane = threadIdx.x & 31, e = lane * 4, group = a.Hq / a.Hk;
  const bool live = e < a.D;
  const Rows qr = rows_of(a.cu_q, b, a.Tq), kr = rows_of(a.cu_k, b, a.Tk);
  const int64_t ahead = kr.count() - qr.count();
  const float c = a.scale * 1.4426950408889634f;
  const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v), *g = static_cast<const T*>(a.dout);
  while (rows) {
    int src[N], own = 0, count = 0;
#pragma unroll
    for (int r = 0; r < N; ++r) {
      src[r] = rows ? __ffs(rows) - 1 : src[0];              // (places without a row do the first one's work)
      count += rows != 0;
      rows &= rows - 1;
      if (lane >> 2 == r) own = src[r];
    }
    // of the row whose sums this lane gets
    const int64_t t_own = __shfl_sync(0xFFFFFFFFu, t, own);
    const float2 known_own = make_float2(__shfl_sync(0xFFFFFFFFu, known.x, own), __shfl_sync(0xFFFFFFFFu, known.y, own));
    // a query sees keys up to `limit`, a key is seen by queries from `limit`
    const int limit = QUERIES ? (int)(a.causal ? max((int64_t)0, min(kr.count(), t_own - qr.begin + 1 + ahead)) : kr.count())
                              : (int)(a.causal ? max((int64_t)0, t_own - kr.begin - ahead) : 0);
    const int from = QUERIES ? 0 : __reduce_min_sync(0xFFFFFFFFu, limit), to = QUERIES ? __reduce_max_sync(0xFFFFFFFFu, limit) : (int)qr.count();
    float x[N][4], y[TWO ? N : 1][4], acc[N][4] = {};
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const int64_t tr = __shfl_sync(0xFFFFFFFFu, t, src[r]);
      const int hr = __shfl_sync(0xFFFFFFFFu, head, src[r]);
      widen4<T>(load4((QUERIES ? q + tr * a.q_stride[0] + hr * a.q_stride[1] : k + tr * a.k_stride[0] + hr * a.k_stride[1]) + e, live), x[r]);
      if (TWO) widen4<T>(load4((QUERIES ? g + tr * a.dout_stride[0] + hr * a.dout_stride[1] : v + tr * a.v_stride[0] + hr * a.v_stride[1]) + e, live), y[TWO ? r : 0]);
    }
    const int kh = QUERIES ? __shfl_sync(0xFFFFFFFFu, head, src[0]) / group : __shfl_sync(0xFFFFFFFFu, head, src[0]);
    bool done = false;
    for (int h = QUERIES ? kh : kh * group; h < (QUERIES ? kh + 1 : (kh + 1) * group) && !done; ++h) {
      const T* first = (QUERIES ? k + kr.begin * a.k_stride[0] + h * a.k_stride[1] : q + qr.begin * a.q_stride[0] + h * a.q_stride[1]) + e;
      const T* second = (QUERIES ? v + kr.begin * a.v_stride[0] + h * a.v_stride[1] : g + qr.begin * a.dout_stride[0] + h * a.dout_stride[1]) + e;
      const int64_t fs = QUERIES ? a.k_stride[0] : a.q_stride[0], ss = QUERIES ? a.v_stride[0] : a.dout_stride[0];
      for (int i0 = from; i0 < to && !done; i0 += U) {
        uint2 wf[U], ws[U];
        float2 st[U];
#pragma unroll
        for (int z = 0; z < U; ++z) {
          const bool in = i0 + z < to;
          wf[z] = load4(first + (i0 + z) * fs, live && in), ws[z] = load4(second + (i0 + z) * ss, live && in);
          st[z] = QUERIES ? known_own : in ? __ldg(stats + (qr.begin + i0 + z) * a.Hq + h) : make_float2(0.0f, 0.0f);
        }
        float weight[U];
        uint32_t sees[U];
#pragma unroll
        for (int z = 0; z < U; ++z) {
          float f[4], s[4], part[N];
          widen4<T>(wf[z], f), widen4<T>(ws[z], s);
#pragma unroll
          for (int r = 0; r < N; ++r) part[r] = __fmaf_rn(x[r][3], f[3], __fmaf_rn(x[r][2], f[2], __fmaf_rn(x[r][1], f[1], __fmul_rn(x[r][0], f[0]))));
          weight[z] = exp2f(__fmaf_rn(sum8(part), c, st[z].x));
          if (TWO) {
#pragma unroll
            for (int r = 0; r < N; ++r) {
              const float(&yr)[4] = y[TWO ? r : 0];
              part[r] = __fmaf_rn(yr[3], s[3], __fmaf_rn(yr[2], s[2], __fmaf_rn(yr[1], s[1], __fmul_rn(yr[0], s[0]))));
            }
            weight[z] = __fmul_rn(weight[z], sum8(part) - st[z].y);
          }
          if (WHAT == AGAIN_OUT) weight[z] = __fmul_rn(weight[z], known_own.y);
          sees[z] = __ballot_sync(0xFFFFFFFFu, i0 + z < to && (QUERIES ? i0 + z < limit : i0 + z >= limit));
        }
#pragma unroll
        for (int z = 0; z < U; ++z) {
          float u[4];
          widen4<T>(FIRST ? wf[z] : ws[z], u);
#pragma unroll
          for (int r = 0; r < N; ++r) {
            const float w = __shfl_sync(0xFFFFFFFFu, weight[z], 4 * r);
            if (sees[z] >> (4 * r) & 1)
#pragma unroll
              for (int n = 0; n < 4; ++n) acc[r][n] = __fmaf_rn(w, u[n], acc[r][n]);
          }
        }
        if ((i0 - from) % 64 == 0) {                         // once every element is NaN, nothing changes it any more
          bool nan = true;
#pragma unroll
          for (int r = 0; r < N; ++r)
#pragma unroll
            for (int n = 0; n < 4; ++n) nan = nan && isnan(acc[r][n]);
          done = __all_sync(0xFFFFFFFFu, nan || !live);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const int64_t tr = __shfl_sync(0xFFFFFFFFu, t, src[r]);
      const int hr = __shfl_sync(0xFFFFFFFFu, head, src[r]);
      if (r >= count || e < d0 || e >= d1) continue;
      const int64_t at = (tr * (QUERIES ? a.Hq : a.Hk) + hr) * a.D + e;
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (TWO) acc[r][n] = __fmul_rn(acc[r][n], a.scale);
      store4(static_cast<T*>(WHAT == AGAIN_OUT ? a.out : WHAT == AGAIN_DQ ? a.dq : WHAT == AGAIN_DK ? a.dk : a.dv) + at, acc[r]);
      if (WHAT == AGAIN_OUT && a.low) {
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[r][n] = rounded_off<T>(acc[r][n]);
        store4(static_cast<T*>(a.low) + at, acc[r]);
      }
    }
  }
}

}  // namespace attn
}  // namespace emu
