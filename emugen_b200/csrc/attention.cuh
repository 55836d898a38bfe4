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

// One row at a time, a warp to a row: lane l holds elements l, l + 32, l + 64 and l + 96 of it.  Nothing that the mask
// hides is read, so that infinities and NaN there reach no result.
struct Lanes {
  float v[4];
};
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
template <typename T> __device__ __forceinline__ Lanes load_row(const T* p, int D) {
  Lanes r;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = lane + 32 * i < D ? widen<T>(p[lane + 32 * i]) : 0.0f;
  return r;
}
__device__ __forceinline__ float dot(const Lanes& a, const Lanes& b) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s = __fmaf_rn(a.v[i], b.v[i], s);
  return warp_sum(s);
}
// Elements [d0, d1) of the row.
template <typename T> __device__ __forceinline__ void store_row(T* p, int d0, int d1, const Lanes& r, float f) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i >= d0 && lane + 32 * i < d1) p[lane + 32 * i] = narrow<T>(__fmul_rn(r.v[i], f));
}
// Whether every element of the row is NaN: nothing that is added changes it any more.
__device__ __forceinline__ bool settled(const Lanes& r, int D) {
  const int lane = threadIdx.x & 31;
  bool nan = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) nan = nan && (isnan(r.v[i]) || lane + 32 * i >= D);
  return __all_sync(0xFFFFFFFFu, nan);
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

// The keys that query t of sequence b sees: the first `n` of the sequence's.
struct Seen {
  Rows k;
  int64_t n;
};
__device__ __forceinline__ Seen seen_by(const AttnArgs& a, int64_t b, int64_t t) {
  const Rows q = rows_of(a.cu_q, b, a.Tq);
  Seen s;
  s.k = rows_of(a.cu_k, b, a.Tk);
  s.n = s.k.count();
  if (a.causal) s.n = max((int64_t)0, min(s.n, t - q.begin + 1 + s.k.count() - q.count()));
  return s;
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

// Elements [d0, d1) of o_t of one head.
template <typename T> __device__ __forceinline__ void row_forward(const AttnArgs& a, int64_t b, int64_t t, int h, int d0, int d1) {
  const T* q = static_cast<const T*>(a.q) + t * a.q_stride[0] + h * a.q_stride[1];
  const int kh = h / (a.Hq / a.Hk);
  const T* k = static_cast<const T*>(a.k) + kh * a.k_stride[1];
  const T* v = static_cast<const T*>(a.v) + kh * a.v_stride[1];
  Seen s{{0, 0}, 0};
  if (b < a.B) s = seen_by(a, b, t);
  const Lanes x = load_row(q, a.D);
  Lanes o{};
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = s.k.begin; j < s.k.begin + s.n; ++j) {
    const float z = __fmul_rn(dot(x, load_row(k + j * a.k_stride[0], a.D)), a.scale);
    const float top = fmaxf(m, z);
    const float shift = top == -INFINITY ? 0.0f : top;
    const float old = expf(m - shift), p = expf(z - shift);
    const Lanes y = load_row(v + j * a.v_stride[0], a.D);
    l = __fmaf_rn(l, old, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = __fmaf_rn(p, y.v[i], __fmul_rn(o.v[i], old));
    m = top;
    if (settled(o, a.D)) break;
  }
  const float f = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  store_row(static_cast<T*>(a.out) + (t * a.Hq + h) * a.D, d0, d1, o, f);
  if (a.low) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = rounded_off<T>(__fmul_rn(o.v[i], f));
    store_row(static_cast<T*>(a.low) + (t * a.Hq + h) * a.D, d0, d1, o, 1.0f);
  }
}

// A query's shift -lse log2 e and its delta, at [t * Hq + h].
__device__ __forceinline__ float2 stat_of(const float2* stats, const AttnArgs& a, int64_t t, int h) { return stats[t * a.Hq + h]; }

// Elements [d0, d1) of dq_t of one head.
template <typename T> __device__ __forceinline__ void row_dq(const AttnArgs& a, const float2* stats, int64_t b, int64_t t, int h, int d0, int d1) {
  const T* q = static_cast<const T*>(a.q) + t * a.q_stride[0] + h * a.q_stride[1];
  const T* g = static_cast<const T*>(a.dout) + t * a.dout_stride[0] + h * a.dout_stride[1];
  const int kh = h / (a.Hq / a.Hk);
  const T* k = static_cast<const T*>(a.k) + kh * a.k_stride[1];
  const T* v = static_cast<const T*>(a.v) + kh * a.v_stride[1];
  Seen s{{0, 0}, 0};
  if (b < a.B) s = seen_by(a, b, t);
  const Lanes x = load_row(q, a.D), y = load_row(g, a.D);
  const float2 st = stat_of(stats, a, t, h);
  const float c = a.scale * 1.4426950408889634f;
  Lanes o{};
  for (int64_t j = s.k.begin; j < s.k.begin + s.n; ++j) {
    const Lanes kj = load_row(k + j * a.k_stride[0], a.D);
    const float p = exp2f(__fmaf_rn(dot(x, kj), c, st.x));
    const float ds = __fmul_rn(p, dot(y, load_row(v + j * a.v_stride[0], a.D)) - st.y);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = __fmaf_rn(ds, kj.v[i], o.v[i]);
    if (settled(o, a.D)) break;
  }
  store_row(static_cast<T*>(a.dq) + (t * a.Hq + h) * a.D, d0, d1, o, a.scale);
}

// dk_t (KEYS) or dv_t of one key head, t a row of the keys.
template <typename T, bool KEYS> __device__ __forceinline__ void row_dkv(const AttnArgs& a, const float2* stats, int64_t b, int64_t t, int kh) {
  Lanes o{};
  if (b < a.B) {
    const Rows q = rows_of(a.cu_q, b, a.Tq), kr = rows_of(a.cu_k, b, a.Tk);
    const Lanes kj = load_row(static_cast<const T*>(a.k) + t * a.k_stride[0] + kh * a.k_stride[1], a.D);
    const Lanes vj = load_row(static_cast<const T*>(a.v) + t * a.v_stride[0] + kh * a.v_stride[1], a.D);
    const int64_t first = a.causal ? max((int64_t)0, (t - kr.begin) - (kr.count() - q.count())) : 0;
    const int group = a.Hq / a.Hk;
    const float c = a.scale * 1.4426950408889634f;
    bool done = false;
    for (int h = kh * group; h < (kh + 1) * group && !done; ++h)
      for (int64_t i = q.begin + first; i < q.end && !done; ++i) {
        const Lanes x = load_row(static_cast<const T*>(a.q) + i * a.q_stride[0] + h * a.q_stride[1], a.D);
        const Lanes g = load_row(static_cast<const T*>(a.dout) + i * a.dout_stride[0] + h * a.dout_stride[1], a.D);
        const float2 st = stat_of(stats, a, i, h);
        const float p = exp2f(__fmaf_rn(dot(x, kj), c, st.x));
        const float w = KEYS ? __fmul_rn(p, dot(g, vj) - st.y) : p;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = __fmaf_rn(w, KEYS ? x.v[e] : g.v[e], o.v[e]);
        done = settled(o, a.D);
      }
  }
  store_row(static_cast<T*>(KEYS ? a.dk : a.dv) + (t * a.Hk + kh) * a.D, 0, a.D, o, KEYS ? a.scale : 1.0f);
}

}  // namespace attn
}  // namespace emu
