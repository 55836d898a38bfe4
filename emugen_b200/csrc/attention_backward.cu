// Gradients of attention over packed sequences (the formulas: attention.cuh) on the 5th-generation tensor cores.
//
// Two kernels walk over the (query, key) tiles, one with the keys' sums in tensor memory, one with the queries': the scores
// and dp are made twice (7 products in place of 5), and in return no sum leaves the CTA that makes it: no additions in
// memory, whose order would change the result from run to run, and no f32 copy of dq.
// Measured: 8192 causal tokens in 3 sequences, 32 heads on 8 of 128, bf16: statistics 31 us (reading out, its rest and dout: a copy's
// rate), dk and dv 418 us, dq 308 us (0.94 and 0.96 PFLOP/s of the products done).  P and ds are rounded to the inputs' type, as
// the products take them.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/emugen.h"
#include "attention.cuh"
#include "attention_tc.cuh"
#include "tc_ptx.cuh"

namespace emu {
namespace {

using namespace attn;

constexpr int THREADS = 384;                                // warps 10, 11 (11 alone) fill up the third warpgroup
constexpr int REG_LOW = 40, REG_HIGH = 232;                 // 128 x 40 + 256 x 232 = 64512 = 384 x 168, the launch's

// fp16: P is held 2^15 times as large, so that weights down to 2^-29 keep all their bits, and ds is multiplied by a power of
// two that puts a bound of it at 2^14: |dp - delta| <= 2 |dO_i| |v_j|, as o_i is a mean of values.  A row of dq has its own |dO_i|, with
// the largest |v_j| of its sequence and key head; dk adds up over rows, and takes the largest |dO_i| of the sequence and key head (with
// one factor for the whole call, a sequence 2^22 times larger left none of its neighbour's bits).  bf16 needs neither.
template <typename T> constexpr float P_LOG2 = std::is_same<T, __half>::value ? 15.0f : 0.0f;

struct Work {
  float2* stats;               // [Tq][Hq]: -lse log2 e, delta
  float* norms;                // from here on fp16.  [Tq][Hq]: |dO_i|^2
  uint32_t* top_g;             // [sequence][key head]: bits of the largest |dO_i|^2
  uint32_t* top_v;             // the same of |v_j|^2
  size_t bytes;
};
__host__ __device__ inline Work work_of(void* p, int64_t Tq, int64_t B, int Hq, int Hk, bool half) {
  uint8_t* base = static_cast<uint8_t*>(p) + 256;
  const size_t rows = (size_t)Tq * Hq, heads = (size_t)B * Hk;
  Work w;
  w.stats = reinterpret_cast<float2*>(base);
  w.norms = reinterpret_cast<float*>(base + rows * 8);
  w.top_g = reinterpret_cast<uint32_t*>(base + rows * 12);
  w.top_v = w.top_g + heads;
  w.bytes = 256 + (half ? rows * 12 + heads * 8 : rows * 8);
  return w;
}
__host__ __device__ inline Work work_of(const AttnArgs& a) { return work_of(a.workspace, a.Tq, a.B, a.Hq, a.Hk, a.dtype == EMU_DTYPE_F16); }

// The factor of ds where |dO_i|^2 <= g and |v_j|^2 <= v.
__device__ __forceinline__ float ds_factor(float g, float v) {
  const float b = 4.0f * g * v;
  return b > 0.0f && b < INFINITY ? exp2f(floorf((28.0f - log2f(b)) * 0.5f)) : 1.0f;
}
// The sequence that holds row t, or B for a row behind the last one.
__device__ __forceinline__ int64_t sequence_of(const int32_t* cu, int64_t B, int64_t t) {
  int64_t lo = 0, hi = B;
  while (lo < hi) {
    const int64_t m = (lo + hi) / 2;
    if ((int64_t)cu[m + 1] > t) hi = m;
    else lo = m + 1;
  }
  return lo;
}

// ------------------------------------------------------------------------------ statistics
// delta of each (token, head), from the output before its rounding where its rest was kept: ds is what is left of
// dp - delta, so that a sequence of 2 tokens had 0.0039 of its gradients' norm off without the rest, 0.0026 with it.  Beside
// the shift of its scores; fp16: its norm.  16 lanes to a row, 8 elements each.
template <typename T> __device__ __forceinline__ void load8(const T* p, bool any, float (&v)[8]) {
  uint4 w = make_uint4(0, 0, 0, 0);
  if (any) w = __ldg(reinterpret_cast<const uint4*>(p));
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = widen<T>(e[i]);
}
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
template <typename T> __global__ void __launch_bounds__(256) attention_stats_kernel(const __grid_constant__ AttnArgs a) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  const Work w = work_of(a);
  const int64_t row = (int64_t)blockIdx.x * 16 + threadIdx.x / 16, nq = a.Tq * a.Hq;
  const int d = (threadIdx.x & 15) * 8;
  const bool in = row < nq;
  const int64_t t = in ? row / a.Hq : 0;
  const int h = in ? (int)(row - t * a.Hq) : 0;
  float o[8], low[8], g[8], s = 0.0f, rest = 0.0f, norm = 0.0f;
  load8(static_cast<const T*>(a.out) + row * a.D + d, in && d < a.D, o);
  load8(static_cast<const T*>(a.low) + row * a.D + d, in && a.low && d < a.D, low);
  load8(static_cast<const T*>(a.dout) + t * a.dout_stride[0] + h * a.dout_stride[1] + d, in && d < a.D, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) s = __fmaf_rn(o[i], g[i], s), rest = __fmaf_rn(low[i], g[i], rest), norm = __fmaf_rn(g[i], g[i], norm);
  s = sum16(__fadd_rn(s, rest));
  if (HALF) norm = sum16(norm);
  const float lse = in ? a.lse[(int64_t)h * a.Tq + t] : -INFINITY;
  if (in && (threadIdx.x & 15) == 0) {
    w.stats[row] = make_float2(lse == -INFINITY ? -INFINITY : -lse * 1.4426950408889634f, s);
    // (-infinity: sees no key, or is behind the last sequence)
    if (HALF) w.norms[row] = lse == -INFINITY || !(norm < INFINITY) ? 0.0f : norm;
  }
}

// fp16: the largest norms of each sequence and key head.  A warp has 32 tokens of a key head, a lane the largest of its token; one lane of
// each of their sequences tells the memory.  (3001 tokens of 12 heads: 16 us with the statistics, 28 where each row told it by itself; with
// rows of one head side by side in the statistics' blocks, to put them together there, 8192 tokens of 32 heads took 53 us for 32.)  In any
// order the same.  b: B where the token has none.
__device__ __forceinline__ void keep_largest(uint32_t* top, int Hk, int64_t B, int64_t b, float norm) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t s = __shfl_down_sync(0xFFFFFFFFu, b, o);
    const float n = __shfl_down_sync(0xFFFFFFFFu, norm, o);
    if (lane + o < 32 && s == b) norm = fmaxf(norm, n);
  }
  // the first token of a sequence now has the largest of them
  const int64_t before = __shfl_up_sync(0xFFFFFFFFu, b, 1);
  if (b >= B || (lane > 0 && before == b)) return;
  const uint32_t bits = __float_as_uint(norm);               // (a positive number's bits grow with it)
  uint32_t* to = top + b * Hk;
  if (bits > __ldcg(to)) atomicMax(to, bits);
}
// Warps of the queries' norms first, then those of the values, which are made here from those that some query sees.
inline int64_t norm_warps(int64_t tokens, int heads) { return (tokens + 31) / 32 * heads; }
__global__ void __launch_bounds__(256) attention_norms_kernel(const __grid_constant__ AttnArgs a, int64_t query_warps, int64_t warps) {
  const Work w = work_of(a);
  int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (i >= warps) return;
  const bool values = i >= query_warps;
  if (values) i -= query_warps;
  const int kh = (int)(i % a.Hk), lane = threadIdx.x & 31;
  const int64_t t0 = i / a.Hk * 32, t = t0 + lane;
  float norm = 0.0f;
  int64_t b = a.B;
  if (!values) {
    const int group = a.Hq / a.Hk;
    if (t < a.Tq) {
      const float* p = w.norms + t * a.Hq + kh * group;
#pragma unroll 4
      for (int g = 0; g < group; ++g) norm = fmaxf(norm, __ldg(p + g));
      b = sequence_of(a.cu_q, a.B, t);
    }
    keep_largest(w.top_g + kh, a.Hk, a.B, b, norm);
    return;
  }
  // a row to 16 lanes, 16 times two rows; the sums change places so that token t0 + l's is in lane l
  const int d = (lane & 15) * 8;
#pragma unroll 1
  for (int r0 = 0; r0 < 16; r0 += 8) {
    uint4 v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t at = t0 + 2 * (r0 + r) + (lane >> 4);
      v[r] = make_uint4(0, 0, 0, 0);
      if (at < a.Tk && d < a.D) v[r] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(a.v) + at * a.v_stride[0] + kh * a.v_stride[1] + d));
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const __half* e = reinterpret_cast<const __half*>(&v[r]);
      float n = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) n = __fmaf_rn(__half2float(e[k]), __half2float(e[k]), n);
      n = sum16(n);
      const float from = __shfl_sync(0xFFFFFFFFu, n, (lane & 1) * 16);
      if (lane >> 1 == r0 + r) norm = from;
    }
  }
  if (!(norm < INFINITY)) norm = 0.0f;
  if (t < a.Tk) b = sequence_of(a.cu_k, a.B, t);
  if (b < a.B && rows_of(a.cu_q, b, a.Tq).count() == 0) b = a.B;
  keep_largest(w.top_v + kh, a.Hk, a.B, b, norm);
}

// ------------------------------------------------------------------------------ the keys' and values' gradients
// A CTA owns 128 keys of a key head and walks over the rows of queries that see them (all heads of the group) in tiles of
// up to 128.  With the keys as the MMA's rows, S^T = K Q^T and dP^T = V dO^T come out with a key to a lane, so that P^T and dS^T
// are the next products' A operands where they lie: dV += P^T dO, dK += dS^T Q.  Tensor memory: S^T (then P^T), dP^T (then
// dS^T), dV, dK.  While the weights of a tile are made, dK and the next dP run; while its ds is made, dV and the next S.
//   warps 0-7   the elements, a thread to a key and half of the tile's queries; at the end a row of dV or dK
//   warp 8      MMA issuer;  warp 9  TMA;  warp 10  the queries' statistics
template <int DP> struct Kv {
  static constexpr int TILE = 128 * DP * 2;
  static constexpr int SLOTS = DP == 128 ? 2 : 4;           // of Q, and of dO
  static constexpr int STAT = 128 * 12 + 16, STATS = 3;     // shift, delta, keys seen; whether all see all
  static constexpr int BARS = 1 + 4 * SLOTS + 2 * STATS + 5;
  static constexpr int SMEM = 1024 + (2 + 2 * SLOTS) * TILE + STATS * STAT + BARS * 8 + 16;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
constexpr uint32_t KV_S = 0, KV_DP = 128, KV_DV = 256;      // dK behind dV

// Tiles of 128 rows by TMA: `heads` x `tokens` rows, zeros in the rest, which is written once here.
__device__ __forceinline__ void zero_rest(uint8_t* tiles, int count, int boxes, int rows) {
  for (int i = threadIdx.x; i < count * boxes * (128 - rows) * 8; i += THREADS) {
    const int box = i / ((128 - rows) * 8), at = i % ((128 - rows) * 8);
    *reinterpret_cast<uint4*>(tiles + box * 16384 + rows * 128 + at * 16) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Which keys' rows of dK (`keys`) or dV with `bad`, that are not finite, have to be made again: those where one of the rows that were
// multiplied but do not see the key is not finite: the tiles' first ones, up to the key's, tokens behind the sequence, heads behind the
// group.  What is not finite by right stays as it is.  (The whole warp.  A function that finds its place again: what the kernel
// would keep for it through its loop would not fit its registers.)
template <typename T> __device__ __noinline__ uint32_t keys_made_again(const AttnArgs& a, const Tiling& tl, bool keys, int key, bool bad) {
  Unit u;
  u.kh = (int)(blockIdx.x % a.Hk);
  find_unit(u, a.cu_k, a.B, a.Tk, 128, blockIdx.x / a.Hk);
  const Rows qr = rows_of(a.cu_q, u.b, a.Tq);
  const int64_t nq = qr.count(), hidden = u.rows.count() - nq, j0 = u.t0 - u.rows.begin;
  const int64_t first = a.causal ? max((int64_t)0, j0 - hidden) / tl.tokens * tl.tokens : 0;
  const int64_t end = min(qr.begin + first + (nq - first + tl.tokens - 1) / tl.tokens * tl.tokens, a.Tq);
  const T* src = static_cast<const T*>(keys ? a.q : a.dout);
  const int64_t ts = keys ? a.q_stride[0] : a.dout_stride[0], hs = keys ? a.q_stride[1] : a.dout_stride[1];
  const int h0 = u.kh * tl.group, h1 = h0 + tl.group, h2 = min(h0 + tl.chunks * tl.heads, a.Hq);
  // the first query that sees the key, of this lane's and of the last one's
  const int64_t sees = a.causal ? max((int64_t)0, j0 + key - hidden) : 0;
  const int64_t most = __shfl_sync(0xFFFFFFFFu, sees, 31 - __clz(__ballot_sync(0xFFFFFFFFu, bad)));
  bool made = false;
#pragma unroll 1
  for (int part = 0; part < 3; ++part) {
    const Span s = not_finite(src, ts, hs, part == 1 ? qr.end : qr.begin + first, part == 0 ? qr.begin + most : part == 1 ? end : qr.end,
                              part == 2 ? h1 : h0, part == 0 ? h1 : h2, 0, a.D);
    made = made || (s.last >= 0 && (part > 0 || first + s.first < sees));
  }
  return __ballot_sync(0xFFFFFFFFu, bad && made);
}

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1) attention_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                                                                  const __grid_constant__ AttnArgs a, const __grid_constant__ Tiling tl) {
  using C = Kv<DP>;
  extern __shared__ uint8_t smem_raw[];
  Unit u;
  u.kh = (int)(blockIdx.x % a.Hk);
  find_unit(u, a.cu_k, a.B, a.Tk, 128, blockIdx.x / a.Hk);
  if (!u.any) return;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Rows kr = u.rows, qr = u.b < a.B ? rows_of(a.cu_q, u.b, a.Tq) : Rows{0, 0};
  const int64_t nq = qr.count(), nk = kr.count(), j0 = u.t0 - kr.begin;
  // the first query that sees the tile's first key
  const int64_t first = a.causal ? max((int64_t)0, j0 - (nk - nq)) / tl.tokens * tl.tokens : 0;
  const int tiles = (int)max((int64_t)0, (nq - first + tl.tokens - 1) / tl.tokens);
  const int steps = tiles * tl.chunks;                       // chunk after chunk

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring_q = smem + 2 * C::TILE;                      // K, V first
  uint8_t* ring_g = ring_q + C::SLOTS * C::TILE;
  uint8_t* stats = ring_g + C::SLOTS * C::TILE;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(stats + C::STATS * C::STAT);
  uint64_t* q_full = kv_full + 1;
  uint64_t* q_empty = q_full + C::SLOTS;
  uint64_t* g_full = q_empty + C::SLOTS;
  uint64_t* g_empty = g_full + C::SLOTS;
  uint64_t* st_full = g_empty + C::SLOTS;
  uint64_t* st_empty = st_full + C::STATS;
  uint64_t* s_full = st_empty + C::STATS;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&map_q), ptx::prefetch_tmap(&map_k), ptx::prefetch_tmap(&map_v), ptx::prefetch_tmap(&map_g);
    ptx::mbar_init(kv_full, 1);
    for (int i = 0; i < C::SLOTS; ++i)
      ptx::mbar_init(&q_full[i], 1), ptx::mbar_init(&q_empty[i], 1), ptx::mbar_init(&g_full[i], 1), ptx::mbar_init(&g_empty[i], 1);
    for (int i = 0; i < C::STATS; ++i) ptx::mbar_init(&st_full[i], 1), ptx::mbar_init(&st_empty[i], 8);
    ptx::mbar_init(s_full, 1), ptx::mbar_init(p_full, 256), ptx::mbar_init(dp_full, 1), ptx::mbar_init(ds_full, 256), ptx::mbar_init(done, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  if (tl.heads * tl.tokens < 128) zero_rest(ring_q, 2 * C::SLOTS, DP / 64, tl.heads * tl.tokens);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp >= 8) {
    ptx::setmaxnreg_dec<REG_LOW>();
    if (warp == 9 && lane == 0 && steps) {
      ptx::mbar_arrive_expect_tx(kv_full, 2 * C::TILE);
      for (int x = 0; x < DP / 64; ++x) {
        ptx::tma_load_3d(smem + x * 16384, &map_k, kv_full, x * 64, u.kh, (int)u.t0);
        ptx::tma_load_3d(smem + C::TILE + x * 16384, &map_v, kv_full, x * 64, u.kh, (int)u.t0);
      }
      const uint32_t bytes = (DP / 64) * tl.heads * tl.tokens * 128;
      Ring<C::SLOTS> r;
      int i = 0, queries = 0, tile = 0, chunk = 0;            // queries, i: tiles of Q and of dO asked for
      for (; i < steps; ++i, r.next()) {
        const int head = u.kh * tl.group + chunk * tl.heads, row = (int)(qr.begin + first + (int64_t)tile * tl.tokens);
        if (i >= C::SLOTS && !wait_or_record(&q_empty[r.at], r.parity ^ 1, tl.wait_limit, WAIT_BACK_SLOT)) break;
        ptx::mbar_arrive_expect_tx(&q_full[r.at], bytes);
        for (int x = 0; x < DP / 64; ++x) ptx::tma_load_3d(ring_q + r.at * C::TILE + x * 16384, &map_q, &q_full[r.at], x * 64, head, row);
        ++queries;
        if (i >= C::SLOTS && !wait_or_record(&g_empty[r.at], r.parity ^ 1, tl.wait_limit, WAIT_BACK_SLOT)) break;
        ptx::mbar_arrive_expect_tx(&g_full[r.at], bytes);
        for (int x = 0; x < DP / 64; ++x) ptx::tma_load_3d(ring_g + r.at * C::TILE + x * 16384, &map_g, &g_full[r.at], x * 64, head, row);
        if (++tile == tiles) tile = 0, ++chunk;
      }
      drain<1>(kv_full, 1), drain<C::SLOTS>(q_full, queries), drain<C::SLOTS>(g_full, i);
    } else if (warp == 10 && steps) {
      const float2* src = work_of(a).stats;
      Ring<C::STATS> r;
      int tile = 0, chunk = 0;
      for (int i = 0; i < steps; ++i, r.next()) {
        if (i >= C::STATS && !warp_wait_or_record(&st_empty[r.at], r.parity ^ 1, tl.wait_limit, WAIT_BACK_SLOT)) break;
        float* shift = reinterpret_cast<float*>(stats + r.at * C::STAT);
        float* delta = shift + 128;
        int* seen = reinterpret_cast<int*>(delta + 128);
        bool all = true;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = lane + 32 * k, gh = chunk * tl.heads + row % tl.heads;
          const int64_t q = first + (int64_t)tile * tl.tokens + row / tl.heads;
          const bool in = row < tl.heads * tl.tokens && gh < tl.group && q < nq;
          const float2 s = in ? src[(qr.begin + q) * a.Hq + u.kh * tl.group + gh] : make_float2(0.0f, 0.0f);
          // keys of the tile that the row sees
          const int n = !in ? 0 : a.causal ? (int)max((int64_t)0, min((int64_t)128, q + 1 + nk - nq - j0)) : 128;
          shift[row] = s.x + P_LOG2<T>;
          delta[row] = s.y;
          seen[row] = n;
          all = all && n == 128;
        }
        all = __all_sync(0xFFFFFFFFu, all);
        if (lane == 0) seen[128] = all;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&st_full[r.at]);
        if (++tile == tiles) tile = 0, ++chunk;
      }
    } else if (warp == 8 && steps) {
      const uint32_t tmem = *tmem_slot;
      constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
      const uint32_t id_s = ptx::idesc_16_f32(128, 128, BF, false), id_d = ptx::idesc_16_f32(128, tl.d16, BF, true);
      const int ks = tl.d16 / 16;
      auto outer = [&](uint32_t d, const uint8_t* x, const uint8_t* y) {       // [keys][queries] = x y^T over the head
        const uint32_t xa = ptx::smem_u32(x), ya = ptx::smem_u32(y);
        for (int s = 0; s < ks; ++s) {
          const uint32_t at = (s / 4) * 16384 + (s % 4) * 32;
          ptx::mma_f16(tmem + d, ptx::smem_desc_sw128(xa + at), ptx::smem_desc_sw128(ya + at), id_s, s > 0);
        }
      };
      auto inner = [&](uint32_t d, uint32_t p, const uint8_t* y, bool more) {  // [keys][d] += p y over the queries
        const uint64_t b = ptx::smem_desc_mn_sw128(ptx::smem_u32(y), 16384);
#pragma unroll
        for (int s = 0; s < 8; ++s) ptx::mma_f16_ta(tmem + d, tmem + p + (s / 4) * 64 + (s % 4) * 8, b + s * 128, id_d, more || s > 0);
      };
      bool ok = warp_wait_or_record(kv_full, 0, tl.wait_limit, WAIT_BACK_FIXED);
      ok = ok && warp_wait_or_record(&q_full[0], 0, tl.wait_limit, WAIT_BACK_TILE);
      ok = ok && warp_wait_or_record(&g_full[0], 0, tl.wait_limit, WAIT_BACK_TILE);
      ptx::tc_fence_after();
      if (ok && ptx::elect_one()) {
        outer(KV_S, smem, ring_q);
        if (!tl.hold_first_ready) ptx::mma_commit(s_full);
        outer(KV_DP, smem + C::TILE, ring_g);
        ptx::mma_commit(dp_full);
      }
      __syncwarp();
      Ring<C::SLOTS> r, n;                                   // this tile and the next
      for (int i = 0; i < steps && ok; ++i, r.next()) {
        const bool next = i + 1 < steps;
        n.next();
        if (!warp_wait_or_record(p_full, i & 1, tl.wait_limit, WAIT_BACK_P)) { ok = false; break; }
        if (next && !warp_wait_or_record(&q_full[n.at], n.parity, tl.wait_limit, WAIT_BACK_TILE)) { ok = false; break; }
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          inner(KV_DV, KV_S, ring_g + r.at * C::TILE, i > 0);
          ptx::mma_commit(&g_empty[r.at]);
          if (next) {
            outer(KV_S, smem, ring_q + n.at * C::TILE);
            ptx::mma_commit(s_full);
          }
        }
        __syncwarp();
        if (!warp_wait_or_record(ds_full, i & 1, tl.wait_limit, WAIT_BACK_DS)) { ok = false; break; }
        if (next && !warp_wait_or_record(&g_full[n.at], n.parity, tl.wait_limit, WAIT_BACK_TILE)) { ok = false; break; }
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          inner(KV_DV + DP, KV_DP, ring_q + r.at * C::TILE, i > 0);
          ptx::mma_commit(&q_empty[r.at]);
          if (next) {
            outer(KV_DP, smem + C::TILE, ring_g + n.at * C::TILE);
            ptx::mma_commit(dp_full);
          }
        }
        __syncwarp();
      }
      if (ptx::elect_one()) ptx::mma_commit(done);           // after a failed wait too: the MMAs in flight are waited for
      __syncwarp();
      warp_wait_or_record(done, 0, DRAIN_LIMIT, WAIT_DRAIN);
    }
  } else {
    ptx::setmaxnreg_inc<REG_HIGH>();
    const uint32_t tmem = *tmem_slot;
    const int half = warp >> 2, key = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + KV_S + half * 64, dp_at = lanes + KV_DP + half * 64;
    const Work w = work_of(a);
    constexpr bool HALF = std::is_same<T, __half>::value;
    auto factor_of = [&] {
      const int64_t top = u.b * a.Hk + u.kh;
      return HALF && steps ? ds_factor(__uint_as_float(__ldg(w.top_g + top)), __uint_as_float(__ldg(w.top_v + top))) : 1.0f;
    };
    const float c = a.scale * 1.4426950408889634f, factor = factor_of() * exp2f(-P_LOG2<T>);
    const uint64_t c2 = ptx::join2(__float_as_uint(c), __float_as_uint(c));
    const uint64_t f2 = ptx::join2(__float_as_uint(factor), __float_as_uint(factor));
    const uint64_t minus = ptx::join2(0xBF800000u, 0xBF800000u);
    Ring<C::STATS> r;
    bool ok = true;
    for (int i = 0; i < steps; ++i, r.next()) {
      if (!warp_wait_or_record(&st_full[r.at], r.parity, tl.wait_limit, WAIT_BACK_STATS)) { ok = false; break; }
      const float* shift = reinterpret_cast<const float*>(stats + r.at * C::STAT) + half * 64;
      const float* delta = shift + 128;
      const int* seen = reinterpret_cast<const int*>(delta + 128);
      const bool all = seen[128 - half * 64] != 0;
      if (!warp_wait_or_record(s_full, i & 1, tl.wait_limit, WAIT_BACK_S)) { ok = false; break; }
      ptx::tc_fence_after();
      uint32_t s[2][32];
#pragma unroll
      for (int x = 0; x < 2; ++x) ptx::tmem_ld_regs(s_at + 32 * x, s[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x) ptx::tmem_wait_regs(s[x]);
      // P
      {
        uint32_t p[32];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 sh = *reinterpret_cast<const float4*>(shift + x * 32 + e);
            const uint64_t z0 = ptx::fma2(ptx::join2(s[x][e], s[x][e + 1]), c2, ptx::join2(__float_as_uint(sh.x), __float_as_uint(sh.y)));
            const uint64_t z1 = ptx::fma2(ptx::join2(s[x][e + 2], s[x][e + 3]), c2, ptx::join2(__float_as_uint(sh.z), __float_as_uint(sh.w)));
            s[x][e] = __float_as_uint(exp2_approx(ptx::lo2(z0))), s[x][e + 1] = __float_as_uint(exp2_approx(ptx::hi2(z0)));
            s[x][e + 2] = __float_as_uint(exp2_approx(ptx::lo2(z1))), s[x][e + 3] = __float_as_uint(exp2_approx(ptx::hi2(z1)));
          }
        if (!all) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const int4 n = *reinterpret_cast<const int4*>(seen + x * 32 + e);
              if (key >= n.x) s[x][e] = 0;
              if (key >= n.y) s[x][e + 1] = 0;
              if (key >= n.z) s[x][e + 2] = 0;
              if (key >= n.w) s[x][e + 3] = 0;
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 32; e += 2) p[x * 16 + e / 2] = pack2<T>(__uint_as_float(s[x][e]), __uint_as_float(s[x][e + 1]));
        ptx::tmem_st_regs(s_at, p);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(p_full);
      if (!warp_wait_or_record(dp_full, i & 1, tl.wait_limit, WAIT_BACK_DP)) { ok = false; break; }
      ptx::tc_fence_after();
      // dS
      {
        uint32_t g[2][32];
#pragma unroll
        for (int x = 0; x < 2; ++x) ptx::tmem_ld_regs(dp_at + 32 * x, g[x]);
#pragma unroll
        for (int x = 0; x < 2; ++x) ptx::tmem_wait_regs(g[x]);
        uint32_t p[32];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 dl = *reinterpret_cast<const float4*>(delta + x * 32 + e);
            uint64_t y0 = ptx::fma2(ptx::join2(__float_as_uint(dl.x), __float_as_uint(dl.y)), minus, ptx::join2(g[x][e], g[x][e + 1]));
            uint64_t y1 = ptx::fma2(ptx::join2(__float_as_uint(dl.z), __float_as_uint(dl.w)), minus, ptx::join2(g[x][e + 2], g[x][e + 3]));
            uint64_t p0 = ptx::join2(s[x][e], s[x][e + 1]), p1 = ptx::join2(s[x][e + 2], s[x][e + 3]);
            if (HALF) p0 = ptx::mul2(p0, f2), p1 = ptx::mul2(p1, f2);
            y0 = ptx::mul2(p0, y0), y1 = ptx::mul2(p1, y1);
            g[x][e] = (uint32_t)y0, g[x][e + 1] = (uint32_t)(y0 >> 32), g[x][e + 2] = (uint32_t)y1, g[x][e + 3] = (uint32_t)(y1 >> 32);
          }
        if (!all) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const int4 n = *reinterpret_cast<const int4*>(seen + x * 32 + e);
              if (key >= n.x) g[x][e] = 0;
              if (key >= n.y) g[x][e + 1] = 0;
              if (key >= n.z) g[x][e + 2] = 0;
              if (key >= n.w) g[x][e + 3] = 0;
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 32; e += 2) p[x * 16 + e / 2] = pack2<T>(__uint_as_float(g[x][e]), __uint_as_float(g[x][e + 1]));
        ptx::tmem_st_regs(dp_at, p);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(ds_full);
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&st_empty[r.at]);
    }
    if (ok && steps) ok = warp_wait_or_record(done, 0, tl.wait_limit, WAIT_BACK_DONE);
    ptx::tc_fence_after();
    // the first warpgroup's rows are of dV, the second's of dK
    const int64_t t = u.t0 + key;
    const bool keys = half == 1;
    void* base = keys ? a.dk : a.dv;
    const bool mine = ok && base && t < kr.end;
    RowsOut<DP / 8> rows_out{smem + half * C::TILE + (warp & 3) * 32 * DP * 2};      // (the places of K and V: their products are done)
    const float f = keys ? a.scale / factor_of() : exp2f(-P_LOG2<T>);
    const uint64_t out2 = ptx::join2(__float_as_uint(f), __float_as_uint(f));
    uint64_t worst = 0;                                      // NaN where a gradient is NaN or infinite
#pragma unroll
    for (int x = 0; x < DP; x += 32) {
      uint32_t o[32];
      if (steps) {
        ptx::tmem_ld_regs(lanes + KV_DV + half * DP + x, o);
        ptx::tmem_wait_regs(o);
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8)
        if (x + e < a.D) {
          uint32_t v[4];
          round8<T>(o + e, out2, false, worst, v);
          if (!steps) v[0] = v[1] = v[2] = v[3] = 0;         // whatever its place held
          rows_out.put((x + e) / 8, v);
        }
    }
    rows_out.store(static_cast<T*>(base) + (t * a.Hk + u.kh) * a.D, mine, a.D / 8);
    // A query that does not see the key was multiplied by 0, which infinities and NaN turn into NaN: such rows are made
    // again from the queries that see them alone.
    const bool bad = mine && steps && (ptx::lo2(worst) != 0.0f || ptx::hi2(worst) != 0.0f);
    const uint32_t rows = __any_sync(0xFFFFFFFFu, bad) ? keys_made_again<T>(a, tl, keys, key, bad) : 0;
    if (rows && keys) make_again<T, AGAIN_DK>(a, w.stats, rows, u.b, t, u.kh, make_float2(0.0f, 0.0f), 0, a.D);
    else if (rows) make_again<T, AGAIN_DV>(a, w.stats, rows, u.b, t, u.kh, make_float2(0.0f, 0.0f), 0, a.D);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(*tmem_slot, 512);
  }
}

// ------------------------------------------------------------------------------ the queries' gradients
// A CTA owns a tile of up to 128 rows of queries (all heads of a group) and walks over the keys that they see in tiles of 128:
// S = Q K^T, dP = dO V^T, dQ += dS K, with dS from tensor memory.  Tensor memory: S twice, dP (then dS), dQ.
//   warps 0-7   the elements, a thread to a row and half of the tile's keys; at the end half of a row of dQ
//   warp 8      MMA issuer;  warp 9  TMA
template <int DP> struct Dq {
  static constexpr int TILE = 128 * DP * 2;
  static constexpr int K_SLOTS = DP == 128 ? 3 : 5, V_SLOTS = DP == 128 ? 2 : 5;
  static constexpr int BARS = 1 + 2 * K_SLOTS + 2 * V_SLOTS + 5;
  static constexpr int SMEM = 1024 + (2 + K_SLOTS + V_SLOTS) * TILE + BARS * 8 + 16;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
constexpr uint32_t DQ_S = 0, DQ_DP = 256, DQ_SUM = 384;

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1) attention_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                                                                 const __grid_constant__ AttnArgs a, const __grid_constant__ Tiling tl) {
  using C = Dq<DP>;
  extern __shared__ uint8_t smem_raw[];
  const Unit u = unit_of(a, tl, a.cu_q, a.Tq, 1);
  if (!u.any) return;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Rows qr = u.rows, kr = u.b < a.B ? rows_of(a.cu_k, u.b, a.Tk) : Rows{0, 0};
  const int64_t nq = qr.count(), nk = kr.count();
  const int64_t last = min(u.t0 + tl.tokens, qr.end) - 1 - qr.begin;
  const int64_t most = a.causal ? max((int64_t)0, min(nk, last + 1 + nk - nq)) : nk;
  const int tiles = (int)((most + 127) / 128);

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring_k = smem + 2 * C::TILE;                      // Q, dO first
  uint8_t* ring_v = ring_k + C::K_SLOTS * C::TILE;
  uint64_t* fixed = reinterpret_cast<uint64_t*>(ring_v + C::V_SLOTS * C::TILE);
  uint64_t* k_full = fixed + 1;
  uint64_t* k_empty = k_full + C::K_SLOTS;
  uint64_t* v_full = k_empty + C::K_SLOTS;
  uint64_t* v_empty = v_full + C::V_SLOTS;
  uint64_t* s_full = v_empty + C::V_SLOTS;                   // two
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&map_q), ptx::prefetch_tmap(&map_k), ptx::prefetch_tmap(&map_v), ptx::prefetch_tmap(&map_g);
    ptx::mbar_init(fixed, 1);
    for (int i = 0; i < C::K_SLOTS; ++i) ptx::mbar_init(&k_full[i], 1), ptx::mbar_init(&k_empty[i], 1);
    for (int i = 0; i < C::V_SLOTS; ++i) ptx::mbar_init(&v_full[i], 1), ptx::mbar_init(&v_empty[i], 1);
    ptx::mbar_init(&s_full[0], 1), ptx::mbar_init(&s_full[1], 1), ptx::mbar_init(dp_full, 1), ptx::mbar_init(ds_full, 256), ptx::mbar_init(done, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp >= 8) {
    ptx::setmaxnreg_dec<REG_LOW>();
    if (warp == 9 && lane == 0 && tiles) {
      const int head = u.kh * tl.group + u.chunk * tl.heads;
      ptx::mbar_arrive_expect_tx(fixed, 2 * (DP / 64) * tl.heads * tl.tokens * 128);
      for (int x = 0; x < DP / 64; ++x) {
        ptx::tma_load_3d(smem + x * 16384, &map_q, fixed, x * 64, head, (int)u.t0);
        ptx::tma_load_3d(smem + C::TILE + x * 16384, &map_g, fixed, x * 64, head, (int)u.t0);
      }
      Ring<C::K_SLOTS> k;
      Ring<C::V_SLOTS> v;
      int keys = 0, j = 0;                                   // tiles of K and of V asked for
      for (; j < tiles; ++j, k.next(), v.next()) {
        const int row = (int)(kr.begin + (int64_t)j * 128);
        if (j >= C::K_SLOTS && !wait_or_record(&k_empty[k.at], k.parity ^ 1, tl.wait_limit, WAIT_BACK_SLOT)) break;
        ptx::mbar_arrive_expect_tx(&k_full[k.at], C::TILE);
        for (int x = 0; x < DP / 64; ++x) ptx::tma_load_3d(ring_k + k.at * C::TILE + x * 16384, &map_k, &k_full[k.at], x * 64, u.kh, row);
        ++keys;
        if (j >= C::V_SLOTS && !wait_or_record(&v_empty[v.at], v.parity ^ 1, tl.wait_limit, WAIT_BACK_SLOT)) break;
        ptx::mbar_arrive_expect_tx(&v_full[v.at], C::TILE);
        for (int x = 0; x < DP / 64; ++x) ptx::tma_load_3d(ring_v + v.at * C::TILE + x * 16384, &map_v, &v_full[v.at], x * 64, u.kh, row);
      }
      drain<1>(fixed, 1), drain<C::K_SLOTS>(k_full, keys), drain<C::V_SLOTS>(v_full, j);
    } else if (warp == 8 && tiles) {
      const uint32_t tmem = *tmem_slot;
      constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
      const uint32_t id_s = ptx::idesc_16_f32(128, 128, BF, false), id_d = ptx::idesc_16_f32(128, tl.d16, BF, true);
      const int ks = tl.d16 / 16;
      auto outer = [&](uint32_t d, const uint8_t* x, const uint8_t* y) {       // [queries][keys] = x y^T over the head
        const uint32_t xa = ptx::smem_u32(x), ya = ptx::smem_u32(y);
        for (int s = 0; s < ks; ++s) {
          const uint32_t at = (s / 4) * 16384 + (s % 4) * 32;
          ptx::mma_f16(tmem + d, ptx::smem_desc_sw128(xa + at), ptx::smem_desc_sw128(ya + at), id_s, s > 0);
        }
      };
      bool ok = warp_wait_or_record(fixed, 0, tl.wait_limit, WAIT_BACK_FIXED);
      ok = ok && warp_wait_or_record(&k_full[0], 0, tl.wait_limit, WAIT_BACK_TILE);
      ok = ok && warp_wait_or_record(&v_full[0], 0, tl.wait_limit, WAIT_BACK_TILE);
      ptx::tc_fence_after();
      if (ok && ptx::elect_one()) {
        outer(DQ_S, smem, ring_k);
        if (!tl.hold_first_ready) ptx::mma_commit(&s_full[0]);
        outer(DQ_DP, smem + C::TILE, ring_v);
        ptx::mma_commit(dp_full);
        ptx::mma_commit(&v_empty[0]);
      }
      __syncwarp();
      Ring<C::K_SLOTS> k, kn;
      Ring<C::V_SLOTS> vn;
      for (int j = 0; j < tiles && ok; ++j, k.next()) {
        const bool next = j + 1 < tiles;
        kn.next(), vn.next();
        if (next) {
          // S's other half: its last tile, j - 1, has been read, as ds of that tile was there
          if (!warp_wait_or_record(&k_full[kn.at], kn.parity, tl.wait_limit, WAIT_BACK_TILE)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            outer(DQ_S + ((j + 1) & 1) * 128, smem, ring_k + kn.at * C::TILE);
            ptx::mma_commit(&s_full[(j + 1) & 1]);
          }
          __syncwarp();
        }
        if (!warp_wait_or_record(ds_full, j & 1, tl.wait_limit, WAIT_BACK_DS)) { ok = false; break; }
        if (next && !warp_wait_or_record(&v_full[vn.at], vn.parity, tl.wait_limit, WAIT_BACK_TILE)) { ok = false; break; }
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          const uint64_t b = ptx::smem_desc_mn_sw128(ptx::smem_u32(ring_k + k.at * C::TILE), 16384);
#pragma unroll
          for (int s = 0; s < 8; ++s)
            ptx::mma_f16_ta(tmem + DQ_SUM, tmem + DQ_DP + (s / 4) * 64 + (s % 4) * 8, b + s * 128, id_d, j > 0 || s > 0);
          ptx::mma_commit(&k_empty[k.at]);
          if (next) {
            outer(DQ_DP, smem + C::TILE, ring_v + vn.at * C::TILE);
            ptx::mma_commit(dp_full);
            ptx::mma_commit(&v_empty[vn.at]);
          }
        }
        __syncwarp();
      }
      if (ptx::elect_one()) ptx::mma_commit(done);           // after a failed wait too: the MMAs in flight are waited for
      __syncwarp();
      warp_wait_or_record(done, 0, DRAIN_LIMIT, WAIT_DRAIN);
    }
  } else {
    ptx::setmaxnreg_inc<REG_HIGH>();
    const uint32_t tmem = *tmem_slot;
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t dp_at = lanes + DQ_DP + half * 64;
    const int64_t t = u.t0 + r / tl.heads;
    const int gh = u.chunk * tl.heads + r % tl.heads, h = u.kh * tl.group + gh;
    const bool mine = r < tl.heads * tl.tokens && gh < tl.group && t < qr.end;
    const int64_t n = !mine ? 0 : a.causal ? max((int64_t)0, min(nk, t - qr.begin + 1 + nk - nq)) : nk;
    const int64_t first = a.causal ? u.t0 - qr.begin + 1 + nk - nq : nk;     // keys that every row sees
    const Work w = work_of(a);
    const float2 st = mine ? w.stats[t * a.Hq + h] : make_float2(0.0f, 0.0f);
    const bool scaled = std::is_same<T, __half>::value && mine && u.b < a.B;
    const float factor = scaled ? ds_factor(w.norms[t * a.Hq + h], __uint_as_float(__ldg(w.top_v + u.b * a.Hk + u.kh))) : 1.0f;
    const float c = a.scale * 1.4426950408889634f;
    const uint64_t c2 = ptx::join2(__float_as_uint(c), __float_as_uint(c)), sh2 = ptx::join2(__float_as_uint(st.x), __float_as_uint(st.x));
    const uint64_t dl2 = ptx::join2(__float_as_uint(-st.y), __float_as_uint(-st.y)), f2 = ptx::join2(__float_as_uint(factor), __float_as_uint(factor));
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      if (!warp_wait_or_record(&s_full[j & 1], (j >> 1) & 1, tl.wait_limit, WAIT_BACK_S)) { ok = false; break; }
      ptx::tc_fence_after();
      const uint32_t s_at = lanes + DQ_S + (j & 1) * 128 + half * 64;
      uint32_t s[2][32];
#pragma unroll
      for (int x = 0; x < 2; ++x) ptx::tmem_ld_regs(s_at + 32 * x, s[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x) ptx::tmem_wait_regs(s[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t z = ptx::fma2(ptx::join2(s[x][e], s[x][e + 1]), c2, sh2);
          s[x][e] = __float_as_uint(exp2_approx(ptx::lo2(z))), s[x][e + 1] = __float_as_uint(exp2_approx(ptx::hi2(z)));
        }
      if (!warp_wait_or_record(dp_full, j & 1, tl.wait_limit, WAIT_BACK_DP)) { ok = false; break; }
      ptx::tc_fence_after();
      uint32_t g[2][32], p[32];
#pragma unroll
      for (int x = 0; x < 2; ++x) ptx::tmem_ld_regs(dp_at + 32 * x, g[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x) ptx::tmem_wait_regs(g[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          uint64_t y = ptx::add2(ptx::join2(g[x][e], g[x][e + 1]), dl2), q = ptx::join2(s[x][e], s[x][e + 1]);
          if (std::is_same<T, __half>::value) q = ptx::mul2(q, f2);
          y = ptx::mul2(q, y);
          g[x][e] = (uint32_t)y, g[x][e + 1] = (uint32_t)(y >> 32);
        }
      if ((int64_t)(j + 1) * 128 > first || (int64_t)(j + 1) * 128 > nk) {
        const int lim = (int)max((int64_t)0, min((int64_t)128, n - (int64_t)j * 128)) - half * 64;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (x * 32 + e >= lim) g[x][e] = 0;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 32; e += 2) p[x * 16 + e / 2] = pack2<T>(__uint_as_float(g[x][e]), __uint_as_float(g[x][e + 1]));
      ptx::tmem_st_regs(dp_at, p);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(ds_full);
    }
    if (ok && tiles) ok = warp_wait_or_record(done, 0, tl.wait_limit, WAIT_BACK_DONE);
    ptx::tc_fence_after();
    constexpr int HALF = DP / 2;
    RowsOut<HALF / 8> rows_out{smem + (half * 128 + (warp & 3) * 32) * HALF * 2};    // (Q's place: its products are done)
    const float f = a.scale / factor;
    const uint64_t out2 = ptx::join2(__float_as_uint(f), __float_as_uint(f));
    uint64_t worst = 0;                                      // NaN where a gradient is NaN or infinite
#pragma unroll
    for (int x = 0; x < HALF; x += 32) {
      uint32_t o[32];
      if (tiles) {
        ptx::tmem_ld_regs(lanes + DQ_SUM + half * HALF + x, o);
        ptx::tmem_wait_regs(o);
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8)
        if (half * HALF + x + e < a.D) {
          uint32_t v[4];
          round8<T>(o + e, out2, false, worst, v);
          if (n <= 0) v[0] = v[1] = v[2] = v[3] = 0;         // whatever its place held
          rows_out.put((x + e) / 8, v);
        }
    }
    rows_out.store(static_cast<T*>(a.dq) + (t * a.Hq + h) * a.D + half * HALF, mine && ok, (a.D - half * HALF) / 8);
    // a hidden key that is infinite or NaN: the row again, from the keys that it sees alone (this thread's half of it)
    const bool redo = mine && ok && n > 0 && (ptx::lo2(worst) != 0.0f || ptx::hi2(worst) != 0.0f);
    const int d0 = half * HALF, d1 = min(a.D, (half + 1) * HALF);
    const uint32_t rows = __any_sync(0xFFFFFFFFu, redo) ? rows_made_again<T, false>(a, redo, u.b, (int)n, (int64_t)tiles * 128, u.kh, d0, d1, static_cast<T*>(nullptr)) : 0;
    if (rows) make_again<T, AGAIN_DQ>(a, w.stats, rows, u.b, t, h, st, d0, d1);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(*tmem_slot, 512);
  }
}

template <typename T, int DP> cudaError_t launch(const AttnArgs& a, cudaStream_t stream) {
  CUtensorMap mq, mk, mv, mg;
  const Tiling tl = tiling_of(a);
  const cudaError_t bound = bind_context();
  if (bound != cudaSuccess) return bound;
  if (!make_rows_map(&mq, a.q, a.Tq, a.Hq, a.D, a.q_stride, a.dtype, tl.heads, tl.tokens) ||
      !make_rows_map(&mg, a.dout, a.Tq, a.Hq, a.D, a.dout_stride, a.dtype, tl.heads, tl.tokens) ||
      !make_rows_map(&mk, a.k, a.Tk, a.Hk, a.D, a.k_stride, a.dtype, 1, 128) || !make_rows_map(&mv, a.v, a.Tk, a.Hk, a.D, a.v_stride, a.dtype, 1, 128))
    return cudaErrorUnknown;
  attention_stats_kernel<T><<<(unsigned)((a.Tq * a.Hq + 15) / 16), 256, 0, stream>>>(a);
  if (std::is_same<T, __half>::value) {
    const cudaError_t e = cudaMemsetAsync(work_of(a).top_g, 0, (size_t)a.B * a.Hk * 8, stream);
    if (e != cudaSuccess) return e;
    const int64_t queries = norm_warps(a.Tq, a.Hk), warps = queries + norm_warps(a.Tk, a.Hk);
    attention_norms_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(a, queries, warps);
  }
  if ((a.dk || a.dv) && a.Tk) {
    auto kernel = attention_dkv_kernel<T, DP>;
    static std::atomic<uint64_t> set{0};
    const cudaError_t e = allow_shared(kernel, Kv<DP>::SMEM, set);
    if (e != cudaSuccess) return e;
    const int64_t grid = units(a.Tk, a.B, 128) * a.Hk;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    kernel<<<(unsigned)grid, THREADS, Kv<DP>::SMEM, stream>>>(mq, mk, mv, mg, a, tl);
  }
  if (a.dq) {
    auto kernel = attention_dq_kernel<T, DP>;
    static std::atomic<uint64_t> set{0};
    const cudaError_t e = allow_shared(kernel, Dq<DP>::SMEM, set);
    if (e != cudaSuccess) return e;
    const int64_t grid = units(a.Tq, a.B, tl.tokens) * tl.chunks * a.Hk;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    kernel<<<(unsigned)grid, THREADS, Dq<DP>::SMEM, stream>>>(mq, mk, mv, mg, a, tl);
  }
  return cudaGetLastError();
}

}  // namespace

size_t attention_backward_workspace(int64_t Tq, int64_t B, int Hq, int Hk, int dtype) { return work_of(nullptr, Tq, B, Hq, Hk, dtype == EMU_DTYPE_F16).bytes; }

cudaError_t take_attention_backward_wait_error(int* code) { return take_error(code); }

cudaError_t launch_attention_backward(const AttnArgs& a, cudaStream_t stream) {
  const bool half = a.dtype == EMU_DTYPE_F16;
  if (a.D <= 64) return half ? launch<__half, 64>(a, stream) : launch<__nv_bfloat16, 64>(a, stream);
  return half ? launch<__half, 128>(a, stream) : launch<__nv_bfloat16, 128>(a, stream);
}

}  // namespace emu
