// Attention over packed sequences, forward pass (the formulas: attention.cuh), on the 5th-generation tensor cores.
//
// A CTA owns two tiles of up to 128 rows and walks over the keys in tiles of 128: S = Q K^T into tensor memory, one pass
// over S by the tile's warpgroup with the running maximum and sum of the softmax, P in 16 bits back into S's place, O += P V
// with P from tensor memory.  A row is (token, query head of the group): the tile holds all heads that share a key head, so
// that K and V are staged once for them and few queries still fill it.
//
//   warps 0-3, 4-7   softmax of the first and the second tile, a thread to a row; at the end its row's output
//   warp 8           MMA issuer: for each tile in turn O += P V of the tile of keys before, then S of the next, so that
//                    the tensor cores work on one tile while the other's softmax runs.  Owns the tensor memory.
//   warp 9           TMA: Q once, then K and V tiles through a ring
//
// Bound by the tensor cores, and on long inputs by power: 16384 causal tokens, 32 heads on 8 of 128, bf16: 2.0 ms, 1.10 PFLOP/s (79%
// of a sustained library product's rate; the SM clock falls to 1.4 .. 1.7 GHz).  8192 tokens in 3 sequences, with
// the rest for a backward pass, 249 us.  S is
// not rounded, l and O are held in f32; the weights are rounded to the inputs' type (by up to 2^-8 or 2^-11 of them), which is
// what the second product takes.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "../../include/emugen.h"
#include "attention.cuh"
#include "attention_tc.cuh"
#include "tc_ptx.cuh"

namespace emu {
namespace {

using namespace attn;

constexpr int THREADS = 384;                                // the third warpgroup's rest fills it up
// 128 threads x 40 + 256 x 232 = 64512 = 384 x 168, what the CTA is launched with
constexpr int REG_LOW = 40, REG_HIGH = 232;

template <int DP> struct Fwd {
  static constexpr int TILE = 128 * DP * 2;                 // 128 rows of DP elements, as DP / 64 boxes of 128 x 128 bytes
  static constexpr int SLOTS = DP == 128 ? 5 : 8;           // ring of K and V tiles in turn
  static constexpr int BARS = 1 + 2 * SLOTS + 2 + 2 + 2;
  static constexpr int SMEM = 1024 + 2 * TILE + SLOTS * TILE + BARS * 8 + 16;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
// fp16: P, and with it l and O, is held 2^7 times as large.  P is below 2^8 (the maximum is held up to that factor), so that it
// stays below 2^15, and weights down to 2^-21 keep all their bits, those down to 2^-31 some; without it they were lost from 2^-14 and
// gone below 2^-25, and 16384 keys 18 below a first one came out as zeros.  bf16 has f32's range.
template <typename T> __device__ __forceinline__ float held_shift(float m, float c) {
  return std::is_same<T, __half>::value ? shift_of(m, c) + 7.0f : shift_of(m, c);
}

// tensor memory columns: S (and P) of both tiles, O of both tiles
constexpr uint32_t S_COL = 0, O_COL = 256;

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1) attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a,
                                                              const __grid_constant__ Tiling tl) {
  using C = Fwd<DP>;
  extern __shared__ uint8_t smem_raw[];
  const Unit u = unit_of(a, tl, a.cu_q, a.Tq, 2);
  if (!u.any) return;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Rows qr = u.rows;
  const Rows kr = u.b < a.B ? rows_of(a.cu_k, u.b, a.Tk) : Rows{0, 0};
  const int64_t nq = qr.count(), nk = kr.count();
  // keys that the unit's last token sees
  const int64_t last = min(u.t0 + 2 * tl.tokens, qr.end) - 1 - qr.begin;
  const int64_t most = a.causal ? max((int64_t)0, min(nk, last + 1 + nk - nq)) : nk;
  const int tiles = (int)((most + 127) / 128);

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = smem + 2 * C::TILE;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + C::SLOTS * C::TILE);
  uint64_t* kv_full = q_full + 1;
  uint64_t* kv_empty = kv_full + C::SLOTS;
  uint64_t* s_full = kv_empty + C::SLOTS;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&map_q), ptx::prefetch_tmap(&map_k), ptx::prefetch_tmap(&map_v);
    ptx::mbar_init(q_full, 1);
    for (int i = 0; i < C::SLOTS; ++i) ptx::mbar_init(&kv_full[i], 1), ptx::mbar_init(&kv_empty[i], 1);
    for (int i = 0; i < 2; ++i) ptx::mbar_init(&s_full[i], 1), ptx::mbar_init(&p_full[i], 128), ptx::mbar_init(&o_full[i], 1);
    ptx::fence_mbar_init();
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // no load may be in flight across the register split: the TMEM address is read after it
  if (warp >= 8) {
    ptx::setmaxnreg_dec<REG_LOW>();
    if (warp == 9 && lane == 0 && tiles) {
      const int head = u.kh * tl.group + u.chunk * tl.heads;
      ptx::mbar_arrive_expect_tx(q_full, 2 * (DP / 64) * tl.heads * tl.tokens * 128);
      for (int i = 0; i < 2; ++i)
        for (int x = 0; x < DP / 64; ++x)
          ptx::tma_load_3d(smem + i * C::TILE + x * 16384, &map_q, q_full, x * 64, head, (int)(u.t0 + i * tl.tokens));
      Ring<C::SLOTS> r;
      int i = 0;
      for (; i < 2 * tiles; ++i, r.next()) {
        if (i >= C::SLOTS && !wait_or_record(&kv_empty[r.at], r.parity ^ 1, tl.wait_limit, WAIT_FWD_SLOT)) break;
        ptx::mbar_arrive_expect_tx(&kv_full[r.at], C::TILE);
        for (int x = 0; x < DP / 64; ++x)
          ptx::tma_load_3d(ring + r.at * C::TILE + x * 16384, i & 1 ? &map_v : &map_k, &kv_full[r.at], x * 64, u.kh, (int)(kr.begin + (i >> 1) * 128));
      }
      drain<1>(q_full, 1), drain<C::SLOTS>(kv_full, i);
    } else if (warp == 8 && tiles) {
      const uint32_t tmem = *tmem_slot;
      constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
      const uint32_t id_s = ptx::idesc_16_f32(128, 128, BF, false), id_o = ptx::idesc_16_f32(128, tl.d16, BF, true);
      const int steps = tl.d16 / 16;
      bool ok = warp_wait_or_record(q_full, 0, tl.wait_limit, WAIT_FWD_Q);
      auto scores = [&](int i, int slot) {                   // S_i = Q_i K^T
        const uint32_t q = ptx::smem_u32(smem + i * C::TILE), k = ptx::smem_u32(ring + slot * C::TILE);
        for (int s = 0; s < steps; ++s) {
          const uint32_t at = (s / 4) * 16384 + (s % 4) * 32;
          ptx::mma_f16(tmem + S_COL + i * 128, ptx::smem_desc_sw128(q + at), ptx::smem_desc_sw128(k + at), id_s, s > 0);
        }
      };
      auto values = [&](int i, int slot, bool more) {        // O_i += P_i V
        const uint64_t v = ptx::smem_desc_mn_sw128(ptx::smem_u32(ring + slot * C::TILE), 16384);
#pragma unroll
        for (int s = 0; s < 8; ++s)
          ptx::mma_f16_ta(tmem + O_COL + i * DP, tmem + S_COL + i * 128 + s * 8, v + s * 128, id_o, more || s > 0);
      };
      Ring<C::SLOTS> k, v;                                   // of the keys and of the values before them
      v.next();
      uint32_t parity = 0;                                   // of P
      for (int j = 0; j < tiles && ok; ++j) {
        if (j > 0 && !warp_wait_or_record(&kv_full[v.at], v.parity, tl.wait_limit, WAIT_FWD_V)) { ok = false; break; }
        if (!warp_wait_or_record(&kv_full[k.at], k.parity, tl.wait_limit, WAIT_FWD_K)) { ok = false; break; }
        for (int i = 0; i < 2 && ok; ++i) {
          if (j > 0 && !warp_wait_or_record(&p_full[i], parity ^ 1, tl.wait_limit, WAIT_FWD_P)) ok = false;
          ptx::tc_fence_after();
          if (ok && ptx::elect_one()) {
            if (j > 0) values(i, v.at, j > 1);
            scores(i, k.at);
            if (!(j == 0 && i == 0 && tl.hold_first_ready)) ptx::mma_commit(&s_full[i]);
          }
          __syncwarp();
        }
        if (ok && ptx::elect_one()) {
          if (j > 0) ptx::mma_commit(&kv_empty[v.at]);
          ptx::mma_commit(&kv_empty[k.at]);
        }
        __syncwarp();
        k.next(), k.next();
        if (j > 0) v.next(), v.next();
        parity ^= 1;
      }
      if (ok) ok = warp_wait_or_record(&kv_full[v.at], v.parity, tl.wait_limit, WAIT_FWD_V);
      for (int i = 0; i < 2; ++i) {
        if (ok) ok = warp_wait_or_record(&p_full[i], parity ^ 1, tl.wait_limit, WAIT_FWD_P);
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          if (ok) values(i, v.at, tiles > 1);
          ptx::mma_commit(&o_full[i]);                       // after a failed wait too: the MMAs in flight are waited for
        }
        __syncwarp();
      }
      warp_wait_or_record(&o_full[1], 0, DRAIN_LIMIT, WAIT_DRAIN);
    }
  } else {
    ptx::setmaxnreg_inc<REG_HIGH>();
    const uint32_t tmem = *tmem_slot;
    // softmax of tile i, row r
    const int i = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + S_COL + i * 128, o_at = lanes + O_COL + i * DP;
    const int64_t t = u.t0 + i * tl.tokens + r / tl.heads;
    const int gh = u.chunk * tl.heads + r % tl.heads, h = u.kh * tl.group + gh;
    const bool mine = r < tl.heads * tl.tokens && gh < tl.group && t < qr.end;
    // this row sees the first n keys
    const int64_t n = !mine ? 0 : a.causal ? max((int64_t)0, min(nk, t - qr.begin + 1 + nk - nq)) : nk;
    // all rows of the tile see the first n0
    const int64_t first = a.causal ? u.t0 + i * tl.tokens - qr.begin + 1 + nk - nq : nk;
    const float c = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      if (!warp_wait_or_record(&s_full[i], j & 1, tl.wait_limit, WAIT_FWD_S)) { ok = false; break; }
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_ld_regs(s_at + 32 * x, s[x]);
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_wait_regs(s[x]);
      if ((int64_t)(j + 1) * 128 > first || (int64_t)(j + 1) * 128 > nk) {      // the same for the whole tile
        const int lim = (int)max((int64_t)0, min((int64_t)128, n - (int64_t)j * 128));
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (x * 32 + e >= lim) s[x][e] = 0xFF800000u;
      }
      float top[4] = {m, m, m, m};
#pragma unroll
      for (int e = 0; e < 32; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) top[x] = fmaxf(top[x], __uint_as_float(s[x][e]));
      const float tm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      // The weights are held to the maximum up to a factor of 2^8: P, l and O stay in range, and most
      // tiles need no correction of O.
      const bool grow = (tm - m) * c > 8.0f;
      if (__any_sync(0xFFFFFFFFu, grow)) {
        const float f = tm == -INFINITY ? 1.0f : exp2f((m - tm) * c);
        l *= f;
        m = tm;
        if (j > 0) {
#pragma unroll
          for (int x = 0; x < DP; x += 32) {
            uint32_t o[32];
            ptx::tmem_ld_regs(o_at + x, o);
            ptx::tmem_wait_regs(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            ptx::tmem_st_regs(o_at + x, o);
          }
        }
      }
      const float shift = held_shift<T>(m, c);
      const uint64_t c2 = ptx::join2(__float_as_uint(c), __float_as_uint(c)), sh2 = ptx::join2(__float_as_uint(shift), __float_as_uint(shift));
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int x = 0; x < 4; x += 2) {
        uint32_t p[32];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint64_t z = ptx::fma2(ptx::join2(s[x + y][e], s[x + y][e + 1]), c2, sh2);
            const float p0 = exp2_approx(ptx::lo2(z)), p1 = exp2_approx(ptx::hi2(z));
            sum[y] = ptx::add2(sum[y], ptx::join2(__float_as_uint(p0), __float_as_uint(p1)));
            p[y * 16 + e / 2] = pack2<T>(p0, p1);
          }
        ptx::tmem_st_regs(s_at + 16 * x, p);
      }
      const uint64_t all = ptx::add2(sum[0], sum[1]);
      l += ptx::lo2(all) + ptx::hi2(all);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(&p_full[i]);
    }
    bool redo = false;
    if (ok && tiles) ok = warp_wait_or_record(&o_full[i], 0, tl.wait_limit, WAIT_FWD_O);
    ptx::tc_fence_after();
    const float f = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    const uint64_t f2 = ptx::join2(__float_as_uint(f), __float_as_uint(f));
    uint64_t worst = 0;                                      // NaN where an output is NaN or infinite
    RowsOut<DP / 8> rows_out{smem + i * C::TILE + (warp & 3) * 32 * DP * 2};         // (Q's place: its products are done)
    for (int pass = 0; pass < (a.low ? 2 : 1); ++pass) {     // the output, and what its rounding took away
#pragma unroll
      for (int x = 0; x < DP; x += 32) {
        uint32_t o[32];
        if (tiles) {
          ptx::tmem_ld_regs(o_at + x, o);
          ptx::tmem_wait_regs(o);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          if (x + e < a.D) {
            uint32_t v[4];
            round8<T>(o + e, f2, pass, worst, v);
            if (n <= 0) v[0] = v[1] = v[2] = v[3] = 0;                 // whatever its place held
            rows_out.put((x + e) / 8, v);
          }
      }
      rows_out.store(static_cast<T*>(pass ? a.low : a.out) + (t * a.Hq + h) * a.D, mine && ok, a.D / 8);
    }
    if (mine && ok && a.lse) a.lse[(int64_t)h * a.Tq + t] = n == 0 || l == 0.0f ? -INFINITY : l > 0.0f ? (log2f(l) - held_shift<T>(m, c)) * 0.6931471805599453f : l;
    // A value that the mask hides was multiplied by 0, which infinities and NaN turn into NaN: such rows are made again
    // from the keys that they see alone.  (Where the sum is NaN, the scores are, and the row is NaN by right.)
    redo = mine && ok && n > 0 && (ptx::lo2(worst) != 0.0f || ptx::hi2(worst) != 0.0f) && l > 0.0f;
    T* low = a.low ? static_cast<T*>(a.low) + (t * a.Hq + h) * a.D : nullptr;
    const uint32_t rows = __any_sync(0xFFFFFFFFu, redo) ? rows_made_again<T, true>(a, redo, u.b, (int)n, (int64_t)tiles * 128, u.kh, 0, a.D, low) : 0;
    if (rows) make_again<T, AGAIN_OUT>(a, nullptr, rows, u.b, t, h, make_float2(held_shift<T>(m, c), f), 0, a.D);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(*tmem_slot, 512);
  }
}

// ------------------------------------------------------------------------------ few tiles of rows
// Where there are fewer pairs of tiles than SMs, a CTA owns one tile of rows and its two warpgroups take the tiles of keys in
// turn, so that a tile of rows takes half the time.  Tensor memory holds S (and P) of three tiles of keys beside O: a tile's
// products run ahead of and behind its softmax.
//
//   warps 0-3, 4-7   softmax of every other tile of keys, a thread to a row; at the end half of its row's output each
//   warps 8, 10      MMA issuers, of S and of O += P V: an issuer is held up while its MMAs run, and the other's waits pass
//                    meanwhile (one for both: 650 of 1690 clocks a tile without an MMA).  Warp 8 owns the tensor memory.
//   warp 9           TMA: Q once, then K and V tiles through two rings
template <int DP> struct Few {
  static constexpr int TILE = 128 * DP * 2;                 // 128 rows of DP elements, as DP / 64 boxes of 128 x 128 bytes
  static constexpr int SLOTS = DP == 128 ? 3 : 5;           // of K, and of V
  static constexpr int BARS = 1 + 4 * SLOTS + 3 + 3 + 3 + 2 + 1 + 2;
  static constexpr int SMEM = 1024 + (1 + 2 * SLOTS) * TILE + BARS * 8 + 16 + 3 * 128 * 4;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
constexpr uint32_t FEW_O = 384;                             // tensor memory columns: S (and P) of three tiles, O

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1) attention_few_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a,
                                                              const __grid_constant__ Tiling tl) {
  using C = Few<DP>;
  extern __shared__ uint8_t smem_raw[];
  const Unit u = unit_of(a, tl, a.cu_q, a.Tq, 1);
  if (!u.any) return;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Rows qr = u.rows;
  const Rows kr = u.b < a.B ? rows_of(a.cu_k, u.b, a.Tk) : Rows{0, 0};
  const int64_t nq = qr.count(), nk = kr.count();
  // keys that the unit's last token sees
  const int64_t last = min(u.t0 + tl.tokens, qr.end) - 1 - qr.begin;
  const int64_t most = a.causal ? max((int64_t)0, min(nk, last + 1 + nk - nq)) : nk;
  const int tiles = (int)((most + 127) / 128);

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring_k = smem + C::TILE;
  uint8_t* ring_v = ring_k + C::SLOTS * C::TILE;
  float* ref = reinterpret_cast<float*>(ring_v + C::SLOTS * C::TILE);             // [row]: the maximum that the weights are held to
  float* sums = ref + 128;                                   // [warpgroup][row], at the end
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sums + 256);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + C::SLOTS;
  uint64_t* v_full = k_empty + C::SLOTS;
  uint64_t* v_empty = v_full + C::SLOTS;
  uint64_t* s_full = v_empty + C::SLOTS;                     // [place]
  uint64_t* p_full = s_full + 3;                             // [place]
  uint64_t* p_free = p_full + 3;                             // [place]: its weights' product, and so all before it, is in O
  uint64_t* ref_full = p_free + 3;                           // [warpgroup]: it has written `ref` of its tile
  uint64_t* o_full = ref_full + 2;
  uint64_t* drained = o_full + 1;                            // [issuer]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&map_q), ptx::prefetch_tmap(&map_k), ptx::prefetch_tmap(&map_v);
    ptx::mbar_init(q_full, 1), ptx::mbar_init(o_full, 1);
    for (int i = 0; i < C::SLOTS; ++i)
      ptx::mbar_init(&k_full[i], 1), ptx::mbar_init(&k_empty[i], 1), ptx::mbar_init(&v_full[i], 1), ptx::mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 3; ++i) ptx::mbar_init(&s_full[i], 1), ptx::mbar_init(&p_full[i], 128), ptx::mbar_init(&p_free[i], 1);
    for (int i = 0; i < 2; ++i) ptx::mbar_init(&ref_full[i], 128), ptx::mbar_init(&drained[i], 1);
    ptx::fence_mbar_init();
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // no load may be in flight across the register split: the TMEM address is read after it
  if (warp >= 8) {
    ptx::setmaxnreg_dec<REG_LOW>();
    if (warp == 9 && lane == 0 && tiles) {
      const int head = u.kh * tl.group + u.chunk * tl.heads;
      ptx::mbar_arrive_expect_tx(q_full, (DP / 64) * tl.heads * tl.tokens * 128);
      for (int x = 0; x < DP / 64; ++x) ptx::tma_load_3d(smem + x * 16384, &map_q, q_full, x * 64, head, (int)u.t0);
      Ring<C::SLOTS> k, v;
      int keys = 0, values = 0;                              // tiles asked for
      auto load = [&](const CUtensorMap* map, uint8_t* ring, uint64_t* full, uint64_t* empty, Ring<C::SLOTS>& r, int& j) {
        if (j >= C::SLOTS && !wait_or_record(&empty[r.at], r.parity ^ 1, tl.wait_limit, WAIT_FWD_SLOT)) return false;
        ptx::mbar_arrive_expect_tx(&full[r.at], C::TILE);
        for (int x = 0; x < DP / 64; ++x) ptx::tma_load_3d(ring + r.at * C::TILE + x * 16384, map, &full[r.at], x * 64, u.kh, (int)(kr.begin + (int64_t)j * 128));
        r.next(), ++j;
        return true;
      };
      // in the order of their use: K_0, K_1, K_2, V_0, K_3, V_1, ..
      bool ok = true;
      while (keys < min(3, tiles) && ok) ok = load(&map_k, ring_k, k_full, k_empty, k, keys);
      while (values < tiles && ok) {
        ok = load(&map_v, ring_v, v_full, v_empty, v, values);
        if (ok && keys < tiles) ok = load(&map_k, ring_k, k_full, k_empty, k, keys);
      }
      drain<1>(q_full, 1), drain<C::SLOTS>(k_full, keys), drain<C::SLOTS>(v_full, values);
    } else if ((warp == 8 || warp == 10) && tiles) {
      const uint32_t tmem = *tmem_slot;
      constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
      Ring<C::SLOTS> slot;
      Ring<3> place;
      bool ok = true;
      if (warp == 8) {                                       // S = Q K^T
        const uint32_t id = ptx::idesc_16_f32(128, 128, BF, false);
        const int ks = tl.d16 / 16;
        // descriptors of the first slot; a slot or a step of the sums further on is an addition to them
        const uint64_t q_desc = ptx::smem_desc_sw128(ptx::smem_u32(smem)), k_desc = ptx::smem_desc_sw128(ptx::smem_u32(ring_k));
        ok = warp_wait_or_record(q_full, 0, tl.wait_limit, WAIT_FWD_Q);
        for (int j = 0; j < tiles && ok; ++j, slot.next(), place.next()) {
          if (!warp_wait_or_record(&k_full[slot.at], slot.parity, tl.wait_limit, WAIT_FWD_K)) { ok = false; break; }
          // the weights of tile j - 3, in the same place, have been used
          if (j >= 3 && !warp_wait_or_record(&p_free[place.at], place.parity ^ 1, tl.wait_limit, WAIT_FWD_P)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t kd = k_desc + (uint32_t)(slot.at * (C::TILE >> 4));
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
              constexpr int BOX = 16384 >> 4, STEP = 32 >> 4;
              if (s < ks) ptx::mma_f16(tmem + place.at * 128, q_desc + (s / 4) * BOX + (s % 4) * STEP, kd + (s / 4) * BOX + (s % 4) * STEP, id, s > 0);
            }
            if (!(j == 0 && tl.hold_first_ready)) ptx::mma_commit(&s_full[place.at]);
            ptx::mma_commit(&k_empty[slot.at]);
          }
          __syncwarp();
        }
      } else {                                               // O += P V
        const uint32_t id = ptx::idesc_16_f32(128, tl.d16, BF, true);
        const uint64_t v_desc = ptx::smem_desc_mn_sw128(ptx::smem_u32(ring_v), 16384);
        for (int j = 0; j < tiles && ok; ++j, slot.next(), place.next()) {
          if (!warp_wait_or_record(&v_full[slot.at], slot.parity, tl.wait_limit, WAIT_FWD_V)) { ok = false; break; }
          if (!warp_wait_or_record(&p_full[place.at], place.parity, tl.wait_limit, WAIT_FWD_P)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t vd = v_desc + (uint32_t)(slot.at * (C::TILE >> 4));
#pragma unroll
            for (int s = 0; s < 8; ++s) ptx::mma_f16_ta(tmem + FEW_O, tmem + place.at * 128 + s * 8, vd + s * 128, id, j > 0 || s > 0);
            ptx::mma_commit(&p_free[place.at]);
            ptx::mma_commit(&v_empty[slot.at]);
            if (j + 1 == tiles) ptx::mma_commit(o_full);
          }
          __syncwarp();
        }
      }
      if (!ok) {                                             // the MMAs in flight are waited for
        uint64_t* bar = &drained[warp == 10];
        if (ptx::elect_one()) ptx::mma_commit(bar);
        __syncwarp();
        warp_wait_or_record(bar, 0, DRAIN_LIMIT, WAIT_DRAIN);
      }
    }
  } else {
    ptx::setmaxnreg_inc<REG_HIGH>();
    const uint32_t tmem = *tmem_slot;
    // softmax of row r, tiles w, w + 2, ..
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int64_t t = u.t0 + r / tl.heads;
    const int gh = u.chunk * tl.heads + r % tl.heads, h = u.kh * tl.group + gh;
    const bool mine = r < tl.heads * tl.tokens && gh < tl.group && t < qr.end;
    // this row sees the first n keys
    const int64_t n = !mine ? 0 : a.causal ? max((int64_t)0, min(nk, t - qr.begin + 1 + nk - nq)) : nk;
    // all rows of the tile see the first ones
    const int64_t first = a.causal ? u.t0 - qr.begin + 1 + nk - nq : nk;
    const float c = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = w; j < tiles; j += 2) {
      const int place = j % 3;
      const uint32_t s_at = lanes + place * 128;
      if (!warp_wait_or_record(&s_full[place], (j / 3) & 1, tl.wait_limit, WAIT_FWD_S)) { ok = false; break; }
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_ld_regs(s_at + 32 * x, s[x]);
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_wait_regs(s[x]);
      if ((int64_t)(j + 1) * 128 > first || (int64_t)(j + 1) * 128 > nk) {      // the same for the whole tile
        const int lim = (int)max((int64_t)0, min((int64_t)128, n - (int64_t)j * 128));
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (x * 32 + e >= lim) s[x][e] = 0xFF800000u;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) top[x] = fmaxf(top[x], __uint_as_float(s[x][e]));
      // The weights are held to the maximum up to a factor of 2^8: P, l and O stay in range, and most
      // tiles need no correction of O.  The other warpgroup has left what its tile, the one before, was held to.
      if (j > 0 && !warp_wait_or_record(&ref_full[w ^ 1], ((j - 1) >> 1) & 1, tl.wait_limit, WAIT_FWD_S)) { ok = false; break; }
      float now = j > 0 ? ref[r] : -INFINITY;
      const float tm = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), now);
      if (__any_sync(0xFFFFFFFFu, (tm - now) * c > 8.0f)) {
        if (j > 0) {
          // Tile j - 1's product has to be there; this tile's waits for its weights.  A wait for a parity tells a round from the
          // one before it alone, so the barrier may be at tile j - 1's round or the next, and it is: S of tile j - 1 waited for
          // the round before, and the next one's end, tile j + 2's product, is behind this tile's, which needs this warp.
          if (!warp_wait_or_record(&p_free[(j - 1) % 3], ((j - 1) / 3) & 1, tl.wait_limit, WAIT_FWD_O)) { ok = false; break; }
          ptx::tc_fence_after();
          const float f = tm == -INFINITY ? 1.0f : exp2f((now - tm) * c);
#pragma unroll
          for (int x = 0; x < DP; x += 32) {
            uint32_t o[32];
            ptx::tmem_ld_regs(lanes + FEW_O + x, o);
            ptx::tmem_wait_regs(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            ptx::tmem_st_regs(lanes + FEW_O + x, o);
          }
        }
        now = tm;
      }
      ref[r] = now;
      ptx::mbar_arrive(&ref_full[w]);
      if (__any_sync(0xFFFFFFFFu, now != m)) {               // this warpgroup's sum, from its own tile before
        l *= now == -INFINITY ? 1.0f : exp2f((m - now) * c);
        m = now;
      }
      const float shift = held_shift<T>(m, c);
      const uint64_t c2 = ptx::join2(__float_as_uint(c), __float_as_uint(c)), sh2 = ptx::join2(__float_as_uint(shift), __float_as_uint(shift));
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t p[32];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint64_t z = ptx::fma2(ptx::join2(s[2 * x + y][e], s[2 * x + y][e + 1]), c2, sh2);
            const float p0 = exp2_approx(ptx::lo2(z)), p1 = exp2_approx(ptx::hi2(z));
            sum[y] = ptx::add2(sum[y], ptx::join2(__float_as_uint(p0), __float_as_uint(p1)));
            p[y * 16 + e / 2] = pack2<T>(p0, p1);
          }
        ptx::tmem_st_regs(s_at + 32 * x, p);
      }
      const uint64_t all = ptx::add2(sum[0], sum[1]);
      l += ptx::lo2(all) + ptx::hi2(all);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(&p_full[place]);
    }
    // both warpgroups' sums, held to the last tile's maximum
    if (ok && tiles) ok = warp_wait_or_record(o_full, 0, tl.wait_limit, WAIT_FWD_O);
    ptx::tc_fence_after();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float last_m = tiles ? ref[r] : -INFINITY;
    sums[w * 128 + r] = m == last_m ? l : l * exp2f((m - last_m) * c);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    m = last_m, l = sums[r] + sums[128 + r];
    const float f = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    const uint64_t f2 = ptx::join2(__float_as_uint(f), __float_as_uint(f));
    uint64_t worst = 0;                                      // NaN where an output is NaN or infinite
    constexpr int HALF = DP / 2;
    RowsOut<HALF / 8> rows_out{smem + (w * 128 + (warp & 3) * 32) * HALF * 2};       // (Q's place: its products are done)
    for (int pass = 0; pass < (a.low ? 2 : 1); ++pass) {     // the output, and what its rounding took away
#pragma unroll
      for (int x = 0; x < HALF; x += 32) {
        uint32_t o[32];
        if (tiles) {
          ptx::tmem_ld_regs(lanes + FEW_O + w * HALF + x, o);
          ptx::tmem_wait_regs(o);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          if (w * HALF + x + e < a.D) {
            uint32_t v[4];
            round8<T>(o + e, f2, pass, worst, v);
            if (n <= 0) v[0] = v[1] = v[2] = v[3] = 0;                 // whatever its place held
            rows_out.put((x + e) / 8, v);
          }
      }
      rows_out.store(static_cast<T*>(pass ? a.low : a.out) + (t * a.Hq + h) * a.D + w * HALF, mine && ok, (a.D - w * HALF) / 8);
    }
    if (mine && ok && a.lse && w == 0) a.lse[(int64_t)h * a.Tq + t] = n == 0 || l == 0.0f ? -INFINITY : l > 0.0f ? (log2f(l) - held_shift<T>(m, c)) * 0.6931471805599453f : l;
    // A value that the mask hides was multiplied by 0, which infinities and NaN turn into NaN: such rows are made again
    // from the keys that they see alone (this thread's half).  (Where the sum is NaN, the scores are, and the row is NaN by right.)
    const bool redo = mine && ok && n > 0 && (ptx::lo2(worst) != 0.0f || ptx::hi2(worst) != 0.0f) && l > 0.0f;
    const int d0 = w * HALF, d1 = min(a.D, (w + 1) * HALF);
    T* low = a.low ? static_cast<T*>(a.low) + (t * a.Hq + h) * a.D : nullptr;
    const uint32_t rows = __any_sync(0xFFFFFFFFu, redo) ? rows_made_again<T, true>(a, redo, u.b, (int)n, (int64_t)tiles * 128, u.kh, d0, d1, low) : 0;
    if (rows) make_again<T, AGAIN_OUT>(a, nullptr, rows, u.b, t, h, make_float2(held_shift<T>(m, c), f), d0, d1);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(*tmem_slot, 512);
  }
}

template <typename T, int DP> cudaError_t launch(const AttnArgs& a, cudaStream_t stream) {
  CUtensorMap mq, mk, mv;
  const Tiling tl = tiling_of(a);
  const cudaError_t bound = bind_context();
  if (bound != cudaSuccess) return bound;
  if (!make_rows_map(&mq, a.q, a.Tq, a.Hq, a.D, a.q_stride, a.dtype, tl.heads, tl.tokens) ||
      !make_rows_map(&mk, a.k, a.Tk, a.Hk, a.D, a.k_stride, a.dtype, 1, 128) || !make_rows_map(&mv, a.v, a.Tk, a.Hk, a.D, a.v_stride, a.dtype, 1, 128))
    return cudaErrorUnknown;
  // One tile to a CTA while the pairs of tiles would not fill the SMs, or not twice with several sequences, whose lengths may
  // differ: 32 heads on 8 of 128, causal, us: 512 tokens 12.3 against 16.4, 1024 22.8 against 24.7, 1536 37 against 31.5,
  // 4096 137 against 132; 9 sequences of 2051 queries and 20011 keys, 20 heads on 4 of 80: 59 against 90.
  const int64_t heads = (int64_t)tl.chunks * a.Hk, pairs = units(a.Tq, a.B, 2 * tl.tokens) * heads, sms = sm_count();
  const bool few = pairs <= (a.B > 1 ? sms + sms / 2 : sms);
  const int64_t grid = few ? units(a.Tq, a.B, tl.tokens) * heads : pairs;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  static std::atomic<uint64_t> done[2] = {{0}, {0}};
  auto start = [&](auto kernel, int bytes, std::atomic<uint64_t>& set) {
    const cudaError_t e = allow_shared(kernel, bytes, set);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)grid, THREADS, bytes, stream>>>(mq, mk, mv, a, tl);
    return cudaGetLastError();
  };
  return few ? start(attention_few_kernel<T, DP>, Few<DP>::SMEM, done[1]) : start(attention_kernel<T, DP>, Fwd<DP>::SMEM, done[0]);
}

}  // namespace

cudaError_t take_attention_wait_error(int* code) { return take_error(code); }

cudaError_t launch_attention(const AttnArgs& a, cudaStream_t stream) {
  const bool half = a.dtype == EMU_DTYPE_F16;
  if (a.D <= 64) return half ? launch<__half, 64>(a, stream) : launch<__nv_bfloat16, 64>(a, stream);
  return half ? launch<__half, 128>(a, stream) : launch<__nv_bfloat16, 128>(a, stream);
}

}  // namespace emu
