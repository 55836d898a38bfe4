// Matrix product of 8-bit floating-point operands with one f32 scale per block of 128, on the
// 5th-generation tensor cores (tcgen05 + TMEM + TMA), sm_100a:
//
//   out[m][n] = sum_kb sa[m][kb] * sb[n or n / 128][kb] * sum_{k in block kb} A[m][k] * B[n][k]
//
// The inner sum of one 128-wide block is four MMAs into a fresh TMEM accumulator; CUDA cores multiply
// it by the two scales and add it to f32 accumulators in registers, so neither the scaled block sums nor the
// sum over blocks pass through fewer than 32 bits.  The scales may be any f32: see "Order of the factors".
//
// Few rows of A (gemm_fp8_skinny_kernel): the rows of B are the MMA's 128 lanes and BN rows of A its columns
// ("weights by tokens"), so that few rows of A cost few columns; the blocks of K are split over the CTAs
// of a cluster where the tiles alone would leave SMs idle, their partial sums meeting in distributed
// shared memory in rank order (the same result every run).
//
//   warp 0      TMA: a 128 x 128 tile of B and a BN x 128 tile of A per block of K into a ring; bulk copies
//               of the block's scales into a second ring
//   warps 1, 6  MMA issuers in turn (warp 1 owns the TMEM)
//   warps 2-5   epilogue: a thread owns one row of B (a TMEM lane) and BN accumulators
// Bound: reading B.  B200: 1 x 128256 x 4096 83 us (96% of the measured copy rate), 32 x 14336 x 4096 16.9 us (floor 9.2;
// about 5 us are the launch, the pipeline's fill and the parts' exchange: 1 x 512 x 4096 takes 5.4).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace emu {
namespace {

constexpr int BK = 128;                         // bytes of K per stage: one scale block, one 128-byte swizzle row
constexpr int LANES = 128;
constexpr int THREADS = 224;
constexpr long long DRAIN_LIMIT = 1ll << 31;    // waits for copies / MMAs already in flight

struct Params {
  const float* sa;      // [kb][lda_s]: block after block, a row of A each
  const float* sb;      // row blocks: as sa; tiles: [n / 128][ldb_s]
  int64_t ldsa, ldsb;
  int64_t M, N;
  int kb_count;
  int b_rows;           // sb holds a scale per row of B
  uint32_t idesc;
  void* out;
  int64_t ldo;
  int out_mode;         // EMU_DTYPE_*
  long long wait_limit;
  int hold_first_ready;
};

__device__ int g_fp8_wait_error;   // code of the first wait that ran out since the last read (0 = none)

__device__ __forceinline__ bool wait_or_record(uint64_t* bar, uint32_t parity, long long limit, int code) {
  if (ptx::mbar_wait(bar, parity, limit)) return true;
  atomicCAS(&g_fp8_wait_error, 0, code);
  return false;
}
// The same for a whole warp: every lane gets the same answer, so that the warp stays together.
__device__ __forceinline__ bool warp_wait_or_record(uint64_t* bar, uint32_t parity, long long limit, int code) {
  return __all_sync(0xFFFFFFFFu, wait_or_record(bar, parity, limit, code));
}

__device__ __forceinline__ void store_out(void* out, int64_t i, float v, int mode) {
  if (mode == EMU_DTYPE_F32) static_cast<float*>(out)[i] = v;
  else if (mode == EMU_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(out)[i] = __float2half_rn(v);
}

// ------------------------------------------------------------------------------ Order of the factors
// sum * sa * sb must not leave f32's range on the way where the result does not.  A block sum is 0 or between 2^-32 (two
// smallest E5M2 codes) and 2^39 (128 products of the largest), so
//   * times a scale in [2^-94, 2^89] it stays a normal number, and the other scale may be anything;
//   * times a smaller scale it is off by at most 2^-150, which a second scale of at most 1 leaves below f32's last place
//     (blocks of zeros have the quantiser's smallest scale, 2^-126, and are in this form as a rule);
//   * where sa * sb is a normal number, the sum may be multiplied by that product;
//   * where it is smaller, by the larger scale first: that is below 2^23 (the other is at least 2^-149), and where it takes
//     the sum below the normal range, both are below 2^-94 and the result below 2^-150 (a scale of 0 goes first instead:
//     the other may be anything);
//   * where it is larger, by the smaller scale first: that is at least 1, so an overflow is the result's own.
// Which of these an element takes depends on its own two scales and not on what else a warp adds up (but for the last
// place of results below f32's normal range).
constexpr float SCALE_LOW = 0x1p-94f, SCALE_HIGH = 0x1p89f;

__device__ __forceinline__ bool in_range(float s) { return fabsf(s) >= SCALE_LOW && fabsf(s) <= SCALE_HIGH; }
__device__ __forceinline__ bool normal_product(float f) {
  return fabsf(f) >= 0x1p-126f && fabsf(f) <= 3.402823466e38f;       // NaN: no
}
struct Factors {
  float first, second;
};
// The last three of these cases.
__device__ __forceinline__ Factors factors(float sa, float sb) {
  const float f = __fmul_rn(sa, sb);
  if (normal_product(f)) return {1.0f, f};
  const bool larger_first = fabsf(f) < 0x1p-126f && sa != 0.0f && sb != 0.0f;
  return (fabsf(sa) > fabsf(sb)) == larger_first ? Factors{sa, sb} : Factors{sb, sa};
}
// All of them: `first` before `second` where the first two say so.
__device__ __forceinline__ Factors factors_in_order(float first, float second) {
  const float m = fabsf(first);
  return (m >= SCALE_LOW || fabsf(second) <= 1.0f) && m <= SCALE_HIGH ? Factors{first, second} : factors(first, second);
}
// Four sums added up, each in its own order (out of line: rare, and its code many times over would cost the usual path
// registers: 118 -> 137 us at 4096^3 with row scales of both operands).
__device__ __noinline__ float4 add_any4(float4 x, float first, float4 second, float4 acc) {
  const Factors a = factors_in_order(first, second.x), b = factors_in_order(first, second.y);
  const Factors c = factors_in_order(first, second.z), d = factors_in_order(first, second.w);
  return make_float4(__fmaf_rn(__fmul_rn(x.x, a.first), a.second, acc.x), __fmaf_rn(__fmul_rn(x.y, b.first), b.second, acc.y),
                     __fmaf_rn(__fmul_rn(x.z, c.first), c.second, acc.z), __fmaf_rn(__fmul_rn(x.w, d.first), d.second, acc.w));
}
// The whole warp.  Sums of 0 are 0 (or NaN) in any order, so rows of zeros beside columns of any scale stay quick: 4096^3
// with such rows and columns of scales above 1 in every warp 194 us; 1400 where every sum has to be looked at.
template <int N> __device__ __forceinline__ void add_any(const uint32_t (&x)[N], float first, const float* second, float* acc) {
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) bits |= x[j];
  const bool easy = __all_sync(0xFFFFFFFFu, in_range(first) || (bits & 0x7FFFFFFFu) == 0);
  // the test once for the pairs (194 against 431 us), for every four in the skinny kernel, whose usual path then is as
  // quick as without (64 x 4096 x 4096: 12.8 against 13.1 us)
  constexpr bool ONCE = N > 16;
  if (ONCE && easy) {
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = __fmaf_rn(__fmul_rn(__uint_as_float(x[j]), first), second[j], acc[j]);
    return;
  }
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 s = *reinterpret_cast<const float4*>(second + j);
    const float4 v = make_float4(__uint_as_float(x[j]), __uint_as_float(x[j + 1]), __uint_as_float(x[j + 2]), __uint_as_float(x[j + 3]));
    float4 r = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    if (!ONCE && easy) {
      r.x = __fmaf_rn(__fmul_rn(v.x, first), s.x, r.x);
      r.y = __fmaf_rn(__fmul_rn(v.y, first), s.y, r.y);
      r.z = __fmaf_rn(__fmul_rn(v.z, first), s.z, r.z);
      r.w = __fmaf_rn(__fmul_rn(v.w, first), s.w, r.w);
    } else {
      r = add_any4(v, first, s, r);
    }
    acc[j] = r.x, acc[j + 1] = r.y, acc[j + 2] = r.z, acc[j + 3] = r.w;
  }
}
// For the second case: whether this lane's share of the first n of `second` (shared memory; n <= 128) is at most 1.
__device__ __forceinline__ bool at_most_one(const float* second, int n, int lane) {
  bool ok = true;
  if (lane * 4 < n) {
    const float4 s = *reinterpret_cast<const float4*>(second + lane * 4);
    const int j = n - lane * 4;
    ok = fabsf(s.x) <= 1.0f && (j < 2 || fabsf(s.y) <= 1.0f) && (j < 3 || fabsf(s.z) <= 1.0f) && (j < 4 || fabsf(s.w) <= 1.0f);
  }
  return ok;
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BN> struct Cfg {
  static constexpr int STAGE = (LANES + BN) * BK;
  static constexpr int NSTAGE = BN <= 32 ? 5 : 4;                    // ~100 KB: two CTAs share an SM
  static constexpr int NSCALE = 8;                                    // scale slots: BN + 128 floats each
  static constexpr int SCALE = (BN + LANES) * 4;
  static constexpr int NACC = 4;                                      // TMEM accumulators
  static constexpr int TMEM_COLS = NACC * BN;                         // <= 256: two CTAs share an SM's 512
  static constexpr int BARS = 2 * NSTAGE + 2 * NSCALE + 2 * NACC + 1;
  static constexpr int SMEM = 1024 + NSTAGE * STAGE + NSCALE * SCALE + BARS * 8 + 16;
  static_assert(NSTAGE * STAGE >= BN * LANES * 4, "the ring holds the partial sums afterwards");
};

template <int BN>
__global__ void __launch_bounds__(THREADS, 2) gemm_fp8_skinny_kernel(const __grid_constant__ CUtensorMap map_b,
                                                                  const __grid_constant__ CUtensorMap map_a,
                                                                  const Params p) {
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* scales = reinterpret_cast<float*>(smem + C::NSTAGE * C::STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::NSTAGE * C::STAGE + C::NSCALE * C::SCALE);
  uint64_t* empty = full + C::NSTAGE;
  uint64_t* s_full = empty + C::NSTAGE;
  uint64_t* s_empty = s_full + C::NSCALE;
  uint64_t* acc_full = s_empty + C::NSCALE;
  uint64_t* acc_empty = acc_full + C::NACC;
  uint64_t* drained = acc_empty + C::NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* failed = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t split = gridDim.x, rank = blockIdx.x;             // the cluster spans grid.x
  const int64_t n0 = (int64_t)blockIdx.y * LANES;
  const int64_t m0 = (int64_t)blockIdx.z * BN;
  const int kb0 = (int)((int64_t)p.kb_count * rank / split), kb1 = (int)((int64_t)p.kb_count * (rank + 1) / split);
  const int steps = kb1 - kb0;

  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&map_a);
    ptx::prefetch_tmap(&map_b);
    for (int i = 0; i < C::NSTAGE; ++i) ptx::mbar_init(&full[i], 1), ptx::mbar_init(&empty[i], 1);
    for (int i = 0; i < C::NSCALE; ++i) ptx::mbar_init(&s_full[i], 1), ptx::mbar_init(&s_empty[i], 4);
    for (int i = 0; i < C::NACC; ++i) ptx::mbar_init(&acc_full[i], 1), ptx::mbar_init(&acc_empty[i], 4);
    ptx::mbar_init(drained, 2);
    *failed = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, C::TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  float acc[BN];
#pragma unroll
  for (int j = 0; j < BN; ++j) acc[j] = 0.0f;

  if (warp == 0) {
    if (lane == 0) {
      // scale copies are whole 16-byte pieces: rows of sa / sb start on 16 bytes and are padded to 4 floats
      const int64_t m_pad = (p.M + 3) & ~(int64_t)3, n_pad = (p.N + 3) & ~(int64_t)3;
      const uint32_t a_bytes = (uint32_t)min((int64_t)BN, m_pad - m0) * 4;
      const uint32_t b_bytes = p.b_rows ? (uint32_t)min((int64_t)LANES, n_pad - n0) * 4 : 0;
      int i = 0;
      for (; i < steps; ++i) {
        const int st = i % C::NSTAGE, sc = i % C::NSCALE, kb = kb0 + i;
        if (i >= C::NSCALE && !wait_or_record(&s_empty[sc], (i / C::NSCALE - 1) & 1, p.wait_limit, 10)) break;
        if (i >= C::NSTAGE && !wait_or_record(&empty[st], (i / C::NSTAGE - 1) & 1, p.wait_limit, 11)) break;
        float* slot = scales + sc * (C::SCALE / 4);
        ptx::mbar_arrive_expect_tx(&s_full[sc], a_bytes + b_bytes);
        ptx::bulk_load(slot, p.sa + kb * p.ldsa + m0, a_bytes, &s_full[sc]);
        if (b_bytes) ptx::bulk_load(slot + BN, p.sb + kb * p.ldsb + n0, b_bytes, &s_full[sc]);
        ptx::mbar_arrive_expect_tx(&full[st], C::STAGE);
        ptx::tma_load_2d(smem + st * C::STAGE, &map_b, &full[st], kb * BK, (int)n0);
        ptx::tma_load_2d(smem + st * C::STAGE + LANES * BK, &map_a, &full[st], kb * BK, (int)m0);
      }
      // every copy has landed before the ring is reused for the partial sums or the CTA exits
      for (int j = max(0, i - C::NSTAGE); j < i; ++j)
        wait_or_record(&full[j % C::NSTAGE], (j / C::NSTAGE) & 1, DRAIN_LIMIT, 12);
      for (int j = max(0, i - C::NSCALE); j < i; ++j)
        wait_or_record(&s_full[j % C::NSCALE], (j / C::NSCALE) & 1, DRAIN_LIMIT, 12);
    }
  } else if (warp == 1 || warp == 6) {
    if (lane == 0) {
      // Two issuers, blocks in turn: NACC is even, so each has its own accumulators.  The accumulator is
      // waited for first: it is free once block i - NACC has been read, so the stage's last block, i - NSTAGE,
      // has landed, and the parity of the stage's barrier cannot be that of two rounds before.
      static_assert(C::NACC % 2 == 0 && C::NSTAGE >= C::NACC, "see above");
      for (int i = warp == 1 ? 0 : 1; i < steps; i += 2) {
        const int st = i % C::NSTAGE, ac = i % C::NACC;
        if (i >= C::NACC && !wait_or_record(&acc_empty[ac], (i / C::NACC - 1) & 1, p.wait_limit, 13)) break;
        if (!wait_or_record(&full[st], (i / C::NSTAGE) & 1, p.wait_limit, 14)) break;
        ptx::tc_fence_after();
        const uint64_t da = ptx::smem_desc_sw128(ptx::smem_u32(smem + st * C::STAGE));
        const uint64_t db = ptx::smem_desc_sw128(ptx::smem_u32(smem + st * C::STAGE + LANES * BK));
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)                          // 32 bytes of K per MMA: +2 in the descriptor
          ptx::mma_f8(tmem + ac * BN, da + 2 * k, db + 2 * k, p.idesc, k > 0);
        if (!(i == 0 && p.hold_first_ready)) ptx::mma_commit(&acc_full[ac]);
        ptx::mma_commit(&empty[st]);
      }
      ptx::mma_commit(drained);
      wait_or_record(drained, 0, DRAIN_LIMIT, 15);
    }
  } else {
    const int quarter = warp & 3;                                  // the TMEM lanes this warp may read
    const int64_t n = n0 + quarter * 32 + lane;
    const float* sb_tile = p.sb + (n0 / 128) * p.ldsb;
    const int columns = (int)min((int64_t)BN, p.M - m0);
    // The blocks whose sums may be multiplied by the scale of B's row first, up to one whose scales need more care; from
    // there on each element in its own order.
    int i = 0;
    auto add_up = [&](auto any_scales) {
      constexpr bool ANY = decltype(any_scales)::value;
      for (; i < steps; ++i) {
        const int sc = i % C::NSCALE, ac = i % C::NACC;
        const float sb_t = p.b_rows ? 0.0f : __ldg(sb_tile + kb0 + i);
        if (!warp_wait_or_record(&s_full[sc], (i / C::NSCALE) & 1, p.wait_limit, 16)) {
          *failed = 1;
          return;
        }
        const float* slot = scales + sc * (C::SCALE / 4);
        const float sb = !p.b_rows ? sb_t : n < p.N ? slot[BN + quarter * 32 + lane] : 1.0f;   // lanes past N have no scale
        // one vote for the wait and the scales
        const bool full_now = wait_or_record(&acc_full[ac], (i / C::NACC) & 1, p.wait_limit, 17);
        if (!__all_sync(0xFFFFFFFFu, full_now && (ANY || in_range(sb)))) {
          if (!__all_sync(0xFFFFFFFFu, full_now)) {
            *failed = 1;
            return;
          }
          if (!__all_sync(0xFFFFFFFFu, fabsf(sb) <= SCALE_HIGH && at_most_one(slot, columns, lane))) return;
        }
        ptx::tc_fence_after();
#pragma unroll
        for (int j = 0; j < BN; j += 16) {
          uint32_t v[16];
          ptx::tmem_ld_regs(tmem + ((uint32_t)(quarter * 32) << 16) + ac * BN + j, v);
          ptx::tmem_wait_regs(v);
          if constexpr (ANY) {
            add_any(v, sb, slot + j, acc + j);
          } else {
#pragma unroll
            for (int u = 0; u < 16; u += 4) {
              const float4 s4 = *reinterpret_cast<const float4*>(slot + j + u);
              const float s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[j + u + e] = __fmaf_rn(__fmul_rn(__uint_as_float(v[u + e]), sb), s[e], acc[j + u + e]);
            }
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(&acc_empty[ac]);
          ptx::mbar_arrive(&s_empty[sc]);
        }
      }
    };
    add_up(std::false_type{});
    if (i < steps && !*failed) add_up(std::true_type{});
    if (split == 1 && n < p.N && !*failed) {
      auto write = [&](auto* out) {
        out += m0 * p.ldo + n;
#pragma unroll
        for (int j = 0; j < BN; ++j, out += p.ldo)
          if (j < columns) *out = from_float<std::remove_pointer_t<decltype(out)>>(acc[j]);
      };
      if (p.out_mode == EMU_DTYPE_BF16) write(static_cast<__nv_bfloat16*>(p.out));
      else if (p.out_mode == EMU_DTYPE_F16) write(static_cast<__half*>(p.out));
      else write(static_cast<float*>(p.out));
    }
  }

  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();                                                 // copies landed, MMAs done, TMEM read
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::TMEM_COLS);
  }
  if (split == 1) return;

  // partial sums: [column][lane] in the ring's place, then each CTA adds up its share of the columns
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2 && warp < 6) {
    const int l = (warp & 3) * 32 + lane;
#pragma unroll
    for (int j = 0; j < BN; ++j) part[j * LANES + l] = *failed ? __int_as_float(0x7FC00000) : acc[j];
  }
  ptx::cluster_sync();
  if (warp >= 2 && warp < 6) {
    const int l = (warp & 3) * 32 + lane;
    const int64_t n = n0 + l;
    auto add_up = [&](auto parts) {
      constexpr int S = decltype(parts)::value;
      constexpr int COLS = BN / S, CH = COLS < 8 ? COLS : 8;       // this CTA's columns, loads of CH of them at once
      uint32_t base[S];
#pragma unroll
      for (int r = 0; r < S; ++r) base[r] = ptx::map_shared(ptx::smem_u32(part + (int)rank * COLS * LANES + l), r);
      for (int j = 0; j < COLS; j += CH) {
        float v[S][CH];
#pragma unroll
        for (int r = 0; r < S; ++r)
#pragma unroll
          for (int c = 0; c < CH; ++c) v[r][c] = ptx::ld_shared_cluster(base[r] + (j + c) * (LANES * 4));
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float sum = v[0][c];
#pragma unroll
          for (int r = 1; r < S; ++r) sum = __fadd_rn(sum, v[r][c]);
          const int64_t m = m0 + (int)rank * COLS + j + c;
          if (n < p.N && m < p.M) store_out(p.out, m * p.ldo + n, sum, p.out_mode);
        }
      }
    };
    if (split == 8) add_up(std::integral_constant<int, 8>{});
    else if (split == 4) add_up(std::integral_constant<int, 4>{});
    else add_up(std::integral_constant<int, 2>{});
  }
  ptx::cluster_sync();                                             // no CTA leaves while its sums are read
}


// ------------------------------------------------------------------------------ large products
// A pair of CTAs computes a 256 x 256 output tile with cta_group::2 MMAs: each CTA stages 128 rows of A
// and 128 of B (32 KB per block of K instead of 48 KB for the same MMA time alone, so that L2 keeps up)
// and holds the 128 x 256 accumulators of its rows of A, twice.  Persistent: one pair per two SMs.
//   warp 0      producer: TMA into the ring (signalling the leader's barriers); B_ROWS: bulk copies of the column scales
//   warps 1, 2  in the leader, the MMA issuers, one for each accumulator: a block's waits, four MMAs and
//               commit take one thread ~970 clocks, the MMAs themselves 512, so two threads take turns
//               (warp 1 owns the TMEM)
//   warps 4-11  epilogue: a thread owns one row and 128 columns in registers; per block of K it reads
//               them from TMEM and adds scale * block sum.  (The f32x2 form of the multiply-add was slower:
//               its register pairs cost a move each, 484 against 268 us for the epilogue alone at 8192^3.)
//               B_ROWS = false: 128 columns share one scale of B, so the factor is one number per thread;
//               B_ROWS = true: the block sum is multiplied by the row's scale, then by the column's.
// Bound: the epilogue's turn-around.  A block's MMAs take 512 clocks; its sums reach the epilogue about 450 clocks
// after that, take 270 to load (TMEM's rate) and 400 to add up, so with two accumulators a block comes every
// 850 clocks or so.  B200: 4096^3 74 us (1.86 PFLOP/s; 121 with column scales), 8192^3 500 us (2.20 PFLOP/s, the clock
// already lowered by the power limit: MMAs and loads alone take 366); without the test of the scales' range 73, 120
// and 493.  Other splits were no faster: 128-column MMAs with four accumulators 72, sixteen epilogue warps of 64
// columns 95, one issuer 89 us at 4096^3.
constexpr int P_STAGE = 2 * 128 * BK;            // one CTA's 128 rows of A and of B
constexpr int P_NSTAGE = 5;                      // at least 4: see the issuers' waits
constexpr int P_NSCALE = 8;
constexpr int P_SCALE = 256 * 4;                 // column scales (B_ROWS)
constexpr int P_STORE = 8 * 32 * 128;            // per epilogue warp: 32 rows x 128 bytes of output
constexpr int P_BARS = 2 * P_NSTAGE + 2 * P_NSCALE + 2 + 1;
constexpr int P_SMEM = 1024 + P_NSTAGE * P_STAGE + P_STORE + P_NSCALE * P_SCALE + P_BARS * 8 + 16;
constexpr int P_THREADS = 384;
// 128 threads x 40 + 256 x 232 = 64512 = 384 x 168, what the CTA is launched with
constexpr int P_REG_LOW = 40, P_REG_HIGH = 232;
constexpr int P_BAND = 8;                        // tile raster: bands of 8 row tiles (2048 rows of A stay in L2)
static_assert(P_SMEM <= 232448, "shared memory per CTA");

__device__ __forceinline__ void pair_tile(int64_t t, int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn) {
  const int64_t per_band = P_BAND * tiles_n, band = t / per_band, first = band * P_BAND;
  const int64_t gm = min(tiles_m - first, (int64_t)P_BAND), idx = t % per_band;
  tm = first + idx % gm;
  tn = idx / gm;
}

// A place in a ring of N barriers and the parity of its current round; a division by N for each block would
// put a chain of multiplications in every role's loop.
template <int N> struct Ring {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) at = 0, parity ^= 1;
  }
};

template <bool B_ROWS>
__global__ void __launch_bounds__(P_THREADS, 1) gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b,
                                                                     const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* store = smem + P_NSTAGE * P_STAGE;
  float* scales = reinterpret_cast<float*>(store + P_STORE);
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + P_NSCALE * (P_SCALE / 4));
  // a block's MMAs have completed: its stage may be filled again (producers), its accumulator read (epilogue)
  uint64_t* done = full + P_NSTAGE;
  uint64_t* s_full = done + P_NSTAGE;
  uint64_t* s_empty = s_full + P_NSCALE;
  uint64_t* acc_empty = s_empty + P_NSCALE;
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int64_t tiles_m = (p.M + 255) / 256, tiles_n = (p.N + 255) / 256, tiles = tiles_m * tiles_n;
  const int64_t first = blockIdx.x / 2, stride = gridDim.x / 2;

  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&map_a);
    ptx::prefetch_tmap(&map_b);
    for (int i = 0; i < P_NSTAGE; ++i) ptx::mbar_init(&full[i], 1), ptx::mbar_init(&done[i], 1);
    for (int i = 0; i < P_NSCALE; ++i) ptx::mbar_init(&s_full[i], 1), ptx::mbar_init(&s_empty[i], 8);
    for (int i = 0; i < 2; ++i) ptx::mbar_init(&acc_empty[i], 16);   // both CTAs' warps
    ptx::mbar_init(drained, 2);
    ptx::fence_mbar_init();
  }
  __syncwarp();
  ptx::cluster_sync();                                               // barriers of both CTAs exist
  if (warp == 1) {
    ptx::tmem_alloc2(tmem_slot, 512);
    ptx::tmem_relinquish2();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();

  // no load may be in flight across the register split: the TMEM address is read after it
  if (warp < 4) {
    ptx::setmaxnreg_dec<P_REG_LOW>();
    if (warp == 0 && lane == 0) {
      const int64_t n_pad = (p.N + 3) & ~(int64_t)3;
      bool ok = true;
      Ring<P_NSTAGE> st;
      Ring<P_NSCALE> sc;
      int filled = 0, s_filled = 0;                                  // slots in their first round need no wait
      for (int64_t t = first; t < tiles && ok; t += stride) {
        int64_t tm, tn;
        pair_tile(t, tiles_m, tiles_n, tm, tn);
        const int64_t m0 = tm * 256 + rank * 128, n0 = tn * 256;
        const uint32_t b_bytes = (uint32_t)min((int64_t)256, n_pad - n0) * 4;
        for (int kb = 0; kb < p.kb_count; ++kb) {
          if (B_ROWS && s_filled == P_NSCALE && !wait_or_record(&s_empty[sc.at], sc.parity ^ 1, p.wait_limit, 10)) { ok = false; break; }
          if (filled == P_NSTAGE && !wait_or_record(&done[st.at], st.parity ^ 1, p.wait_limit, 11)) { ok = false; break; }
          const uint32_t bar = ptx::map_shared(ptx::smem_u32(&full[st.at]), 0);
          if (rank == 0) ptx::mbar_arrive_expect_tx(&full[st.at], 2 * P_STAGE);   // both CTAs' bytes
          ptx::tma_load_2d_pair(smem + st.at * P_STAGE, &map_a, bar, kb * BK, (int)m0);
          ptx::tma_load_2d_pair(smem + st.at * P_STAGE + 128 * BK, &map_b, bar, kb * BK, (int)(n0 + rank * 128));
          if (B_ROWS) {
            ptx::mbar_arrive_expect_tx(&s_full[sc.at], b_bytes);
            ptx::bulk_load(scales + sc.at * (P_SCALE / 4), p.sb + kb * p.ldsb + n0, b_bytes, &s_full[sc.at]);
          }
          st.next();
          sc.next();
          if (filled < P_NSTAGE) ++filled;
          if (s_filled < P_NSCALE) ++s_filled;
        }
      }
      // every copy has landed before the CTA may exit: the leader's barriers count both CTAs' tiles, the
      // final cluster barrier holds the other CTA until then.  After a failed wait the CTAs may have
      // stopped at different blocks: then time for copies in flight.
      const Ring<P_NSCALE> sc_end = sc;
      for (int j = 0; j < P_NSCALE; ++j, sc.next())                  // oldest first: slots of the round before, then of this one
        if (B_ROWS && j >= P_NSCALE - s_filled)
          wait_or_record(&s_full[sc.at], sc.at < sc_end.at ? sc_end.parity : sc_end.parity ^ 1, DRAIN_LIMIT, 12);
      if (ok && rank == 0) {
        const Ring<P_NSTAGE> st_end = st;
        for (int j = 0; j < P_NSTAGE; ++j, st.next())
          if (j >= P_NSTAGE - filled)
            ok = ok && wait_or_record(&full[st.at], st.at < st_end.at ? st_end.parity : st_end.parity ^ 1, p.wait_limit, 12);
      }
      if (!ok) {
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) {}
      }
    } else if ((warp == 1 || warp == 2) && rank == 0) {
      // The whole warp walks the blocks and one elected lane issues: descriptors then stay in uniform
      // registers, from which the MMAs take them.
      const uint32_t tmem = *tmem_slot + (warp - 1) * 256;
      uint64_t* acc_free = &acc_empty[warp - 1];
      bool ok = true, first_block = true;
      Ring<P_NSTAGE> st;
      uint32_t parity = 1;                                           // of the accumulator's round before: free at first
      int turn = 1;
      for (int64_t t = first; t < tiles && ok; t += stride) {
        for (int kb = 0; kb < p.kb_count; ++kb, st.next(), turn ^= 3) {
          if (turn != warp) continue;                                // the other warp's block
          // The stage first: it filled long ago as a rule, the accumulator comes free last.  The parity of
          // the stage's barrier cannot be that of two rounds before, although the round between was the
          // other issuer's: this one has waited for the accumulator of block i - 2, that is for block i - 4
          // to be read, so the stage's last block, i - 5, has landed.
          static_assert(P_NSTAGE >= 4, "see above");
          if (!warp_wait_or_record(&full[st.at], st.parity, p.wait_limit, 14)) { ok = false; break; }
          if (!warp_wait_or_record(acc_free, parity, p.wait_limit, 13)) { ok = false; break; }
          parity ^= 1;
          ptx::tc_fence_after();
          const uint64_t da = ptx::smem_desc_sw128(ptx::smem_u32(smem + st.at * P_STAGE));
          const uint64_t db = ptx::smem_desc_sw128(ptx::smem_u32(smem + st.at * P_STAGE + 128 * BK));
          if (ptx::elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 32; ++k) ptx::mma2_f8(tmem, da + 2 * k, db + 2 * k, p.idesc, k > 0);
            if (!(first_block && warp == 1 && p.hold_first_ready)) ptx::mma2_commit_both(&done[st.at]);
          }
          __syncwarp();
          first_block = false;
        }
      }
      if (ptx::elect_one()) ptx::mma2_commit_both(drained);
      __syncwarp();
      warp_wait_or_record(drained, 0, DRAIN_LIMIT, 15);
    }
  } else {
    ptx::setmaxnreg_inc<P_REG_HIGH>();
    const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;     // TMEM lanes, columns
    const uint32_t lane_base = *tmem_slot + ((uint32_t)(quarter * 32) << 16) + half * 128;
    uint8_t* buf = store + ew * (32 * 128);
    const int64_t blocks_n = (p.N + 127) / 128;
    const uint32_t empty_bar = ptx::map_shared(ptx::smem_u32(acc_empty), 0);
    constexpr int LD = 32, CHUNKS = 128 / LD;                        // columns of one TMEM load
    bool ok = true;
    Ring<P_NSTAGE> st;
    Ring<P_NSCALE> sc;
    uint32_t ac = 0;                                                 // TMEM column of the block's accumulator
    for (int64_t t = first; t < tiles && ok; t += stride) {
      int64_t tm, tn;
      pair_tile(t, tiles_m, tiles_n, tm, tn);
      const int64_t nb = min(tn * 2 + half, blocks_n - 1);
      const float* sb_tile = p.sb + nb * p.ldsb;
      const int columns = (int)max((int64_t)0, min((int64_t)128, p.N - (tn * 2 + half) * 128));
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
      // this row's scale and the column block's, read three blocks ahead
      const float* sa_row = p.sa + min(tm * 256 + rank * 128 + quarter * 32 + lane, p.M - 1);
      float sa1 = __ldg(sa_row), sa2 = p.kb_count > 1 ? __ldg(sa_row + p.ldsa) : 0.0f;
      float sa3 = p.kb_count > 2 ? __ldg(sa_row + 2 * p.ldsa) : 0.0f, sb3 = B_ROWS || p.kb_count < 3 ? 1.0f : __ldg(sb_tile + 2);
      float sb1 = B_ROWS ? 1.0f : __ldg(sb_tile), sb2 = B_ROWS || p.kb_count < 2 ? 1.0f : __ldg(sb_tile + 1);
      // B_ROWS = false: a row whose first block has the quantiser's smallest scale (zeros, as a rule all along the row) would
      // make the product of the scales too small.  Such a row is added up 2^100 times as large, while its factors stay
      // below 2^60; so rows of zeros among others cost nothing (4096^3: 74 us; in the last loop below 90).
      float up = !B_ROWS && fabsf(__fmul_rn(sa1, sb1)) < 0x1p-126f ? 0x1p100f : 1.0f;
      const float low = up == 1.0f ? 0x1p-126f : 0.0f;
      if (!B_ROWS) sa1 = __fmul_rn(sa1, up);
      auto next_scales = [&](int kb) {
        sa1 = B_ROWS ? sa2 : __fmul_rn(sa2, up), sb1 = sb2, sa2 = sa3, sb2 = sb3;
        if (kb + 3 < p.kb_count) {
          sa3 = __ldg(sa_row + (kb + 3) * p.ldsa);
          if (!B_ROWS) sb3 = __ldg(sb_tile + kb + 3);
        }
      };
      auto factor = [&] { return B_ROWS ? sa1 : __fmul_rn(sa1, sb1); };
      auto fine = [&](float f) { return B_ROWS ? in_range(f) : fabsf(f) >= low && fabsf(f) <= 0x1p60f; };
      // B_ROWS: rows of scales below the range, beside columns of scales up to 1 (4096^3 with such a row in every warp 152 us)
      auto fine_beside = [&](float f) { return fabsf(f) <= SCALE_HIGH && at_most_one(scales + sc.at * (P_SCALE / 4) + half * 128, columns, lane); };
      uint32_t v[2][LD];
      if (!warp_wait_or_record(&done[st.at], st.parity, p.wait_limit, 17)) { ok = false; break; }
      ptx::tc_fence_after();
      ptx::tmem_ld_regs(lane_base + ac, v[0]);
      int kb = 0;
      float f = factor();
      bool usual = __all_sync(0xFFFFFFFFu, fine(f));
      if (B_ROWS && !usual) {
        if (!warp_wait_or_record(&s_full[sc.at], sc.parity, p.wait_limit, 16)) { ok = false; break; }
        usual = __all_sync(0xFFFFFFFFu, fine_beside(f));
      }
      // The blocks of K, up to one whose scales need more care (see "Order of the factors")
      for (; usual && kb < p.kb_count; ++kb) {
        const bool more = kb + 1 < p.kb_count;
        next_scales(kb);
        const float f1 = factor();                                   // the next block's
        const bool fine1 = fine(f1);
        if (B_ROWS && !warp_wait_or_record(&s_full[sc.at], sc.parity, p.wait_limit, 16)) { ok = false; break; }
        const float* slot = scales + sc.at * (P_SCALE / 4) + half * 128;
        st.next();
        bool next = false;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          ptx::tmem_wait_regs(v[c & 1]);
          // the next columns travel while these are added up
          if (c + 1 < CHUNKS) {
            ptx::tmem_ld_regs(lane_base + ac + (c + 1) * LD, v[(c + 1) & 1]);
          } else {
            ptx::tc_fence_before();                                  // all of this block is in registers
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(empty_bar + ac / 32);   // 8 bytes per 256 columns
            ac ^= 256;
            if (more) {
              // (one vote for both, without a branch: a second vote for the scales cost 72 -> 75 us at 4096^3)
              next = __all_sync(0xFFFFFFFFu, (int)ptx::mbar_test_wait(&done[st.at], st.parity) & (int)fine1);
              if (next) {
                ptx::tc_fence_after();
                ptx::tmem_ld_regs(lane_base + ac, v[0]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < LD; j += 4) {
            float x[4], s[4] = {f, f, f, f};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[c & 1][j + e]);
            if (B_ROWS) {
              // two products per instruction: here the pairs lie as they were loaded
              const float4 s4 = *reinterpret_cast<const float4*>(slot + c * LD + j);
              s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
              const uint64_t ff = ptx::join2(__float_as_uint(f), __float_as_uint(f));
              const uint64_t lo = ptx::mul2(ptx::join2(v[c & 1][j], v[c & 1][j + 1]), ff);
              const uint64_t hi = ptx::mul2(ptx::join2(v[c & 1][j + 2], v[c & 1][j + 3]), ff);
              x[0] = ptx::lo2(lo), x[1] = ptx::hi2(lo), x[2] = ptx::lo2(hi), x[3] = ptx::hi2(hi);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c * LD + j + e] = __fmaf_rn(x[e], s[e], acc[c * LD + j + e]);
          }
        }
        if (B_ROWS) {
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&s_empty[sc.at]);
          sc.next();
        }
        f = f1;
        if (more && !next) {
          if (!warp_wait_or_record(&done[st.at], st.parity, p.wait_limit, 17)) { ok = false; break; }
          ptx::tc_fence_after();
          ptx::tmem_ld_regs(lane_base + ac, v[0]);
          usual = __all_sync(0xFFFFFFFFu, fine(f));
          if (B_ROWS && !usual) {
            if (!warp_wait_or_record(&s_full[sc.at], sc.parity, p.wait_limit, 16)) { ok = false; break; }
            usual = __all_sync(0xFFFFFFFFu, fine_beside(f));
          }
        }
      }
      if (!B_ROWS && !__all_sync(0xFFFFFFFFu, up == 1.0f)) {
        const float down = up == 1.0f ? 1.0f : 0x1p-100f;
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] = __fmul_rn(acc[j], down);
        if (kb < p.kb_count) sa1 = __ldg(sa_row + kb * p.ldsa);
        up = 1.0f;
      }
      // The rest: each element in its own order (no load is in flight over add_any's calls)
      for (; ok && kb < p.kb_count; ++kb) {
        const float sa = sa1;
        const Factors fs = factors(sa1, sb1);
        next_scales(kb);
        if (B_ROWS && !warp_wait_or_record(&s_full[sc.at], sc.parity, p.wait_limit, 16)) { ok = false; break; }
        const float* slot = scales + sc.at * (P_SCALE / 4) + half * 128;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          ptx::tmem_wait_regs(v[0]);
          if (B_ROWS) {
            add_any(v[0], sa, slot + c * LD, acc + c * LD);
          } else {
#pragma unroll
            for (int j = 0; j < LD; ++j) acc[c * LD + j] = __fmaf_rn(__fmul_rn(__uint_as_float(v[0][j]), fs.first), fs.second, acc[c * LD + j]);
          }
          if (c + 1 < CHUNKS) ptx::tmem_ld_regs(lane_base + ac + (c + 1) * LD, v[0]);
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive_cluster(empty_bar + ac / 32);
          if (B_ROWS) ptx::mbar_arrive(&s_empty[sc.at]);
        }
        ac ^= 256;
        st.next();
        if (B_ROWS) sc.next();
        if (kb + 1 < p.kb_count) {
          if (!warp_wait_or_record(&done[st.at], st.parity, p.wait_limit, 17)) { ok = false; break; }
          ptx::tc_fence_after();
          ptx::tmem_ld_regs(lane_base + ac, v[0]);
        }
      }
      if (!ok) break;
      // output: 128 bytes of each of the warp's 32 rows at a time, turned in shared memory so that a
      // row's bytes leave together; 16-byte pieces are spread over the banks by the row's low bits
      const int64_t row0 = tm * 256 + rank * 128 + quarter * 32, col0 = tn * 256 + half * 128;
      const int rows = (int)max((int64_t)0, min((int64_t)32, p.M - row0));
      auto write = [&](auto* out) {
        using O = std::remove_pointer_t<decltype(out)>;
        constexpr int PER = 16 / sizeof(O), COLS = 8 * PER;          // elements of a piece, of 128 bytes
        out += row0 * p.ldo + col0;
        const int cols = (int)min((int64_t)128, p.N - col0);
        const uintptr_t mis = reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.ldo * sizeof(O));
#pragma unroll
        for (int c = 0; c < 128; c += COLS) {
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (sizeof(O) == 4) {
                w[e] = __float_as_uint(acc[c + 4 * u + e]);
              } else if constexpr (std::is_same<O, __half>::value) {
                const __half2 h = __floats2half2_rn(acc[c + 8 * u + 2 * e], acc[c + 8 * u + 2 * e + 1]);
                w[e] = reinterpret_cast<const uint32_t&>(h);
              } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(acc[c + 8 * u + 2 * e], acc[c + 8 * u + 2 * e + 1]);
                w[e] = reinterpret_cast<const uint32_t&>(h);
              }
            }
            *reinterpret_cast<uint4*>(buf + lane * 128 + ((u ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          if ((mis & 15) == 0) {
            // 8 lanes write 128 bytes of a row
            const int u = lane & 7, col = c + u * PER;
            O* dst = out + (lane >> 3) * p.ldo + col;
#pragma unroll
            for (int r4 = 0; r4 < 8; ++r4, dst += 4 * p.ldo) {
              const int r = r4 * 4 + (lane >> 3);
              if (r >= rows || col >= cols) continue;
              const uint4 w = *reinterpret_cast<const uint4*>(buf + r * 128 + ((u ^ (r & 7)) * 16));
              if (col + PER <= cols) {
                *reinterpret_cast<uint4*>(dst) = w;
              } else {
                const O* x = reinterpret_cast<const O*>(buf + r * 128 + ((u ^ (r & 7)) * 16));
                for (int e = 0; col + e < cols; ++e) dst[e] = x[e];
              }
            }
          } else {
            // rows that do not start on 16 bytes: the warp writes a row's 128 bytes, 4 to a lane (or two
            // 16-bit elements by themselves where rows start on 2 bytes)
            constexpr int EL = 4 / sizeof(O);
            const int col = c + lane * EL;
            O* dst = out + col;
#pragma unroll 4
            for (int r = 0; r < rows; ++r, dst += p.ldo) {
              const uint8_t* x = buf + r * 128 + (((lane >> 2) ^ (r & 7)) * 16) + (lane & 3) * 4;
              if ((mis & 3) == 0 && col + EL <= cols) {
                *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(x);
              } else {
#pragma unroll
                for (int e = 0; e < EL; ++e)
                  if (col + e < cols) dst[e] = reinterpret_cast<const O*>(x)[e];
              }
            }
          }
        }
      };
      if (p.out_mode == EMU_DTYPE_BF16) write(static_cast<__nv_bfloat16*>(p.out));
      else if (p.out_mode == EMU_DTYPE_F16) write(static_cast<__half*>(p.out));
      else write(static_cast<float*>(p.out));
    }
  }

  __syncwarp();
  ptx::tc_fence_before();
  ptx::cluster_sync();                                               // both CTAs are done with both memories
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc2(*tmem_slot, 512);
    // the leader's last signal to this CTA's shared memory has arrived before it goes
    if (rank == 1 && lane == 0) wait_or_record(drained, 0, DRAIN_LIMIT, 15);
  }
}

// ------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode() {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(ptr);
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

// rows x K bytes with 128-byte swizzle, boxes of box_rows x 128 bytes; bytes past K and rows past the end
// read as zero.
bool make_map(CUtensorMap* m, const uint8_t* base, int64_t rows, int64_t K, int64_t ld, int box_rows) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {BK, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Raises a kernel's shared-memory limit, once for each device.
template <typename Kernel> cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <int BN>
cudaError_t launch_skinny(const Fp8GemmArgs& g, Params p, int sms, cudaStream_t stream) {
  CUtensorMap ma, mb;
  if (!make_map(&mb, g.b, g.N, g.K, g.ldb, LANES) || !make_map(&ma, g.a, g.M, g.K, g.lda, BN)) return cudaErrorUnknown;
  auto kernel = gemm_fp8_skinny_kernel<BN>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared(kernel, Cfg<BN>::SMEM, done);
  if (e != cudaSuccess) return e;
  p.idesc = ptx::idesc_f8_f32(LANES, BN, g.b_type, g.a_type);
  const int64_t tiles_n = (g.N + LANES - 1) / LANES, tiles_m = (g.M + BN - 1) / BN;
  // split K (in powers of two: the kernel adds up 2, 4 or 8 parts) while the CTAs fit twice into the SMs and
  // each keeps at least two blocks
  int split = 1;
  while (split < 8 && tiles_n * tiles_m * split * 2 <= 2 * sms && p.kb_count >= split * 4) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)split, (unsigned)tiles_n, (unsigned)tiles_m);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Cfg<BN>::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, mb, ma, p);
}

template <bool B_ROWS>
cudaError_t launch_pair(const Fp8GemmArgs& g, Params p, int sms, cudaStream_t stream) {
  CUtensorMap ma, mb;
  if (!make_map(&ma, g.a, g.M, g.K, g.lda, 128) || !make_map(&mb, g.b, g.N, g.K, g.ldb, 128)) return cudaErrorUnknown;
  auto kernel = gemm_fp8_pair_kernel<B_ROWS>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared(kernel, P_SMEM, done);
  if (e != cudaSuccess) return e;
  p.idesc = ptx::idesc_f8_f32(256, 256, g.a_type, g.b_type);
  const int64_t tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, sms / 2)));
  cfg.blockDim = dim3(P_THREADS);
  cfg.dynamicSmemBytes = P_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, p);
}

}  // namespace

cudaError_t take_fp8_wait_error(int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_fp8_wait_error, sizeof(int));
  if (e != cudaSuccess || *code == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_fp8_wait_error, &zero, sizeof(int));
}

cudaError_t launch_gemm_fp8(const Fp8GemmArgs& g, cudaStream_t stream) {
  const int sms = sm_count();
  Params p{};
  p.sa = g.sa, p.sb = g.sb, p.ldsa = g.ldsa, p.ldsb = g.ldsb;
  p.M = g.M, p.N = g.N;
  p.kb_count = (int)((g.K + BK - 1) / BK);
  p.b_rows = g.b_rows;
  p.out = g.out, p.ldo = g.ldo, p.out_mode = g.out_dtype;
  p.wait_limit = current_wait_limit();
  p.hold_first_ready = current_hold_first_ready();
  // Up to 64 rows of A are one column tile of the skinny kernel: each byte of B is read once.  Beyond, the two
  // kernels' times by what they do, in us: the skinny one 6.5 + its tiles' blocks of K / 300, the pairs 3.5 + for each
  // wave of tiles 0.53 (0.8 with a scale per row of B) a block + 2.3 to store.  A rough rule: over 124 sizes of 65 .. 4096
  // rows the median error is 14% (skinny; at worst 46%, it knows neither the split nor its own waves) and 9% (pairs;
  // 27%), and 14 times the kernel taken is over 5% slower than the other, at worst 1.45 times.  E.g. 128 x 4096 x 4096:
  // 14.3 against 21.1; 128 x 14336 x 4096: 26.6 against 23.2; 1024 x 4096 x 4096: 48 against 23.4.
  const int64_t kb = p.kb_count;
  const int64_t tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256), pairs = std::max(1, sms / 2);
  const double t_pair = 3.5 + (double)((tiles + pairs - 1) / pairs) * ((g.b_rows ? 0.8 : 0.53) * kb + 2.3);
  const double t_skinny = 6.5 + (double)((g.M + 63) / 64) * (double)((g.N + 127) / 128) * (double)kb / 300.0;
  if (g.M > 64 && t_pair < t_skinny)
    return g.b_rows ? launch_pair<true>(g, p, sms, stream) : launch_pair<false>(g, p, sms, stream);
  if (g.M <= 16) return launch_skinny<16>(g, p, sms, stream);
  if (g.M <= 32) return launch_skinny<32>(g, p, sms, stream);
  return launch_skinny<64>(g, p, sms, stream);
}

}  // namespace emu
