// Matrix product of 8-bit floating-point operands with one f32 scale per block of 128, on the
// 5th-generation tensor cores (tcgen05 + TMEM + TMA), sm_100a:
//
//   out[m][n] = sum_kb sa[m][kb] * sb[n or n / 128][kb] * sum_{k in block kb} A[m][k] * B[n][k]
//
// The inner sum of one 128-wide block is four MMAs into a fresh TMEM accumulator; CUDA cores multiply
// it by the two scales and add it to f32 accumulators in registers, so the scales' f32 product and the
// sum over blocks never pass through fewer than 32 bits.
//
// One kernel (this file's first form): the rows of B are the MMA's 128 lanes and BN rows of A its columns
// ("weights by tokens"), so that few rows of A cost few columns; the blocks of K are split over the CTAs
// of a cluster where the tiles alone would leave SMs idle, their partial sums meeting in distributed
// shared memory in rank order (the same result every run).
//
//   warp 0      TMA: a 128 x 128 tile of B and a BN x 128 tile of A per block of K into a ring; bulk copies
//               of the block's scales into a second ring
//   warp 1      TMEM owner and MMA issuer
//   warps 2-5   epilogue: a thread owns one row of B (a TMEM lane) and BN accumulators
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace emu {
namespace {

constexpr int BK = 128;                         // bytes of K per stage: one scale block, one 128-byte swizzle row
constexpr int LANES = 128;
constexpr int THREADS = 192;
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

template <int BN> struct Cfg {
  static constexpr int STAGE = (LANES + BN) * BK;
  static constexpr int NSTAGE = BN <= 32 ? 5 : BN == 64 ? 4 : 3;     // ~100 KB: two CTAs share an SM
  static constexpr int NSCALE = 8;                                    // scale slots: BN + 128 floats each
  static constexpr int SCALE = (BN + LANES) * 4;
  static constexpr int NACC = BN <= 64 ? 4 : 2;                       // TMEM accumulators
  static constexpr int TMEM_COLS = NACC * BN < 32 ? 32 : NACC * BN;   // <= 256: two CTAs share an SM's 512
  static constexpr int BARS = 2 * NSTAGE + 2 * NSCALE + 2 * NACC + 1;
  static constexpr int SMEM = 1024 + NSTAGE * STAGE + NSCALE * SCALE + BARS * 8 + 16;
  static_assert(NSTAGE * STAGE >= BN * LANES * 4, "the ring holds the partial sums afterwards");
};

template <int BN>
__global__ void __launch_bounds__(THREADS) gemm_fp8_skinny_kernel(const __grid_constant__ CUtensorMap map_b,
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
    ptx::mbar_init(drained, 1);
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
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < steps; ++i) {
        const int st = i % C::NSTAGE, ac = i % C::NACC;
        if (i >= C::NACC && !wait_or_record(&acc_empty[ac], (i / C::NACC - 1) & 1, p.wait_limit, 13)) break;
        if (!wait_or_record(&full[st], (i / C::NSTAGE) & 1, p.wait_limit, 14)) break;
        ptx::tc_fence_after();
        const uint64_t da = ptx::smem_desc_sw128(ptx::smem_u32(smem + st * C::STAGE));
        const uint64_t db = ptx::smem_desc_sw128(ptx::smem_u32(smem + st * C::STAGE + LANES * BK));
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)                          // 32 bytes of K per MMA: +2 in the descriptor
          ptx::mma_f8(tmem + ac * BN, da + 2 * k, db + 2 * k, p.idesc, k > 0);
        ptx::mma_commit(&empty[st]);
        if (!(i == 0 && p.hold_first_ready)) ptx::mma_commit(&acc_full[ac]);
      }
      ptx::mma_commit(drained);
      wait_or_record(drained, 0, DRAIN_LIMIT, 15);
    }
  } else {
    const int quarter = warp & 3;                                  // the TMEM lanes this warp may read
    const int64_t n = n0 + quarter * 32 + lane;
    const float* sb_tile = p.sb + (n0 / 128) * p.ldsb;
    for (int i = 0; i < steps; ++i) {
      const int sc = i % C::NSCALE, ac = i % C::NACC;
      const float sb_t = p.b_rows ? 0.0f : __ldg(sb_tile + kb0 + i);
      if (!warp_wait_or_record(&s_full[sc], (i / C::NSCALE) & 1, p.wait_limit, 16) ||
          !warp_wait_or_record(&acc_full[ac], (i / C::NACC) & 1, p.wait_limit, 17)) {
        *failed = 1;
        break;
      }
      ptx::tc_fence_after();
      const float* slot = scales + sc * (C::SCALE / 4);
      const float sb = p.b_rows ? slot[BN + quarter * 32 + lane] : sb_t;
#pragma unroll
      for (int j = 0; j < BN; j += 16) {
        float v[16];
        ptx::tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + ac * BN + j, v);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int u = 0; u < 16; u += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(slot + j + u);
          acc[j + u] = __fmaf_rn(v[u], __fmul_rn(sb, s4.x), acc[j + u]);
          acc[j + u + 1] = __fmaf_rn(v[u + 1], __fmul_rn(sb, s4.y), acc[j + u + 1]);
          acc[j + u + 2] = __fmaf_rn(v[u + 2], __fmul_rn(sb, s4.z), acc[j + u + 2]);
          acc[j + u + 3] = __fmaf_rn(v[u + 3], __fmul_rn(sb, s4.w), acc[j + u + 3]);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(&acc_empty[ac]);
        ptx::mbar_arrive(&s_empty[sc]);
      }
    }
    if (split == 1 && n < p.N && !*failed) {
#pragma unroll
      for (int j = 0; j < BN; ++j)
        if (m0 + j < p.M) store_out(p.out, (m0 + j) * p.ldo + n, acc[j], p.out_mode);
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
  if (warp >= 2) {
    const int l = (warp & 3) * 32 + lane;
#pragma unroll
    for (int j = 0; j < BN; ++j) part[j * LANES + l] = *failed ? __int_as_float(0x7FC00000) : acc[j];
  }
  ptx::cluster_sync();
  if (warp >= 2) {
    const int l = (warp & 3) * 32 + lane;
    const int64_t n = n0 + l;
    const int j0 = BN * rank / split, j1 = BN * (rank + 1) / split;
    for (int j = j0; j < j1; ++j) {
      const uint32_t at = ptx::smem_u32(part + j * LANES + l);
      float s = 0.0f;
      for (uint32_t r = 0; r < split; ++r) s = __fadd_rn(s, ptx::ld_shared_cluster(ptx::map_shared(at, r)));
      if (n < p.N && m0 + j < p.M) store_out(p.out, (m0 + j) * p.ldo + n, s, p.out_mode);
    }
  }
  ptx::cluster_sync();                                             // no CTA leaves while its sums are read
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

template <int BN>
cudaError_t launch_skinny(const Fp8GemmArgs& g, Params p, int sms, cudaStream_t stream) {
  CUtensorMap ma, mb;
  if (!make_map(&mb, g.b, g.N, g.K, g.ldb, LANES) || !make_map(&ma, g.a, g.M, g.K, g.lda, BN)) return cudaErrorUnknown;
  auto kernel = gemm_fp8_skinny_kernel<BN>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::SMEM);
  if (e != cudaSuccess) return e;
  p.idesc = ptx::idesc_f8_f32(LANES, BN, g.b_type, g.a_type);
  const int64_t tiles_n = (g.N + LANES - 1) / LANES, tiles_m = (g.M + BN - 1) / BN;
  // split K while CTAs fit twice into the SMs and each keeps at least two blocks
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

}  // namespace

cudaError_t take_fp8_wait_error(int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_fp8_wait_error, sizeof(int));
  if (e != cudaSuccess || *code == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_fp8_wait_error, &zero, sizeof(int));
}

cudaError_t launch_gemm_fp8(const Fp8GemmArgs& g, cudaStream_t stream) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  Params p{};
  p.sa = g.sa, p.sb = g.sb, p.ldsa = g.ldsa, p.ldsb = g.ldsb;
  p.M = g.M, p.N = g.N;
  p.kb_count = (int)((g.K + BK - 1) / BK);
  p.b_rows = g.b_rows;
  p.out = g.out, p.ldo = g.ldo, p.out_mode = g.out_dtype;
  p.wait_limit = current_wait_limit();
  p.hold_first_ready = current_hold_first_ready();
  if (g.M <= 16) return launch_skinny<16>(g, p, sms, stream);
  if (g.M <= 32) return launch_skinny<32>(g, p, sms, stream);
  if (g.M <= 64) return launch_skinny<64>(g, p, sms, stream);
  return launch_skinny<128>(g, p, sms, stream);
}

}  // namespace emu
