// What the tensor-core kernels of attention share: their work units, tensor maps, waits and conversions.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attention.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace emu {
namespace attn {

constexpr long long DRAIN_LIMIT = 1ll << 31;    // waits for copies / MMAs already in flight

// Codes of the waits (emu_device_status).
enum {
  WAIT_FWD_SLOT = 18, WAIT_FWD_Q, WAIT_FWD_K, WAIT_FWD_V, WAIT_FWD_P, WAIT_FWD_S, WAIT_FWD_O, WAIT_DRAIN,
  WAIT_BACK_SLOT, WAIT_BACK_FIXED, WAIT_BACK_TILE, WAIT_BACK_STATS, WAIT_BACK_S, WAIT_BACK_P, WAIT_BACK_DP, WAIT_BACK_DS, WAIT_BACK_DONE,
};

static __device__ int g_wait_error;             // code of the first wait that ran out since the last read (0 = none)

__device__ __forceinline__ bool wait_or_record(uint64_t* bar, uint32_t parity, long long limit, int code) {
  if (ptx::mbar_wait(bar, parity, limit)) return true;
  atomicCAS(&g_wait_error, 0, code);
  return false;
}
// The same for a whole warp: every lane gets the same answer, so that the warp stays together.
__device__ __forceinline__ bool warp_wait_or_record(uint64_t* bar, uint32_t parity, long long limit, int code) {
  return __all_sync(0xFFFFFFFFu, wait_or_record(bar, parity, limit, code));
}

// A place in a ring of N barriers and the parity of its current round.
template <int N> struct Ring {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) at = 0, parity ^= 1;
  }
};

// The copies into a ring of N slots, filled in turn by `issued` loads, have all landed: a CTA does not exit before (after a failed
// wait nothing else may have waited for them).
template <int N> __device__ __forceinline__ void drain(uint64_t* full, int issued) {
  for (int j = max(0, issued - N); j < issued; ++j) wait_or_record(&full[j % N], (j / N) & 1, DRAIN_LIMIT, WAIT_DRAIN);
}

// How rows of queries are put into tiles of up to 128: `tokens` consecutive tokens, `heads` query heads of each, row
// token * heads + head.  All heads of a group as a rule; groups of more than 128 in `chunks`.
struct Tiling {
  int group, heads, chunks, tokens;
  int d16;                      // head size up to a multiple of 16
  long long wait_limit;
  int hold_first_ready;
};

// A unit of work is `tiles` tiles of one sequence, or of the rows behind the last one.  Sequence b's first unit is
// floor(begin_b / W) + b, W tokens to a unit: that leaves room for all of its units whatever the lengths, and finding a
// unit's sequence is a search of the cumulative lengths, without a sum over them.
inline int64_t units(int64_t total, int64_t B, int64_t width) { return total / width + B + 1; }

struct Unit {
  bool any;
  int64_t b, t0;
  Rows rows;
  int kh, chunk;
};
__device__ __forceinline__ int64_t unit_start(const int32_t* cu, int64_t b, int64_t total, int64_t width) {
  return min(max((int64_t)cu[b], (int64_t)0), total) / width + b;
}
// Sequence and first row of unit `index` of a list of rows; `any`: there are rows in it.
__device__ __forceinline__ void find_unit(Unit& u, const int32_t* cu, int64_t B, int64_t total, int64_t width, int64_t index) {
  int64_t lo = 0, hi = B;                       // the last b whose units start at or before index
  while (lo < hi) {
    const int64_t m = (lo + hi + 1) / 2;
    if (unit_start(cu, m, total, width) <= index) lo = m;
    else hi = m - 1;
  }
  u.b = lo;
  if (lo < B) u.rows = rows_of(cu, lo, total);
  else u.rows = {min(max((int64_t)cu[B], (int64_t)0), total), total};
  u.t0 = u.rows.begin + (index - unit_start(cu, lo, total, width)) * width;
  u.any = index >= unit_start(cu, lo, total, width) && u.t0 < u.rows.end;
}
// This CTA's unit of queries: key heads first, then chunks, the sequences' last tiles (with a causal mask the longest)
// before their first.
__device__ __forceinline__ Unit unit_of(const AttnArgs& a, const Tiling& tl, const int32_t* cu, int64_t total, int tiles) {
  Unit u;
  const int64_t width = (int64_t)tiles * tl.tokens;
  const int64_t per = (int64_t)a.Hk * tl.chunks, index = total / width + a.B - blockIdx.x / per;
  const int rest = (int)(blockIdx.x % per);
  u.kh = rest % a.Hk;
  u.chunk = rest / a.Hk;
  find_unit(u, cu, a.B, total, width, index);
  return u;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float shift_of(float m, float c) { return m == -INFINITY ? 0.0f : -m * c; }

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight sums times f (twice, f2) in 16 bits, or with `rest` what that rounding takes away.  worst: NaN once one of them is infinite
// or NaN (a rest of an infinite value is).
template <typename T> __device__ __forceinline__ uint64_t widen2(uint32_t w);
template <> __device__ __forceinline__ uint64_t widen2<__nv_bfloat16>(uint32_t w) { return ptx::join2(w << 16, w & 0xFFFF0000u); }
template <> __device__ __forceinline__ uint64_t widen2<__half>(uint32_t w) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return ptx::join2(__float_as_uint(v.x), __float_as_uint(v.y));
}
template <typename T> __device__ __forceinline__ void round8(const uint32_t* o, uint64_t f2, bool rest, uint64_t& worst, uint32_t (&w)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint64_t v = ptx::mul2(ptx::join2(o[2 * k], o[2 * k + 1]), f2);
    w[k] = pack2<T>(ptx::lo2(v), ptx::hi2(v));
    if (rest) {
      v = ptx::fma2(widen2<T>(w[k]), ptx::join2(0xBF800000u, 0xBF800000u), v);
      w[k] = pack2<T>(ptx::lo2(v), ptx::hi2(v));
    }
    worst = ptx::fma2(v, 0, worst);
  }
}

// A warp's 32 rows, one to a lane, on their way out through 32 x CHUNKS x 16 bytes of shared memory: stored by the lanes that have
// them, each 16-byte piece would be a memory line of its own, and the stores were an eighth of the forward pass.
template <int CHUNKS> struct RowsOut {
  uint8_t* at;
  static __device__ __forceinline__ int place(int row, int k) { return (row * CHUNKS + (k ^ (CHUNKS == 4 ? row >> 1 & 3 : row & 7))) * 16; }
  __device__ __forceinline__ void put(int k, const uint32_t (&v)[4]) { *reinterpret_cast<uint4*>(at + place(threadIdx.x & 31, k)) = make_uint4(v[0], v[1], v[2], v[3]); }
  // To `to` of each lane that has `any`, the first `count` pieces.  (The whole warp.)
  __device__ __forceinline__ void store(void* to, bool any, int count) {
    const int lane = threadIdx.x & 31, k = lane % CHUNKS;
    const uint32_t rows = __ballot_sync(0xFFFFFFFFu, any);   // (the warp's writes above come before the reads below)
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < 32; i += 32 / CHUNKS) {
      const int row = i + lane / CHUNKS;
      uint8_t* p = reinterpret_cast<uint8_t*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(to), row));
      const uint4 v = *reinterpret_cast<const uint4*>(at + place(row, k));
      if ((rows >> row & 1) && k < count) *reinterpret_cast<uint4*>(p + 16 * k) = v;
    }
    __syncwarp();
  }
};

// ------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode() {
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

// Makes the current device's context this thread's: encoding a tensor map is a driver call, which takes what is current, and
// in a thread without earlier CUDA calls (an autograd worker) nothing is.
inline cudaError_t bind_context() {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  return e == cudaSuccess ? cudaSetDevice(dev) : e;
}

// Rows [tokens][heads][D] of 16-bit elements with 128-byte swizzle: boxes of 64 elements x box_heads x box_tokens; what is
// past D, the heads or the tokens reads as zero.  (A tensor without rows gets a map of one row that no load reaches.)
inline bool make_rows_map(CUtensorMap* m, const void* base, int64_t tokens, int64_t heads, int64_t D, const int64_t* stride, int dtype, int box_heads, int box_tokens) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return false;
  alignas(16) static const uint8_t nothing[16] = {};
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)std::max<int64_t>(tokens, 1)};
  cuuint64_t strides[2] = {(cuuint64_t)stride[1] * 2, (cuuint64_t)stride[0] * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  cuuint32_t es[3] = {1, 1, 1};
  return enc(m, dtype == EMU_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<void*>(tokens ? base : nothing), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static inline cudaError_t take_error(int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_wait_error, sizeof(int));
  if (e != cudaSuccess || *code == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_wait_error, &zero, sizeof(int));
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

inline Tiling tiling_of(const AttnArgs& a) {
  Tiling t{};
  t.group = a.Hq / a.Hk;
  t.chunks = (t.group + 127) / 128;
  t.heads = (t.group + t.chunks - 1) / t.chunks;
  t.tokens = 128 / t.heads;
  t.d16 = (a.D + 15) / 16 * 16;
  t.wait_limit = current_wait_limit();
  t.hold_first_ready = current_hold_first_ready();
  return t;
}

}  // namespace attn
}  // namespace emu
