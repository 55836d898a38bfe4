// Attention of one new token for each sequence over the quantised key/value cache.
//
// With s_j = scale q . k_j over the cached rows j < len of the sequence whose page exists, k_j = code * scale as it is
// stored:  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), m = max_j s_j   (no row: o = 0, lse = -inf)
//
// Bound: reading the cache once.  The query heads that share a key head (16 to an item) are the rows of m16n8k16 MMAs, so
// that each code is converted once for all of them; the codes become fp16, which holds all of their values, without
// their scales:
//   scores   q is multiplied by a power of two that puts its row's largest element into [2^14, 2^15) (exact for both 16-bit
//            types but for elements 2^-24 and more below the largest) and the sum over a block is multiplied by the
//            key's scale of that block in f32;
//   values   the scale goes into the weight: p * scale, relative to the largest scale that the warp has met in that
//            block of the head, rounded to fp16 (2^-11 relative; weights of up to 2^-30 of the largest keep all their bits)
// A step of this size is bound by bytes and not by products (about 90 MACs per byte for 16 heads), which mma.sync serves
// from registers; tcgen05 would want the converted codes in shared memory first.
//
// The work is cut into tiles of 64 keys and dealt out evenly over the CTAs, whatever the lengths: a CTA takes a run of tiles
// of one or several (sequence, head)s.  Where a run is not all of a (sequence, head), its sums go to the workspace, and a
// second kernel joins them in the tiles' order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/emugen.h"
#include "kernels.h"

namespace emu {
namespace {

constexpr int WARPS = 4, NT = WARPS * 32, KEYS = 16, TILE = WARPS * KEYS;

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^e, 0 below f32's normal range, for e <= 127
__device__ __forceinline__ float pow2(int e) { return __int_as_float(e < -126 ? 0 : (e + 127) << 23); }

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two codes -> two fp16 (the low byte's first)
__device__ __forceinline__ uint32_t half2_of_e4m3(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t half2_of_e2m1(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)two, __NV_E2M1);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, bool any) {
  const int n = any ? 16 : 0;                                // 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// The shapes of a format at a padded head size.
template <int FORMAT, int DP> struct Shape {
  static constexpr bool FP8 = FORMAT == EMU_KV_FP8;
  static constexpr int ROW = FP8 ? DP : DP / 2;              // bytes of a row of codes
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int BLOCKS = FP8 ? (DP + 127) / 128 : DP / 32;
  static constexpr int CODES = KEYS * ROW;                   // keys (or values) of a stage
  static constexpr int SCALES = BLOCKS * KEYS * 4;           // [block][key], 32 bits each
  static constexpr int STAGE = 2 * (CODES + SCALES);
  static constexpr int STAGES = FP8 && DP == 256 ? 3 : 4;    // two or three CTAs to an SM, see ctas_per_sm
  static constexpr int JOIN = 16 * (DP + 4) * 4;             // a warp's sums
  static constexpr int WARP = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
  static constexpr int SMEM = WARPS * WARP + WARPS * 16 * 8 + WARPS * STAGES * 4 + 64;
};
// Where chunk `c` of row r lies: lines of 128 bytes, the chunk's place in its line turned so that the lanes that read
// together meet all banks (K: 8 rows and 4 neighbours each; V: every other row and 8 neighbours).
template <int FORMAT, int DP, bool VALUES> __device__ __forceinline__ uint32_t place(int r, int c) {
  using S = Shape<FORMAT, DP>;
  const int at = r * S::CHUNKS + c, line = at >> 3;
  int turn;
  if (S::FP8) {
    if (DP == 64) turn = (line * 2) & 7;
    else turn = VALUES ? r & 7 : (r & 1) * 4;
  } else {
    turn = DP == 64 ? line & 1 : DP == 128 ? line & 3 : r & 7;
  }
  return (uint32_t)(line * 128 + ((at & 7) ^ turn) * 16);
}

// The tiles of a sequence (of each of its heads).
__device__ __forceinline__ int64_t tiles_of(const KvAttendArgs& a, int64_t b) {
  const int64_t len = min((int64_t)a.lens[b], a.table_cols * a.page_size);
  return len > 0 ? (len + TILE - 1) / TILE : 0;
}
// Sum over the block of v, and the sum over the threads before this one.  (All threads.)
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* tmp, int64_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t n = __shfl_up_sync(0xFFFFFFFFu, s, o);
    if (lane >= o) s += n;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = s;
  __syncthreads();
  int64_t before = 0;
  all = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += tmp[w];
    all += tmp[w];
  }
  return before + s - v;
}
struct Place {
  int64_t total;               // tiles of all (sequence, head)s
  int64_t lo, hi;              // this CTA's run of them
  int64_t b, first;            // the sequence of tile `lo`, and its first tile
};
// CTA `cta`'s run, of heads * the sequences' tiles.  (All threads; found: 2 words of shared memory.)
__device__ __forceinline__ Place locate(const KvAttendArgs& a, int heads, int cta, int ctas, int64_t* tmp, int64_t* found) {
  Place p;
  int64_t sum = 0;
  for (int64_t i = threadIdx.x; i < a.B; i += blockDim.x) sum += tiles_of(a, i);
  block_scan(sum, tmp, p.total);
  p.total *= heads;
  p.lo = p.total * cta / ctas, p.hi = p.total * (cta + 1) / ctas;
  p.b = p.first = 0;
  if (p.lo >= p.hi) return p;
  int64_t base = 0;
  for (int64_t b0 = 0; b0 < a.B && base <= p.lo; b0 += blockDim.x) {
    const int64_t n = b0 + threadIdx.x < a.B ? tiles_of(a, b0 + threadIdx.x) * heads : 0;
    int64_t all;
    const int64_t before = base + block_scan(n, tmp, all);
    if (before <= p.lo && p.lo < before + n) found[0] = b0 + threadIdx.x, found[1] = before;
    base += all;
  }
  __syncthreads();
  p.b = found[0], p.first = found[1];
  return p;
}

struct Parts {
  float* o;                    // [slot][rows][D]
  float2* ml;                  // [slot][rows]: maximum (of log2 scores), sum
};
__host__ __device__ inline Parts parts_of(void* workspace, int64_t slots, int rows) {
  Parts p;
  p.ml = static_cast<float2*>(workspace);
  p.o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (slots * rows * sizeof(float2) + 255) / 256 * 256);
  return p;
}
struct Plan {
  int ctas, groups, rows;      // CTAs, items of up to 16 query heads to a key head, rows of an item
  bool wide_scales;            // MXFP4: a row's scale bytes may be read at once
  uint32_t page_size;          // up to 2^31 (more than any length)
};

// As many as registers (and shared memory) allow.
constexpr int ctas_per_sm(int DP, bool two) { return DP == 256 || (DP == 128 && two) ? 2 : 3; }
constexpr int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

template <typename T, int FORMAT, int DP, bool TWO>
__global__ void __launch_bounds__(NT, ctas_per_sm(DP, TWO)) kv_attend_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ Plan pl) {
  using S = Shape<FORMAT, DP>;
  constexpr int STAGES = S::STAGES, NB = S::BLOCKS, STEPS = DP / 16, NTS = DP / 8, PER = NTS / NB, R = TWO ? 2 : 1;   // PER: MMAs of a block of values
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t tmp[WARPS], found[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint8_t* mine = smem + warp * S::WARP;
  float2* join_ml = reinterpret_cast<float2*>(smem + WARPS * S::WARP);            // [warp][16]
  uint32_t* live = reinterpret_cast<uint32_t*>(join_ml + WARPS * 16) + warp * STAGES;
  const uint32_t mine_u = (uint32_t)__cvta_generic_to_shared(mine);
  const int D = a.D, HV = a.Hk * pl.groups, group = a.Hq / a.Hk;

  // sequences that have nothing
  for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x)
    if (tiles_of(a, b) == 0) {
      for (int64_t x = threadIdx.x; x < (int64_t)a.Hq * D; x += NT) static_cast<T*>(a.out)[b * a.Hq * D + x] = narrow<T>(0.0f);
      if (a.lse)
        for (int h = threadIdx.x; h < a.Hq; h += NT) a.lse[b * a.Hq + h] = -INFINITY;
    }
  // this CTA's run of tiles
  const Place run = locate(a, HV, blockIdx.x, pl.ctas, tmp, found);
  int64_t b = run.b, first = run.first, at = run.lo;         // `at` in the list of all tiles
  const int64_t hi = run.hi;
  const Parts parts = parts_of(a.workspace, 2 * (int64_t)pl.ctas, pl.rows);

  while (at < hi) {
    const int64_t per = tiles_of(a, b);
    if (per == 0 || at >= first + per * HV) {
      first += per * HV;
      ++b;
      continue;
    }
    const int hv = (int)((at - first) / per);
    const int64_t tile0 = at - first - hv * per, tile1 = min(per, tile0 + (hi - at));
    const int kh = hv / pl.groups, h0 = kh * group + (hv % pl.groups) * 16, rows = min(16, group - (hv % pl.groups) * 16);
    const int len = (int)min((int64_t)a.lens[b], a.table_cols * a.page_size);
    const int32_t* table = a.table + b * a.table_stride;

    // ---- q: this lane's elements of rows g and g + 8, as the MMAs' A operands
    uint32_t q[STEPS][2 * R];
    float qf[R];                                             // what a score of the row is multiplied by
    {
      auto place_of = [&](int s) {                           // the first of a step's two pairs
        return S::FP8 ? (c + 4 * (s >> 2)) * 16 + (s & 3) * 4 : (s >> 1) * 32 + c * 8 + (s & 1) * 4;
      };
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = g + 8 * r;
        const T* src = static_cast<const T*>(a.q) + b * a.q_stride[0] + (int64_t)(h0 + row) * a.q_stride[1];
        float v[STEPS][4], top = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[s][e] = row < rows && place_of(s) + e < D ? widen<T>(src[place_of(s) + e]) : 0.0f;
            top = fmaxf(top, fabsf(v[s][e]));
          }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        int e2 = top > 0.0f && top < INFINITY ? ilogbf(top) : 14;
        e2 = max(e2, -113);
        const float f = pow2(14 - e2);
        qf[r] = a.scale * 1.4426950408889634f * pow2(max(e2 - 14, -126));
        if (e2 - 14 < -126) qf[r] *= pow2(e2 - 14 + 126);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          q[s][r] = pack_half(v[s][0] * f, v[s][1] * f);
          q[s][R + r] = pack_half(v[s][2] * f, v[s][3] * f);
        }
      }
    }

    float o[NTS][2 * R] = {}, m[R], l[R] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -INFINITY;
    int ref[NB];                                             // exponent of the largest scale of values so far
#pragma unroll
    for (int k = 0; k < NB; ++k) ref[k] = -1000;

    // ---- steps of 16 keys; the warps take them in turn
    const int key0 = (int)(tile0 * TILE) + warp * KEYS, end = (int)min((int64_t)len, tile1 * TILE);
    const int steps = (int)(tile1 - tile0);
    const int my = lane & 15;
    auto page_of = [&](int i) {                              // the page of this lane's key of step i
      const int key = key0 + i * TILE + my;
      return i < steps && key < end ? __ldg(table + (uint32_t)key / pl.page_size) : -1;
    };
    const int RB = S::FP8 ? D : D / 2, nb = S::FP8 ? (D + 127) / 128 : D / 32, chunks = RB / 16;
    uint32_t sc[NB];                                         // scales on their way: lanes 0-15 keys', 16-31 values'
    // codes of step i into its stage, its scales into registers
    auto fetch = [&](int i, int page) {
      const int key = key0 + i * TILE + my;
      const bool ok = page >= 0 && page < a.num_pages;       // (page is -1 past the end)
      const int64_t row = ok ? ((int64_t)page * a.page_size + (uint32_t)key % pl.page_size) * a.Hk + kh : 0;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, ok) & 0xFFFFu;
      const int64_t at_row = row * RB;
      const uint32_t st = mine_u + (i % STAGES) * S::STAGE;
#pragma unroll
      for (int x = 0; x < KEYS * S::CHUNKS / 32; ++x) {
        const int idx = lane + 32 * x, r = idx / S::CHUNKS, ch = idx % S::CHUNKS;
        const int64_t src = __shfl_sync(0xFFFFFFFFu, at_row, r);
        const bool any = (mask >> r & 1) && ch < chunks;
        copy16(st + place<FORMAT, DP, false>(r, ch), a.cache[0] + (any ? src + ch * 16 : 0), any);
        copy16(st + S::CODES + place<FORMAT, DP, true>(r, ch), a.cache[1] + (any ? src + ch * 16 : 0), any);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      const void* src = lane < 16 ? a.scales[0] : a.scales[1];
      if (S::FP8) {
#pragma unroll
        for (int k = 0; k < NB; ++k) sc[k] = ok && k < nb ? __float_as_uint(__ldg(static_cast<const float*>(src) + row * nb + k)) : 0;
      } else {
        const uint8_t* p = static_cast<const uint8_t*>(src) + row * nb;
        if (pl.wide_scales) {
          uint64_t w = 0;
          if (ok) w = NB == 2 ? __ldg(reinterpret_cast<const uint16_t*>(p)) : NB == 4 ? __ldg(reinterpret_cast<const uint32_t*>(p)) : __ldg(reinterpret_cast<const unsigned long long*>(p));
#pragma unroll
          for (int k = 0; k < NB; ++k) sc[k] = (uint32_t)(w >> (8 * k)) & 255u;
        } else {
#pragma unroll
          for (int k = 0; k < NB; ++k) sc[k] = ok && k < nb ? __ldg(p + k) : 0;
        }
      }
      if (lane == 0) live[i % STAGES] = mask;
    };
    // the scales that `fetch` of step i asked for
    auto put_scales = [&](int i) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(mine + (i % STAGES) * S::STAGE + 2 * S::CODES + (lane < 16 ? 0 : S::SCALES));
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        // MXFP4 keys: 2^(byte - 127); byte 0 is f32's subnormal 2^-127, byte 255 infinity.  Values: the byte.
        const uint32_t v = S::FP8 || lane >= 16 ? sc[k] : sc[k] ? sc[k] << 23 : 0x00400000u;
        dst[k * KEYS + my] = v;
      }
    };
    int page = page_of(0);
    for (int i = 0; i < STAGES - 1; ++i) {
      const int next = page_of(i + 1);
      fetch(i, page);
      page = next;
      put_scales(i);
    }
    for (int i = 0; i < steps; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      // the next step to fetch, into the stage that was read last
      const int next = page_of(i + STAGES);
      fetch(i + STAGES - 1, page);
      page = next;
      const uint8_t* kc = mine + (i % STAGES) * S::STAGE;
      const uint8_t* vc = kc + S::CODES;
      const float* ks = reinterpret_cast<const float*>(kc + 2 * S::CODES);
      const uint32_t* vs = reinterpret_cast<const uint32_t*>(kc + 2 * S::CODES + S::SCALES);
      const uint32_t mask = live[i % STAGES];
      // ---- scores of rows g (and g + 8) with keys 8 t + 2 c and 8 t + 2 c + 1
      float s[2][2 * R];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int e = 0; e < 2 * R; ++e) s[t][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          float acc[4] = {};
          if (S::FP8) {
#pragma unroll
            for (int x = 2 * k; x < 2 * k + 2 && x < DP / 64; ++x) {
              const uint4 w = *reinterpret_cast<const uint4*>(kc + place<FORMAT, DP, false>(8 * t + g, c + 4 * x));
              const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int st = 4 * x + y;
                mma(acc, q[st][0], TWO ? q[st][1] : 0, q[st][R], TWO ? q[st][R + R - 1] : 0, half2_of_e4m3(ws[y] & 0xFFFFu), half2_of_e4m3(ws[y] >> 16));
              }
            }
          } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + place<FORMAT, DP, false>(8 * t + g, k) + 4 * c);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int st = 2 * k + y;
              mma(acc, q[st][0], TWO ? q[st][1] : 0, q[st][R], TWO ? q[st][R + R - 1] : 0, half2_of_e2m1(w >> (16 * y) & 255u), half2_of_e2m1(w >> (16 * y + 8) & 255u));
            }
          }
          const float2 f = *reinterpret_cast<const float2*>(ks + k * KEYS + 8 * t + 2 * c);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            s[t][2 * r] = __fmaf_rn(acc[2 * r], f.x, s[t][2 * r]);
            s[t][2 * r + 1] = __fmaf_rn(acc[2 * r + 1], f.y, s[t][2 * r + 1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2 * R; ++e)
          s[t][e] = mask >> (8 * t + 2 * c + (e & 1)) & 1 ? __fmul_rn(s[t][e], qf[e >> 1]) : -INFINITY;
      }
      // ---- the running maximum: held up to a factor of 2^8
      bool grow = false;
      float top[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        grow = grow || top[r] - m[r] > 8.0f;
      }
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 1));
          top[r] = fmaxf(m[r], fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 2)));
          const float f = top[r] == -INFINITY ? 1.0f : exp2_approx(m[r] - top[r]);
          m[r] = top[r];
          l[r] *= f;
#pragma unroll
          for (int n = 0; n < NTS; ++n) o[n][2 * r] *= f, o[n][2 * r + 1] *= f;
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float sh = m[r] == -INFINITY ? 0.0f : m[r];
          s[t][2 * r] = exp2_approx(s[t][2 * r] - sh), s[t][2 * r + 1] = exp2_approx(s[t][2 * r + 1] - sh);
          l[r] += s[t][2 * r] + s[t][2 * r + 1];
        }
      // ---- values, block by block: weight = p * scale / 2^ref * 2^6 (below 2^8 * 2 * 2^6)
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        float f[4];                                          // keys 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c
        {
          const uint2 lo2 = *reinterpret_cast<const uint2*>(vs + k * KEYS + 2 * c), hi2 = *reinterpret_cast<const uint2*>(vs + k * KEYS + 8 + 2 * c);
          const uint32_t w[4] = {lo2.x, lo2.y, hi2.x, hi2.y};
          int e[4], most = -1000;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            e[x] = S::FP8 ? (int)(w[x] >> 23 & 255u) : (int)w[x];
            if (e[x] != 255) most = max(most, e[x]);         // (infinities and NaN go through as they are)
          }
          if (__any_sync(0xFFFFFFFFu, most > ref[k])) {
            most = __reduce_max_sync(0xFFFFFFFFu, most);
            const float down = ref[k] < 0 ? 1.0f : pow2(ref[k] - most);
#pragma unroll
            for (int n = k * PER; n < (k + 1) * PER; ++n)
#pragma unroll
              for (int y = 0; y < 2 * R; ++y) o[n][y] *= down;
            ref[k] = most;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (S::FP8) {
              const int up = 133 - max(ref[k], 0);                   // 2^(6 - (ref - 127)), in two factors that both exist
              f[x] = __uint_as_float(w[x]) * pow2(up / 2) * pow2(up - up / 2);
            } else {
              f[x] = e[x] == 255 ? INFINITY : pow2(e[x] - ref[k] + 6);
            }
          }
        }
        uint32_t p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          p[2 * t] = pack_half(s[t][0] * f[2 * t], s[t][1] * f[2 * t + 1]);
          p[2 * t + 1] = TWO ? pack_half(s[t][2 * R - 2] * f[2 * t], s[t][2 * R - 1] * f[2 * t + 1]) : 0;
        }
        const int rv[4] = {2 * c, 2 * c + 1, 8 + 2 * c, 9 + 2 * c};
        if (S::FP8) {
          // block k's codes of lane g: elements 128 k + g * PER .. of the four rows, as pairs of rows
          {
            uint32_t w[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              if (DP == 64) {
                const uint2 v = *reinterpret_cast<const uint2*>(vc + place<FORMAT, DP, true>(rv[y], g >> 1) + (g & 1) * 8);
                w[y][0] = v.x, w[y][1] = v.y, w[y][2] = w[y][3] = 0;
              } else {
                const uint4 v = *reinterpret_cast<const uint4*>(vc + place<FORMAT, DP, true>(rv[y], 8 * k + g));
                w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
              }
            }
#pragma unroll
            for (int z = 0; z < (DP == 64 ? 2 : 4); ++z) {
              const uint32_t a0 = __byte_perm(w[0][z], w[1][z], 0x5140), a1 = __byte_perm(w[0][z], w[1][z], 0x7362);
              const uint32_t b0 = __byte_perm(w[2][z], w[3][z], 0x5140), b1 = __byte_perm(w[2][z], w[3][z], 0x7362);
              const int n = k * PER + z * 4;
              auto step = [&](int at_n, uint32_t u, uint32_t v) {
                float acc[4] = {o[at_n][0], o[at_n][1], TWO ? o[at_n][2 * R - 2] : 0.0f, TWO ? o[at_n][2 * R - 1] : 0.0f};
                mma(acc, p[0], p[1], p[2], p[3], half2_of_e4m3(u), half2_of_e4m3(v));
                o[at_n][0] = acc[0], o[at_n][1] = acc[1];
                if (TWO) o[at_n][2 * R - 2] = acc[2], o[at_n][2 * R - 1] = acc[3];
              };
              step(n, a0 & 0xFFFFu, b0 & 0xFFFFu);
              step(n + 1, a0 >> 16, b0 >> 16);
              step(n + 2, a1 & 0xFFFFu, b1 & 0xFFFFu);
              step(n + 3, a1 >> 16, b1 >> 16);
            }
          }
        } else {
          // block k: elements 32 k + 4 g .. + 3 of the four rows
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) w[y] = *reinterpret_cast<const uint16_t*>(vc + place<FORMAT, DP, true>(rv[y], k) + 2 * g);
          // pairs of rows: nibbles of two rows side by side in a byte
          const uint32_t even0 = (w[0] & 0x0F0Fu) | (w[1] & 0x0F0Fu) << 4, odd0 = (w[0] >> 4 & 0x0F0Fu) | (w[1] & 0xF0F0u);
          const uint32_t even1 = (w[2] & 0x0F0Fu) | (w[3] & 0x0F0Fu) << 4, odd1 = (w[2] >> 4 & 0x0F0Fu) | (w[3] & 0xF0F0u);
          auto step = [&](int at_n, uint32_t u, uint32_t v) {
            float acc[4] = {o[at_n][0], o[at_n][1], TWO ? o[at_n][2 * R - 2] : 0.0f, TWO ? o[at_n][2 * R - 1] : 0.0f};
            mma(acc, p[0], p[1], p[2], p[3], half2_of_e2m1(u), half2_of_e2m1(v));
            o[at_n][0] = acc[0], o[at_n][1] = acc[1];
            if (TWO) o[at_n][2 * R - 2] = acc[2], o[at_n][2 * R - 1] = acc[3];
          };
          step(4 * k, even0 & 255u, even1 & 255u);
          step(4 * k + 1, odd0 & 255u, odd1 & 255u);
          step(4 * k + 2, even0 >> 8, even1 >> 8);
          step(4 * k + 3, odd0 >> 8, odd1 >> 8);
        }
      }
      // the scales asked for above; their stage is read next in STAGES - 1 steps
      put_scales(i + STAGES - 1);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- join the warps
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
    }
    __syncwarp();
    float* sums = reinterpret_cast<float*>(mine);            // [row][DP + 4], over the warp's own stages
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (c == 0) join_ml[warp * 16 + g + 8 * r] = make_float2(m[r], l[r]);
#pragma unroll
      for (int n = 0; n < NTS; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int col = 2 * c + y;
          const int d = (n / PER) * 8 * PER + col * PER + n % PER;
          const int up = max(ref[n / PER], 0) - 133;                   // 2^(ref - 127 - 6)
          sums[(g + 8 * r) * (DP + 4) + d] = o[n][2 * r + y] * pow2(up / 2) * pow2(up - up / 2);
        }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == per;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (tile0 == 0 ? 1 : 0);
    for (int x = threadIdx.x; x < rows * D; x += NT) {
      const int row = x / D, d = x - row * D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, join_ml[w * 16 + row].x);
      const float sh = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, v = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float2 ml = join_ml[w * 16 + row];
        const float f = exp2_approx(ml.x - sh);
        sum = __fmaf_rn(ml.y, f, sum);
        v = __fmaf_rn(reinterpret_cast<const float*>(smem + w * S::WARP)[row * (DP + 4) + d], f, v);
      }
      if (whole) {
        const int64_t i = b * a.Hq + h0 + row;
        static_cast<T*>(a.out)[i * D + d] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
        if (d == 0 && a.lse) a.lse[i] = sum > 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
      } else {
        parts.o[(slot * pl.rows + row) * D + d] = v;
        if (d == 0) parts.ml[slot * pl.rows + row] = make_float2(top, sum);
      }
    }
    __syncthreads();
    at += tile1 - tile0;
  }
}

// Joins the sums of each (sequence, head) that lies in several CTAs, in the order of its tiles: CTA (i, row) those of one row
// where the run of the attention's CTA i ends it and another began it.
constexpr int JOIN_NT = 512;
template <typename T> __global__ void __launch_bounds__(JOIN_NT) kv_attend_join_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ Plan pl, int lanes) {
  __shared__ int64_t tmp[JOIN_NT / 32], found[2];
  __shared__ float so[JOIN_NT], sl[JOIN_NT], stop[JOIN_NT / 32];
  const int group = a.Hq / a.Hk, HV = a.Hk * pl.groups, row = blockIdx.y;
  const Place run = locate(a, HV, blockIdx.x, pl.ctas, tmp, found);
  if (run.lo >= run.hi) return;
  const int64_t b = run.b, per = tiles_of(a, b);
  const int hv = (int)((run.lo - run.first) / per);
  const int64_t first = run.first + hv * per;
  if (first == run.lo || first + per > run.hi) return;       // begins here, or does not end here
  const int hq = hv % pl.groups * 16 + row, h = hv / pl.groups * group + hq;
  if (hq >= group) return;
  int64_t c0 = first * pl.ctas / run.total;                  // the CTA of its first tile
  while (run.total * (c0 + 1) / pl.ctas <= first) ++c0;
  while (run.total * c0 / pl.ctas > first) --c0;
  const Parts parts = parts_of(a.workspace, 2 * (int64_t)pl.ctas, pl.rows);
  const int n = (int)(blockIdx.x - c0) + 1;
  auto slot = [&](int i) { return (2 * (c0 + i) + (i == 0 ? 1 : 0)) * pl.rows + row; };
  // (where there are fewer tiles than CTAs, some have none and no part)
  auto has = [&](int i) { return run.total * (c0 + i) / pl.ctas < run.total * (c0 + i + 1) / pl.ctas; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < n; i += JOIN_NT)
    if (has(i)) top = fmaxf(top, parts.ml[slot(i)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if ((threadIdx.x & 31) == 0) stop[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < JOIN_NT / 32; ++w) top = fmaxf(top, stop[w]);
  const float sh = top == -INFINITY ? 0.0f : top;
  const int d = threadIdx.x % lanes, part = threadIdx.x / lanes, step = JOIN_NT / lanes;
  float v = 0.0f, sum = 0.0f;
  for (int i = part; i < n; i += step)
    if (has(i)) {
      const float2 ml = parts.ml[slot(i)];
      const float f = exp2_approx(ml.x - sh);
      sum = __fmaf_rn(ml.y, f, sum);
      if (d < a.D) v = __fmaf_rn(parts.o[slot(i) * a.D + d], f, v);
    }
  so[threadIdx.x] = v;
  if (d == 0) sl[part] = sum;
  __syncthreads();
  if (threadIdx.x < a.D) {
    v = 0.0f, sum = 0.0f;
    for (int x = 0; x < step; ++x) v = __fadd_rn(v, so[x * lanes + threadIdx.x]), sum = __fadd_rn(sum, sl[x]);
    const int64_t i = b * a.Hq + h;
    static_cast<T*>(a.out)[i * a.D + threadIdx.x] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
    if (threadIdx.x == 0 && a.lse) a.lse[i] = sum > 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
  }
}

Plan plan_of(int Hq, int Hk, int D) {
  Plan p{};
  const int group = Hq / Hk;
  p.groups = (group + 15) / 16;
  p.rows = std::min(group, 16);
  p.ctas = ctas_per_sm(padded(D), p.rows > 8) * sm_count();
  return p;
}

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

template <typename T, int FORMAT, int DP, bool TWO> cudaError_t launch(const KvAttendArgs& a, Plan pl, cudaStream_t stream) {
  using S = Shape<FORMAT, DP>;
  auto kernel = kv_attend_kernel<T, FORMAT, DP, TWO>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_shared(kernel, S::SMEM, done);
  if (e != cudaSuccess) return e;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.scales[0]) | reinterpret_cast<uintptr_t>(a.scales[1]);
  pl.wide_scales = FORMAT == EMU_KV_MXFP4 && a.D == DP && at % S::BLOCKS == 0;
  pl.page_size = (uint32_t)std::min<int64_t>(a.page_size, 1ll << 31);
  kernel<<<pl.ctas, NT, S::SMEM, stream>>>(a, pl);
  kv_attend_join_kernel<T><<<dim3(pl.ctas, pl.rows), JOIN_NT, 0, stream>>>(a, pl, DP);
  return cudaGetLastError();
}
template <typename T, int FORMAT> cudaError_t launch_sized(const KvAttendArgs& a, cudaStream_t stream) {
  const Plan pl = plan_of(a.Hq, a.Hk, a.D);
  const bool two = pl.rows > 8;
  if (a.D <= 64) return two ? launch<T, FORMAT, 64, true>(a, pl, stream) : launch<T, FORMAT, 64, false>(a, pl, stream);
  if (a.D <= 128) return two ? launch<T, FORMAT, 128, true>(a, pl, stream) : launch<T, FORMAT, 128, false>(a, pl, stream);
  return two ? launch<T, FORMAT, 256, true>(a, pl, stream) : launch<T, FORMAT, 256, false>(a, pl, stream);
}

}  // namespace

size_t kv_attend_workspace(int64_t, int Hq, int Hk, int D) {
  const Plan p = plan_of(Hq, Hk, D);
  const int64_t slots = 2 * (int64_t)p.ctas;
  return (slots * p.rows * sizeof(float2) + 255) / 256 * 256 + slots * p.rows * D * sizeof(float);
}

cudaError_t launch_kv_attend(const KvAttendArgs& a, cudaStream_t stream) {
  const bool half = a.dtype == EMU_DTYPE_F16;
  if (a.format == EMU_KV_FP8) return half ? launch_sized<__half, EMU_KV_FP8>(a, stream) : launch_sized<__nv_bfloat16, EMU_KV_FP8>(a, stream);
  return half ? launch_sized<__half, EMU_KV_MXFP4>(a, stream) : launch_sized<__nv_bfloat16, EMU_KV_MXFP4>(a, stream);
}

}  // namespace emu
