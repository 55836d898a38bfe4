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
  static constexpr int STAGES = FP8 && DP >= 128 ? 3 : 4;    // what ctas_per_sm leaves room for
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
  return len > 0 && a.num_pages > 0 ? (len + TILE - 1) / TILE : 0;
}
// What a (sequence, head) counts for when the work is dealt out: its tiles and EXTRA places before them, for what
// starting and joining it costs.
constexpr int EXTRA = 2;
__device__ __forceinline__ int64_t places_of(const KvAttendArgs& a, int64_t b) {
  const int64_t n = tiles_of(a, b);
  return n ? n + EXTRA : 0;
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
// `total` places over `ctas` CTAs: CTA i's first one, and the CTA that has a place.
struct Deal {
  int64_t base;
  int rest;
  __device__ __forceinline__ Deal(int64_t total, int ctas) {
    base = total <= 0x7FFFFFFF ? (int64_t)((uint32_t)total / (uint32_t)ctas) : total / ctas;
    rest = (int)(total - base * ctas);
  }
  __device__ __forceinline__ int64_t begin(int i) const { return base * i + min(i, rest); }
  __device__ __forceinline__ int owner(int64_t place) const {
    const int64_t big = (base + 1) * rest;                   // places of the CTAs with one more
    if (place < big) return (int)(place / (base + 1));
    return rest + (int)((place - big) / base);
  }
};

// The workspace: what each CTA ends, and the sums of its first and its last (sequence, head) where they are parts.
struct Ending;
struct Parts {
  Ending* endings;             // [CTA]
  float2* ml;                  // [slot][rows]: maximum (of log2 scores), sum
  float* o;                    // [slot][rows][D]
  size_t bytes;
};
__host__ __device__ inline Parts parts_of(void* workspace, int64_t ctas, int rows, int D) {
  uint8_t* base = static_cast<uint8_t*>(workspace);
  const size_t ml = (size_t)(ctas * 16 + 255) / 256 * 256, o = ml + (2 * ctas * rows * sizeof(float2) + 255) / 256 * 256;
  return {reinterpret_cast<Ending*>(base), reinterpret_cast<float2*>(base + ml), reinterpret_cast<float*>(base + o), o + 2 * ctas * rows * D * sizeof(float)};
}
struct Plan {
  int ctas, groups, rows;      // CTAs, items of up to 16 query heads to a key head, rows of an item
  bool wide_scales;            // MXFP4: a row's scale bytes may be read at once
  bool whole_steps;            // a step's 16 keys lie in one page
  uint32_t page_size;          // up to 2^31 (more than any length)
};
// What a CTA leaves for the join: where its run ends a (sequence, head) that another CTA began.
struct Ending {
  int64_t out;                 // the first row of the outputs
  int rows, first;             // rows (0: nothing to join), the CTA that began it
};

// As many as registers (and shared memory) allow.
constexpr int ctas_per_sm(int DP, bool two) { return DP == 256 ? 2 : DP == 128 && two ? 3 : 4; }
constexpr int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

template <typename T, int FORMAT, int DP, bool TWO>
__global__ void __launch_bounds__(NT, ctas_per_sm(DP, TWO)) kv_attend_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ Plan pl) {
  using S = Shape<FORMAT, DP>;
  // d-tiles of 16 (DT), those of a block of values (PER), groups of 8 heads (R)
  constexpr int STAGES = S::STAGES, NB = S::BLOCKS, STEPS = DP / 16, DT = DP / 16, PER = DT / NB, R = TWO ? 2 : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t tmp[WARPS], found[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint8_t* mine = smem + warp * S::WARP;
  float2* join_ml = reinterpret_cast<float2*>(smem + WARPS * S::WARP);            // [warp][16]
  uint32_t* live = reinterpret_cast<uint32_t*>(join_ml + WARPS * 16) + warp * STAGES;
  const uint32_t mine_u = (uint32_t)__cvta_generic_to_shared(mine);
  const int D = a.D, HV = a.Hk * pl.groups, group = a.Hq / a.Hk;
  const Parts parts = parts_of(a.workspace, pl.ctas, pl.rows, D);

  asm volatile("griddepcontrol.launch_dependents;");        // the join's CTAs may come when there is room
  // this CTA's run of places
  int64_t total = 0, b = 0, first = 0;                       // sequence b's first place
  {
    int64_t base = 0;
    if (a.B <= NT) {
      const int64_t n = threadIdx.x < a.B ? places_of(a, threadIdx.x) * HV : 0;
      const int64_t before = block_scan(n, tmp, total);
      const int64_t lo = Deal(total, pl.ctas).begin(blockIdx.x);
      if (before <= lo && lo < before + n) found[0] = threadIdx.x, found[1] = before;
    } else {
      int64_t sum = 0;
      for (int64_t i = threadIdx.x; i < a.B; i += NT) sum += places_of(a, i);
      block_scan(sum * HV, tmp, total);
      const int64_t lo = Deal(total, pl.ctas).begin(blockIdx.x);
      for (int64_t b0 = 0; b0 < a.B && base <= lo; b0 += NT) {
        const int64_t n = b0 + threadIdx.x < a.B ? places_of(a, b0 + threadIdx.x) * HV : 0;
        int64_t all;
        const int64_t before = base + block_scan(n, tmp, all);
        if (before <= lo && lo < before + n) found[0] = b0 + threadIdx.x, found[1] = before;
        base += all;
      }
    }
    __syncthreads();
  }
  const Deal deal(total, pl.ctas);
  int64_t at = deal.begin(blockIdx.x);                       // `at` in the list of all places
  const int64_t hi = deal.begin(blockIdx.x + 1);
  if (at < hi) b = found[0], first = found[1];
  Ending ending{0, 0, 0};

  while (at < hi) {
    const int64_t per = places_of(a, b);
    if (per == 0 || at >= first + per * HV) {
      first += per * HV;
      ++b;
      continue;
    }
    const int hv = at - first <= 0xFFFFFFFF ? (int)((uint32_t)(at - first) / (uint32_t)per) : (int)((at - first) / per);
    const int64_t start = first + hv * per, stop = start + per;                    // this (sequence, head)'s places
    const int64_t tile0 = max((int64_t)0, at - start - EXTRA), tile1 = min(hi, stop) - start - EXTRA;
    at = min(hi, stop);
    if (tile1 <= tile0) continue;
    const int kh = hv / pl.groups, h0 = kh * group + (hv % pl.groups) * 16, rows = min(16, group - (hv % pl.groups) * 16);
    const int len = (int)min((int64_t)a.lens[b], a.table_cols * a.page_size);
    const int32_t* table = a.table + b * a.table_stride;

    // ---- steps of 16 keys; the warps take them in turn
    const int key0 = (int)(tile0 * TILE) + warp * KEYS, end = (int)min((int64_t)len, tile1 * TILE);
    const int steps = (int)(tile1 - tile0);
    const int my = lane & 15;
    // the page of this lane's key of step i (of all of the step's keys); -1 past the end
    auto page_of = [&](int i) {
      const int key = key0 + i * TILE + (pl.whole_steps ? 0 : my);
      return i < steps && key < end ? __ldg(table + (uint32_t)key / pl.page_size) : -1;
    };
    const int RB = S::FP8 ? D : D / 2, nb = S::FP8 ? (D + 127) / 128 : D / 32, chunks = RB / 16;
    uint32_t sc[NB];                                         // scales on their way: lanes 0-15 keys', 16-31 values'
    // codes of step i into its stage, its scales into registers
    auto fetch = [&](int i, int stage, int page) {
      const int key = key0 + i * TILE;
      const bool page_ok = page >= 0 && page < a.num_pages;
      const uint32_t st = mine_u + stage * S::STAGE;
      const int rem = (int)((uint32_t)(key + (pl.whole_steps ? 0 : my)) % pl.page_size);
      int64_t row = page_ok ? ((int64_t)page * a.page_size + rem) * a.Hk + kh : 0;
      uint32_t mask;
      if (pl.whole_steps) {
        const int n = page_ok ? min(KEYS, end - key) : 0;
        mask = (1u << n) - 1;
        const int64_t base = row * RB;
#pragma unroll
        for (int x = 0; x < KEYS * S::CHUNKS / 32; ++x) {
          const int idx = lane + 32 * x, r = idx / S::CHUNKS, ch = idx % S::CHUNKS;
          const bool any = r < n && ch < chunks;
          const int64_t src = any ? base + (int64_t)r * a.Hk * RB + ch * 16 : 0;
          copy16(st + place<FORMAT, DP, false>(r, ch), a.cache[0] + src, any);
          copy16(st + S::CODES + place<FORMAT, DP, true>(r, ch), a.cache[1] + src, any);
        }
        row += (int64_t)my * a.Hk;
      } else {
        mask = __ballot_sync(0xFFFFFFFFu, page_ok) & 0xFFFFu;
        const int64_t base = row * RB;
#pragma unroll
        for (int x = 0; x < KEYS * S::CHUNKS / 32; ++x) {
          const int idx = lane + 32 * x, r = idx / S::CHUNKS, ch = idx % S::CHUNKS;
          const int64_t from = __shfl_sync(0xFFFFFFFFu, base, r);
          const bool any = (mask >> r & 1) && ch < chunks;
          const int64_t src = any ? from + ch * 16 : 0;
          copy16(st + place<FORMAT, DP, false>(r, ch), a.cache[0] + src, any);
          copy16(st + S::CODES + place<FORMAT, DP, true>(r, ch), a.cache[1] + src, any);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      const bool ok = mask >> my & 1;
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
      if (lane == 0) live[stage] = mask;
    };
    // the scales that the last `fetch` asked for
    auto put_scales = [&](int stage) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(mine + stage * S::STAGE + 2 * S::CODES + (lane < 16 ? 0 : S::SCALES));
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        // MXFP4 keys: 2^(byte - 127); byte 0 is f32's subnormal 2^-127, byte 255 infinity.  Values: the byte.
        const uint32_t v = S::FP8 || lane >= 16 ? sc[k] : sc[k] ? sc[k] << 23 : 0x00400000u;
        dst[k * KEYS + my] = v;
      }
    };
    int page;
    uint32_t held[STAGES - 1][NB];
    {
      int pages[STAGES];
#pragma unroll
      for (int i = 0; i < STAGES; ++i) pages[i] = page_of(i);
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) {
        fetch(i, i, pages[i]);
#pragma unroll
        for (int k = 0; k < NB; ++k) held[i][k] = sc[k];
      }
      page = pages[STAGES - 1];
    }

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
        float top = 0.0f;
        uint32_t raw[STEPS][2];                              // pairs as they were read
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool in = row < rows && place_of(s) < D;   // (D is a multiple of 16)
            const uint16_t* p = reinterpret_cast<const uint16_t*>(src) + place_of(s) + 2 * e;
            raw[s][e] = in ? (uint32_t)p[0] | (uint32_t)p[1] << 16 : 0;
          }
        auto value = [&](uint32_t w, int i) {
          const uint16_t u = (uint16_t)(i ? w >> 16 : w);
          return widen<T>(*reinterpret_cast<const T*>(&u));
        };
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) top = fmaxf(top, fmaxf(fabsf(value(raw[s][e], 0)), fabsf(value(raw[s][e], 1))));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        int e2 = top > 0.0f && top < INFINITY ? (int)(__float_as_uint(top) >> 23) - 127 : 14;
        e2 = max(e2, -113);
        const float f = pow2(14 - e2);
        qf[r] = a.scale * 1.4426950408889634f * pow2(max(e2 - 14, -126));
        if (e2 - 14 < -126) qf[r] *= pow2(e2 - 14 + 126);
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) q[s][e * R + r] = pack_half(value(raw[s][e], 0) * f, value(raw[s][e], 1) * f);
      }
    }
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
#pragma unroll
      for (int k = 0; k < NB; ++k) sc[k] = held[i][k];
      put_scales(i);
    }

    // o[n][r]: elements d (rows of the MMA) of heads 8 r + 2 c and 8 r + 2 c + 1; m and l are those of heads g + 8 r
    float o[DT][R][4] = {}, m[R], l[R] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -INFINITY;
    int ref[NB];                                             // exponent of the largest scale of values so far
    float up0[NB], up1[NB];                                  // FP8: 2^(6 - (ref - 127)), in two factors that both exist
#pragma unroll
    for (int k = 0; k < NB; ++k) ref[k] = -1000, up0[k] = up1[k] = 1.0f;

    int st = 0, st_new = STAGES - 1;                         // the stage that is read, and the one that is filled
    for (int i = 0; i < steps; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      // the next step to fetch, into the stage that was read last
      const int next = page_of(i + STAGES);
      fetch(i + STAGES - 1, st_new, page);
      page = next;
      const uint8_t* kc = mine + st * S::STAGE;
      const uint8_t* vc = kc + S::CODES;
      const float* ks = reinterpret_cast<const float*>(kc + 2 * S::CODES);
      const uint32_t* vs = reinterpret_cast<const uint32_t*>(kc + 2 * S::CODES + S::SCALES);
      const uint32_t mask = live[st];
      // ---- scores of rows g (and g + 8) with keys 8 t + 2 c and 8 t + 2 c + 1
      float s[2][2 * R];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
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
                const int z = 4 * x + y;
                mma(acc, q[z][0], TWO ? q[z][1] : 0, q[z][R], TWO ? q[z][2 * R - 1] : 0, half2_of_e4m3(ws[y] & 0xFFFFu), half2_of_e4m3(ws[y] >> 16));
              }
            }
          } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + place<FORMAT, DP, false>(8 * t + g, k) + 4 * c);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int z = 2 * k + y;
              mma(acc, q[z][0], TWO ? q[z][1] : 0, q[z][R], TWO ? q[z][2 * R - 1] : 0, half2_of_e2m1(w >> (16 * y) & 255u), half2_of_e2m1(w >> (16 * y + 8) & 255u));
            }
          }
          const float2 f = *reinterpret_cast<const float2*>(ks + k * KEYS + 8 * t + 2 * c);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            s[t][2 * r] = k ? __fmaf_rn(acc[2 * r], f.x, s[t][2 * r]) : __fmul_rn(acc[2 * r], f.x);
            s[t][2 * r + 1] = k ? __fmaf_rn(acc[2 * r + 1], f.y, s[t][2 * r + 1]) : __fmul_rn(acc[2 * r + 1], f.y);
          }
        }
#pragma unroll
        for (int e = 0; e < 2 * R; ++e) s[t][e] = __fmul_rn(s[t][e], qf[e >> 1]);
      }
      if (mask != 0xFFFFu) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2 * R; ++e)
            if (!(mask >> (8 * t + 2 * c + (e & 1)) & 1)) s[t][e] = -INFINITY;
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
          const float fx = __shfl_sync(0xFFFFFFFFu, f, 8 * c), fy = __shfl_sync(0xFFFFFFFFu, f, 8 * c + 4);   // heads 2 c, 2 c + 1
#pragma unroll
          for (int n = 0; n < DT; ++n) o[n][r][0] *= fx, o[n][r][1] *= fy, o[n][r][2] *= fx, o[n][r][3] *= fy;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float sh = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          s[t][2 * r] = exp2_approx(s[t][2 * r] - sh), s[t][2 * r + 1] = exp2_approx(s[t][2 * r + 1] - sh);
          l[r] += s[t][2 * r] + s[t][2 * r + 1];
        }
      }
      // ---- values, block by block: O^T += V^T P^T, weight = p * scale / 2^ref * 2^6 (below 2^8 * 2 * 2^6)
      const int rv[4] = {2 * c, 2 * c + 1, 8 + 2 * c, 9 + 2 * c};                  // this lane's keys
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const uint2 w0 = *reinterpret_cast<const uint2*>(vs + k * KEYS + 2 * c), w1 = *reinterpret_cast<const uint2*>(vs + k * KEYS + 8 + 2 * c);
        const uint32_t sw[4] = {w0.x, w0.y, w1.x, w1.y};
        int most = -1000;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int e = S::FP8 ? (int)(sw[x] >> 23 & 255u) : (int)sw[x];
          if (e != 255) most = max(most, e);                 // (infinities and NaN go through as they are)
        }
        if (__any_sync(0xFFFFFFFFu, most > ref[k])) {
          most = __reduce_max_sync(0xFFFFFFFFu, most);
          const float down = ref[k] < 0 ? 1.0f : pow2(ref[k] - most);
#pragma unroll
          for (int n = k * PER; n < (k + 1) * PER; ++n)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int y = 0; y < 4; ++y) o[n][r][y] *= down;
          ref[k] = most;
          const int up = 133 - most;
          up0[k] = pow2(up / 2), up1[k] = pow2(up - up / 2);
        }
        float f[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          f[x] = S::FP8 ? __uint_as_float(sw[x]) * up0[k] * up1[k] : sw[x] == 255 ? INFINITY : pow2((int)sw[x] - ref[k] + 6);
        uint32_t p[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) p[r][t] = pack_half(s[t][2 * r] * f[2 * t], s[t][2 * r + 1] * f[2 * t + 1]);
        // a tile of 16 elements: rows g and g + 8 of the MMA are two neighbours of this lane's, keys in pairs
        auto step = [&](int n, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
          for (int r = 0; r < R; ++r) mma(o[n][r], a0, a1, a2, a3, p[r][0], p[r][1]);
        };
        if (S::FP8) {
          // block k's codes of lane g: elements 128 k + 2 PER g .. of the four rows
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
          for (int z = 0; z < PER / 2; ++z) {
            const uint32_t x0 = __byte_perm(w[0][z], w[1][z], 0x5140), x1 = __byte_perm(w[0][z], w[1][z], 0x7362);
            const uint32_t y0 = __byte_perm(w[2][z], w[3][z], 0x5140), y1 = __byte_perm(w[2][z], w[3][z], 0x7362);
            step(k * PER + 2 * z, half2_of_e4m3(x0 & 0xFFFFu), half2_of_e4m3(x0 >> 16), half2_of_e4m3(y0 & 0xFFFFu), half2_of_e4m3(y0 >> 16));
            step(k * PER + 2 * z + 1, half2_of_e4m3(x1 & 0xFFFFu), half2_of_e4m3(x1 >> 16), half2_of_e4m3(y1 & 0xFFFFu), half2_of_e4m3(y1 >> 16));
          }
        } else {
          // block k: elements 32 k + 4 g .. + 3 of the four rows
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) w[y] = *reinterpret_cast<const uint16_t*>(vc + place<FORMAT, DP, true>(rv[y], k) + 2 * g);
          // pairs of rows: their nibbles side by side in a byte
          const uint32_t x0 = (w[0] & 0x0F0Fu) | (w[1] & 0x0F0Fu) << 4, x1 = (w[0] >> 4 & 0x0F0Fu) | (w[1] & 0xF0F0u);
          const uint32_t y0 = (w[2] & 0x0F0Fu) | (w[3] & 0x0F0Fu) << 4, y1 = (w[2] >> 4 & 0x0F0Fu) | (w[3] & 0xF0F0u);
          step(2 * k, half2_of_e2m1(x0 & 255u), half2_of_e2m1(x1 & 255u), half2_of_e2m1(y0 & 255u), half2_of_e2m1(y1 & 255u));
          step(2 * k + 1, half2_of_e2m1(x0 >> 8), half2_of_e2m1(x1 >> 8), half2_of_e2m1(y0 >> 8), half2_of_e2m1(y1 >> 8));
        }
      }
      // the scales asked for above; their stage is read next in STAGES - 1 steps
      put_scales(st_new);
      st_new = st;
      if (++st == STAGES) st = 0;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- join the warps
    __syncwarp();
    float* sums = reinterpret_cast<float*>(mine);            // [row][DP + 4], over the warp's own stages
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
      if (c == 0) join_ml[warp * 16 + g + 8 * r] = make_float2(m[r], l[r]);
#pragma unroll
      for (int n = 0; n < DT; ++n) {
        const int up = max(ref[n / PER], 0) - 133;           // 2^(ref - 127 - 6)
        const float f0 = pow2(up / 2), f1 = pow2(up - up / 2);
        const int d = (n / PER) * 16 * PER + g * 2 * PER + 2 * (n % PER);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          *reinterpret_cast<float2*>(sums + (8 * r + 2 * c + y) * (DP + 4) + d) = make_float2(o[n][r][y] * f0 * f1, o[n][r][2 + y] * f0 * f1);
      }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == per - EXTRA;
    // a CTA's first segment may be the rest of a (sequence, head), its last one the beginning of one
    const int64_t slot = 2 * (int64_t)blockIdx.x + (tile0 == 0 ? 1 : 0);
    if (!whole && tile1 == per - EXTRA) ending = {b * a.Hq + h0, rows, deal.owner(start + EXTRA)};
    for (int row = 0; row < rows; ++row) {
      float2 ml[WARPS];
      float t = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) ml[w] = join_ml[w * 16 + row], t = fmaxf(t, ml[w].x);
      const float sh = t == -INFINITY ? 0.0f : t;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) ml[w].x = exp2_approx(ml[w].x - sh), sum = __fmaf_rn(ml[w].y, ml[w].x, sum);
      const int64_t i = b * a.Hq + h0 + row;
      for (int d = threadIdx.x; d < D; d += NT) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v = __fmaf_rn(reinterpret_cast<const float*>(smem + w * S::WARP)[row * (DP + 4) + d], ml[w].x, v);
        if (whole) static_cast<T*>(a.out)[i * D + d] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
        else parts.o[(slot * pl.rows + row) * D + d] = v;
      }
      if (threadIdx.x == 0) {
        if (!whole) parts.ml[slot * pl.rows + row] = make_float2(t, sum);
        else if (a.lse) a.lse[i] = sum > 0.0f ? (t + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) parts.endings[blockIdx.x] = ending;
  // sequences that have nothing
  for (int64_t i = blockIdx.x; i < a.B; i += gridDim.x)
    if (tiles_of(a, i) == 0) {
      for (int64_t x = threadIdx.x; x < (int64_t)a.Hq * D; x += NT) static_cast<T*>(a.out)[i * a.Hq * D + x] = narrow<T>(0.0f);
      if (a.lse)
        for (int h = threadIdx.x; h < a.Hq; h += NT) a.lse[i * a.Hq + h] = -INFINITY;
    }
}

// Joins the sums of each (sequence, head) that lies in several CTAs, in the order of its tiles: CTA (i, y) the rows y, y +
// gridDim.y, .. of the one that the run of the attention's CTA i ends.  Threads [part][element]; then a sum over the parts' shares.
constexpr int JOIN_NT = 512;
template <typename T> __global__ void __launch_bounds__(JOIN_NT) kv_attend_join_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ Plan pl, int lanes) {
  __shared__ float so[JOIN_NT], sl[JOIN_NT], stop[JOIN_NT / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");         // the attention's results are there
  const Parts parts = parts_of(a.workspace, pl.ctas, pl.rows, a.D);
  const Ending e = parts.endings[blockIdx.x];
  const int n = (int)blockIdx.x - e.first + 1;
  const int d = threadIdx.x % lanes, part = threadIdx.x / lanes, step = JOIN_NT / lanes;
  for (int row = blockIdx.y; row < e.rows; row += gridDim.y) {
    auto slot = [&](int i) { return (2 * (int64_t)(e.first + i) + (i == 0 ? 1 : 0)) * pl.rows + row; };
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += JOIN_NT) top = fmaxf(top, parts.ml[slot(i)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if ((threadIdx.x & 31) == 0) stop[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_NT / 32; ++w) top = fmaxf(top, stop[w]);
    const float sh = top == -INFINITY ? 0.0f : top;
    float v = 0.0f, sum = 0.0f;
#pragma unroll 8
    for (int i = part; i < n; i += step) {
      const float2 ml = parts.ml[slot(i)];
      const float x = d < a.D ? parts.o[slot(i) * a.D + d] : 0.0f;
      const float f = exp2_approx(ml.x - sh);
      sum = __fmaf_rn(ml.y, f, sum);
      v = __fmaf_rn(x, f, v);
    }
    so[threadIdx.x] = v;
    if (d == 0) sl[part] = sum;
    __syncthreads();
    if (threadIdx.x < a.D) {
      v = 0.0f, sum = 0.0f;
      for (int x = 0; x < step; ++x) v = __fadd_rn(v, so[x * lanes + threadIdx.x]), sum = __fadd_rn(sum, sl[x]);
      const int64_t i = e.out + row;
      static_cast<T*>(a.out)[i * a.D + threadIdx.x] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
      if (threadIdx.x == 0 && a.lse) a.lse[i] = sum > 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
    }
    __syncthreads();
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
  pl.whole_steps = a.page_size % KEYS == 0;
  kernel<<<pl.ctas, NT, S::SMEM, stream>>>(a, pl);
  // launched early, so that its CTAs wait where the attention's finish
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.ctas, std::min(pl.rows, 4));
  cfg.blockDim = dim3(JOIN_NT);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kv_attend_join_kernel<T>, a, pl, DP);
  if (e != cudaSuccess) return e;
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
  return parts_of(nullptr, p.ctas, p.rows, D).bytes;
}

cudaError_t launch_kv_attend(const KvAttendArgs& a, cudaStream_t stream) {
  const bool half = a.dtype == EMU_DTYPE_F16;
  if (a.format == EMU_KV_FP8) return half ? launch_sized<__half, EMU_KV_FP8>(a, stream) : launch_sized<__nv_bfloat16, EMU_KV_FP8>(a, stream);
  return half ? launch_sized<__half, EMU_KV_MXFP4>(a, stream) : launch_sized<__nv_bfloat16, EMU_KV_MXFP4>(a, stream);
}

}  // namespace emu
