// Attention of one new token for each sequence over the quantised key/value cache.
//
// With s_j = scale q . k_j over the cached rows j < len of the sequence whose page exists, k_j = code * scale as it is
// stored:  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), m = max_j s_j   (no row: o = 0, lse = -inf)
//
// Bound: reading the cache once.  The query heads that share a key head (16 to an item) are the columns of m16n8k16 MMAs, so
// that each code is converted once for all of them.  The codes become fp16, which holds all of their values:
//   scores   S^T = K Q^T, a step of 16 keys to a warp.  q is multiplied by a power of two that puts its row's largest element
//            into [2^14, 2^15) (exact for both 16-bit types but for elements 2^-24 and more below the largest).  FP8: the sum
//            over a block is multiplied by the key's scale of that block in f32.  MXFP4: the scales, powers of two, go into the
//            codes, relative to the largest that the warp has met: exact down to 2^-31 of it
//   values   O^T += V^T P^T, P^T by a transposition of S^T's fp16 pairs.  FP8: the scale goes into the weight, p * scale relative to
//            the largest scale that the warp has met in that block of the head, rounded to fp16 (2^-11 relative; weights of
//            up to 2^-30 of the largest keep all their bits).  MXFP4: the scales go into the codes, the weights are p
// Products of this size (about 90 MACs per byte for 16 heads) are served by mma.sync from registers; tcgen05 would want the
// converted codes in shared memory first.
//
// The work is cut into tiles of 64 keys and dealt out evenly over the CTAs, whatever the lengths: a CTA takes a run of tiles
// of one or several (sequence, head)s.  Where a run is not all of a (sequence, head), its sums go to the workspace, and a
// second kernel joins them in the tiles' order.  Neighbouring heads go to neighbouring CTAs where a slot's row is long.
//
// Measured, both kernels: 64 sequences, 262144 slots of 8 heads of 128 in FP8, 32 query heads: 113 .. 120 us for 555 MB (4.7 TB/s, 72%
// of a copy's rate; the first kernel 105 us at 5.3 TB/s: memory waits, issue slots 48% busy).  4 sequences, 400001 slots on one
// head, 16 query heads: 43 us (106 MB): 21 steps to a warp, so that starting and joining count.  4 bits, 33 sequences, 100003
// slots of 4 heads of 64: 33 us (27 MB), 10 steps to a warp, each of which waits for the scale bytes that it asked for.
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
// A word's codes -> fp16 pairs, the low byte's first.
__device__ __forceinline__ void halves_of_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void halves_of_e2m1(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Copies into shared memory that are waited for later.
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, bool any) {
  const int n = any ? 16 : 0;                                // 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const uint8_t* src, bool any) {
  const int n = any ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int N> __device__ __forceinline__ void read_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}
// two fp16 factors of a power of two each
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// An 8 x 8 matrix of fp16 pairs, row lane / 4 and columns 2 (lane % 4) and the next, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// 2^e as fp16 bits: subnormal below -14, 0 below -24, infinity above 15
__device__ __forceinline__ uint32_t half_pow2(int e) { return e > 15 ? 0x7C00u : e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u; }

// Who holds which of a row's DP elements.  Keys (k = 16 to an MMA, 4 lanes to a key): lane c's are KX places of KW words.
// Values (8 lanes to a row): lane g's are VX places of VW words.  A stage holds 16 rows of keys, 16 of values and their scales; its
// rows are 16 bytes further apart than they are long, so that the lanes that read together meet different banks.
template <int FORMAT, int DP> struct Shape {
  static constexpr bool FP8 = FORMAT == EMU_KV_FP8;
  static constexpr int ROW = FP8 ? DP : DP / 2;              // bytes of a row of codes
  static constexpr int KW = ROW >= 64 ? 4 : 2, KX = ROW / (16 * KW);
  static constexpr int VW = ROW >= 128 ? 4 : ROW / 32, VX = ROW / (32 * VW);
  static constexpr int BLOCKS = FP8 ? (DP + 127) / 128 : 1;  // separately scaled sums of the scores, weights of the values
  static constexpr int CODES = FP8 ? 4 : 8;                  // codes in a word
  static constexpr int PITCH = ROW + 16, SCALE = FP8 ? 4 * BLOCKS : DP == 256 ? 8 : 4;   // bytes from row to row, of a row's scales
  static constexpr int STAGE = 2 * KEYS * (PITCH + SCALE);
  static constexpr int STAGES = FP8 && DP >= 128 ? 3 : 4;    // what ctas_per_sm leaves room for
  static constexpr int CHUNKS = ROW / 16, COPIES = KEYS * CHUNKS / 32;   // 16-byte copies of a row, of keys (values) to a lane
  static_assert(CHUNKS <= 32 && COPIES >= 1, "a lane copies at least one chunk of a step");
  // bytes of lane c's place x
  static __host__ __device__ constexpr int key_place(int c, int x) { return (KX == 1 ? c : 8 * (x / 2) + 2 * c + x % 2) * 4 * KW; }
  static __host__ __device__ constexpr int value_place(int g, int x) { return (g + 8 * x) * 4 * VW; }
};
constexpr int JOIN = 4;                                      // floats between the rows of the join's buffer

// The tiles of a sequence (of each of its heads).
__device__ __forceinline__ int64_t tiles_of(const KvAttendArgs& a, int64_t b) {
  const int64_t len = min((int64_t)a.lens[b], a.table_cols * a.page_size);
  return len > 0 && a.num_pages > 0 ? (len + TILE - 1) / TILE : 0;
}
// What a (sequence, head) counts for when the work is dealt out: its tiles and EXTRA places before them, for what
// starting and joining it costs.  Calls with EXTRA 0, 2, 4, 8, us: 33 sequences, 100003 slots in 4 bits 50, 42, 40, 40; 64 sequences,
// 16384 slots of 8 heads 38, 34, 32, 32; 262144 in 4 bits 138, 134, 130, 132; 400001 slots on one head 52, 52, 50, 48.
constexpr int EXTRA = 4;
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
  Ending* endings;             // [sequence][head]
  float2* ml;                  // [slot][rows]: maximum (of log2 scores), sum
  float* o;                    // [slot][rows][D]
  size_t bytes;
};
__host__ __device__ inline Parts parts_of(void* workspace, int64_t items, int64_t ctas, int rows, int D) {
  uint8_t* base = static_cast<uint8_t*>(workspace);
  const size_t ml = (size_t)(items * 8 + 255) / 256 * 256, o = ml + (2 * ctas * rows * sizeof(float2) + 255) / 256 * 256;
  return {reinterpret_cast<Ending*>(base), reinterpret_cast<float2*>(base + ml), reinterpret_cast<float*>(base + o), o + 2 * ctas * rows * D * sizeof(float)};
}
struct Plan {
  int ctas, groups, rows;      // CTAs, items of up to 16 query heads to a key head, rows of an item
  int side_bits, sets;         // sets of 2^side_bits CTAs that take the same keys of neighbouring heads
  bool wide_q;                 // four elements of q may be read at once
  bool wide_scales;            // MXFP4: a row's scale bytes may be read at once
  bool whole_steps;            // a step's 16 keys lie in one page
  uint32_t page_size;          // up to 2^31 (more than any length)
  uint32_t tile_columns, tile_off;                           // pages in a tile of keys, and what is left
};
// What the CTA that ends a (sequence, head) leaves for the join: the first and the last CTA of it (the same: nothing to join).
struct Ending {
  int first, last;
};

// As many as registers (and shared memory) allow; 16 heads of 128 in FP8 two, without spills (262144 rows of 8 heads: 164 us
// against 170 with three; MXFP4 three, 51 against 53).
constexpr int ctas_per_sm(int format, int DP, bool two) {
  return DP == 256 || (DP == 128 && two && format == EMU_KV_FP8) ? 2 : DP == 128 && (two || format == EMU_KV_FP8) ? 3 : 4;
}
constexpr int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

template <typename T, int FORMAT, int DP, bool TWO>
__global__ void __launch_bounds__(NT, ctas_per_sm(FORMAT, DP, TWO)) kv_attend_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ Plan pl) {
  using S = Shape<FORMAT, DP>;
  // d-tiles of 16 (DT), those of a block of values (PER), groups of 8 heads (R)
  constexpr int NB = S::BLOCKS, STEPS = DP / 16, DT = DP / 16, PER = DT / NB, R = TWO ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t tmp[WARPS], found[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  constexpr int STAGES = S::STAGES, RING = STAGES * S::STAGE;
  static_assert(RING >= 8 * (DP + JOIN) * 4, "the ring holds the warp's sums afterwards");
  uint8_t* ring = smem + warp * RING;
  const uint32_t ring_u = (uint32_t)__cvta_generic_to_shared(ring);
  float* sums = reinterpret_cast<float*>(ring);              // [8 rows][DP + 4]
  float2* join_ml = reinterpret_cast<float2*>(smem + WARPS * RING);                // [warp][8]
  const int D = a.D, HV = a.Hk * pl.groups, group = a.Hq / a.Hk;
  const int set = blockIdx.x >> pl.side_bits, side = blockIdx.x & ((1 << pl.side_bits) - 1), HS = HV >> pl.side_bits;            // (sequence, set of heads)s of a sequence
  const Parts parts = parts_of(a.workspace, a.B * HV, pl.ctas, pl.rows, D);

  asm volatile("griddepcontrol.launch_dependents;");        // the join's CTAs may come when there is room
  // this CTA's run of places
  int64_t total = 0, b = 0, first = 0;                       // sequence b's first place
  {
    int64_t base = 0;
    if (a.B <= NT) {
      const int64_t n = threadIdx.x < a.B ? places_of(a, threadIdx.x) * HS : 0;
      const int64_t before = block_scan(n, tmp, total);
      const int64_t lo = Deal(total, pl.sets).begin(set);
      if (before <= lo && lo < before + n) found[0] = threadIdx.x, found[1] = before;
    } else {
      int64_t sum = 0;
      for (int64_t i = threadIdx.x; i < a.B; i += NT) sum += places_of(a, i);
      block_scan(sum * HS, tmp, total);
      const int64_t lo = Deal(total, pl.sets).begin(set);
      for (int64_t b0 = 0; b0 < a.B && base <= lo; b0 += NT) {
        const int64_t n = b0 + threadIdx.x < a.B ? places_of(a, b0 + threadIdx.x) * HS : 0;
        int64_t all;
        const int64_t before = base + block_scan(n, tmp, all);
        if (before <= lo && lo < before + n) found[0] = b0 + threadIdx.x, found[1] = before;
        base += all;
      }
    }
    __syncthreads();
  }
  const Deal deal(total, pl.sets);
  int64_t at = deal.begin(set);                              // `at` in the list of all places
  const int64_t hi = set < pl.sets ? deal.begin(set + 1) : at;
  if (at < hi) b = found[0], first = found[1];

  while (at < hi) {
    const int64_t per = places_of(a, b);
    if (per == 0 || at >= first + per * HS) {
      first += per * HS;
      ++b;
      continue;
    }
    const int hs = at - first <= 0xFFFFFFFF ? (int)((uint32_t)(at - first) / (uint32_t)per) : (int)((at - first) / per);
    const int64_t start = first + hs * per, stop = start + per;                    // this (sequence, set of heads)'s places
    const int64_t tile0 = max((int64_t)0, at - start - EXTRA), tile1 = min(hi, stop) - start - EXTRA;
    at = min(hi, stop);
    if (tile1 <= tile0) continue;
    const int kh = (hs / pl.groups << pl.side_bits) + side, part = hs % pl.groups, hv = kh * pl.groups + part;
    const int h0 = kh * group + part * 16, rows = min(16, group - part * 16);
    const int len = (int)min((int64_t)a.lens[b], a.table_cols * a.page_size);
    const int32_t* table = a.table + b * a.table_stride;

    // ---- this lane's elements of q's rows g and g + 8 as they are, asked for before the cache's
    uint32_t raw[R][STEPS][2];
    {
      auto place_of = [&](int z) {                           // the first of a step's two pairs
        constexpr int PER_PLACE = S::KW * S::CODES / 4;      // steps of one place
        return S::key_place(c, z / PER_PLACE) / 4 * S::CODES + z % PER_PLACE * 4;
      };
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = g + 8 * r;
        const T* src = static_cast<const T*>(a.q) + b * a.q_stride[0] + (int64_t)(h0 + row) * a.q_stride[1];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          raw[r][s][0] = raw[r][s][1] = 0;
          if (row < rows && place_of(s) < D) {               // (D is a multiple of 16)
            if (pl.wide_q) {
              const uint2 w = __ldg(reinterpret_cast<const uint2*>(src + place_of(s)));
              raw[r][s][0] = w.x, raw[r][s][1] = w.y;
            } else {
              const uint16_t* p = reinterpret_cast<const uint16_t*>(src) + place_of(s);
              raw[r][s][0] = (uint32_t)p[0] | (uint32_t)p[1] << 16;
              raw[r][s][1] = (uint32_t)p[2] | (uint32_t)p[3] << 16;
            }
          }
        }
      }
    }

    // ---- steps of 16 keys; the warps take them in turn
    const int key0 = (int)(tile0 * TILE) + warp * KEYS, end = (int)min((int64_t)len, tile1 * TILE);
    const int steps = (int)(tile1 - tile0);
    const int RB = S::FP8 ? D : D / 2, nb = S::FP8 ? (D + 127) / 128 : D / 32;
    constexpr int SZ = S::FP8 ? 4 : 1;                       // bytes of a scale
    // from slot to slot, in bytes (16 slots stay below 2^32)
    const uint32_t head_row = (uint32_t)(a.Hk * RB), head_scale = (uint32_t)(a.Hk * nb * SZ);
    // The step whose page is looked up next: its key (of a step in several pages its key lane % 16) counted back from the end,
    // and its place in the table and in the page, which move on by additions alone (divisions were a tenth of the
    // kernel's instructions).
    const int key_first = key0 + (pl.whole_steps ? 0 : lane & 15);
    struct Look {
      int left, column, page;
      uint32_t off;
    } look{end - key_first, (int)((uint32_t)key_first / pl.page_size), 0, (uint32_t)key_first % pl.page_size};
    auto look_up = [&]() {
      Look r = look;
      r.page = look.left > 0 ? __ldg(table + look.column) : -1;
      look.left -= TILE, look.column += pl.tile_columns, look.off += pl.tile_off;
      if (look.off >= pl.page_size) look.off -= pl.page_size, ++look.column;
      return r;
    };
    // This lane's rows: keys g and 8 + g for the scores' operand; keys 2 c, 2 c + 1, 8 + 2 c and 9 + 2 c for the values' and for what
    // is known of a score.
    struct Step {
      uint32_t live;                                         // a bit for each key that is seen
      int64_t slot;                                          // of the first key (of key lane % 16)
    };
    auto step_of = [&](const Look& k) {
      Step t;
      const bool ok = k.page >= 0 && k.page < a.num_pages;
      t.slot = ok ? (int64_t)k.page * a.page_size + k.off : 0;
      t.live = pl.whole_steps ? (ok ? (1u << min(KEYS, k.left)) - 1 : 0) : __ballot_sync(0xFFFFFFFFu, ok) & 0xFFFFu;
      return t;
    };
    // A step's codes and scales on their way into stage `st`.  Where all of its keys are seen and lie behind one another and D
    // fills the places, without a test for each copy: addresses and tests were half of the kernel's instructions.
    const bool full = pl.whole_steps && D == DP;
    constexpr int ROWS = 32 / S::CHUNKS;                     // rows that the warp copies at once
    const int my_row = lane / S::CHUNKS, my_chunk = lane % S::CHUNKS, my = lane & 15;
    const uint32_t my_src = (uint32_t)my_row * head_row + my_chunk * 16, my_dst = my_row * S::PITCH + my_chunk * 16;
    uint32_t held[2];                                        // MXFP4: scale bytes of key (value) lane % 16 until they are put down
    auto fetch = [&](const Step& t, int st) {
      const uint32_t dst = ring_u + st * S::STAGE, dst_s = dst + 2 * KEYS * S::PITCH + (lane >> 4) * KEYS * S::SCALE + my * S::SCALE;
      const uint8_t* scales = static_cast<const uint8_t*>(lane < 16 ? a.scales[0] : a.scales[1]) + kh * nb * SZ;
      const bool seen = t.live >> my & 1;
      if (full && t.live == 0xFFFFu) {
        const int64_t base = t.slot * head_row + kh * RB;
        const uint8_t* k = a.cache[0] + base;
        const uint8_t* v = a.cache[1] + base;
#pragma unroll
        for (int x = 0; x < S::COPIES; ++x) {
          const uint32_t from = my_src + x * ROWS * head_row;
          copy16(dst + my_dst + x * ROWS * S::PITCH, k + from);
          copy16(dst + KEYS * S::PITCH + my_dst + x * ROWS * S::PITCH, v + from);
        }
        scales += (t.slot + my) * head_scale;
      } else {
#pragma unroll
        for (int x = 0; x < S::COPIES; ++x) {
          const int r = my_row + x * ROWS;
          const int64_t slot = pl.whole_steps ? t.slot + r : __shfl_sync(0xFFFFFFFFu, t.slot, r);
          const bool any = (t.live >> r & 1) && my_chunk * 16 < RB;
          const int64_t from = any ? slot * head_row + kh * RB + my_chunk * 16 : 0;
          copy16(dst + my_dst + x * ROWS * S::PITCH, a.cache[0] + from, any);
          copy16(dst + KEYS * S::PITCH + my_dst + x * ROWS * S::PITCH, a.cache[1] + from, any);
        }
        scales += seen ? (pl.whole_steps ? t.slot + my : t.slot) * head_scale : 0;
      }
      if (S::FP8) {
#pragma unroll
        for (int k = 0; k < NB; ++k) copy4(dst_s + 4 * k, k < nb ? scales + 4 * k : scales, seen && k < nb);
      } else {
        held[0] = held[1] = 0;
        if (seen && pl.wide_scales) {
          if (DP == 64) held[0] = __ldg(reinterpret_cast<const uint16_t*>(scales));
          else held[0] = __ldg(reinterpret_cast<const uint32_t*>(scales));
          if (DP == 256) held[1] = __ldg(reinterpret_cast<const uint32_t*>(scales) + 1);
        } else if (seen) {
#pragma unroll
          for (int k = 0; k < DP / 32; ++k)
            if (k < nb) held[k / 4] |= (uint32_t)__ldg(scales + k) << (8 * (k & 3));
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto put_scales = [&](int st) {
      if (S::FP8) return;
      uint32_t* dst = reinterpret_cast<uint32_t*>(ring + st * S::STAGE + 2 * KEYS * S::PITCH + (lane >> 4) * KEYS * S::SCALE + my * S::SCALE);
#pragma unroll
      for (int k = 0; k < S::SCALE / 4; ++k) dst[k] = held[k];
    };
    uint32_t lives[STAGES];                                  // of the steps under way, the next one first
    Look next;
    {
      Look pages[STAGES];
#pragma unroll
      for (int i = 0; i < STAGES; ++i) pages[i] = look_up();
      uint32_t early[STAGES][2];
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) {
        const Step t = step_of(pages[i]);
        lives[i] = t.live;
        fetch(t, i);
        early[i][0] = held[0], early[i][1] = held[1];
      }
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) {
        held[0] = early[i][0], held[1] = early[i][1];
        put_scales(i);
      }
      next = pages[STAGES - 1];
    }

    // ---- q as the MMAs' A operands: fp16, multiplied by a power of two
    uint32_t q[STEPS][2 * R];
    float qf[R];                                             // what a score of the row is multiplied by
#pragma unroll
    for (int r = 0; r < R; ++r) {
      auto value = [&](uint32_t w, int i) {
        const uint16_t u = (uint16_t)(i ? w >> 16 : w);
        return widen<T>(*reinterpret_cast<const T*>(&u));
      };
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) top = fmaxf(top, fmaxf(fabsf(value(raw[r][s][e], 0)), fabsf(value(raw[r][s][e], 1))));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      int e2 = top > 0.0f && top < INFINITY ? (int)(__float_as_uint(top) >> 23) - 127 : 14;
      e2 = max(e2, -113);
      const float f = pow2(14 - e2);
      qf[r] = a.scale * 1.4426950408889634f * pow2(max(e2 - 14, -126));
      if (e2 - 14 < -126) qf[r] *= pow2(e2 - 14 + 126);
      qf[r] = fmaxf(qf[r], 1.4e-45f);                        // -inf times it stays -inf
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) q[s][e * R + r] = pack_half(value(raw[r][s][e], 0) * f, value(raw[r][s][e], 1) * f);
    }

    // o[n][r]: elements d (rows of the MMA) of heads 8 r + 2 c and 8 r + 2 c + 1, as are m, l and what a score is multiplied by (up_s: MXFP4 with
    // 2^(kref - 127 - 8))
    float o[DT][R][4] = {}, m[R][2], l[R][2] = {}, up_q[R][2], up_s[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int y = 0; y < 2; ++y) m[r][y] = -INFINITY, up_s[r][y] = up_q[r][y] = __shfl_sync(0xFFFFFFFFu, qf[r], 8 * c + 4 * y);
    // FP8: the exponent of the largest scale of values so far, for each block, the same in the whole warp; MXFP4: that of
    // this lane's block.  up: FP8, 2^(6 - (ref - 127)), in two factors that both exist; limit: the smallest scale past ref.
    int ref[NB], kref = -1000;                               // kref: MXFP4, the largest exponent of the keys' scales so far
    float up0[NB], up1[NB], limit[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) ref[k] = -1000, up0[k] = up1[k] = 1.0f, limit[k] = 0.0f;

    int st = 0, st_new = STAGES - 1;                         // the stage that is read, and the one that is filled
    for (int i = 0; i < steps; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      // the step to fetch next, into the stage that was read last
      const uint32_t live = lives[0];
#pragma unroll
      for (int x = 0; x + 2 < STAGES; ++x) lives[x] = lives[x + 1];
      {
        const Step t = step_of(next);
        next = look_up();
        lives[STAGES - 2] = t.live;
        fetch(t, st_new);
      }
      const uint8_t* keys = ring + st * S::STAGE;
      const uint8_t* values = keys + KEYS * S::PITCH;
      const uint8_t* key_scales = values + KEYS * S::PITCH;
      const uint8_t* value_scales = key_scales + KEYS * S::SCALE;
      uint32_t ksc[2][S::FP8 ? NB : S::KX], vsc[S::FP8 ? 2 : 4][NB];
#pragma unroll
      for (int y = 0; y < 2; ++y) {                          // keys g and 8 + g
        if (S::FP8) {
          uint32_t w[NB];
          read_words(key_scales + (8 * y + g) * S::SCALE, w);
#pragma unroll
          for (int k = 0; k < NB; ++k) ksc[y][k] = w[k];
          read_words(value_scales + (8 * y + g) * S::SCALE, w);
#pragma unroll
          for (int k = 0; k < NB; ++k) vsc[y][k] = w[k];
        } else {
#pragma unroll
          for (int x = 0; x < S::KX; ++x) ksc[y][x] = key_scales[(8 * y + g) * S::SCALE + S::key_place(c, x) / 16];
        }
      }
      if (!S::FP8) {
#pragma unroll
        for (int y = 0; y < 4; ++y) vsc[y][0] = value_scales[(y / 2 * 8 + 2 * c + y % 2) * S::SCALE + S::value_place(g, 0) / 16];
      }
      // ---- scores, S^T = K Q^T: keys g and 8 + g with heads 8 r + 2 c and 8 r + 2 c + 1
      float s[R][4];
      if (!S::FP8) {
        int most = -1000;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int x = 0; x < S::KX; ++x)
            if (ksc[y][x] != 255) most = max(most, (int)ksc[y][x]);
        // codes are up to 6: 2^(8 + 4) times that is still an fp16
        if (__any_sync(0xFFFFFFFFu, most > kref + 4)) {
          kref = __reduce_max_sync(0xFFFFFFFFu, most);
          const int up = max(kref, 0) - 135;
          // (held inside f32: past it scores are infinite, far below it all the same)
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int y = 0; y < 2; ++y) up_s[r][y] = fmaxf(fminf(up_q[r][y] * pow2(up / 2) * pow2(up - up / 2), 3.4028235e38f), 1.4e-45f);
        }
      }
      uint32_t kw[2][S::KX][S::KW];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < S::KX; ++x) read_words(keys + (8 * t + g) * S::PITCH + S::key_place(c, x), kw[t][x]);
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        constexpr int CHAINS = 2 / R;                        // MMAs one after the other wait for one another's sums
        float acc[R][CHAINS][4] = {};
        if (S::FP8) {
#pragma unroll
          for (int x = 2 * k; x < 2 * k + 2 && x < S::KX; ++x)
#pragma unroll
            for (int y = 0; y < S::KW; ++y) {
              const int z = S::KW * x + y;
              uint32_t h[4];
              halves_of_e4m3(kw[0][x][y], h[0], h[2]);
              halves_of_e4m3(kw[1][x][y], h[1], h[3]);
#pragma unroll
              for (int r = 0; r < R; ++r) mma(acc[r][z % CHAINS], h[0], h[1], h[2], h[3], q[z][r], q[z][R + r]);
            }
        } else {
#pragma unroll
          for (int x = 0; x < S::KX; ++x) {
            uint32_t f[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) f[t] = half_pow2(ksc[t][x] == 255 ? 16 : (int)ksc[t][x] - kref + 8) * 0x10001u;
#pragma unroll
            for (int y = 0; y < S::KW; ++y) {
              const int z = 2 * (S::KW * x + y);
              uint32_t h0[4], h1[4];
              halves_of_e2m1(kw[0][x][y], h0);
              halves_of_e2m1(kw[1][x][y], h1);
#pragma unroll
              for (int e = 0; e < 4; ++e) h0[e] = mul_half2(h0[e], f[0]), h1[e] = mul_half2(h1[e], f[1]);
#pragma unroll
              for (int r = 0; r < R; ++r) {
                mma(acc[r][0], h0[0], h1[0], h0[1], h1[1], q[z][r], q[z][R + r]);
                mma(acc[r][CHAINS - 1], h0[2], h1[2], h0[3], h1[3], q[z + 1][r], q[z + 1][R + r]);
              }
            }
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = CHAINS == 2 ? __fadd_rn(acc[r][0][e], acc[r][CHAINS - 1][e]) : acc[r][0][e];
            if (S::FP8) {
              const float f = __uint_as_float(ksc[e >> 1][k]);
              s[r][e] = k ? __fmaf_rn(v, f, s[r][e]) : __fmul_rn(v, f);
            } else {
              s[r][e] = v;
            }
          }
      }
      if (live != 0xFFFFu) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (!(live >> (8 * t + g) & 1)) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][2 * t] = s[r][2 * t + 1] = -INFINITY;
          }
      }
      // ---- the running maximum: held up to a factor of 2^8
      bool grow = false;
      float top[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          top[r][y] = __fmul_rn(fmaxf(s[r][y], s[r][2 + y]), up_s[r][y]);
          grow = grow || top[r][y] - m[r][y] > 8.0f;
        }
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float t = top[r][y];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, x));
            t = fmaxf(m[r][y], t);
            const float f = t == -INFINITY ? 1.0f : exp2_approx(m[r][y] - t);
            m[r][y] = t;
            l[r][y] *= f;
#pragma unroll
            for (int n = 0; n < DT; ++n) o[n][r][y] *= f, o[n][r][2 + y] *= f;
          }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float sh = m[r][y] == -INFINITY ? 0.0f : -m[r][y];
#pragma unroll
          for (int e = y; e < 4; e += 2) s[r][e] = exp2_approx(__fmaf_rn(s[r][e], up_s[r][y], sh));
          l[r][y] += s[r][y] + s[r][2 + y];
        }
      // ---- values: O^T += V^T P^T
      uint32_t vw[4][S::VX][S::VW];
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < S::VX; ++x) read_words(values + (y / 2 * 8 + 2 * c + y % 2) * S::PITCH + S::value_place(g, x), vw[y][x]);
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        int most = -1000;
        bool past;
        if (S::FP8) {
          past = fmaxf(fabsf(__uint_as_float(vsc[0][k])), fabsf(__uint_as_float(vsc[1][k]))) >= limit[k];
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (vsc[x][0] != 255) most = max(most, (int)vsc[x][0]);
          past = most > ref[k];
        }
        if (__any_sync(0xFFFFFFFFu, past)) {
          if (S::FP8) {                                      // (infinities and NaN go through as they are)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int e = (int)(vsc[x][k] >> 23 & 255u);
              if (e != 255) most = max(most, e);
            }
            most = max(__reduce_max_sync(0xFFFFFFFFu, most), ref[k]);
          } else {
            // the four lanes that share the rows g of the MMAs have the same block and the same ref
            most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
            most = max(max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2)), ref[k]);
          }
          const float down = ref[k] < 0 ? 1.0f : pow2(ref[k] - most);
#pragma unroll
          for (int n = k * PER; n < (k + 1) * PER; ++n)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int y = 0; y < 4; ++y) o[n][r][y] *= down;
          ref[k] = most;
          const int up = 133 - max(most, 0);
          up0[k] = pow2(up / 2), up1[k] = pow2(up - up / 2);
          limit[k] = __uint_as_float((uint32_t)(max(most, 0) + 1) << 23);
        }
        // weights as fp16.  FP8: p * scale / 2^ref * 2^6 (below 2^8 * 2 * 2^6).  MXFP4: p * 2^7, and the codes are multiplied
        // by scale / 2^ref * 2^8.
        uint32_t p[R][2], f01 = 0, f23 = 0;
        float f[2] = {128.0f, 128.0f};
        if (S::FP8) {
#pragma unroll
          for (int t = 0; t < 2; ++t) f[t] = __uint_as_float(vsc[t][k]) * up0[k] * up1[k];
        } else {
          uint32_t h[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) h[x] = half_pow2(vsc[x][0] == 255 ? 16 : (int)vsc[x][0] - ref[0] + 8);
          f01 = h[0] | h[1] << 16, f23 = h[2] | h[3] << 16;
        }
        // from a key's heads to a head's keys
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) p[r][t] = transposed(pack_half(s[r][2 * t] * f[t], s[r][2 * t + 1] * f[t]));
        // a tile of 16 elements: rows g and g + 8 of the MMA are two neighbours of this lane's, keys in pairs
        auto step = [&](int n, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
          for (int r = 0; r < R; ++r) mma(o[n][r], a0, a1, a2, a3, p[r][0], p[r][1]);
        };
        if (S::FP8) {
          const int x = DP == 256 ? k : 0;
#pragma unroll
          for (int z = 0; z < S::VW; ++z) {
            const uint32_t x0 = __byte_perm(vw[0][x][z], vw[1][x][z], 0x5140), x1 = __byte_perm(vw[0][x][z], vw[1][x][z], 0x7362);
            const uint32_t y0 = __byte_perm(vw[2][x][z], vw[3][x][z], 0x5140), y1 = __byte_perm(vw[2][x][z], vw[3][x][z], 0x7362);
            uint32_t h[4];
            halves_of_e4m3(x0, h[0], h[1]), halves_of_e4m3(y0, h[2], h[3]);
            step(k * PER + 2 * z, h[0], h[1], h[2], h[3]);
            halves_of_e4m3(x1, h[0], h[1]), halves_of_e4m3(y1, h[2], h[3]);
            step(k * PER + 2 * z + 1, h[0], h[1], h[2], h[3]);
          }
        } else {
#pragma unroll
          for (int z = 0; z < S::VW; ++z) {
            // pairs of rows: their nibbles side by side in a byte, elements 0, 2, 4, 6 of the word and 1, 3, 5, 7
            const uint32_t w0 = vw[0][0][z], w1 = vw[1][0][z], w2 = vw[2][0][z], w3 = vw[3][0][z];
            const uint32_t x0 = (w0 & 0x0F0F0F0Fu) | (w1 << 4 & 0xF0F0F0F0u), x1 = (w0 >> 4 & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u);
            const uint32_t y0 = (w2 & 0x0F0F0F0Fu) | (w3 << 4 & 0xF0F0F0F0u), y1 = (w2 >> 4 & 0x0F0F0F0Fu) | (w3 & 0xF0F0F0F0u);
            uint32_t hx0[4], hx1[4], hy0[4], hy1[4];
            halves_of_e2m1(x0, hx0), halves_of_e2m1(x1, hx1), halves_of_e2m1(y0, hy0), halves_of_e2m1(y1, hy1);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              step(4 * z + e, mul_half2(hx0[e], f01), mul_half2(hx1[e], f01), mul_half2(hy0[e], f23), mul_half2(hy1[e], f23));
          }
        }
      }
      put_scales(st_new);                                    // asked for above; their stage is read in STAGES - 1 steps
      st_new = st;
      if (++st == STAGES) st = 0;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();

    // ---- join the warps, 8 heads at a time
    const bool whole = tile0 == 0 && tile1 == per - EXTRA;
    // a CTA's first segment may be the rest of a (sequence, head), its last one the beginning of one
    const int64_t slot = 2 * (int64_t)blockIdx.x + (tile0 == 0 ? 1 : 0);
    if (tile1 == per - EXTRA && threadIdx.x == 0) parts.endings[b * HV + hv] = {whole ? (int)blockIdx.x : (deal.owner(start + EXTRA) << pl.side_bits) + side, (int)blockIdx.x};
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[r][y] += __shfl_xor_sync(0xFFFFFFFFu, l[r][y], x);
        if (g == 0) join_ml[warp * 8 + 2 * c + y] = make_float2(m[r][y], l[r][y]);
      }
#pragma unroll
      for (int n = 0; n < DT; ++n) {
        const int up = max(ref[n / PER], 0) - (S::FP8 ? 133 : 142);                // 2^(ref - 127 - 6), MXFP4: - 7 - 8
        const float f0 = pow2(up / 2), f1 = pow2(up - up / 2);
        const int d = (n / PER) * 16 * PER + g * 2 * PER + 2 * (n % PER);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          *reinterpret_cast<float2*>(sums + (2 * c + y) * (DP + JOIN) + d) = make_float2(o[n][r][y] * f0 * f1, o[n][r][2 + y] * f0 * f1);
      }
      __syncthreads();
      for (int row = 0; row < min(8, rows - 8 * r); ++row) {
        float2 ml[WARPS];
        float t = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) ml[w] = join_ml[w * 8 + row], t = fmaxf(t, ml[w].x);
        const float sh = t == -INFINITY ? 0.0f : t;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) ml[w].x = exp2_approx(ml[w].x - sh), sum = __fmaf_rn(ml[w].y, ml[w].x, sum);
        const int64_t i = b * a.Hq + h0 + 8 * r + row, at_slot = slot * pl.rows + 8 * r + row;
        for (int d = threadIdx.x; d < D; d += NT) {
          float v = 0.0f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) v = __fmaf_rn(reinterpret_cast<const float*>(smem + w * RING)[row * (DP + JOIN) + d], ml[w].x, v);
          if (whole) static_cast<T*>(a.out)[i * D + d] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
          else parts.o[at_slot * D + d] = v;
        }
        if (threadIdx.x == 0) {
          if (!whole) parts.ml[at_slot] = make_float2(t, sum);
          else if (a.lse) a.lse[i] = sum > 0.0f ? (t + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
        }
      }
      __syncthreads();
    }
  }
  // sequences that have nothing
  for (int64_t i = blockIdx.x; i < a.B; i += gridDim.x)
    if (tiles_of(a, i) == 0) {
      for (int x = threadIdx.x; x < HV; x += NT) parts.endings[i * HV + x] = {0, 0};
      for (int64_t x = threadIdx.x; x < (int64_t)a.Hq * D; x += NT) static_cast<T*>(a.out)[i * a.Hq * D + x] = narrow<T>(0.0f);
      if (a.lse)
        for (int h = threadIdx.x; h < a.Hq; h += NT) a.lse[i * a.Hq + h] = -INFINITY;
    }
}

// Joins the sums of each (sequence, head) that lies in several CTAs, in the order of its tiles.  A CTA to a row of an item (where
// there are many, to every gridDim.x-th item): the parts' factors first, then threads [part][element], then a sum over
// the parts' shares.
constexpr int JOIN_NT = 512, JOIN_PARTS = 1024, FEW = 8;
template <typename T, bool MANY> __global__ void __launch_bounds__(JOIN_NT) kv_attend_join_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ Plan pl, int lanes) {
  __shared__ float so[JOIN_NT], factor[JOIN_PARTS], part_sum[JOIN_NT / 32], part_top[JOIN_NT / 32];
  const int HV = a.Hk * pl.groups, group = a.Hq / a.Hk, row = blockIdx.y, warp = threadIdx.x >> 5;
  const Parts parts = parts_of(a.workspace, a.B * HV, pl.ctas, pl.rows, a.D);
  asm volatile("griddepcontrol.wait;" ::: "memory");         // the attention's results are there
  for (int64_t item = blockIdx.x; item < a.B * HV; item += gridDim.x) {
    const Ending e = parts.endings[item];
    const int n = ((e.last - e.first) >> pl.side_bits) + 1;
    const int64_t b = item / HV;
    const int hv = (int)(item - b * HV);
    if (n < 2) continue;
    const int d = threadIdx.x % lanes, shares = JOIN_NT / lanes;
    if (n <= FEW) {                                          // as many rows at once as there are threads for
      const int r = row + threadIdx.x / lanes, hq = hv % pl.groups * 16 + r;
      if (row % shares || r >= pl.rows || hq >= group || d >= a.D) continue;
      auto slot = [&](int i) { return (2 * (int64_t)(e.first + (i << pl.side_bits)) + (i == 0 ? 1 : 0)) * pl.rows + r; };
      float top = -INFINITY, sum = 0.0f, v = 0.0f;
      for (int i = 0; i < n; ++i) top = fmaxf(top, parts.ml[slot(i)].x);
      const float sh = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float2 ml = parts.ml[slot(i)];
        const float f = exp2_approx(ml.x - sh);
        sum = __fmaf_rn(ml.y, f, sum);
        v = __fmaf_rn(parts.o[slot(i) * a.D + d], f, v);
      }
      const int64_t i = b * a.Hq + hv / pl.groups * group + hq;
      static_cast<T*>(a.out)[i * a.D + d] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
      if (d == 0 && a.lse) a.lse[i] = sum > 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
      continue;
    }
    const int hq = hv % pl.groups * 16 + row;
    if (hq >= group) continue;
    // a CTA's first (sequence, head) is in its even slot; this one's first part is the last of its CTA
    const int64_t slot0 = (2 * (int64_t)e.first) * pl.rows + row, step = 2 * pl.rows << pl.side_bits;
    auto slot = [&](int i) { return slot0 + i * step + (i == 0 ? pl.rows : 0); };
    // MANY: the first parts' shares are asked for before the factors are known
    const int share = threadIdx.x / lanes;
    constexpr int EARLY = MANY ? 24 : 0;
    float early[MANY ? EARLY : 1];
#pragma unroll
    for (int x = 0; x < EARLY; ++x) {
      const int i = share + x * shares;
      early[x] = i < n && d < a.D ? parts.o[slot(i) * a.D + d] : 0.0f;
    }
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += JOIN_NT) top = fmaxf(top, parts.ml[slot(i)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if ((threadIdx.x & 31) == 0) part_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_NT / 32; ++w) top = fmaxf(top, part_top[w]);
    const float sh = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < n; i += JOIN_NT) {
      const float2 ml = parts.ml[slot(i)];
      factor[i] = exp2_approx(ml.x - sh);
      sum = __fmaf_rn(ml.y, factor[i], sum);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xFFFFFFFFu, sum, o));
    if ((threadIdx.x & 31) == 0) part_sum[warp] = sum;
    __syncthreads();
    float v = 0.0f;
    if (d < a.D) {
#pragma unroll
      for (int x = 0; x < EARLY; ++x)
        if (share + x * shares < n) v = __fmaf_rn(early[x], factor[share + x * shares], v);
#pragma unroll 8
      for (int i = share + EARLY * shares; i < n; i += shares) v = __fmaf_rn(parts.o[slot(i) * a.D + d], factor[i], v);
    }
    so[threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.x < a.D) {
      v = 0.0f, sum = 0.0f;
      for (int x = 0; x < shares; ++x) v = __fadd_rn(v, so[x * lanes + threadIdx.x]);
      for (int w = 0; w < JOIN_NT / 32; ++w) sum = __fadd_rn(sum, part_sum[w]);
      const int64_t i = b * a.Hq + hv / pl.groups * group + hq;
      static_cast<T*>(a.out)[i * a.D + threadIdx.x] = narrow<T>(sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
      if (threadIdx.x == 0 && a.lse) a.lse[i] = sum > 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : sum == 0.0f ? -INFINITY : sum;
    }
    __syncthreads();
  }
}

Plan plan_of(int format, int Hq, int Hk, int D) {
  Plan p{};
  const int group = Hq / Hk;
  p.groups = (group + 15) / 16;
  p.rows = std::min(group, 16);
  p.ctas = std::min(JOIN_PARTS, ctas_per_sm(format, padded(D), p.rows > 8) * sm_count());
  const int row = format == EMU_KV_FP8 ? D : D / 2;
  // Neighbouring heads side by side where a slot's row is long: CTAs that read its pieces at about the same time find the memory's
  // rows open (64 sequences, 262144 slots of 8 heads of 128 bytes: 128 -> 117 us; sets of 8 118; of 64 bytes, 512 in all, 120 -> 89 us a
  // call; 4 heads of 128 bytes 84 -> 81).  Shorter rows would gain too (524288 slots of 4 heads of 64 bytes 107 -> 87, of 2 of 128 83 ->
  // 79); they have not been put so yet.
  while (p.side_bits < 2 && Hk % (2 << p.side_bits) == 0 && Hk * row >= 512) ++p.side_bits;
  p.sets = p.ctas >> p.side_bits;
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
  constexpr int SMEM = WARPS * (S::STAGES * S::STAGE + 8 * 8);
  auto kernel = kv_attend_kernel<T, FORMAT, DP, TWO>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t set = allow_shared(kernel, SMEM, done);
  if (set != cudaSuccess) return set;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.scales[0]) | reinterpret_cast<uintptr_t>(a.scales[1]);
  pl.wide_scales = FORMAT == EMU_KV_MXFP4 && a.D == DP && at % std::min(4, DP / 32) == 0;
  pl.wide_q = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride[0] * 2) | (uintptr_t)(a.q_stride[1] * 2)) & 7) == 0;
  pl.page_size = (uint32_t)std::min<int64_t>(a.page_size, 1ll << 31);
  pl.tile_columns = TILE / pl.page_size, pl.tile_off = TILE % pl.page_size;
  pl.whole_steps = a.page_size % KEYS == 0;
  kernel<<<pl.ctas, NT, SMEM, stream>>>(a, pl);
  // launched early, so that its CTAs wait where the attention's finish
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(a.B * a.Hk * pl.groups, std::max(1, 4096 / pl.rows)), pl.rows);
  cfg.blockDim = dim3(JOIN_NT);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  // MANY where most (sequence, head)s lie in more than FEW CTAs (400001 keys on one head 47 -> 43 us; a call of one sequence of 8192 on 8 heads
  // 26 -> 22, 8 sequences of 100000 on 2 heads 34 -> 32); its registers leave room for fewer CTAs, which costs where there are many
  // (262144 keys 113 -> 122 us; calls of 16 sequences of 131072 on 4 heads 52 -> 58, 64 of 16384 on 8 32 -> 40).
  const bool many = pl.ctas > FEW * a.B * a.Hk * pl.groups;
  const cudaError_t e = many ? cudaLaunchKernelEx(&cfg, kv_attend_join_kernel<T, true>, a, pl, DP) : cudaLaunchKernelEx(&cfg, kv_attend_join_kernel<T, false>, a, pl, DP);
  if (e != cudaSuccess) return e;
  return cudaGetLastError();
}
template <typename T, int FORMAT> cudaError_t launch_sized(const KvAttendArgs& a, cudaStream_t stream) {
  const Plan pl = plan_of(FORMAT, a.Hq, a.Hk, a.D);
  const bool two = pl.rows > 8;
  if (a.D <= 64) return two ? launch<T, FORMAT, 64, true>(a, pl, stream) : launch<T, FORMAT, 64, false>(a, pl, stream);
  if (a.D <= 128) return two ? launch<T, FORMAT, 128, true>(a, pl, stream) : launch<T, FORMAT, 128, false>(a, pl, stream);
  return two ? launch<T, FORMAT, 256, true>(a, pl, stream) : launch<T, FORMAT, 256, false>(a, pl, stream);
}

}  // namespace

size_t kv_attend_workspace(int64_t B, int Hq, int Hk, int D) {
  // (both formats' of the head size: the larger one)
  Plan p = plan_of(EMU_KV_MXFP4, Hq, Hk, D);
  p.ctas = std::max(p.ctas, plan_of(EMU_KV_FP8, Hq, Hk, D).ctas);
  return parts_of(nullptr, B * Hk * p.groups, p.ctas, p.rows, D).bytes;
}

cudaError_t launch_kv_attend(const KvAttendArgs& a, cudaStream_t stream) {
  const bool half = a.dtype == EMU_DTYPE_F16;
  if (a.format == EMU_KV_FP8) return half ? launch_sized<__half, EMU_KV_FP8>(a, stream) : launch_sized<__nv_bfloat16, EMU_KV_FP8>(a, stream);
  return half ? launch_sized<__half, EMU_KV_MXFP4>(a, stream) : launch_sized<__nv_bfloat16, EMU_KV_MXFP4>(a, stream);
}

}  // namespace emu
