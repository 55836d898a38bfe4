// Gradients of attention over packed sequences (the formulas: attention.cuh), a warp to a row.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/emugen.h"
#include "attention.cuh"

namespace emu {
namespace {

using namespace attn;

enum { DELTA, DQ, DKDV };

template <typename T, int WHAT> __global__ void __launch_bounds__(256) attention_rows_kernel(const __grid_constant__ AttnArgs a) {
  const int heads = WHAT == DKDV ? a.Hk : a.Hq;
  const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), total = WHAT == DKDV ? a.Tk : a.Tq;
  if (u >= total * heads) return;
  const int64_t t = u / heads;
  const int h = (int)(u - t * heads);
  float* delta = static_cast<float*>(a.workspace);
  if (WHAT == DELTA) {
    const Lanes o = load_row(static_cast<const T*>(a.out) + (t * a.Hq + h) * a.D, a.D);
    const float d = dot(o, load_row(static_cast<const T*>(a.dout) + t * a.dout_stride[0] + h * a.dout_stride[1], a.D));
    if ((threadIdx.x & 31) == 0) delta[(int64_t)h * a.Tq + t] = d;
    return;
  }
  const int64_t b = sequence_of(WHAT == DKDV ? a.cu_k : a.cu_q, a.B, t);
  if (WHAT == DQ) row_dq<T>(a, delta, b, t, h);
  else if (WHAT == DKDV) row_dkdv<T>(a, delta, b, t, h);
}

template <typename T, int WHAT> void launch_rows(const AttnArgs& a, cudaStream_t stream) {
  const int64_t rows = WHAT == DKDV ? a.Tk * a.Hk : a.Tq * a.Hq;
  if (rows) attention_rows_kernel<T, WHAT><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(a);
}
template <typename T> void launch_back(const AttnArgs& a, cudaStream_t stream) {
  launch_rows<T, DELTA>(a, stream);
  if (a.dq) launch_rows<T, DQ>(a, stream);
  if (a.dk || a.dv) launch_rows<T, DKDV>(a, stream);
}

}  // namespace

size_t attention_backward_workspace(int64_t Tq, int64_t, int Hq, int) { return (size_t)Tq * Hq * sizeof(float); }

cudaError_t launch_attention_backward(const AttnArgs& a, cudaStream_t stream) {
  if (a.dtype == EMU_DTYPE_F16) launch_back<__half>(a, stream);
  else launch_back<__nv_bfloat16>(a, stream);
  return cudaGetLastError();
}

}  // namespace emu
