// Attention over a cache or a prompt (yb_lm.h, yb_attn_run): one warp per row.
#include <cmath>

#include "attn_lm.h"
#include "attn_row.cuh"

namespace yb {
namespace {

template <typename T>
__global__ void __launch_bounds__(128) attn_rows_kernel(const yb_attn_args a) {
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(a.B) * a.Sq * a.Hq) return;
  const int h = static_cast<int>(row % a.Hq);
  const int i = static_cast<int>(row / a.Hq % a.Sq), b = static_cast<int>(row / a.Hq / a.Sq);
  const int q_len = clamp_len(a.q_len, b, a.Sq), k_len = clamp_len(a.k_len, b, a.Sk);
  if (i >= q_len) return;
  const RowSpan s = row_span(a, b, i, q_len, k_len);
  const RowAcc r = attn_row<T>(a, b, i, h, s.pos, s.lo, s.hi);
  const int d = 4 * (threadIdx.x & 31);
  if (d >= a.D) return;
  T* o = static_cast<T*>(a.o) + b * a.o_stride[0] + i * a.o_stride[1] + h * a.o_stride[2] + d;
  for (int e = 0; e < 4; ++e) o[e] = from_f<T>(r.l == 0.f ? 0.f : r.o[e] / r.l);
}

}  // namespace

cudaError_t launch_attn_rows(const yb_attn_args& a, cudaStream_t s) {
  const long long rows = static_cast<long long>(a.B) * a.Sq * a.Hq;
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (a.dtype == YB_F16)
    attn_rows_kernel<__half><<<grid, 128, 0, s>>>(a);
  else
    attn_rows_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace yb
