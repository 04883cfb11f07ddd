// One attention row on one warp, key after key: the definition of yb_attn
// (yb_lm.h) read off directly.  Masked keys are never loaded, so whatever they
// hold cannot reach the row.
#pragma once
#include "lm.h"

namespace yb {

// Visible keys [lo, hi) of row i of sequence b, and its position.
struct RowSpan {
  int lo = 0, hi = 0, pos = 0;
};

__device__ __forceinline__ int clamp_len(const int* len, int b, int most) {
  return len ? min(max(len[b], 0), most) : most;
}

__device__ __forceinline__ RowSpan row_span(const yb_attn_args& a, int b, int i, int q_len, int k_len) {
  RowSpan s;
  s.pos = k_len - q_len + i;
  s.lo = 0;
  s.hi = k_len;
  if (a.causal) {
    s.hi = min(s.hi, s.pos + 1);
    if (a.prefix) s.hi = max(s.hi, min(a.prefix[b], k_len));
  }
  if (a.key_range) {
    const int2 r = *reinterpret_cast<const int2*>(a.key_range + 2 * (static_cast<long long>(b) * a.Sq + i));
    s.lo = max(s.lo, r.x);
    s.hi = min(s.hi, r.y);
  }
  s.hi = max(s.hi, s.lo);
  return s;
}

// Running softmax of a row: maximum (log2 units), sum, and the four dimensions
// [4 lane, 4 lane + 4) of the weighted values.
struct RowAcc {
  float m, l, o[4];
};

template <typename T>
__device__ RowAcc attn_row(const yb_attn_args& a, int b, int i, int h, int pos, int lo, int hi) {
  constexpr float kLog2e = 1.44269504f;
  const int lane = threadIdx.x & 31, d = 4 * lane;
  const bool has = d < a.D;
  const int hk = h / (a.Hq / a.Hkv);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2];
  float qf[4] = {0.f, 0.f, 0.f, 0.f};
  if (has)
    for (int e = 0; e < 4; ++e) qf[e] = to_f(q[d + e]);
  const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  RowAcc r;
  r.m = -INFINITY;
  r.l = 0.f;
  for (int e = 0; e < 4; ++e) r.o[e] = 0.f;
  for (int j = lo; j < hi; ++j) {
    float s = 0.f, vf[4] = {0.f, 0.f, 0.f, 0.f};
    if (has) {
      const T* kj = k + j * a.k_stride[1] + d;
      const T* vj = v + j * a.v_stride[1] + d;
      for (int e = 0; e < 4; ++e) {
        s = fmaf(qf[e], to_f(kj[e]), s);
        vf[e] = to_f(vj[e]);
      }
    }
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
    s *= a.scale;
    if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
    s *= kLog2e;
    if (a.slopes) s -= slope * static_cast<float>(abs(pos - j));
    const float m = fmaxf(r.m, s), base = m == -INFINITY ? 0.f : m;
    const float c = exp2f(r.m - base), p = exp2f(s - base);
    r.l = r.l * c + p;
    for (int e = 0; e < 4; ++e) r.o[e] = fmaf(p, vf[e], r.o[e] * c);
    r.m = m;
  }
  return r;
}

}  // namespace yb
