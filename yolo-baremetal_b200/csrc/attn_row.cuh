// One attention row on one warp, 32 keys at a time: the definition of yb_attn
// (yb_lm.h) in fp32.  Masked keys are never loaded, so whatever they hold cannot
// reach the row.
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

// Running softmax of a row: reference of the weights (log2 units), their sum, and
// the four dimensions [4 lane, 4 lane + 4) of the weighted values.  The reference
// is kRoom above the maximum, so that the sum over 2^30 keys of values near the
// end of bf16 stays in fp32 (it is divided by a sum that is as much smaller).
constexpr float kRoom = 30.0f;
struct RowAcc {
  float m, l, o[4];
};

// Sum of the products of eight neighbours.
template <typename T>
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float sum) {
  const T* x = reinterpret_cast<const T*>(&a);
  const T* y = reinterpret_cast<const T*>(&b);
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = fmaf(to_f(x[i]), to_f(y[i]), sum);
  return sum;
}

// A lane scores one key of 32, then all lanes walk their values: 0.12 us a key
// and row at D = 64 (key after key on the whole warp 0.37).
template <typename T>
__device__ RowAcc attn_row(const yb_attn_args& a, int b, int i, int h, int pos, int lo, int hi) {
  constexpr float kLog2e = 1.44269504f;
  const int lane = threadIdx.x & 31, d = 4 * lane;
  const bool has = d < a.D;
  const int hk = h / (a.Hq / a.Hkv);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2] + d;
  const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  RowAcc r;
  r.m = -INFINITY;
  r.l = 0.f;
  for (int e = 0; e < 4; ++e) r.o[e] = 0.f;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int n = min(32, hi - j0), j = j0 + lane;
    float s = -INFINITY;
    if (lane < n) {
      const uint4* kj = reinterpret_cast<const uint4*>(k + j * a.k_stride[1]);
      const uint4* qi = reinterpret_cast<const uint4*>(q);
      float dot = 0.f;
      for (int e = 0; e < a.D / 8; e += 4) {  // four loads of each in flight
        uint4 x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int at = min(e + u, a.D / 8 - 1);
          x[u] = qi[at];
          y[u] = kj[at];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (e + u < a.D / 8) dot = dot8<T>(x[u], y[u], dot);
      }
      s = dot * a.scale;
      if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
      s *= kLog2e;
      if (a.slopes) s -= slope * static_cast<float>(abs(pos - j));
    }
    float m = s;  // a NaN score is passed over here and enters the sums
    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
    m = fmaxf(r.m, m + kRoom);
    const float base = m == -INFINITY ? 0.f : m;
    const float c = exp2f(r.m - base), p = lane < n ? exp2f(s - base) : 0.f;
    float sum = p;
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
    r.l = fmaf(r.l, c, sum);
    for (int e = 0; e < 4; ++e) r.o[e] *= c;
    for (int x = 0; x < n; x += 8) {  // eight loads in flight
      uint2 raw[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        raw[u] = make_uint2(0u, 0u);
        if (has && x + u < n) raw[u] = *reinterpret_cast<const uint2*>(v + (j0 + x + u) * a.v_stride[1]);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __shfl_sync(0xFFFFFFFFu, p, x + u);  // 0 from n on
        const T* vj = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int e = 0; e < 4; ++e) r.o[e] = fmaf(w, to_f(vj[e]), r.o[e]);
      }
    }
    r.m = m;
  }
  return r;
}

}  // namespace yb
