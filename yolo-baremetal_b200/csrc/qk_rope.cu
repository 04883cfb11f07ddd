// Norm of each query and key head, rotation by position, and the write into
// the cache, in one pass (yb_lm.h, yb_qk_norm_rope).
//
// A head row is read once into registers: a group of lanes holds it, each lane
// both members of its pairs (two chunks of kVec neighbours: d and d + R/2, or
// 2 kVec neighbours when interleaved), so the rotation needs no exchange and
// the norm one butterfly sum over the group.  Angles are formed once per token
// and shared by all its heads: position * inv_freq in fp64, reduced to one
// turn there (in fp32 a position of 10^6 would leave 0.06 radian of error),
// then sincospif of the reduced turn with its fp32 rounding put back to first
// order.  Norm and rotation are fp32, rounded once on the way out.
#include <cmath>
#include <string>

#include "lm.h"

namespace yb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 4;  // per CTA
constexpr int kMaxD = 256;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
  T v[VEC];
};

template <typename T, int VEC, int NS>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const yb_qk_args a, int group_log, int tokens) {
  __shared__ float2 turn[kMaxTokens * (kMaxD / 2)];  // cos, sin of each token's pairs
  const int half = a.R / 2;
  const long long total = static_cast<long long>(a.B) * a.S;
  const long long first = static_cast<long long>(blockIdx.x) * tokens;
  for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
    const int k = i / half, f = i - k * half;
    if (first + k >= total) break;
    const int b = static_cast<int>((first + k) / a.S), t = static_cast<int>(first + k - static_cast<long long>(b) * a.S);
    const long long pos =
        a.positions ? a.positions[first + k] : (a.start ? static_cast<long long>(a.start[b]) : 0ll) + t;
    const double turns = static_cast<double>(pos) * a.inv_freq[f] * 0.15915494309189533577;  // 1 / (2 pi)
    const double r = turns - rint(turns);
    const float hi = static_cast<float>(r), lo = static_cast<float>(r - static_cast<double>(hi)) * 6.28318531f;
    float s, c;
    sincospif(2.0f * hi, &s, &c);
    turn[i] = make_float2(c - s * lo, s + c * lo);
  }
  __syncthreads();

  const int group = 1 << group_log, lane = threadIdx.x & (group - 1);
  const int slots = a.D / 2 / VEC;
  const int rows = a.Hq + a.Hkv * (a.v ? 2 : 1);
  const int end = tokens * rows;
  // Every lane of a warp makes the same number of rounds (the sums shuffle).
  const int rounds = (end + (kThreads >> group_log) - 1) / (kThreads >> group_log);
  for (int n = 0; n < rounds; ++n) {
    const int item = n * (kThreads >> group_log) + (threadIdx.x >> group_log);
    const int k = item / rows, head = item - k * rows;
    bool live = item < end && first + k < total;
    int b = 0, t = 0;
    if (live) {
      b = static_cast<int>((first + k) / a.S);
      t = static_cast<int>(first + k - static_cast<long long>(b) * a.S);
      live = !a.length || t < a.length[b];
    }
    const int kind = head < a.Hq ? 0 : head < a.Hq + a.Hkv ? 1 : 2;
    const T* src = nullptr;
    T* dst = nullptr;
    if (live) {
      const int h = kind == 0 ? head : kind == 1 ? head - a.Hq : head - a.Hq - a.Hkv;
      const void* in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
      void* out = kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out;
      const long long* si = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
      const long long* so = kind == 0 ? a.q_out_stride : kind == 1 ? a.k_out_stride : a.v_out_stride;
      long long row = t;
      if (kind) {
        if (a.start) row += a.start[b];
        live = row >= 0 && row < a.cache_rows;
      }
      src = static_cast<const T*>(in) + b * si[0] + t * si[1] + h * si[2];
      dst = static_cast<T*>(out) + b * so[0] + row * so[1] + h * so[2];
    }
    Chunk<T, VEC> c0[NS], c1[NS];
    int o0[NS], o1[NS], f0[NS];  // offsets of the two chunks, first pair (-1: not rotated)
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int slot = s * group + lane;
      f0[s] = -1;
      if (a.interleaved) {
        o0[s] = 2 * slot * VEC;
        o1[s] = o0[s] + VEC;
        if (o0[s] < a.R) f0[s] = slot * VEC;
      } else if (slot * VEC < half) {
        o0[s] = slot * VEC;
        o1[s] = half + slot * VEC;
        f0[s] = slot * VEC;
      } else {
        o0[s] = a.R + slot * VEC - half;
        o1[s] = o0[s] + (a.D - a.R) / 2;
      }
      if (live && slot < slots) {
        c0[s] = *reinterpret_cast<const Chunk<T, VEC>*>(src + o0[s]);
        c1[s] = *reinterpret_cast<const Chunk<T, VEC>*>(src + o1[s]);
        if (kind < 2) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float x = to_f(c0[s].v[e]), y = to_f(c1[s].v[e]);
            sum = fmaf(x, x, sum);
            sum = fmaf(y, y, sum);
          }
        }
      }
    }
    for (int m = group >> 1; m; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
    if (!live) continue;
    const float r = 1.0f / sqrtf(sum / static_cast<float>(a.D) + a.eps);
    const float* w = kind == 0 ? a.q_weight : a.k_weight;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if (s * group + lane >= slots) continue;
      if (kind < 2) {
        float y[2 * VEC];
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) {
          const int d = e < VEC ? o0[s] + e : o1[s] + e - VEC;
          const float x = to_f(e < VEC ? c0[s].v[e] : c1[s].v[e - VEC]);
          y[e] = x * r * ((w ? w[d] : 1.0f) + a.weight_add);
        }
        if (f0[s] >= 0) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float2 cs = turn[k * half + f0[s] + e];
            float p, q;
            if (a.interleaved) {
              p = y[2 * e];
              q = y[2 * e + 1];
            } else {
              p = y[e];
              q = y[e + VEC];
            }
            const float u = p * cs.x - q * cs.y, z = q * cs.x + p * cs.y;
            if (a.interleaved) {
              y[2 * e] = u;
              y[2 * e + 1] = z;
            } else {
              y[e] = u;
              y[e + VEC] = z;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          c0[s].v[e] = from_f<T>(y[e]);
          c1[s].v[e] = from_f<T>(y[e + VEC]);
        }
      }
      *reinterpret_cast<Chunk<T, VEC>*>(dst + o0[s]) = c0[s];
      *reinterpret_cast<Chunk<T, VEC>*>(dst + o1[s]) = c1[s];
    }
  }
}

// Whether pointers and strides let the rows move in 16-byte chunks, and the
// two halves of the rotated and of the plain part split into whole chunks.
template <typename T>
bool chunks_fit(const yb_qk_args& a) {
  constexpr int vec = 16 / static_cast<int>(sizeof(T));
  if (a.interleaved) {
    if (a.R % (2 * vec) || a.D % (2 * vec)) return false;
  } else if ((a.R / 2) % vec || (a.D - a.R) / 2 % vec) {
    return false;
  }
  auto fits = [](const void* p, const long long* s) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % vec == 0 && s[1] % vec == 0 && s[2] % vec == 0;
  };
  if (!fits(a.q, a.q_stride) || !fits(a.q_out, a.q_out_stride)) return false;
  if (a.Hkv && (!fits(a.k, a.k_stride) || !fits(a.k_out, a.k_out_stride))) return false;
  return !a.v || (fits(a.v, a.v_stride) && fits(a.v_out, a.v_out_stride));
}

template <typename T, int VEC, int NS>
cudaError_t launch(const yb_qk_args& a, cudaStream_t s) {
  const int slots = a.D / 2 / VEC;
  int group_log = 0;
  while (group_log < 5 && (1 << group_log) < slots) ++group_log;
  const long long total = static_cast<long long>(a.B) * a.S;
  // A token per CTA spreads a decode step over the SMs; four share the
  // launch and the angle stage once the grid is many waves deep.
  const int tokens = total >= 4096 ? kMaxTokens : 1;
  qk_norm_rope_kernel<T, VEC, NS>
      <<<static_cast<unsigned>((total + tokens - 1) / tokens), kThreads, 0, s>>>(a, group_log, tokens);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dispatch(const yb_qk_args& a, cudaStream_t s) {
  // 16-byte chunks: at most 32 a row (fp32, D = 256); element by element, 128.
  if (chunks_fit<T>(a)) return launch<T, 16 / sizeof(T), 1>(a, s);
  return launch<T, 1, 4>(a, s);
}

bool strides_ok(const long long* s) { return s[0] >= 0 && s[1] >= 0 && s[2] >= 0; }

}  // namespace
}  // namespace yb

using namespace yb;

extern "C" status_t yb_qk_norm_rope(const yb_qk_args* p, void* stream) {
  if (!p) return ERROR_NULL_POINTER;
  yb_qk_args a = *p;
  if (a.B < 0 || a.S < 0 || a.Hq < 0 || a.Hkv < 0 || a.cache_rows < 0 || a.D < 2 || a.D > kMaxD || a.D % 2 ||
      a.R < 0 || a.R > a.D || a.R % 2) {
    set_error("qk_norm_rope: sizes not negative, D even in [2, 256], R even in [0, D]");
    return ERROR_INVALID_DIMS;
  }
  if (a.Hq > 65536 || a.Hkv > 65536 || static_cast<long long>(a.B) * a.S > (1LL << 31) - 1) {
    set_error("qk_norm_rope: at most 65536 heads and 2^31 - 1 tokens");
    return ERROR_INVALID_DIMS;
  }
  if (a.dtype < YB_F32 || a.dtype > YB_BF16 || (a.interleaved != 0 && a.interleaved != 1) || !std::isfinite(a.eps) ||
      a.eps < 0.f || !std::isfinite(a.weight_add)) {
    set_error("qk_norm_rope: dtype YB_F32, YB_F16 or YB_BF16, interleaved 0 or 1, eps >= 0 and finite");
    return ERROR_INVALID_DIMS;
  }
  if (!strides_ok(a.q_stride) || !strides_ok(a.k_stride) || !strides_ok(a.v_stride) || !strides_ok(a.q_out_stride) ||
      !strides_ok(a.k_out_stride) || !strides_ok(a.v_out_stride)) {
    set_error("qk_norm_rope: negative stride");
    return ERROR_INVALID_DIMS;
  }
  if (a.B == 0 || a.S == 0 || (a.Hq == 0 && a.Hkv == 0)) return SUCCESS;
  if (a.Hkv == 0) a.k = a.v = nullptr, a.k_out = a.v_out = nullptr;
  if ((a.Hq && (!a.q || !a.q_out)) || (a.Hkv && (!a.k || !a.k_out)) || (a.R && !a.inv_freq) || !a.v != !a.v_out)
    return ERROR_NULL_POINTER;
  auto same = [](const long long* x, const long long* y) { return x[0] == y[0] && x[1] == y[1] && x[2] == y[2]; };
  if ((a.Hq && a.q == a.q_out && !same(a.q_stride, a.q_out_stride)) ||
      (a.Hkv && a.k == a.k_out && (a.start || !same(a.k_stride, a.k_out_stride))) ||
      (a.v && a.v == a.v_out && (a.start || !same(a.v_stride, a.v_out_stride)))) {
    set_error("qk_norm_rope: an output may be its input only with the same strides and without start");
    return ERROR_INVALID_DIMS;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case YB_F32: return cuda_status(dispatch<float>(a, s), "qk_norm_rope");
    case YB_F16: return cuda_status(dispatch<__half>(a, s), "qk_norm_rope");
    default: return cuda_status(dispatch<__nv_bfloat16>(a, s), "qk_norm_rope");
  }
}
