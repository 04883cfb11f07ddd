// Norm of each query and key head, rotation by position, and the write into
// the cache, in one pass (yb_lm.h, yb_qk_norm_rope).
//
// A head row is read once into registers: a group of lanes holds it, each lane
// both members of its pairs (two chunks of VEC neighbours: d and d + R/2, or
// 2 VEC neighbours when interleaved), so the rotation needs no exchange and the
// norm one butterfly sum over the group.  Angles are formed once per token and
// shared by all its heads: position * inv_freq in fp64, reduced to one turn
// there (in fp32 a position of 10^6 would leave 0.06 radian of error), then
// sincospif of the reduced turn with its fp32 rounding put back to first order.
// Norm and rotation are fp32 on pairs, rounded once on the way out.
//
// The bound is DRAM (each row read and written once): 8,191 tokens of 48 bf16
// head rows of 128 take 53.5 to 54.5 us, 3.7 TB/s, 0.57 of the measured copy rate.
// What is in the way is instructions, two thirds of the issue slots before
// addresses moved into a per-token table, the weights into shared memory and
// the arithmetic onto pairs (62 us then).
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

// VEC floats of shared memory (16-byte aligned where VEC is 4 or 8).
template <int VEC>
__device__ __forceinline__ void shared_words(const float* p, float* v) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + e);
      v[e] = x.x, v[e + 1] = x.y, v[e + 2] = x.z, v[e + 3] = x.w;
    }
  } else {
    v[0] = *p;
  }
}

// A token of the CTA: where its first head rows of q, k and v come from and go
// to (null: not in use, or outside the cache), and its position.
struct Token {
  const void* src[3];
  void* dst[3];
  long long pos;
  int live;
};

template <typename T, int VEC, int NS, bool INTER>
__global__ void __launch_bounds__(kThreads, NS == 1 ? 4 : 3)
    qk_norm_rope_kernel(const __grid_constant__ yb_qk_args a, int group_log, int tokens) {
  // cos and sin of each token's pairs, and both weights: read as whole 16-byte
  // words.
  __shared__ __align__(16) float turn_c[kMaxTokens * (kMaxD / 2)], turn_s[kMaxTokens * (kMaxD / 2)];
  __shared__ __align__(16) float weights[2][kMaxD];
  __shared__ Token token[kMaxTokens];
  const int half = a.R / 2;
  const int pitch = (half + 3) & ~3;  // of a token's angles
  const long long total = static_cast<long long>(a.B) * a.S;
  const long long first = static_cast<long long>(blockIdx.x) * tokens;
  if (threadIdx.x < static_cast<unsigned>(tokens)) {
    const long long x = first + threadIdx.x;
    Token k{};
    if (x < total) {
      const int b = static_cast<int>(x / a.S), t = static_cast<int>(x - static_cast<long long>(b) * a.S);
      const int length = a.length ? a.length[b] : a.S, start = a.start ? a.start[b] : 0;
      const int at = a.positions ? a.positions[x] : 0;  // three loads in flight
      k.live = t < length;
      const long long row = static_cast<long long>(start) + t;
      k.pos = a.positions ? static_cast<long long>(at) : row;
      if (k.live) {
        auto from = [&](const void* p, const long long* st) {
          return static_cast<const void*>(static_cast<const T*>(p) + b * st[0] + t * st[1]);
        };
        auto to = [&](void* p, const long long* st, long long r) {
          return static_cast<void*>(static_cast<T*>(p) + b * st[0] + r * st[1]);
        };
        if (a.q) {
          k.src[0] = from(a.q, a.q_stride);
          k.dst[0] = to(a.q_out, a.q_out_stride, t);
        }
        if (row >= 0 && row < a.cache_rows) {
          if (a.k) {
            k.src[1] = from(a.k, a.k_stride);
            k.dst[1] = to(a.k_out, a.k_out_stride, row);
          }
          if (a.v) {
            k.src[2] = from(a.v, a.v_stride);
            k.dst[2] = to(a.v_out, a.v_out_stride, row);
          }
        }
      }
    }
    token[threadIdx.x] = k;
  }
  for (int d = threadIdx.x; d < a.D; d += kThreads) {
    weights[0][d] = (a.q_weight ? a.q_weight[d] : 1.0f) + a.weight_add;
    weights[1][d] = (a.k_weight ? a.k_weight[d] : 1.0f) + a.weight_add;
  }
  __syncthreads();

  // This lane's chunks of any row: offsets, and first pair (-1: not rotated).
  const int group = 1 << group_log, lane = threadIdx.x & (group - 1);
  const int slots = a.D / 2 / VEC;
  int o0[NS], o1[NS], f0[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int slot = s * group + lane;
    f0[s] = -1;
    if (INTER) {
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
  }

  // Rows (head rows of q, k and v of the CTA's tokens) go round the groups;
  // the next one's loads are under way while one is worked on, the first one's
  // while the angles are formed.
  const int rows = a.Hq + a.Hkv * (a.v ? 2 : 1);
  const int groups = kThreads >> group_log;
  // Every lane of a warp makes the same number of rounds (the sums shuffle).
  const int rounds = (tokens * rows + groups - 1) / groups;
  int k = 0, head = threadIdx.x >> group_log;  // of the row to fetch next
  struct Row {
    Chunk<T, VEC> c0[NS], c1[NS];
    T* dst;
    int k, kind;
    bool live;
  };
  auto fetch = [&](Row& r) {
    while (head >= rows) head -= rows, ++k;
    r.k = k;
    r.kind = head < a.Hq ? 0 : head < a.Hq + a.Hkv ? 1 : 2;
    const int h = head - (r.kind == 0 ? 0 : r.kind == 1 ? a.Hq : a.Hq + a.Hkv);
    const T* src = k < tokens ? static_cast<const T*>(token[k].src[r.kind]) : nullptr;
    r.live = src != nullptr;
    if (r.live) {
      src += h * (r.kind == 0 ? a.q_stride[2] : r.kind == 1 ? a.k_stride[2] : a.v_stride[2]);
      r.dst = static_cast<T*>(token[k].dst[r.kind]) +
              h * (r.kind == 0 ? a.q_out_stride[2] : r.kind == 1 ? a.k_out_stride[2] : a.v_out_stride[2]);
#pragma unroll
      for (int s = 0; s < NS; ++s)
        if (s * group + lane < slots) {
          r.c0[s] = *reinterpret_cast<const Chunk<T, VEC>*>(src + o0[s]);
          r.c1[s] = *reinterpret_cast<const Chunk<T, VEC>*>(src + o1[s]);
        }
    }
    head += groups;
  };
  Row cur, next;
  fetch(cur);

  // One token's angles after another, a quarter of the CTA on each of four.
  const int quarter = kThreads / kMaxTokens;
  for (int i = threadIdx.x; i < kMaxTokens * (tokens == 1 ? kThreads : quarter); i += kThreads) {
    const int x = tokens == 1 ? 0 : i / quarter;
    if (x >= tokens || !token[x].live) continue;
    for (int f = tokens == 1 ? i : i - x * quarter; f < half; f += tokens == 1 ? kThreads : quarter) {
      const double turns = static_cast<double>(token[x].pos) * a.inv_freq[f] * 0.15915494309189533577;  // 1 / (2 pi)
      const double r = turns - rint(turns);
      const float hi = static_cast<float>(r), lo = static_cast<float>(r - static_cast<double>(hi)) * 6.28318531f;
      float s, c;
      sincospif(2.0f * hi, &s, &c);
      turn_c[x * pitch + f] = c - s * lo;
      turn_s[x * pitch + f] = s + c * lo;
    }
  }
  __syncthreads();

  const float inv_d = 1.0f / static_cast<float>(a.D);
  for (int n = 0; n < rounds; ++n) {
    if (n + 1 < rounds) fetch(next);
    float2 squares = make_float2(0.f, 0.f);
    if (cur.live && cur.kind < 2) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
        if (s * group + lane < slots) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float2 x = make_float2(to_f(cur.c0[s].v[e]), to_f(cur.c1[s].v[e]));
            squares = __ffma2_rn(x, x, squares);
          }
        }
    }
    float sum = squares.x + squares.y;
    for (int m = group >> 1; m; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
    if (cur.live) {
      const float r = rsqrtf(fmaf(sum, inv_d, a.eps));
      const float* w = weights[cur.kind == 0 ? 0 : 1];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        if (s * group + lane >= slots) continue;
        if (cur.kind < 2) {
          // y[e] = (chunk 0's element e, chunk 1's element e).
          float2 y[VEC];
          float w0[VEC], w1[VEC];
          shared_words<VEC>(w + o0[s], w0);
          shared_words<VEC>(w + o1[s], w1);
          const float2 r2 = make_float2(r, r);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            y[e] = __fmul2_rn(__fmul2_rn(make_float2(to_f(cur.c0[s].v[e]), to_f(cur.c1[s].v[e])), r2),
                              make_float2(w0[e], w1[e]));
          if (f0[s] >= 0) {
            float tc[VEC], ts[VEC];
            shared_words<VEC>(turn_c + cur.k * pitch + f0[s], tc);
            shared_words<VEC>(turn_s + cur.k * pitch + f0[s], ts);
            if constexpr (!INTER) {
#pragma unroll
              for (int e = 0; e < VEC; ++e)  // (p c - q s, q c + p s)
                y[e] = __ffma2_rn(make_float2(y[e].y, y[e].x), make_float2(-ts[e], ts[e]),
                                  __fmul2_rn(y[e], make_float2(tc[e], tc[e])));
            } else if constexpr (VEC == 1) {
              y[0] = make_float2(y[0].x * tc[0] - y[0].y * ts[0], y[0].y * tc[0] + y[0].x * ts[0]);
            } else {
#pragma unroll
              for (int e = 0; e < VEC; e += 2) {  // pairs e / 2 of chunk 0 and (VEC + e) / 2 of chunk 1
                const float2 c2 = make_float2(tc[e / 2], tc[(VEC + e) / 2]), s2 = make_float2(ts[e / 2], ts[(VEC + e) / 2]);
                const float2 p = y[e], q = y[e + 1];
                y[e] = __ffma2_rn(q, make_float2(-s2.x, -s2.y), __fmul2_rn(p, c2));
                y[e + 1] = __ffma2_rn(p, s2, __fmul2_rn(q, c2));
              }
            }
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            cur.c0[s].v[e] = from_f<T>(y[e].x);
            cur.c1[s].v[e] = from_f<T>(y[e].y);
          }
        }
        *reinterpret_cast<Chunk<T, VEC>*>(cur.dst + o0[s]) = cur.c0[s];
        *reinterpret_cast<Chunk<T, VEC>*>(cur.dst + o1[s]) = cur.c1[s];
      }
    }
    cur = next;
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
  // A token per CTA spreads a decode step over the SMs; four share what comes
  // before their rows once there are CTAs enough for two on each of 148 SMs
  // (3,003 fp32 tokens: 20.6 us one by one, 14.4 by fours).
  const int tokens = total >= 2 * 148 * kMaxTokens ? kMaxTokens : 1;
  const unsigned grid = static_cast<unsigned>((total + tokens - 1) / tokens);
  if (a.interleaved)
    qk_norm_rope_kernel<T, VEC, NS, true><<<grid, kThreads, 0, s>>>(a, group_log, tokens);
  else
    qk_norm_rope_kernel<T, VEC, NS, false><<<grid, kThreads, 0, s>>>(a, group_log, tokens);
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
  if (!on_boundary(a.dtype == YB_F32 ? 4 : 2, a.q, a.k, a.v, a.q_out, a.k_out, a.v_out) || !on_boundary(8, a.inv_freq) ||
      !on_boundary(4, a.q_weight, a.k_weight, a.start, a.length, a.positions)) {
    set_error("qk_norm_rope: a pointer is not aligned to its element");
    return ERROR_INVALID_DIMS;
  }
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
