// Token sampling (yb_lm.h, yb_sample): temperature, top-k, top-p and min-p,
// then the inverse of the running sum at a given random number.
//
// Weights are fixed point, W = rint(2^44 exp((x - max) / T)), at most 2^44
// each and 2^62 for a row of 2^18, so every sum below is exact whatever its
// order: results do not depend on the cluster size, on atomics or on how the
// row is cut, and a border between two tokens lies within V 2^-45 of where
// the real sum has it (fp32 sums would move it by up to V 2^-24, which at
// 100,000 tokens is a whole token).
//
// One cluster of C CTAs per row; each keeps its slice of the row in shared
// memory as order-preserving 32-bit keys, so the logits are read once.
//   1 keys, and the row's largest (key, lowest index);
//   2 with top-k or top-p: a histogram of counts and weights over 1/16-octave
//     steps below the maximum, summed over the cluster; the step that holds
//     the border is either listed (at most kList tokens, ranked by comparing
//     all pairs) or split again into kBins by its composites (key, ~index),
//     which are all distinct, so ties need no rule of their own;
//   3 sums of the kept weights per warp and CTA, then the one warp that holds
//     the border walks its tokens.
#include <cooperative_groups.h>

#include <atomic>
#include <cfloat>
#include <cmath>
#include <string>

#include "lm.h"
#include "pdl.cuh"

namespace cg = cooperative_groups;

namespace yb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kList = 512;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = YB_SAMPLE_MAX_VOCAB / kMaxCluster;
constexpr double kOne = 17592186044416.0;  // 2^44

using u64 = unsigned long long;

struct SampleSmem {
  u64 tmass[kBins];   // cluster totals
  uint32_t tcnt[kBins];
  uint32_t cnt[kBins];      // own slice; the weights' sums in three 15-bit parts
  uint32_t part[3][kBins];  // (2^15 tokens of a slice: 30 bits each)
  u64 list[kList];
  u64 list_w[kList];
  double table[64];  // 2^(j / 64)
  u64 warp_a[kWarps], warp_b[kWarps];
  u64 slot_a[kMaxCluster], slot_b[kMaxCluster];
  u64 result[2];
  int found[1];
  int n_list;
};

__device__ __forceinline__ uint32_t key_of(float x) {
  // NaN and -infinity: 0, which no kept logit has.
  if (!(x >= -FLT_MAX)) return 0u;
  x = fminf(x, FLT_MAX) + 0.0f;  // -0 and 0 are equal
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float val_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

struct Row {
  double best = 0, c = 0;  // largest logit, log2(e) / T
  float bestf = 0, cf = 0;
};

// rint(2^44 2^y), y = (x - best) log2(e) / T <= 0.  2^y = 2^n 2^(j/64) e^r with
// |r| <= ln 2 / 128 (table-driven, after Tang 1989): the Taylor polynomial of
// degree 6 leaves r^7 / 5040 < 2^-64.
__device__ __forceinline__ u64 weight(uint32_t key, const Row& r, const double* table) {
  if (key == 0u) return 0ull;
  const double y = (static_cast<double>(val_of(key)) - r.best) * r.c;
  if (!(y > -46.0)) return 0ull;
  const double t = rint(y * 64.0);
  const int k = static_cast<int>(t);
  const double q = (y - t * 0.015625) * 0.69314718055994530942;
  double p = fma(q, 1.0 / 720.0, 1.0 / 120.0);
  p = fma(p, q, 1.0 / 24.0);
  p = fma(p, q, 1.0 / 6.0);
  p = fma(p, q, 0.5);
  p = fma(p, q, 1.0);
  p = fma(p, q, 1.0);
  const double s = __longlong_as_double(static_cast<long long>(1023 + 44 + (k >> 6)) << 52);
  return static_cast<u64>(__double2ull_rn(p * table[k & 63] * s));
}

// Step of 1/16 octave below the maximum: rises as the key falls.
__device__ __forceinline__ int step_of(uint32_t key, const Row& r) {
  const float d = (r.bestf - val_of(key)) * r.cf * 16.0f;
  return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
}

__device__ __forceinline__ u64 composite(uint32_t key, uint32_t idx) {
  return (static_cast<u64>(key) << 32) | (0xFFFFFFFFu - idx);
}

__device__ __forceinline__ u64 shfl_xor64(u64 v, int m) { return __shfl_xor_sync(0xFFFFFFFFu, v, m); }

template <typename Op>
__device__ __forceinline__ u64 block_reduce(u64 v, u64* warps, u64 id, Op op) {
  for (int m = 16; m; m >>= 1) v = op(v, shfl_xor64(v, m));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = id;
  for (int w = 0; w < kWarps; ++w) r = op(r, warps[w]);
  return r;
}

struct MaxOp {
  __device__ u64 operator()(u64 a, u64 b) const { return a > b ? a : b; }
};
struct MinOp {
  __device__ u64 operator()(u64 a, u64 b) const { return a < b ? a : b; }
};
struct AddOp {
  __device__ u64 operator()(u64 a, u64 b) const { return a + b; }
};

// The same value in every thread of the cluster.  Each use of a slot array is
// separated from the next by the cluster barrier of the other kind of use.
template <typename Op>
__device__ u64 cluster_reduce(cg::cluster_group& cl, u64 v, SampleSmem& S, u64* slot, u64 id, Op op) {
  const u64 b = block_reduce(v, S.warp_a, id, op);
  const unsigned C = cl.num_blocks(), me = cl.block_rank();
  cl.sync();  // earlier readers of the slots are done
  if (threadIdx.x < C) cl.map_shared_rank(slot, threadIdx.x)[me] = b;
  cl.sync();
  u64 r = id;
  for (unsigned i = 0; i < C; ++i) r = op(r, slot[i]);
  return r;
}

struct Picker {
  cg::cluster_group& cl;
  SampleSmem& S;
  const uint32_t* keys;
  int n;          // tokens of the slice
  uint32_t base;  // index of its first
  Row row;

  // Adds one token to bin b of the own histogram.
  __device__ void add(int b, u64 w, bool with_mass) {
    atomicAdd(&S.cnt[b], 1u);
    if (with_mass) {
      const uint32_t p0 = w & 0x7FFFu, p1 = (w >> 15) & 0x7FFFu, p2 = static_cast<uint32_t>(w >> 30);
      if (p0) atomicAdd(&S.part[0][b], p0);
      if (p1) atomicAdd(&S.part[1][b], p1);
      if (p2) atomicAdd(&S.part[2][b], p2);
    }
  }
  __device__ void clear() {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      S.cnt[b] = 0;
      S.part[0][b] = S.part[1][b] = S.part[2][b] = 0;
    }
    __syncthreads();
  }
  // Cluster totals of the histogram into tcnt, tmass of every CTA: CTA r sums
  // the bins congruent to its share and writes them to all.
  __device__ void total(bool with_mass) {
    const int C = static_cast<int>(cl.num_blocks()), me = static_cast<int>(cl.block_rank());
    cl.sync();
    const int share = kBins / C;
    for (int i = threadIdx.x; i < share; i += kThreads) {
      const int b = me * share + i;
      uint32_t c = 0;
      u64 m = 0;
      for (int r = 0; r < C; ++r) {
        const SampleSmem* o = cl.map_shared_rank(&S, r);
        c += o->cnt[b];
        if (with_mass)
          m += o->part[0][b] + (static_cast<u64>(o->part[1][b]) << 15) + (static_cast<u64>(o->part[2][b]) << 30);
      }
      for (int r = 0; r < C; ++r) {
        SampleSmem* o = cl.map_shared_rank(&S, r);
        o->tcnt[b] = c;
        if (with_mass) o->tmass[b] = m;
      }
    }
    cl.sync();
  }
  // First bin in which the running sum of `what` reaches `target` (>= 1), with
  // the sums before it.  Two bins a thread.
  __device__ int border(u64 target, bool by_mass, bool with_mass, u64* before_cnt, u64* before_mass) {
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    const u64 c0 = S.tcnt[2 * t], c1 = S.tcnt[2 * t + 1];
    const u64 m0 = with_mass ? S.tmass[2 * t] : 0, m1 = with_mass ? S.tmass[2 * t + 1] : 0;
    u64 sc = c0 + c1, sm = m0 + m1;
    for (int d = 1; d < 32; d <<= 1) {
      const u64 a = __shfl_up_sync(0xFFFFFFFFu, sc, d), b = __shfl_up_sync(0xFFFFFFFFu, sm, d);
      if (lane >= d) sc += a, sm += b;
    }
    __syncthreads();
    if (t == 0) S.found[0] = kBins - 1;
    if (lane == 31) S.warp_a[w] = sc, S.warp_b[w] = sm;
    __syncthreads();
    for (int i = 0; i < w; ++i) sc += S.warp_a[i], sm += S.warp_b[i];
    // sums before bin 2t, 2t + 1 and after it
    const u64 e0c = sc - c0 - c1, e0m = sm - m0 - m1, e1c = sc - c1, e1m = sm - m1;
    const u64 a0 = by_mass ? e0m : e0c, a1 = by_mass ? e1m : e1c, a2 = by_mass ? sm : sc;
    if (a0 < target && target <= a1) S.found[0] = 2 * t, S.result[0] = e0c, S.result[1] = e0m;
    if (a1 < target && target <= a2) S.found[0] = 2 * t + 1, S.result[0] = e1c, S.result[1] = e1m;
    __syncthreads();
    const int b = S.found[0];
    *before_cnt = S.result[0];
    *before_mass = S.result[1];
    __syncthreads();
    return b;
  }

  // The lowest composite kept when the tokens are taken in falling order while
  // fewer than `target` of them (by_mass: of their weight) came before.
  // tcnt / tmass hold the 1/16-octave histogram, whose whole sum is above
  // target.  *kept_mass: the weight down to the cut.
  __device__ u64 cut(u64 target, bool by_mass, bool with_mass, u64* kept_mass) {
    u64 bc, bm;
    const int step = border(target, by_mass, with_mass, &bc, &bm);
    uint32_t inside = S.tcnt[step];
    u64 lo = 0, hi = ~0ull;  // composites that are still candidates
    while (inside > kList) {
      u64 mn = ~0ull, mx = 0;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t k = keys[i];
        const u64 c = composite(k, base + i);
        if (k && c >= lo && c <= hi && step_of(k, row) == step && weight(k, row, S.table)) {
          mn = c < mn ? c : mn;
          mx = c > mx ? c : mx;
        }
      }
      mn = cluster_reduce(cl, mn, S, S.slot_a, ~0ull, MinOp());
      mx = cluster_reduce(cl, mx, S, S.slot_b, 0ull, MaxOp());
      int shift = 0;  // at least half of the bins span [mn, mx]
      while (((mx - mn) >> shift) >= kBins) ++shift;
      clear();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t k = keys[i];
        const u64 c = composite(k, base + i);
        if (k && c >= mn && c <= mx && step_of(k, row) == step) {
          const u64 w = weight(k, row, S.table);
          if (w) add(static_cast<int>((mx - c) >> shift), w, with_mass);
        }
      }
      total(with_mass);
      u64 c2, m2;
      const u64 rest = target - (by_mass ? bm : bc);
      const int b = border(rest, by_mass, with_mass, &c2, &m2);
      bc += c2;
      bm += m2;
      inside = S.tcnt[b];
      hi = mx - (static_cast<u64>(b) << shift);
      const u64 span = (1ull << shift) - 1;
      lo = hi - mn > span ? hi - span : mn;
    }
    // The candidates to CTA 0, in any order.
    SampleSmem* head = cl.map_shared_rank(&S, 0);
    if (threadIdx.x == 0) S.n_list = 0;
    cl.sync();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t k = keys[i];
      const u64 c = composite(k, base + i);
      if (k && c >= lo && c <= hi && step_of(k, row) == step) {
        const u64 w = weight(k, row, S.table);
        if (w) {
          const int at = atomicAdd(&head->n_list, 1);
          if (at < kList) {
            head->list[at] = c;
            head->list_w[at] = w;
          }
        }
      }
    }
    cl.sync();
    if (cl.block_rank() == 0) {
      const int m = S.n_list < kList ? S.n_list : kList;
      u64 mine = ~0ull, w = 0;
      if (static_cast<int>(threadIdx.x) < m) {
        const u64 c = S.list[threadIdx.x];
        u64 rank = 0, pre = 0;
        for (int j = 0; j < m; ++j)
          if (S.list[j] > c) ++rank, pre += S.list_w[j];
        if ((by_mass ? bm + pre : bc + rank) < target) mine = c, w = S.list_w[threadIdx.x];
      }
      const u64 low = block_reduce(mine, S.warp_a, ~0ull, MinOp());
      const u64 mass = bm + block_reduce(w, S.warp_b, 0ull, AddOp());
      if (threadIdx.x < cl.num_blocks()) {
        SampleSmem* o = cl.map_shared_rank(&S, threadIdx.x);
        o->slot_a[0] = low;
        o->slot_b[0] = mass;
      }
    }
    cl.sync();
    const u64 low = S.slot_a[0];
    *kept_mass = S.slot_b[0];
    cl.sync();
    return low;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const yb_sample_args a, int slice) {
  extern __shared__ __align__(16) uint8_t sample_raw[];
  SampleSmem& S = *reinterpret_cast<SampleSmem*>(sample_raw);
  uint32_t* keys = reinterpret_cast<uint32_t*>(sample_raw + sizeof(SampleSmem));
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), me = static_cast<int>(cl.block_rank());
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = min(me * slice, a.V);
  const int n = min(slice, a.V - first);
  const T* x = static_cast<const T*>(a.logits) + static_cast<long long>(b) * a.row_stride + first;

  if (tid < 64) S.table[tid] = exp2(tid / 64.0);
  u64 best = 0;
  for (int i = tid; i < n; i += kThreads) {
    const uint32_t k = key_of(to_f(x[i]));
    keys[i] = k;
    const u64 c = composite(k, first + i);
    best = c > best ? c : best;
  }
  best = cluster_reduce(cl, best, S, S.slot_a, 0ull, MaxOp());
  const uint32_t best_key = static_cast<uint32_t>(best >> 32);
  const float temp = a.temperature ? a.temperature[b] : 1.0f;
  if (best_key == 0u || !(temp > 0.0f)) {
    if (me == 0 && tid == 0) {
      a.token[b] = best_key ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best)) : -1;
      if (a.logprob) a.logprob[b] = best_key ? 0.0f : -INFINITY;
    }
    return;  // every CTA of the cluster, after its last remote access
  }
  Picker P{cl, S, keys, n, static_cast<uint32_t>(first), Row()};
  P.row.bestf = val_of(best_key);
  P.row.best = P.row.bestf;
  P.row.c = 1.4426950408889634074 / static_cast<double>(temp);
  P.row.cf = static_cast<float>(fmin(P.row.c, 1e30));

  const int top_k = a.top_k ? a.top_k[b] : 0;
  const float top_p = a.top_p ? a.top_p[b] : 1.0f;
  const float min_p = a.min_p ? a.min_p[b] : 0.0f;
  const bool use_k = top_k > 0 && top_k < a.V, use_p = top_p < 1.0f;
  u64 cut = 1;  // keys above 0
  if (use_k || use_p) {
    P.clear();
    u64 mass = 0, count = 0;
    for (int i = tid; i < n; i += kThreads) {
      const u64 w = weight(keys[i], P.row, S.table);
      if (w) {
        P.add(step_of(keys[i], P.row), w, use_p);
        mass += w;
        ++count;
      }
    }
    P.total(use_p);
    count = cluster_reduce(cl, count, S, S.slot_a, 0ull, AddOp());
    if (use_p) mass = cluster_reduce(cl, mass, S, S.slot_b, 0ull, AddOp());
    // `cut` may leave a finer histogram in tcnt / tmass; the second search
    // needs the first one again.
    bool fresh = true;
    if (use_k && static_cast<u64>(top_k) < count) {
      u64 kept = 0;
      cut = P.cut(static_cast<u64>(top_k), false, use_p, &kept);
      mass = kept;
      fresh = false;
    }
    if (use_p) {
      const u64 target = static_cast<u64>(fmax(1.0, ceil(static_cast<double>(top_p) * static_cast<double>(mass))));
      if (target < mass) {
        if (!fresh) {
          P.clear();
          for (int i = tid; i < n; i += kThreads) {
            const u64 w = weight(keys[i], P.row, S.table);
            if (w) P.add(step_of(keys[i], P.row), w, true);
          }
          P.total(true);
        }
        u64 kept = 0;
        const u64 c = P.cut(target, true, true, &kept);
        cut = c > cut ? c : cut;
      }
    }
  }
  const u64 least = min_p > 0.0f ? static_cast<u64>(fmin(rint(static_cast<double>(min_p) * kOne), kOne)) : 0ull;

  // Kept weights: each warp owns a contiguous run of the slice.
  const int run = ((slice + kWarps - 1) / kWarps + 31) & ~31;
  const int w0 = min(warp * run, n), w1 = min(w0 + run, n);
  auto kept_weight = [&](int i) -> u64 {
    const uint32_t k = keys[i];
    if (composite(k, first + i) < cut) return 0ull;
    const u64 w = weight(k, P.row, S.table);
    return w >= least ? w : 0ull;
  };
  u64 sum = 0;
  for (int i = w0 + lane; i < w1; i += 32) sum += kept_weight(i);
  for (int m = 16; m; m >>= 1) sum += shfl_xor64(sum, m);
  __syncthreads();
  if (lane == 0) S.warp_b[warp] = sum;
  __syncthreads();
  u64 mine = 0, before_warp = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before_warp += S.warp_b[w];
    mine += S.warp_b[w];
  }
  cl.sync();
  if (tid < C) cl.map_shared_rank(S.slot_a, tid)[me] = mine;
  cl.sync();  // the last remote access
  u64 all = 0, before = 0;
  for (int r = 0; r < C; ++r) {
    if (r < me) before += S.slot_a[r];
    all += S.slot_a[r];
  }
  float u = a.u[b];
  u = u > 0.0f ? u : 0.0f;
  u64 goal = static_cast<u64>(fmin(static_cast<double>(u), 1.0) * static_cast<double>(all));
  if (goal >= all) goal = all - 1;
  before += before_warp;
  if (goal < before || goal - before >= sum) return;
  goal -= before;  // the first token whose running sum exceeds it
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane;
    const u64 w = i < w1 ? kept_weight(i) : 0ull;
    u64 s = w;
    for (int d = 1; d < 32; d <<= 1) {
      const u64 o = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d) s += o;
    }
    const unsigned hit = __ballot_sync(0xFFFFFFFFu, s > goal);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.token[b] = first + i;
        if (a.logprob) a.logprob[b] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(all)));
      }
      return;
    }
    goal -= __shfl_sync(0xFFFFFFFFu, s, 31);
  }
}

template <typename T>
status_t launch_sample(const yb_sample_args& a, cudaStream_t s) {
  // Cluster size: slices of at most kMaxSlice tokens.
  int C = 1;
  while (C < kMaxCluster && (a.V + C - 1) / C > 4096) C *= 2;
  const int slice = ((a.V + C - 1) / C + 31) & ~31;
  const size_t smem = sizeof(SampleSmem) + static_cast<size_t>(slice) * 4;
  static std::atomic<uint64_t> done{0};
  cudaError_t e =
      smem_attr_once(sample_kernel<T>, static_cast<int>(sizeof(SampleSmem) + (kMaxSlice + 32) * 4), done);
  if (e != cudaSuccess) return cuda_status(e, "sample attributes");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.B) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, slice), "sample");
}

}  // namespace
}  // namespace yb

using namespace yb;

extern "C" status_t yb_sample(const yb_sample_args* a, void* stream) {
  if (!a) return ERROR_NULL_POINTER;
  if (a->B < 0 || a->V < 1 || a->V > YB_SAMPLE_MAX_VOCAB || a->B > (1 << 27)) {
    set_error("sample: B in [0, 2^27], V in [1, " + std::to_string(YB_SAMPLE_MAX_VOCAB) + "]");
    return ERROR_INVALID_DIMS;
  }
  if (a->row_stride < 0 || a->dtype < YB_F32 || a->dtype > YB_BF16) {
    set_error("sample: non-negative row stride, dtype YB_F32, YB_F16 or YB_BF16");
    return ERROR_INVALID_DIMS;
  }
  if (a->B == 0) return SUCCESS;
  if (!a->logits || !a->u || !a->token) return ERROR_NULL_POINTER;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case YB_F32: return launch_sample<float>(*a, s);
    case YB_F16: return launch_sample<__half>(*a, s);
    default: return launch_sample<__nv_bfloat16>(*a, s);
  }
}
