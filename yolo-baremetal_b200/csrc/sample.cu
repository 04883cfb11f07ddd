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
// memory, so the logits are read once.
//   1 the row's largest (logit, lowest index);
//   2 with top-k or top-p: a histogram over 1/16-octave steps of the weight
//     below the maximum, summed over the cluster: counts alone (fp32) for
//     top-k, weights as well for top-p; it names the step that holds the
//     border;
//   3a at most kList tokens down to that step (the usual case): all go to CTA 0,
//     which ranks them and finishes the row;
//   3b else the step that holds the border is split further by composites
//     (order-preserving key, ~index), which are all distinct, so ties need no
//     rule of their own, until kList of them are left to rank; what stays
//     above the cut is summed per warp and CTA, and the run of the warp that
//     holds the goal is scanned.
//
// Measured: one row of 32,000 fp32 logits with top-k 50 and top-p 0.95 10.8 us
// in the kernel, of which the cluster's four barriers and the exchange of the
// histogram are about half: latency.  256 unfiltered rows of 131,072 fp32
// logits 87 us (1.5 TB/s): about 50 instructions and 14 fp64 operations a
// token, half of the issue slots; the rest are the barriers between the load,
// the maximum and the sums, with three CTAs an SM to fill them.
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
constexpr int kLive = 46 * 16;  // steps from here on weigh less than 2^-45: never chosen
constexpr int kList = 512;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = YB_SAMPLE_MAX_VOCAB / kMaxCluster;
constexpr int kCopies = 8;  // of the table: few of a warp's look-ups share a bank
constexpr double kOne = 17592186044416.0;  // 2^44

using u64 = unsigned long long;

struct alignas(16) SampleSmem {
  double table[64 * kCopies];  // 2^(j / 64)
  u64 warp_a[kWarps], warp_b[kWarps];
  u64 slot_a[kMaxCluster], slot_b[kMaxCluster], slot_best[kMaxCluster], slot_sum[kMaxCluster];
};
struct alignas(16) FilterSmem {
  u64 tmass[kBins];  // cluster totals
  uint32_t tcnt[kBins];
  uint32_t cnt[kBins];      // own slice; the weights' sums in three 15-bit parts
  uint32_t part[3][kBins];  // (2^15 tokens of a slice: 30 bits each)
  union {
    struct {  // totalling: each CTA's sums of this CTA's share of the bins
      u64 mass[kBins];
      uint32_t cnt[kBins];
    } in;
    struct {  // ranking; in CTA 0 `list` takes the tokens of all
      u64 list[kList];
      u64 own[kList];
    } l;
  };
  u64 result[2];
  u64 rank_sum[2];
  int found, n_own, base, n_list;
};

// NaN, -infinity: -infinity, which is never chosen; +infinity: the largest float.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
__device__ __forceinline__ u64 composite(float x, uint32_t idx) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
  const uint32_t k = b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  return (static_cast<u64>(k) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float value_of(u64 c) {
  const uint32_t k = static_cast<uint32_t>(c >> 32);
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

struct Row {
  double best = 0, c = 0;  // largest logit, log2(e) / T
  float bestf = 0, cf = 0;
  float floor = 0;  // tokens below weigh less than half a unit, none above it is 46 octaves down
};

// rint(2^44 2^y), y = (x - best) log2(e) / T <= 0, as a whole fp64 number; only
// for x >= floor (below, the exponent may wrap: the result is then any number
// and is not used).
// 2^y = 2^n 2^(j/64) 2^r with |r| <= 1/128 (table-driven, after Tang 1989): the
// Taylor polynomial of degree 4 leaves (r ln 2)^5 / 120 < 2^-44.  Rounding to
// whole numbers is done by adding 1.5 2^52 and 2^52: twelve fp64 operations and
// one conversion (they run at a quarter of the fp64 rate), fourteen with the sum.
__device__ __forceinline__ double weight_d(float x, const Row& r, const double* table) {
  const double y = (static_cast<double>(x) - r.best) * r.c;
  const double t = fma(y, 64.0, 6755399441055744.0);
  const int k = __double2loint(t);
  const double q = fma(t - 6755399441055744.0, -0.015625, y);
  double p = fma(q, 9.6181291076284771619e-3, 5.5504108664821579953e-2);  // ln2^4 / 24, ln2^3 / 6
  p = fma(p, q, 0.24022650695910071233);                                  // ln2^2 / 2
  p = fma(p, q, 0.69314718055994530942);
  p = fma(p, q, 1.0);
  p *= table[((k << 3) & (63 * kCopies)) + (threadIdx.x & (kCopies - 1))];  // 2^44 2^(j/64)
  const double v = __hiloint2double(__double2hiint(p) + (k >> 6) * (1 << 20), __double2loint(p));
  return (v + 4503599627370496.0) - 4503599627370496.0;
}
__device__ __forceinline__ u64 weight(float x, const Row& r, const double* table) {
  if (!(x >= r.floor)) return 0ull;
  const double v = weight_d(x, r, table) + 4503599627370496.0;
  return static_cast<u64>(__double_as_longlong(v)) & 0xFFFFFFFFFFFFFull;
}

// Step of 1/16 octave below the maximum: rises as the logit falls.
__device__ __forceinline__ int step_of(float x, const Row& r) {
  const float d = (r.bestf - x) * r.cf;
  return d < static_cast<float>(kLive) ? static_cast<int>(d) : kLive;
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

// The same value in every thread of the cluster.  The slots' earlier readers
// are done once the caller is behind a cluster barrier of its own (`sync`).
template <typename Op>
__device__ u64 cluster_reduce(cg::cluster_group& cl, u64 v, SampleSmem& S, u64* slot, u64 id, Op op, bool sync) {
  const u64 b = block_reduce(v, S.warp_a, id, op);
  const unsigned C = cl.num_blocks(), me = cl.block_rank();
  if (sync) cl.sync();
  if (threadIdx.x < C) cl.map_shared_rank(slot, threadIdx.x)[me] = b;
  cl.sync();
  u64 r = id;
  for (unsigned i = 0; i < C; ++i) r = op(r, slot[i]);
  return r;
}

struct Settings {
  int top_k = 0;
  float top_p = 1.0f, u = 0.f;
  u64 least = 0;  // min-p as a weight
};

__device__ __forceinline__ u64 mass_target(float top_p, u64 mass) {
  // A token is kept while the weight before it is below top_p times the whole.
  return static_cast<u64>(fmax(1.0, ceil(static_cast<double>(top_p) * static_cast<double>(mass))));
}
__device__ __forceinline__ u64 goal_of(float u, u64 all) {
  const u64 g = static_cast<u64>(fmin(static_cast<double>(u), 1.0) * static_cast<double>(all));
  return g < all ? g : all - 1;
}
// Token of logit x.  Its log-probability comes from the logit: a weight of few
// units of 2^-44 knows it to a few bits only.
__device__ __forceinline__ void answer(const yb_sample_args& a, int b, uint32_t token, float x, const Row& r, u64 all) {
  a.token[b] = static_cast<int>(token);
  if (a.logprob)
    a.logprob[b] = static_cast<float>((static_cast<double>(x) - r.best) * r.c * 0.69314718055994530942 -
                                      log(static_cast<double>(all) / kOne));
}

// Bins 2 t and 2 t + 1 of thread t: what lies before each, and the sums of all.
struct Bins {
  u64 c[3], m[3];  // counts and weights before bin 2 t, before 2 t + 1, after it
  u64 all_c, all_m;
};

struct Picker {
  cg::cluster_group& cl;
  SampleSmem& S;
  FilterSmem& F;
  const float* x;
  int n;          // tokens of the slice
  uint32_t base;  // index of its first
  Row row;

  __device__ void clear(bool with_mass) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      F.cnt[b] = 0;
      if (with_mass) F.part[0][b] = F.part[1][b] = F.part[2][b] = 0;
    }
    __syncthreads();
  }
  // Adds one token to bin b of the own histogram.
  __device__ void add(int b, u64 w, bool with_mass) {
    atomicAdd(&F.cnt[b], 1u);
    if (with_mass) {
      const uint32_t p0 = w & 0x7FFFu, p1 = (w >> 15) & 0x7FFFu, p2 = static_cast<uint32_t>(w >> 30);
      if (p0) atomicAdd(&F.part[0][b], p0);
      if (p1) atomicAdd(&F.part[1][b], p1);
      if (p2) atomicAdd(&F.part[2][b], p2);
    }
  }
  __device__ Bins steps(bool with_mass) {
    clear(with_mass);
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      const int b = step_of(v, row);
      if (b < kLive) add(b, with_mass ? weight(v, row, S.table) : 0ull, with_mass);
    }
    return total(with_mass);
  }
  // Cluster totals of the histogram into tcnt, tmass of every CTA: each CTA
  // sends the bins of another's share there, sums its own share and sends the
  // sums to all (remote stores, which nobody waits for one by one).
  __device__ Bins total(bool with_mass) {
    const int C = static_cast<int>(cl.num_blocks()), me = static_cast<int>(cl.block_rank()), t = threadIdx.x;
    const int share = kBins / C;
    __syncthreads();
    for (int b = t; b < kBins; b += kThreads) {
      FilterSmem* o = cl.map_shared_rank(&F, b / share);
      const int at = me * share + (b & (share - 1));
      o->in.cnt[at] = F.cnt[b];
      if (with_mass)
        o->in.mass[at] = F.part[0][b] + (static_cast<u64>(F.part[1][b]) << 15) + (static_cast<u64>(F.part[2][b]) << 30);
    }
    cl.sync();
    const int group = max(1, kThreads / share);  // threads that share a bin and split the receivers
    for (int i = t & (share - 1); i < share; i += kThreads) {
      uint32_t c = 0;
      u64 m = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < C) {
          c += F.in.cnt[r * share + i];
          if (with_mass) m += F.in.mass[r * share + i];
        }
      for (int r = t / share; r < C; r += group) {
        FilterSmem* o = cl.map_shared_rank(&F, r);
        o->tcnt[me * share + i] = c;
        if (with_mass) o->tmass[me * share + i] = m;
      }
    }
    cl.sync();
    // Running sums.
    const int lane = t & 31, w = t >> 5;
    const u64 c0 = F.tcnt[2 * t], c1 = F.tcnt[2 * t + 1];
    const u64 m0 = with_mass ? F.tmass[2 * t] : 0, m1 = with_mass ? F.tmass[2 * t + 1] : 0;
    u64 sc = c0 + c1, sm = m0 + m1;
    for (int d = 1; d < 32; d <<= 1) {
      const u64 a = __shfl_up_sync(0xFFFFFFFFu, sc, d), b = __shfl_up_sync(0xFFFFFFFFu, sm, d);
      if (lane >= d) sc += a, sm += b;
    }
    if (lane == 31) S.warp_a[w] = sc, S.warp_b[w] = sm;
    __syncthreads();
    Bins r;
    r.all_c = r.all_m = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const u64 a = S.warp_a[i], b = S.warp_b[i];
      if (i < w) sc += a, sm += b;
      r.all_c += a;
      r.all_m += b;
    }
    r.c[0] = sc - c0 - c1, r.c[1] = sc - c1, r.c[2] = sc;
    r.m[0] = sm - m0 - m1, r.m[1] = sm - m1, r.m[2] = sm;
    return r;
  }
  // First bin in which the running sum (of weight when by_mass, else of counts)
  // reaches `target` (at most the whole), with the sums before it.
  __device__ int border(const Bins& r, u64 target, bool by_mass, u64* before_cnt, u64* before_mass) {
    const int t = threadIdx.x;
    if (t == 0) F.found = kBins - 1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if ((by_mass ? r.m[i] : r.c[i]) < target && target <= (by_mass ? r.m[i + 1] : r.c[i + 1])) {
        F.found = 2 * t + i;
        F.result[0] = r.c[i];
        F.result[1] = r.m[i];
      }
    __syncthreads();
    *before_cnt = F.result[0];
    *before_mass = F.result[1];
    return F.found;
  }

  // The tokens of steps [first, last] with composites in [lo, hi] to CTA 0's
  // list, in any order; at most kList by the histogram's count.  n_own and CTA
  // 0's n_list are zero.
  __device__ void gather(int first, int last, u64 lo, u64 hi) {
    FilterSmem* head = cl.map_shared_rank(&F, 0);
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      const int st = step_of(v, row);
      if (st < first || st > last) continue;
      const u64 c = composite(v, base + i);
      if (c < lo || c > hi) continue;
      const int at = atomicAdd(&F.n_own, 1);
      if (at < kList) F.l.own[at] = c;
    }
    __syncthreads();
    const int m = min(F.n_own, kList);
    if (threadIdx.x == 0) F.base = m ? atomicAdd(&head->n_list, m) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kThreads)
      if (F.base + i < kList) head->l.list[F.base + i] = F.l.own[i];
    cl.sync();
  }

  // Sorts the values of the first m threads, all distinct and above 0, falling;
  // the others get 0.  Up to 128 of them by counting, four threads a value (0.6
  // us for 60 values, the network below 1.4); more by a bitonic network (2.7 us
  // for 250, counting 4).
  __device__ u64 sort(u64 v, int m) {
    const int t = threadIdx.x;
    if (m <= kThreads / 4) {
      __syncthreads();
      F.l.own[t] = t < m ? v : 0ull;
      __syncthreads();
      const u64 mine = F.l.own[t >> 2];
      int rank = 0;
#pragma unroll 4
      for (int j = t & 3; j < m; j += 4) rank += F.l.own[j] > mine;
      rank += __shfl_xor_sync(0xFFFFFFFFu, rank, 1);
      rank += __shfl_xor_sync(0xFFFFFFFFu, rank, 2);
      __syncthreads();
      if ((t & 3) == 0 && (t >> 2) < m) F.l.own[rank] = mine;
      __syncthreads();
      return t < m ? F.l.own[t] : 0ull;
    }
    const int size = 1 << (32 - __clz(m - 1));
    if (t >= m) v = 0ull;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j; j >>= 1) {
        u64 o;
        if (j < 32) {
          o = shfl_xor64(v, j);
        } else {
          __syncthreads();
          F.l.own[t] = v;
          __syncthreads();
          o = F.l.own[t ^ j];
        }
        const bool up = (t & k) != 0, low = (t & j) == 0;  // falling runs where !up
        v = (low != up) == (v > o) ? v : o;
      }
    return v;
  }
  // Running sum over the block's threads, this one included.
  __device__ u64 scan(u64 v) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int d = 1; d < 32; d <<= 1) {
      const u64 o = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) S.warp_a[w] = v;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i)
      if (i < w) v += S.warp_a[i];
    return v;
  }
  // CTA 0: its list in falling order, one token a thread, with their weights
  // and running sums; returns the list's length.
  __device__ int ranked(u64* c, u64* w, u64* sum) {
    const int m = min(F.n_list, kList), t = threadIdx.x;
    *c = sort(t < m ? F.l.list[t] : 0ull, m);
    *w = t < m ? weight(value_of(*c), row, S.table) : 0ull;
    *sum = scan(*w);
    return m;
  }

  // The lowest composite kept when the tokens are taken in falling order while
  // fewer than `target` of them (by_mass: of their weight) came before; `step`
  // holds the border, bc and bm are the sums before it.  *kept_mass: the
  // weight down to the cut (with_mass).
  __device__ u64 cut(int step, u64 bc, u64 bm, u64 target, bool by_mass, bool with_mass, u64* kept_mass) {
    uint32_t inside = F.tcnt[step];
    u64 lo = 0, hi = ~0ull;  // composites that are still candidates
    while (inside > kList) {
      u64 mn = ~0ull, mx = 0;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 c = composite(x[i], base + i);
        if (step_of(x[i], row) == step && c >= lo && c <= hi) {
          mn = c < mn ? c : mn;
          mx = c > mx ? c : mx;
        }
      }
      mn = cluster_reduce(cl, mn, S, S.slot_a, ~0ull, MinOp(), true);
      mx = cluster_reduce(cl, mx, S, S.slot_b, 0ull, MaxOp(), true);
      int shift = 0;  // at least half of the bins span [mn, mx]
      while (((mx - mn) >> shift) >= kBins) ++shift;
      clear(with_mass);
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 c = composite(x[i], base + i);
        if (step_of(x[i], row) == step && c >= mn && c <= mx)
          add(static_cast<int>((mx - c) >> shift), with_mass ? weight(x[i], row, S.table) : 0ull, with_mass);
      }
      const Bins r = total(with_mass);
      u64 c2, m2;
      const int b = border(r, target - (by_mass ? bm : bc), by_mass, &c2, &m2);
      bc += c2;
      bm += m2;
      inside = F.tcnt[b];
      hi = mx - (static_cast<u64>(b) << shift);
      const u64 span = (1ull << shift) - 1;
      lo = hi - mn > span ? hi - span : mn;
    }
    gather(step, step, lo, hi);
    if (cl.block_rank() == 0) {
      u64 c, w, sum;
      const int m = ranked(&c, &w, &sum), t = threadIdx.x;
      const bool keep = t < m && (by_mass ? bm + sum - w : bc + t) < target;
      const int last = __syncthreads_count(keep) - 1;
      if (t == last) F.rank_sum[0] = c, F.rank_sum[1] = bm + sum;
      if (t == 0) F.n_list = 0;
      __syncthreads();
      if (t < static_cast<int>(cl.num_blocks())) {
        cl.map_shared_rank(S.slot_a, t)[0] = F.rank_sum[0];
        cl.map_shared_rank(S.slot_b, t)[0] = F.rank_sum[1];
      }
    }
    if (threadIdx.x == 0) F.n_own = 0;
    cl.sync();
    *kept_mass = S.slot_b[0];
    return S.slot_a[0];
  }

  // CTA 0: the row from its list, which holds every token down to some step.
  // mass: the whole weight, when there is no top_k.  What the filters keep is
  // the beginning of the falling order.
  __device__ void finish(const yb_sample_args& a, int b, const Settings& s, u64 mass) {
    u64 c, w, sum;
    const int m = ranked(&c, &w, &sum), t = threadIdx.x;
    if (s.top_k > 0) {
      if (t == s.top_k - 1) F.rank_sum[0] = sum;
      __syncthreads();
      mass = F.rank_sum[0];
    }
    const bool keep = t < m && (s.top_k <= 0 || t < s.top_k) &&
                      (!(s.top_p < 1.0f) || sum - w < mass_target(s.top_p, mass)) && w >= s.least;
    const int kept = __syncthreads_count(keep);
    if (t == kept - 1) F.rank_sum[1] = sum;
    // By rising index: the composite's low half is ~index.
    F.l.list[t] = w;
    F.cnt[t] = __float_as_uint(value_of(c));
    const u64 by_index = sort(t < kept ? (c << 32) | static_cast<uint32_t>(t) : 0ull, kept);
    __syncthreads();
    const u64 all = F.rank_sum[1];
    const u64 wi = t < kept ? F.l.list[static_cast<uint32_t>(by_index)] : 0ull;
    const u64 upto = scan(wi);
    const u64 goal = goal_of(s.u, all);
    if (t < kept && upto > goal && upto - wi <= goal)
      answer(a, b, 0xFFFFFFFFu - static_cast<uint32_t>(by_index >> 32),
             __uint_as_float(F.cnt[static_cast<uint32_t>(by_index)]), row, all);
  }
};

// The slice into shared memory, 16 bytes a load; returns the thread's largest logit.
template <typename T>
__device__ __forceinline__ float load_slice(const T* g, float* x, int n, int head) {
  constexpr int V = 16 / sizeof(T);
  float top = -INFINITY;
  const int vecs = (n - head) / V, tail = head + vecs * V, tid = threadIdx.x;
  if (tid < head) {
    top = clean(to_f(g[tid]));
    x[tid] = top;
  }
  if (tail + tid < n) {
    const float v = clean(to_f(g[tail + tid]));
    x[tail + tid] = v;
    top = fmaxf(top, v);
  }
  constexpr int U = 4;
  const uint4* src = reinterpret_cast<const uint4*>(g + head);
  for (int k0 = tid; k0 < vecs; k0 += U * kThreads) {
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u * kThreads < vecs) r[u] = __ldcs(src + k0 + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * kThreads;
      if (k >= vecs) break;
      const T* e = reinterpret_cast<const T*>(&r[u]);
      float f[V];
#pragma unroll
      for (int d = 0; d < V; ++d) {
        f[d] = clean(to_f(e[d]));
        top = fmaxf(top, f[d]);
      }
#pragma unroll
      for (int d = 0; d < V; d += 4)
        *reinterpret_cast<float4*>(x + head + k * V + d) = make_float4(f[d], f[d + 1], f[d + 2], f[d + 3]);
    }
  }
  return top;
}

template <typename T, bool FILTER>
__global__ void __launch_bounds__(kThreads, FILTER ? 2 : 3) sample_kernel(const yb_sample_args a, int slice) {
  extern __shared__ __align__(16) uint8_t sample_raw[];
  SampleSmem& S = *reinterpret_cast<SampleSmem*>(sample_raw);
  FilterSmem& F = *reinterpret_cast<FilterSmem*>(sample_raw + sizeof(SampleSmem));
  cg::cluster_group cl = cg::this_cluster();
  cl.barrier_arrive();  // remote shared memory may be written once all CTAs are up
  const int C = static_cast<int>(cl.num_blocks()), me = static_cast<int>(cl.block_rank());
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = min(me * slice, a.V);
  const int n = min(slice, a.V - first);
  const T* g = static_cast<const T*>(a.logits) + static_cast<long long>(b) * a.row_stride + first;
  // Elements before the first 16-byte boundary; shared memory is shifted so
  // that it has its boundary at the same element.
  const int head = min(n, static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(g) & 15u)) & 15u) / sizeof(T)));
  const int pad = (4 - (head & 3)) & 3;
  float* raw = reinterpret_cast<float*>(sample_raw + sizeof(SampleSmem) + (FILTER ? sizeof(FilterSmem) : 0));
  float* x = raw + pad;
  // Each warp sums a run of whole 32-token steps; what lies outside the slice
  // holds -infinity.
  const int run = (n + pad + kThreads - 1) / kThreads * 32;

  const float temp = a.temperature ? a.temperature[b] : 1.0f;
  const float top = load_slice(g, x, n, head);
  if (FILTER && tid == 0) F.n_own = F.n_list = 0;
  if (tid < pad) raw[tid] = -INFINITY;
  for (int i = pad + n + tid; i < kWarps * run; i += kThreads) raw[i] = -INFINITY;
  if (tid < 64) {
    const double e = kOne * exp2(tid / 64.0);
    for (int i = 0; i < kCopies; ++i) S.table[tid * kCopies + i] = e;
  }
  cl.barrier_wait();
  u64 best = cluster_reduce(cl, composite(top, 0xFFFFFFFFu), S, S.slot_best, 0ull, MaxOp(), false);
  const float bestf = value_of(best);
  if (!(bestf > -INFINITY) || !(temp > 0.0f)) {
    // The lowest index of the largest logit.
    uint32_t at = 0xFFFFFFFFu;
    if (bestf > -INFINITY)
      for (int i = n - 1 - tid; i >= 0; i -= kThreads)
        if (x[i] == bestf) at = first + i;
    const u64 low = cluster_reduce(cl, at, S, S.slot_a, ~0ull, MinOp(), false);
    if (me == 0 && tid == 0) {
      a.token[b] = bestf > -INFINITY ? static_cast<int>(low) : -1;
      if (a.logprob) a.logprob[b] = bestf > -INFINITY ? 0.0f : -INFINITY;
    }
    return;  // every CTA of the cluster, after its last remote access
  }
  Row row;
  row.bestf = bestf;
  row.best = bestf;
  row.c = 1.4426950408889634074 / static_cast<double>(temp);
  row.cf = static_cast<float>(fmin(16.0 * row.c, 1e30));
  // 2^44 2^-45.5 < 1/2.  Rounded up to fp32, so that the comparison with an
  // fp32 logit is the exact one, also where one step of fp32 below the maximum
  // is many octaves: weight_d's exponent has room for 1,000.
  row.floor = __double2float_ru(fmax(row.best - 45.5 / row.c, -static_cast<double>(FLT_MAX)));

  Settings s;
  s.u = a.u[b] > 0.0f ? a.u[b] : 0.0f;
  u64 cut = 0;  // lowest composite kept
  if constexpr (FILTER) {
    Picker P{cl, S, F, x, n, static_cast<uint32_t>(first), row};
    const float min_p = a.min_p ? a.min_p[b] : 0.0f;
    s.least = min_p > 0.0f ? static_cast<u64>(fmin(rint(static_cast<double>(min_p) * kOne), kOne)) : 0ull;
    s.top_k = a.top_k ? a.top_k[b] : 0;
    s.top_p = a.top_p ? a.top_p[b] : 1.0f;
    if (s.top_k >= a.V) s.top_k = 0;
    const bool use_p = s.top_p < 1.0f;
    u64 mass = 0, bc, bm;
    bool have_k = false;
    if (s.top_k > 0) {
      Bins r = P.steps(false);
      if (static_cast<u64>(s.top_k) < r.all_c) {  // else the rest is never chosen
        int step = P.border(r, s.top_k, false, &bc, &bm);
        if (bc + F.tcnt[step] <= kList) {
          P.gather(0, step, 0ull, ~0ull);
          if (me == 0) P.finish(a, b, s, 0ull);
          return;
        }
        if (use_p) {
          r = P.steps(true);
          step = P.border(r, s.top_k, false, &bc, &bm);
        }
        cut = P.cut(step, bc, bm, s.top_k, false, use_p, &mass);
        have_k = true;
      }
    }
    if (use_p) {
      const Bins r = P.steps(true);
      if (!have_k) mass = r.all_m;
      const u64 target = mass_target(s.top_p, mass);
      if (target < mass) {
        const int step = P.border(r, target, true, &bc, &bm);
        if (!have_k && bc + F.tcnt[step] <= kList) {
          P.gather(0, step, 0ull, ~0ull);
          s.top_k = 0;
          if (me == 0) P.finish(a, b, s, mass);
          return;
        }
        u64 kept = 0;
        const u64 c = P.cut(step, bc, bm, target, true, true, &kept);
        cut = c > cut ? c : cut;
      }
    }
  }

  // Kept weights of each warp's run, as whole fp64 numbers (at most 2^44 times
  // 65 tokens a lane: exact).
  const float edge = cut ? value_of(cut) : -INFINITY;
  const double least = static_cast<double>(s.least);
  auto kept = [&](int j) -> double {  // of raw[j]
    const float v = raw[j];
    if (FILTER && (v < edge || composite(v, first + j - pad) < cut)) return 0.0;
    const double w = weight_d(v, row, S.table);
    return v >= row.floor && (!FILTER || w >= least) ? w : 0.0;
  };
  double part = 0.0;
#pragma unroll 8
  for (int j = warp * run + lane; j < warp * run + run; j += 32) part += kept(j);
  u64 sum = static_cast<u64>(part);
  for (int m = 16; m; m >>= 1) sum += shfl_xor64(sum, m);
  __syncthreads();
  if (lane == 0) S.warp_b[warp] = sum;
  __syncthreads();
  u64 mine = 0;
  for (int w = 0; w < kWarps; ++w) mine += S.warp_b[w];
  if (tid < C) cl.map_shared_rank(S.slot_sum, tid)[me] = mine;
  cl.sync();  // the last remote access
  u64 all = 0, before = 0;
  for (int r = 0; r < C; ++r) {
    if (r < me) before += S.slot_sum[r];
    all += S.slot_sum[r];
  }
  u64 goal = goal_of(s.u, all);
  if (goal < before || goal - before >= mine) return;  // the whole CTA
  goal -= before;
  int at = 0;  // the run that holds the goal
  while (goal >= S.warp_b[at]) goal -= S.warp_b[at++];
  // Its tokens, a few neighbours a thread: the first whose running sum exceeds the goal.
  const int per = (run + kThreads - 1) / kThreads;
  const int j0 = at * run + min(tid * per, run), j1 = at * run + min(tid * per + per, run);
  u64 own = 0;
  for (int j = j0; j < j1; ++j) own += static_cast<u64>(kept(j));
  u64 upto = own;
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) S.warp_a[warp] = upto;
  __syncthreads();
  for (int v = 0; v < kWarps; ++v)
    if (v < warp) upto += S.warp_a[v];
  if (upto <= goal || upto - own > goal) return;
  u64 run_sum = upto - own;
  for (int j = j0; j < j1; ++j) {
    const u64 w = static_cast<u64>(kept(j));
    run_sum += w;
    if (run_sum > goal) {
      answer(a, b, first + j - pad, raw[j], row, all);
      return;
    }
  }
}

template <typename T, bool FILTER>
status_t launch_sample(const yb_sample_args& a, cudaStream_t s) {
  // Slices of at most 16384 tokens; smaller ones while the CTAs do not fill
  // the 148 SMs twice and each thread still has four tokens.
  int C = 1;
  while (C < kMaxCluster && ((a.V + C - 1) / C > 16384 ||
                             (static_cast<long long>(a.B) * C < 2 * 148 && (a.V + C - 1) / C > 4 * kThreads)))
    C *= 2;
  const int slice = ((a.V + C - 1) / C + 31) & ~31;
  constexpr size_t fixed = sizeof(SampleSmem) + (FILTER ? sizeof(FilterSmem) : 0);
  // Up to 3 elements of padding, then whole steps for every warp.
  const auto room = [](int n) { return static_cast<size_t>((n + 3 + kThreads - 1) / kThreads * kThreads) * sizeof(float); };
  static std::atomic<uint64_t> done{0};
  cudaError_t e =
      smem_attr_once(sample_kernel<T, FILTER>, static_cast<int>(fixed + room(kMaxSlice)), done);
  if (e != cudaSuccess) return cuda_status(e, "sample attributes");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.B) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = fixed + room(slice);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, sample_kernel<T, FILTER>, a, slice), "sample");
}

template <typename T>
status_t launch_sample(const yb_sample_args& a, cudaStream_t s) {
  return a.top_k || a.top_p || a.min_p ? launch_sample<T, true>(a, s) : launch_sample<T, false>(a, s);
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
  if (!on_boundary(a->dtype == YB_F32 ? 4 : 2, a->logits) ||
      !on_boundary(4, a->u, a->temperature, a->top_k, a->top_p, a->min_p, a->token, a->logprob)) {
    set_error("sample: a pointer is not aligned to its element");
    return ERROR_INVALID_DIMS;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case YB_F32: return launch_sample<float>(*a, s);
    case YB_F16: return launch_sample<__half>(*a, s);
    default: return launch_sample<__nv_bfloat16>(*a, s);
  }
}
