// Attention over a prompt or a cache (yb_lm.h, yb_attn_run) on the tensor
// cores: S = Q K^T and O += P V as tcgen05.mma kind::f16 (fp16 or bf16
// operands, fp32 accumulation in tensor memory), one pass over the keys with a
// running maximum and sum.
//
// Rows.  A tile is 128 rows: np positions times the gp query heads that share
// a key head, so a key block is read once for all of them, and a step of one
// token still fills gp rows.  Every mask of the operator leaves a row one run
// of keys [lo, hi), so a thread, which owns one row, masks with two compares,
// and only in blocks that some row of its warp does not see whole.
//
// CTA (12 warps): warps 0-3 and 4-7 are two softmax pipelines, warp 8 issues
// the UMMAs (one warp for both in turn: with one each the pipelines fell into
// step and waited for the tensor cores together, 172 -> 191 us), warp 9 the TMA
// loads into a ring of 128-key blocks of K and V.
// Tensor memory: two S buffers of 64 columns a pipeline (half a key block each;
// P overwrites the first half of its S as packed 16-bit pairs and is read back
// as the A operand), O0, O1.  While the softmax works on one buffer the tensor
// cores fill the other; with one buffer of 128 columns a pipeline waited 1,400
// clocks of 3,900 a block at D = 128 for its product and next scores.
//   row mode    the pipelines own two row tiles and share each K and V block;
//   split mode  the pipelines take the even and odd blocks of one row tile, and
//               the blocks of all tiles are dealt out evenly to a grid of one
//               CTA per SM (by the lengths on the device), so a few rows over
//               a long cache still use the whole memory bandwidth.  A tile cut
//               between CTAs leaves (max, sum, O) in scratch, and
//               attn_join_kernel joins the pieces in their order.
//
// Blocks and their halves go from the last keys to the first: with a distance
// bias the nearest, heaviest keys then set the maximum that serves the rest
// (first to last, every half block raised it: 8,191 packed rows with slopes 87
// -> 69 us).  The running maximum is only raised when weights outgrow their
// range (then O is rescaled in place): until then larger weights are as exact,
// and O stays untouched in tensor memory.  The maximum in use never enters the
// result.
//
// A weight of zero times an infinite or NaN value would be NaN, so value rows
// of a block that no row of the tile sees are zeroed in shared memory, and a
// row whose O comes out non-finite under a finite sum (a value that only other
// rows see) is computed again over the keys it does see, which are loaded anew.
//
// Rounding: P is rounded to the operands' type (they enter the same UMMA); its
// sum is taken before that in fp32.  O, maxima and sums are fp32 throughout.
// Against 64 bits the error is up to 1.4 times that of fp32 weights rounded once
// at the end (2 x 4,096 capped rows 0.0022 against 0.0016, one fp16 token over
// 401 keys 0.00028 against 0.00021).
//
// What bounds it.  D = 128: a block pair (256 rows, 128 keys) takes 2,048 clocks
// of tensor work (4,096 multiply-adds a clock) and 2,048 of exponentials (16 a
// clock), which overlap in part, and the scores of 64 keys, whose Q is read
// from shared memory again for each half, take 384 clocks instead of 256: 2 x
// 4,096 capped causal rows of 16 heads 154 to 178 us (0.89 to 0.77 PFLOP/s; the
// longer the more work runs around them).  D = 64: the
// exponentials (about 10 clocks a warp's 32 instead of 8 in practice).  Short
// tiles (documents, a few blocks each): 2 us of start-up and 2 us of output a
// CTA, which nothing overlaps with one CTA per SM.  Split mode: 24 sequences of
// up to 16,384 keys 198 us, 4.2 TB/s, 0.64 of the measured copy rate; the UMMA
// warp's waits and products of 128 rows (4 of them in use) stand between ring
// and memory.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cmath>
#include <mutex>

#include "attn_lm.h"
#include "attn_row.cuh"
#include "pdl.cuh"
#include "sm100.cuh"
#include "split.cuh"

namespace yb {
namespace {

constexpr int kB = kAttnBlock;
constexpr int kH = kB / 2;  // keys of a half block: one S buffer
constexpr int kThreads = 384;
constexpr int kMmaWarp = 8, kLoadWarp = 9;  // 10 and 11 only fill up the warpgroup
// Registers a thread: 384 x 168 at launch, then 256 x 200 + 128 x 104 of them.
constexpr int kSoftmaxRegs = 200, kOtherRegs = 104;
constexpr uint32_t kChunkBytes = kB * 128;  // 128 rows x 64 elements, 128-byte swizzle
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.44269504f;
// A row's weights are 2^(s - m), m its reference: its maximum when that was set,
// for fp16 less 8, so that the largest weights are 2^8 and what falls below the
// type's normal numbers is 2^-22 of them instead of 2^-14.
template <typename T>
constexpr float kHead = std::is_same<T, __half>::value ? 8.0f : 0.0f;
// log2 of a weight up to which a searched maximum leaves the reference alone.
constexpr float kRaise = 15.0f;
// Room for the sum of a tile's pieces, at most two a CTA.
constexpr float kJoinRoom = 8.0f;
// Sum of a half block up to which the reference at hand serves it: fp16 weights
// end at 65504; bf16 ones may be 2^50 above it.  Between references 88 octaves
// apart a join's factor falls out of fp32 (126 less kRoom and kJoinRoom), and
// what it drops is then below 2^-38 a half block.
template <typename T>
constexpr float kFits = std::is_same<T, __half>::value ? 32768.0f : 1.1258999e15f;
constexpr int kSmemMax = 232448;
constexpr int kCtlBytes = 3 * 1024;  // control block, after up to 1 KB of alignment

template <int HDP>
__host__ __device__ constexpr int chunks() { return HDP / 64; }
template <int HDP, bool SPLIT>
__host__ __device__ constexpr int q_bytes() { return (SPLIT ? 1 : 2) * chunks<HDP>() * static_cast<int>(kChunkBytes); }
template <int HDP, bool SPLIT>
__host__ __device__ constexpr int stages() {
  const int n = (kSmemMax - kCtlBytes - q_bytes<HDP, SPLIT>()) / (chunks<HDP>() * static_cast<int>(kChunkBytes));
  return n > 8 ? 8 : n;
}
template <int HDP, bool SPLIT>
__host__ __device__ constexpr int smem_bytes() {
  return q_bytes<HDP, SPLIT>() + stages<HDP, SPLIT>() * chunks<HDP>() * static_cast<int>(kChunkBytes) + kCtlBytes;
}

struct Ctl {
  uint64_t q_full, s_full[2][2], p_full[2][2], o_full[2][2], o_empty, ml_full, drain;
  uint64_t kv_full[8], kv_empty[8];
  uint32_t tmem;
  int abort;
  float2 ml[kB];  // split: second pipeline's maximum and sum
};
static_assert(sizeof(Ctl) + 1024 <= kCtlBytes, "control block plus alignment");

// ------------------------------------------------------------- PTX pieces
// A value that all lanes share, marked as such: what is computed from it can
// stay in uniform registers, where the UMMA's operands have to be.
__device__ __forceinline__ int uni(int x) { return __shfl_sync(0xFFFFFFFFu, x, 0); }
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  tc_mma_bf16(d, ad, bd, idesc, acc);  // kind::f16; the types are in idesc
}
// A from tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void ld32(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr)
      : "memory");
}
// Orders later uses of loaded registers behind the wait for the loads.
__device__ __forceinline__ void ld32_dep(float* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile(""
                 : "+f"(r[i]), "+f"(r[i + 1]), "+f"(r[i + 2]), "+f"(r[i + 3]), "+f"(r[i + 4]), "+f"(r[i + 5]),
                   "+f"(r[i + 6]), "+f"(r[i + 7])
                 :
                 : "memory");
}
// V block as the B operand [keys (K)][dims (N)]: N-major, 128-byte swizzle.
// 64 dims are one 128-byte row of the tile; the next 64 lie a chunk further
// (leading offset), the next 8 keys 1024 bytes further (stride offset).
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kChunkBytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}
// fp32 accumulator, both operands bf16 or both fp16, B N-major when `bn`.
template <typename T>
__device__ __forceinline__ uint32_t idesc_f32(int N, bool bn) {
  constexpr uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (bn ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(kB >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Largest (smallest) of a half block's scores; NaN is passed over.
__device__ __forceinline__ float max_of(const float* s) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = max3(s[i], s[i + 4], s[i + 8]);
#pragma unroll
  for (int e = 12; e + 8 <= kH; e += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max3(m[i], s[e + i], s[e + 4 + i]);
  m[0] = max3(m[0], s[kH - 4], s[kH - 3]);
  m[1] = max3(m[1], s[kH - 2], s[kH - 1]);
  return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}
__device__ __forceinline__ float min_of(const float* s) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = min3(s[i], s[i + 4], s[i + 8]);
#pragma unroll
  for (int e = 12; e + 8 <= kH; e += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = min3(m[i], s[e + i], s[e + 4 + i]);
  m[0] = min3(m[0], s[kH - 4], s[kH - 3]);
  m[1] = min3(m[1], s[kH - 2], s[kH - 1]);
  return fminf(min3(m[0], m[1], m[2]), m[3]);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// ------------------------------------------------------------ work division
// Key blocks of tile qt of sequence b as far as the lengths tell (a document
// range only narrows them); 0 when no row is in use, at least 1 otherwise.
__device__ __forceinline__ int tile_blocks(const AttnPlan& p, int b, int qt) {
  const int q_len = clamp_len(p.a.q_len, b, p.a.Sq), k_len = clamp_len(p.a.k_len, b, p.a.Sk);
  const int i0 = qt * p.np;
  if (i0 >= q_len) return 0;
  int hi = k_len;
  if (p.a.causal) {
    hi = min(k_len, k_len - q_len + min(i0 + p.np, q_len));
    if (p.a.prefix) hi = max(hi, min(p.a.prefix[b], k_len));
  }
  return max(1, (hi + kB - 1) / kB);
}

struct Piece {
  int b = 0, hg = 0, qt = 0;
  int off = 0, take = 0;  // key blocks [off, off + take) of `n`
  int n = 0;
  int slot = -1;  // scratch slot, -1: the whole tile
};

// A CTA's share of the blocks of all tiles, in the order (sequence, tile, head
// group).  Every warp walks it by itself, lanes together.
struct Walk {
  long long total = 0, left = 0;
  int bt = 0, hg = 0, off = 0, ctas = 1;

  // Blocks of all (sequence, tile) pairs per lane, then the lane and pair that hold unit u.
  __device__ void seek(const AttnPlan& p, int cta, int grid) {
    const int lane = threadIdx.x & 31;
    const int pairs = p.a.B * p.tiles;
    if (p.whole) {  // tiles are dealt out whole
      const long long segs = static_cast<long long>(pairs) * p.groups;
      const long long s0 = segs * cta / grid, s1 = segs * (cta + 1) / grid;
      bt = static_cast<int>(s0 / p.groups);
      hg = static_cast<int>(s0 - static_cast<long long>(bt) * p.groups);
      left = s1 - s0;
      return;
    }
    const int per = (pairs + 31) / 32;
    const int x0 = min(lane * per, pairs), x1 = min(x0 + per, pairs);
    long long sum = 0;
    for (int x = x0; x < x1; ++x) sum += tile_blocks(p, x / p.tiles, x % p.tiles);
    sum *= p.groups;
    long long scan = sum;
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xFFFFFFFFu, scan, d);
      if (lane >= d) scan += o;
    }
    total = __shfl_sync(0xFFFFFFFFu, scan, 31);
    const long long want = (total + p.unit_min - 1) / p.unit_min;
    ctas = static_cast<int>(want < 1 ? 1 : want < grid ? want : grid);
    if (cta >= ctas) return;
    const long long u0 = total * cta / ctas, u1 = total * (cta + 1) / ctas;
    left = u1 - u0;
    if (left <= 0) return;
    const unsigned has = __ballot_sync(0xFFFFFFFFu, scan > u0);
    const int who = __ffs(has) - 1;
    long long rest = u0 - (scan - sum);  // of lane `who`
    int at = x0, h = 0, o = 0;
    if (lane == who) {
      for (; at < x1; ++at) {
        const long long n = static_cast<long long>(tile_blocks(p, at / p.tiles, at % p.tiles));
        if (rest < n * p.groups) {
          h = static_cast<int>(rest / n);
          o = static_cast<int>(rest - h * n);
          break;
        }
        rest -= n * p.groups;
      }
    }
    bt = __shfl_sync(0xFFFFFFFFu, at, who);
    hg = __shfl_sync(0xFFFFFFFFu, h, who);
    off = __shfl_sync(0xFFFFFFFFu, o, who);
  }

  __device__ bool next(const AttnPlan& p, Piece* s) {
    while (left > 0 && bt < p.a.B * p.tiles) {
      s->b = bt / p.tiles;
      s->qt = bt - s->b * p.tiles;
      s->n = tile_blocks(p, s->b, s->qt);
      if (s->n == 0) {
        if (p.whole) {
          left -= p.groups - hg;
        }
        ++bt;
        hg = 0;
        continue;
      }
      s->hg = hg;
      s->off = off;
      s->take = p.whole ? s->n : static_cast<int>(min(static_cast<long long>(s->n - off), left));
      s->slot = s->take == s->n ? -1 : s->off ? 0 : 1;
      left -= p.whole ? 1 : s->take;
      off += s->take;
      if (off >= s->n) {
        off = 0;
        if (++hg == p.groups) hg = 0, ++bt;
      }
      return true;
    }
    return false;
  }
};

// Keys that some row of the tile sees: [lo, hi), by a whole warp.
struct Keys {
  int lo, hi;
};
__device__ __forceinline__ Keys tile_keys(const AttnPlan& p, int b, int qt) {
  const int q_len = clamp_len(p.a.q_len, b, p.a.Sq), k_len = clamp_len(p.a.k_len, b, p.a.Sk);
  const int i0 = qt * p.np, i1 = min(i0 + p.np, q_len);
  Keys k{0, 0};
  if (i0 >= i1) return k;
  if (!p.a.key_range) {
    k.hi = max(0, row_span(p.a, b, i1 - 1, q_len, k_len).hi);
    return k;
  }
  int lo = 0x7FFFFFFF, hi = 0;
  const int prefix = p.a.causal && p.a.prefix ? min(p.a.prefix[b], k_len) : 0;
  const int2* range = reinterpret_cast<const int2*>(p.a.key_range) + static_cast<long long>(b) * p.a.Sq;
  int2 own[kB / 32];  // all rows' loads in flight together
#pragma unroll
  for (int x = 0; x < kB / 32; ++x) own[x] = range[min(i0 + 32 * x + static_cast<int>(threadIdx.x & 31), i1 - 1)];
#pragma unroll
  for (int x = 0; x < kB / 32; ++x) {
    const int i = min(i0 + 32 * x + static_cast<int>(threadIdx.x & 31), i1 - 1);
    int end = k_len;  // as row_span
    if (p.a.causal) end = max(min(k_len, k_len - q_len + i + 1), prefix);
    const int first = max(0, own[x].x), last = min(end, own[x].y);
    if (first < last) {
      lo = min(lo, first);
      hi = max(hi, last);
    }
  }
  lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  hi = __reduce_max_sync(0xFFFFFFFFu, hi);
  if (lo < hi) k.lo = lo, k.hi = hi;
  return k;
}

// Block range of a CTA's two pipelines.
struct Blocks {
  int j0[2], j1[2];  // row mode: each tile's; split mode: both hold the piece's
  int lo, hi;        // keys outside need not be finite in V
};
template <bool SPLIT>
__device__ __forceinline__ Blocks block_range(const AttnPlan& p, const Piece& s) {
  Blocks r;
  if constexpr (SPLIT) {
    const Keys k = tile_keys(p, s.b, s.qt);
    int a = k.lo / kB, e = (k.hi + kB - 1) / kB;
    a = max(a, s.off);
    e = max(a, min(e, s.off + s.take));
    r.j0[0] = r.j0[1] = a;
    r.j1[0] = r.j1[1] = e;
    r.lo = k.lo;
    r.hi = k.hi;
  } else {
    r.lo = 0x7FFFFFFF;
    r.hi = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Keys k = tile_keys(p, s.b, s.qt + t);
      r.j0[t] = k.lo / kB;
      r.j1[t] = max(r.j0[t], (k.hi + kB - 1) / kB);
      if (k.lo < k.hi) {
        r.lo = min(r.lo, k.lo);
        r.hi = max(r.hi, k.hi);
      }
    }
    if (r.j0[0] == r.j1[0]) r.j0[0] = r.j1[0] = r.j0[1];  // an empty tile takes no part in the union
    if (r.j0[1] == r.j1[1]) r.j0[1] = r.j1[1] = r.j0[0];
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    r.j0[t] = uni(r.j0[t]);
    r.j1[t] = uni(r.j1[t]);
  }
  r.lo = uni(r.lo);
  r.hi = uni(r.hi);
  return r;
}

__device__ __forceinline__ void raise_error(int* err, volatile int* abort_flag, int code) {
  *abort_flag = 1;
  atomicCAS(err, 0, code);
}

// Position in the ring of key and value blocks.
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  template <int N>
  __device__ __forceinline__ void next() {
    if (++slot == N) slot = 0, phase ^= 1u;
  }
};

// ------------------------------------------------------------------ softmax
struct RowState {
  float m = -INFINITY, l = 0.f;  // reference of the weights (log2 units) and their sum
  int lo = 0, hi = 0, pos = 0;
  float slope = 0.f;
  bool valid = false;
};

struct ScoreConst {
  float sc2;             // scale * log2(e); with a cap: scale / cap
  float cap2;            // cap * log2(e)
  float c0, c1, c2, c3;  // cap2 tanh(sc2 s) = s (c0 + c1 s^2 + c2 s^4 + c3 s^6) for |s| <= near
  float near, near2;
  bool forward;  // causal without prefix: no visible key lies behind its row
};

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// tanh(u) / u = 1 + k1 u^2 + k2 u^4 + k3 u^6 on |u| <= kNear, relative error
// 7.0e-8 (1.2 units of 2^-24): least maximum relative error with the first
// coefficient held at 1 (Remez exchange).
constexpr float kNear = 0.375f;
constexpr float kTanh1 = -0.333323335f, kTanh2 = 0.132897262f, kTanh3 = -0.0484872926f;

// c0 + c1 z + c2 z^2 + c3 z^3 with z = s^2, for a pair.
__device__ __forceinline__ float2 cap_poly(float2 z, const ScoreConst& c) {
  const float2 q = __ffma2_rn(__ffma2_rn(both(c.c3), z, both(c.c2)), z, both(c.c1));
  return __ffma2_rn(q, z, both(c.c0));
}
// cap2 tanh(sc2 s) for any s: the polynomial where it holds (the other form
// loses there what the subtraction cancels: its error is one of the cap, not of
// the score), else 1 - 2 / (1 + e^(2u)).
__device__ __forceinline__ float2 cap_any(float2 s, const ScoreConst& c) {
  const float k = fminf(c.sc2 * (2.0f * kLog2e), 3.4028234e38f);  // finite: 0 times it is 0
  auto large = [&](float x) { return c.cap2 * fmaf(-2.0f, rcp_ftz(1.0f + ex2_ftz(x * k)), 1.0f); };
  const float2 small = __fmul2_rn(cap_poly(__fmul2_rn(s, s), c), s);
  return make_float2(fabsf(s.x) <= c.near ? small.x : large(s.x), fabsf(s.y) <= c.near ? small.y : large(s.y));
}

// Column e of a half block that begins at key0 is visible.
struct Mask {
  uint32_t w[2];
  __device__ __forceinline__ Mask(int key0, int lo, int hi) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // Visible columns [a, b) of this word.
      const int a = min(max(lo - key0 - 32 * i, 0), 32), b = min(max(hi - key0 - 32 * i, 0), 32);
      const uint32_t upto = b == 32 ? 0xFFFFFFFFu : (1u << b) - 1u;
      w[i] = a < b ? upto & (0xFFFFFFFFu << a) : 0u;
    }
  }
  __device__ __forceinline__ bool operator[](int e) const { return (w[e >> 5] >> (e & 31)) & 1u; }
};

// One half block of one row: raw scores in s; the weights go to tensor memory at
// `tp` as packed pairs, the row's reference (its maximum, log2 units) and sum are brought up
// to date.  Returns the factor that O has to be scaled by (1: none).
//
// The maximum in use only has to keep weights in range, so a half block that every
// row of the warp sees whole (or whose hidden scores are -infinity beforehand,
// where no cap follows) is tried with the one at hand, in one sweep
// without a search for its own: its sum, taken anyway, tells whether a weight
// left the range.  Only then and in a row's first half block is the maximum
// searched.
//
// cap tanh(s / cap) is a polynomial on the FMA pipe while all scores of the
// warp's rows lie within 3/8 of the cap, else cap_any, with two more steps of
// the exponential pipe that bounds the sweep.  Either is within 16 2^-24 of the
// capped score, less than the 32-bit dot product before it (a polynomial two
// coefficients shorter was off by 8e-7 of the cap: 2 x 4,096 capped rows 154 us
// instead of 159).  Where scores are capped outside the first try they are so
// in place, ahead of the sweep: inside it, 24 sequences of up to 16,384 keys
// took 221 us instead of 203.
template <typename T, bool CAP, bool BIAS>
__device__ __forceinline__ float softmax_block(float* s, uint32_t tp, RowState& r, const ScoreConst& c, int key0,
                                               bool masked, bool first) {
  float2 sum[2];
  auto sweep = [&](auto transform) {
    sum[0] = sum[1] = both(0.f);
#pragma unroll
    for (int e0 = 0; e0 < kH; e0 += 32) {
      uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 y = transform(make_float2(s[e0 + e], s[e0 + e + 1]), e0 + e);
        const float2 w = make_float2(ex2_ftz(y.x), ex2_ftz(y.y));
        sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], w);
        pk[e >> 1] = pack2<T>(w.x, w.y);
      }
      tc_st_32x32b_x16(tp + e0 / 2, pk);
    }
    const float2 a = __fadd2_rn(sum[0], sum[1]);
    return a.x + a.y;
  };
  const float d0 = static_cast<float>(key0 - r.pos);
  // The bias is slope * (key - pos) where no visible key of the warp's rows
  // lies behind its row, else -slope * |key - pos|.
  const bool linear = BIAS && (c.forward || __all_sync(0xFFFFFFFFu, key0 + kH - 1 <= r.pos || !r.valid));
  bool fits = true;  // the maximum at hand served this row
  if (!(CAP && masked) && !first && (!BIAS || linear) && __all_sync(0xFFFFFFFFu, r.m > -INFINITY || !r.valid)) {
    if (!CAP && masked) {
      const Mask vis(key0, r.lo, r.hi);
#pragma unroll
      for (int e = 0; e < kH; ++e) s[e] = vis[e] ? s[e] : -INFINITY;
    }
    const float2 add = both(BIAS ? fmaf(d0, r.slope, -r.m) : -r.m);
    float far[2] = {0.f, 0.f};
    const float t = sweep([&](float2 x, int e) {
      const float2 at = BIAS ? __ffma2_rn(both(r.slope), make_float2(static_cast<float>(e), static_cast<float>(e + 1)), add)
                             : add;
      if constexpr (CAP) {
        const float2 z = __fmul2_rn(x, x);
        far[(e >> 1) & 1] = max3(far[(e >> 1) & 1], z.x, z.y);
        return __ffma2_rn(cap_poly(z, c), x, at);
      } else {
        return __ffma2_rn(x, both(c.sc2), at);
      }
    });
    fits = t <= kFits<T>;
    if constexpr (CAP) {
      fits = fits && fmaxf(far[0], far[1]) <= c.near2;
    }
    fits = fits || !r.valid;
    if (__all_sync(0xFFFFFFFFu, fits)) {
      r.l += t;
      return 1.0f;
    }
  }

  const Mask vis(key0, r.lo, r.hi);
  if constexpr (CAP) {
    if (masked) {  // NaN takes no part in minima and maxima
#pragma unroll
      for (int e = 0; e < kH; ++e) s[e] = vis[e] ? s[e] : __uint_as_float(0x7FC00000u);
    }
    const float far = fmaxf(fabsf(max_of(s)), fabsf(min_of(s)));
    // Every visible score of the warp's rows lies within 3/8 of the cap.
    const bool near = __all_sync(0xFFFFFFFFu, !(far > c.near) || !r.valid);
    if (near) {
#pragma unroll
      for (int e = 0; e < kH; e += 2) {
        const float2 x = make_float2(s[e], s[e + 1]), y = __fmul2_rn(cap_poly(__fmul2_rn(x, x), c), x);
        s[e] = y.x;
        s[e + 1] = y.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kH; e += 2) {
        const float2 y = cap_any(make_float2(s[e], s[e + 1]), c);
        s[e] = y.x;
        s[e + 1] = y.y;
      }
    }
  }
  if constexpr (BIAS) {
    const float mul = CAP ? 1.0f : c.sc2;
    if (linear) {
#pragma unroll
      for (int e = 0; e < kH; ++e) s[e] = fmaf(r.slope, d0 + static_cast<float>(e), s[e] * mul);
    } else {
#pragma unroll
      for (int e = 0; e < kH; ++e) s[e] = fmaf(-r.slope, fabsf(d0 + static_cast<float>(e)), s[e] * mul);
    }
  }
  if (masked) {
#pragma unroll
    for (int e = 0; e < kH; ++e) s[e] = vis[e] ? s[e] : -INFINITY;
  }
  float m = fmaxf(max_of(s), -INFINITY);
  if constexpr (!CAP && !BIAS) m *= c.sc2;
  float factor = 1.0f;
  if (first) {
    r.m = m - kHead<T>;
  } else if (m > r.m + (fits ? kRaise : kHead<T>)) {
    m -= kHead<T>;
    factor = ex2_ftz(r.m - m);
    r.l *= factor;
    r.m = m;
  }
  const float2 base = both(r.m == -INFINITY ? 0.f : -r.m);
  if constexpr (CAP || BIAS) {
    r.l += sweep([&](float2 x, int) { return __fadd2_rn(x, base); });
  } else {
    r.l += sweep([&](float2 x, int) { return __ffma2_rn(x, both(c.sc2), base); });
  }
  return factor;
}

// ------------------------------------------------------------------- kernel
template <typename T, int HDP, bool CAP, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ AttnPlan p, const __grid_constant__ CUtensorMap tmq,
                   const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  constexpr int NCH = chunks<HDP>(), NST = stages<HDP, SPLIT>();
  constexpr uint32_t kBlockBytes = NCH * kChunkBytes;
  extern __shared__ uint8_t attn_lm_raw[];
  uint8_t* base = attn_lm_raw + ((1024u - (smem_u32(attn_lm_raw) & 1023u)) & 1023u);
  uint8_t* sq = base;
  uint8_t* ring = base + q_bytes<HDP, SPLIT>();
  Ctl& C = *reinterpret_cast<Ctl*>(ring + NST * kBlockBytes);
  const int warp = uni(threadIdx.x >> 5), lane = threadIdx.x & 31;
  volatile int* abort_flag = &C.abort;
  const yb_attn_args& a = p.a;

  Piece pc;
  if constexpr (!SPLIT) {
    // Row mode has one pair of tiles, the last rows (the most keys of a causal
    // prompt) first.  What its roles are about to read is on its way while
    // barriers and tensor memory are set up.
    const int bh = a.B * p.groups, pairs = (p.tiles + 1) / 2;
    const int x = blockIdx.x / bh, y = blockIdx.x - x * bh;
    pc.b = y / p.groups;
    pc.hg = y - pc.b * p.groups;
    pc.qt = 2 * (pairs - 1 - x);
    if (threadIdx.x < 32) {
      if (a.q_len) prefetch_l1(a.q_len + pc.b);
      if (a.k_len) prefetch_l1(a.k_len + pc.b);
      if (a.prefix) prefetch_l1(a.prefix + pc.b);
    }
    const int i = pc.qt * p.np + static_cast<int>(threadIdx.x);
    if (a.key_range && static_cast<int>(threadIdx.x) < 2 * p.np && i < a.Sq)
      prefetch_l1(a.key_range + 2 * (static_cast<long long>(pc.b) * a.Sq + i));
  }
  pdl_trigger();  // the join's blocks may come up meanwhile; they wait for this grid's end
  if (threadIdx.x == 0) {
    mbar_init(&C.q_full, 1);
    for (int t = 0; t < 2; ++t) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&C.s_full[t][h], 1);
        mbar_init(&C.p_full[t][h], 4);
        mbar_init(&C.o_full[t][h], 1);
      }
    }
    mbar_init(&C.o_empty, 4);
    mbar_init(&C.ml_full, 4);
    mbar_init(&C.drain, 1);
    for (int i = 0; i < NST; ++i) {
      mbar_init(&C.kv_full[i], 1);
      mbar_init(&C.kv_empty[i], 1);
    }
    C.abort = 0;
    mbar_fence_init();
    prefetch_tmap(&tmq);
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&C.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = uni(C.tmem);
  const uint32_t ts[2] = {tm, tm + kB}, to[2] = {tm + 2 * kB, tm + 2 * kB + HDP};

  // Pieces of this CTA: split mode walks its share, row mode has its pair.
  Walk walk;
  const int ksteps = (a.D + 15) / 16;
  const int fill = p.gp * p.np;  // rows of a full tile
  bool more;
  if constexpr (SPLIT) {
    walk.seek(p, blockIdx.x, gridDim.x);
    more = walk.next(p, &pc);
  } else {
    more = pc.qt * p.np < clamp_len(a.q_len, pc.b, a.Sq);
  }

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kLoadWarp) {
    // ------------------------------------------------------------- loads
    Ring rg;
    int loads = 0;
    while (more && !p.withhold) {
      const Blocks r = block_range<SPLIT>(p, pc);
      const int j0 = min(r.j0[0], r.j0[1]), j1 = max(r.j1[0], r.j1[1]);
      const int hk = pc.hg * p.gp / (a.Hq / a.Hkv);
      bool ok = true;
      if (lane == 0) {
        auto load = [&](const CUtensorMap* m, int bmul, int j) {
          if (!mbar_wait(&C.kv_empty[rg.slot], rg.phase ^ 1u, abort_flag, p.wait_ns)) {
            if (!*abort_flag) raise_error(p.err, abort_flag, kErrWaitEmpty);
            ok = false;
            return;
          }
          mbar_arrive_expect_tx(&C.kv_full[rg.slot], kBlockBytes);
          uint8_t* dst = ring + rg.slot * kBlockBytes;
#pragma unroll
          for (int c = 0; c < NCH; ++c)
            tma_tile_4d(dst + c * kChunkBytes, m, 64 * c, j * kB, hk, pc.b * bmul, &C.kv_full[rg.slot]);
          ++loads;
          rg.next<NST>();
        };
        // Ring order: K then V of one block after another, the last keys first;
        // in split mode of pairs of blocks, one for each pipeline.
        constexpr int kSet = SPLIT ? 2 : 1;
        for (int j = j1 - 1; j >= j0 && ok; j -= kSet) {
          for (int x = j; x > max(j - kSet, j0 - 1) && ok; --x) load(&tmk, p.k_bmul, x);
          for (int x = j; x > max(j - kSet, j0 - 1) && ok; --x) load(&tmv, p.v_bmul, x);
        }
      }
      ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
      if (!ok) break;
      if constexpr (SPLIT)
        more = walk.next(p, &pc);
      else
        more = false;
    }
    // After an abort, copies may still be landing in shared memory.
    if (lane == 0 && *abort_flag) {
      int dummy = 0;
      const int open = loads < NST ? loads : NST;
      for (int i = 0; i < open; ++i) {
        rg.slot = rg.slot ? rg.slot - 1 : NST - 1;
        if (rg.slot == NST - 1) rg.phase ^= 1u;
        mbar_wait(&C.kv_full[rg.slot], rg.phase, &dummy, p.wait_ns);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // -------------------------------------------------------------- UMMAs
    Ring rg;
    uint32_t p_phase[2] = {0, 0}, q_phase = 0;  // of a pipeline, both halves
    // Pieces with keys.  The others move no barrier, in any role: a role that
    // passed through them alone would get two phases ahead of another's wait.
    int piece = 0;
    bool ok = true, q_open = false;
    const uint32_t id_s = idesc_f32<T>(kH, false), id_o = idesc_f32<T>(16 * ksteps, true);
    const uint32_t q_tx = static_cast<uint32_t>(NCH * 128 * fill);
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
      // The lanes agree, so that none is left behind at a warp barrier.
      if (ok && !__all_sync(0xFFFFFFFFu, mbar_wait(bar, phase, abort_flag, p.wait_ns))) {
        if (lane == 0 && !*abort_flag) raise_error(p.err, abort_flag, code);
        ok = false;
      }
      return ok;
    };
    // Scores of half h of the block in `slot` into the pipeline's buffer h, and
    // the product of the weights there with the values of that half.
    auto scores = [&](int t, int h, int slot) {
      tc_fence_after();
      const uint64_t qd = sw128_kmajor_desc(smem_u32(sq) + (SPLIT ? 0 : t) * kBlockBytes);
      const uint64_t kd = sw128_kmajor_desc(smem_u32(ring) + slot * kBlockBytes + h * (kH * 128));
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k) {
          constexpr uint32_t kc = kChunkBytes >> 4;
          const uint32_t o = (k >> 2) * kc + (k & 3) * 2;  // 16-byte units
          if (k < ksteps) mma_ss(ts[t] + h * kH, qd + o, kd + o, id_s, k > 0);
        }
        tc_commit(&C.s_full[t][h]);
      }
    };
    auto values = [&](int t, int h, int slot, bool first) {
      tc_fence_after();
      const uint64_t vd = v_desc(smem_u32(ring) + slot * kBlockBytes + h * (kH * 128));
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kH / 16; ++k)
          mma_ts(to[t], ts[t] + h * kH + 8 * k, vd + 128 * k, id_o, !first || h == 0 || k > 0);
        tc_commit(&C.o_full[t][h]);
      }
    };
    auto release = [&](int slot) {
      if (elect_one()) tc_commit(&C.kv_empty[slot]);
    };
    // Zeroes the value rows of block j that no row sees.
    auto clean = [&](int slot, int j, const Blocks& r) {
      if (j * kB >= r.lo && (j + 1) * kB <= r.hi) return;
      uint4* v = reinterpret_cast<uint4*>(ring + slot * kBlockBytes);
      for (int k = 0; k < kB; ++k) {
        const int key = j * kB + k;
        if (key >= r.lo && key < r.hi) continue;
        if (lane < 8 * NCH)
          v[(lane >> 3) * (kChunkBytes / 16) + k * 8 + (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    while (more && ok) {
      const Blocks r = block_range<SPLIT>(p, pc);
      const int j0 = min(r.j0[0], r.j0[1]), j1 = max(r.j1[0], r.j1[1]);
      if (j1 > j0) {
        // The earlier piece's scores are done (their weights were waited for).
        if (lane == 0 && !p.withhold) {
          mbar_arrive_expect_tx(&C.q_full, q_tx * (SPLIT ? 1 : (pc.qt + 1 < p.tiles ? 2 : 1)));
          for (int t = 0; t < (SPLIT ? 1 : 2); ++t)
            if (pc.qt + t < p.tiles)
#pragma unroll
              for (int c = 0; c < NCH; ++c)
                tma_tile_4d(sq + t * kBlockBytes + c * kChunkBytes, &tmq, 64 * c, pc.hg * p.gp, (pc.qt + t) * p.np,
                            pc.b * p.q_bmul, &C.q_full);
        }
        q_open = !p.withhold;
        __syncwarp();
        if (!wait(&C.q_full, q_phase, kErrWaitFull)) break;
        q_open = false;
        q_phase ^= 1u;
        // Step by step: one block, which both pipelines share, or in split
        // mode a pair of blocks, one for each.  The scores of a step's halves
        // go out when the weights of the step before them are used up, so the
        // softmax finds its next half ready.
        constexpr int kSet = SPLIT ? 2 : 1;
        const int steps = (j1 - j0 + kSet - 1) / kSet;
        auto takes = [&](int t, int n) {  // pipeline t has a block in step n
          return SPLIT ? n < steps && 2 * n + t < j1 - j0 : n < steps && j1 - 1 - n >= r.j0[t] && j1 - 1 - n < r.j1[t];
        };
        int ks[2] = {0, 0}, vs[2] = {0, 0};
        auto take = [&](int n, int (&slot)[2]) {  // waits for the blocks of step n next in the ring
          for (int x = 0; x < kSet && kSet * n + x < j1 - j0; ++x) {
            if (!wait(&C.kv_full[rg.slot], rg.phase, kErrWaitFull)) return false;
            slot[x] = rg.slot;
            rg.next<NST>();
          }
          return true;
        };
        auto drop = [&](int n, const int (&slot)[2]) {
          for (int x = 0; x < kSet && kSet * n + x < j1 - j0; ++x) release(slot[x]);
        };
        if (!take(0, ks)) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (takes(t, 0)) {
            scores(t, 1, ks[SPLIT ? t : 0]);
            scores(t, 0, ks[SPLIT ? t : 0]);
          }
        drop(0, ks);
        // The earlier piece's O has been read.
        if (SPLIT && piece > 0 && !wait(&C.o_empty, (piece - 1) & 1, kErrWaitAccEmpty)) break;
        for (int n = 0; n < steps && ok; ++n) {
          if (!take(n, vs)) break;
          for (int x = 0; x < kSet && kSet * n + x < j1 - j0; ++x) clean(vs[x], j1 - 1 - kSet * n - x, r);
          if (!SPLIT && n + 1 < steps && !take(n + 1, ks)) break;
#pragma unroll
          for (int h = 1; h >= 0; --h)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (takes(t, n)) {
                if (!wait(&C.p_full[t][h], p_phase[t], kErrWaitAccFull)) break;
                values(t, h, vs[SPLIT ? t : 0], n == 0 || !takes(t, n - 1));
                if (SPLIT && h == 0) release(vs[t]);
              }
              // Split mode is bound by memory: the next keys may come while the
              // first product of the step runs, and slots go back one by one.
              if (SPLIT && h == 1 && t == 0 && n + 1 < steps && !take(n + 1, ks)) break;
              if (takes(t, n + 1)) {
                scores(t, h, ks[SPLIT ? t : 0]);
                if (SPLIT && h == 0) release(ks[t]);
              }
            }
          if (!ok) break;
          for (int t = 0; t < 2; ++t)
            if (takes(t, n)) p_phase[t] ^= 1u;
          if (!SPLIT) {
            drop(n, vs);
            if (n + 1 < steps) drop(n + 1, ks);
          }
        }
        ++piece;
      }
      if (!ok) break;
      if constexpr (SPLIT)
        more = walk.next(p, &pc);
      else
        more = false;
    }
    // Everything issued has to finish before tensor memory goes.
    if (elect_one()) {
      int dummy = 0;
      if (q_open) mbar_wait(&C.q_full, q_phase, &dummy, p.wait_ns);
      tc_commit(&C.drain);
      if (!mbar_wait(&C.drain, 0, &dummy, p.wait_ns)) raise_error(p.err, abort_flag, kErrDrain);
    }
    __syncwarp();
  }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_s = ts[t] + lane_addr;
    ScoreConst c;
    if constexpr (CAP) {
      c.sc2 = a.scale / a.cap;
      c.cap2 = a.cap * kLog2e;
      // The polynomial in s = u / sc2.  For caps of some 2^20 times the scale
      // and more its last coefficients leave the normal numbers: it ends where
      // the next one would count (u^2 / 3 < 2^-24 at 4e-4, and so on).
      const float k2 = c.sc2 * c.sc2;
      c.c0 = a.scale * kLog2e;
      c.c1 = c.c0 * k2 * kTanh1;
      c.c2 = c.c0 * k2 * k2 * kTanh2;
      c.c3 = c.c0 * k2 * k2 * k2 * kTanh3;
      const auto normal = [](float x) { return fabsf(x) >= 1.17549435e-38f; };
      const float reach = normal(c.c3) ? kNear : normal(c.c2) ? 0.1f : normal(c.c1) ? 0.01f : 4e-4f;
      const bool finite = fabsf(c.c1) <= 3.4028234e38f && fabsf(c.c2) <= 3.4028234e38f && fabsf(c.c3) <= 3.4028234e38f;
      c.near = finite ? fminf(reach / c.sc2, 1.8e19f) : -1.0f;
      c.near2 = finite ? c.near * c.near : -1.0f;
    } else {
      c.sc2 = a.scale * kLog2e;
      c.cap2 = c.c0 = c.c1 = c.c2 = c.c3 = c.near = c.near2 = 0.f;
    }
    c.forward = a.causal && !a.prefix;
    uint32_t s_phase = 0;
    int piece = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
      // The lanes agree, so that none is left behind at a warp barrier.
      if (ok && !__all_sync(0xFFFFFFFFu, mbar_wait(bar, phase, abort_flag, p.wait_ns))) {
        if (lane == 0 && !*abort_flag) raise_error(p.err, abort_flag, code);
        ok = false;
      }
      return ok;
    };
    while (more && ok) {
      const Blocks r = block_range<SPLIT>(p, pc);
      const int qt = pc.qt + (SPLIT ? 0 : t);
      const int i = qt * p.np + static_cast<int>(p.fd_gp.div(row)), h = pc.hg * p.gp + row - static_cast<int>(p.fd_gp.div(row)) * p.gp;
      const int q_len = clamp_len(a.q_len, pc.b, a.Sq), k_len = clamp_len(a.k_len, pc.b, a.Sk);
      RowState st;
      st.valid = row < fill && i < q_len;
      int wlo = 0, whi = 0x7FFFFFFF;
      if (st.valid) {
        const RowSpan sp = row_span(a, pc.b, i, q_len, k_len);
        st.lo = wlo = sp.lo;
        st.hi = whi = sp.hi;
        st.pos = sp.pos;
        if constexpr (BIAS) st.slope = a.slopes[h] * kLog2e;
      }
      const bool live = __any_sync(0xFFFFFFFFu, st.valid);
      wlo = __reduce_max_sync(0xFFFFFFFFu, wlo);  // keys [wlo, whi) are seen by every row of the warp
      whi = __reduce_min_sync(0xFFFFFFFFu, whi);
      const int step = SPLIT ? 2 : 1;
      int done = 0;  // half blocks
      for (int j = r.j1[t] - 1 - (SPLIT ? t : 0); j >= r.j0[t] && ok; j -= step) {
#pragma unroll 1
        for (int h = 1; h >= 0; --h, ++done) {
          if (!wait(&C.s_full[t][h], s_phase, kErrWaitAccFull)) break;
          if (live) {
            tc_fence_after();
            const uint32_t buf = my_s + h * kH;
            const int key0 = j * kB + h * kH;
            float s[kH];
#pragma unroll
            for (int e = 0; e < kH; e += 32) ld32(buf + e, s + e);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < kH; e += 32) ld32_dep(s + e);
            const bool masked = key0 < wlo || key0 + kH > whi;
            const float f = softmax_block<T, CAP, BIAS>(s, buf, st, c, key0, masked, done == 0);
            if (__any_sync(0xFFFFFFFFu, f != 1.0f)) {
              // After the product before this one: of this block's upper half,
              // or of the lower half of the block before.  (s_phase is the
              // block's parity; the product before that one was complete when
              // these scores were, so the barrier is never two phases off.)
              if (!wait(&C.o_full[t][h ^ 1], h ? s_phase ^ 1u : s_phase, kErrWaitAccFull)) break;
              tc_fence_after();
              for (int e = 0; e < 16 * ksteps; e += 16) {
                uint32_t o[16];
                tc_ld_32x32b_x16(to[t] + lane_addr + e, o);
                tc_wait_ld();
                tc_ld_dep(o);
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                tc_st_32x32b_x16(to[t] + lane_addr + e, o);
              }
            }
            tc_wait_st();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&C.p_full[t][h]);
        }
        s_phase ^= 1u;
      }
      if (!ok) break;
      if (done) {  // the last block's products
        if (!wait(&C.o_full[t][0], s_phase ^ 1u, kErrWaitAccFull)) break;
        if (!wait(&C.o_full[t][1], s_phase ^ 1u, kErrWaitAccFull)) break;
      }
      float w[2] = {1.f, 0.f}, m = st.m, l = st.l;
      bool have[2] = {done > 0, false};
      const bool work = r.j1[0] > r.j0[0];  // split mode: the piece has keys
      if constexpr (SPLIT) {
        if (t == 1) {
          if (work) {
            if (piece > 0 && !wait(&C.o_empty, (piece - 1) & 1, kErrWaitAccEmpty)) break;
            C.ml[row] = make_float2(st.m, st.l);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&C.ml_full);
            ++piece;
          }
          more = walk.next(p, &pc);
          continue;
        }
        float2 o = make_float2(-INFINITY, 0.f);
        if (work) {
          if (!wait(&C.ml_full, piece & 1, kErrWaitAccFull)) break;
          o = C.ml[row];
        }
        have[1] = r.j1[0] - r.j0[0] > 1;
        m = fmaxf(st.m, o.x);
        const float mb = m == -INFINITY ? 0.f : m;
        w[0] = ex2_ftz(st.m - mb);
        w[1] = ex2_ftz(o.x - mb);
        l = st.l * w[0] + o.y * w[1];
      }
      tc_fence_after();
      const bool part = SPLIT && pc.slot >= 0;
      const float inv = part ? 1.0f : (l == 0.f ? 0.f : 1.0f / l);
      w[0] *= inv;
      w[1] *= inv;
      float* po = nullptr;
      if (SPLIT && part) {
        po = p.ws + (static_cast<size_t>(blockIdx.x) * 2 + pc.slot) * p.rows * (a.D + 4);
      }
      T* out = static_cast<T*>(a.o) + pc.b * a.o_stride[0] + static_cast<long long>(i) * a.o_stride[1] +
               static_cast<long long>(h) * a.o_stride[2];
      bool bad = false;
      if (live) {
        for (int e = 0; e < 16 * ksteps; e += 16) {
          uint32_t x[2][16];
#pragma unroll
          for (int u = 0; u < (SPLIT ? 2 : 1); ++u)
            if (have[u]) tc_ld_32x32b_x16(to[SPLIT ? u : t] + lane_addr + e, x[u]);
          tc_wait_ld();
          float y[16];
#pragma unroll
          for (int d = 0; d < 16; ++d) y[d] = 0.f;
#pragma unroll
          for (int u = 0; u < (SPLIT ? 2 : 1); ++u)
            if (have[u]) {
              tc_ld_dep(x[u]);
#pragma unroll
              for (int d = 0; d < 16; ++d) y[d] = fmaf(__uint_as_float(x[u][d]), w[u], y[d]);
            }
#pragma unroll
          for (int d = 0; d < 16; ++d) bad = bad || !(fabsf(y[d]) <= 3.4028234e38f);
          if (!st.valid) continue;
          if (part) {
            float4* dst = reinterpret_cast<float4*>(po + static_cast<size_t>(row) * a.D + e);
#pragma unroll
            for (int d = 0; d < 16; d += 4)
              if (e + d < a.D) dst[d / 4] = make_float4(y[d], y[d + 1], y[d + 2], y[d + 3]);
          } else {
            uint32_t z[8];
#pragma unroll
            for (int d = 0; d < 8; ++d) z[d] = pack2<T>(y[2 * d], y[2 * d + 1]);
            *reinterpret_cast<uint4*>(out + e) = make_uint4(z[0], z[1], z[2], z[3]);
            if (e + 8 < a.D) *reinterpret_cast<uint4*>(out + e + 8) = make_uint4(z[4], z[5], z[6], z[7]);
          }
        }
        if (part && st.valid)
          *reinterpret_cast<float2*>(po + static_cast<size_t>(p.rows) * a.D + 2 * row) = make_float2(m, l);
        // Rows that a value of keys they do not see has spoilt.
        unsigned again = __ballot_sync(0xFFFFFFFFu, st.valid && bad && l == l);
        while (again) {
          const int who = __ffs(again) - 1;
          again &= again - 1;
          const int wi = __shfl_sync(0xFFFFFFFFu, i, who), wh = __shfl_sync(0xFFFFFFFFu, h, who);
          const int pos = __shfl_sync(0xFFFFFFFFu, st.pos, who);
          int lo = __shfl_sync(0xFFFFFFFFu, st.lo, who), hi = __shfl_sync(0xFFFFFFFFu, st.hi, who);
          if constexpr (SPLIT) {
            lo = max(lo, r.j0[0] * kB);
            hi = min(hi, r.j1[0] * kB);
          }
          const RowAcc x = attn_row<T>(a, pc.b, wi, wh, pos, lo, hi);
          const int d = 4 * lane, wrow = __shfl_sync(0xFFFFFFFFu, row, who);
          if (d < a.D) {
            if (part) {
              *reinterpret_cast<float4*>(po + static_cast<size_t>(wrow) * a.D + d) =
                  make_float4(x.o[0], x.o[1], x.o[2], x.o[3]);
              if (lane == 0)
                *reinterpret_cast<float2*>(po + static_cast<size_t>(p.rows) * a.D + 2 * wrow) = make_float2(x.m, x.l);
            } else {
              T* o = static_cast<T*>(a.o) + pc.b * a.o_stride[0] + static_cast<long long>(wi) * a.o_stride[1] +
                     static_cast<long long>(wh) * a.o_stride[2] + d;
              for (int e = 0; e < 4; ++e) o[e] = from_f<T>(x.l == 0.f ? 0.f : x.o[e] / x.l);
            }
          }
        }
      }
      if constexpr (SPLIT) {
        tc_fence_before();
        __syncwarp();
        if (work) {
          if (lane == 0) mbar_arrive(&C.o_empty);
          ++piece;
        }
        more = walk.next(p, &pc);
      } else {
        more = false;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tm, kTmemCols);
  }
}

// Joins the pieces of a tile that was cut between CTAs of the split mode.
// Block c finds the tile, if any, whose last piece is CTA c's first and which
// began before; its pieces lie in CTAs c0 .. c (a CTA's piece that begins the
// tile in slot 1, later ones in slot 0).  One warp per row.
template <typename T>
__global__ void __launch_bounds__(1024) attn_join_kernel(const __grid_constant__ AttnPlan p) {
  const yb_attn_args& a = p.a;
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Walk w;
  w.seek(p, c, gridDim.x);
  Piece s;
  const bool mine = w.next(p, &s) && s.slot == 0 && s.off + s.take == s.n;
  pdl_wait();
  if (!mine) return;
  const long long u0 = w.total * c / w.ctas - s.off;  // the tile's first unit
  int c0 = c;
  while (c0 > 0 && w.total * c0 / w.ctas > u0) --c0;
  const int q_len = clamp_len(a.q_len, s.b, a.Sq);
  const size_t slot_size = static_cast<size_t>(p.rows) * (a.D + 4);
  const int pieces = c - c0 + 1;
  for (int row = warp; row < p.rows; row += blockDim.x >> 5) {
    const int x = static_cast<int>(p.fd_gp.div(row)), i = s.qt * p.np + x, h = s.hg * p.gp + row - x * p.gp;
    if (i >= q_len) break;
    // A lane per piece for maxima and sums, then all lanes on each piece's row.
    auto piece_ml = [&](int k) {
      const float* sl = p.ws + (2 * static_cast<size_t>(c0 + k) + (k == 0)) * slot_size;
      return *reinterpret_cast<const float2*>(sl + static_cast<size_t>(p.rows) * a.D + 2 * row);
    };
    float m = -INFINITY;
    for (int k = lane; k < pieces; k += 32) m = fmaxf(m, piece_ml(k).x);
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    const float mb = (m == -INFINITY ? 0.f : m) + kJoinRoom;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int d = 4 * lane;
    for (int k0 = 0; k0 < pieces; k0 += 32) {
      const int n = min(32, pieces - k0);
      float f = 0.f;
      if (lane < n) {
        const float2 ml = piece_ml(k0 + lane);
        f = ex2_ftz(ml.x - mb);
        l = fmaf(ml.y, f, l);
      }
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const float w = __shfl_sync(0xFFFFFFFFu, f, k);
        if (d < a.D) {
          const float* sl = p.ws + (2 * static_cast<size_t>(c0 + k0 + k) + (k0 + k == 0)) * slot_size;
          const float4 v = *reinterpret_cast<const float4*>(sl + static_cast<size_t>(row) * a.D + d);
          o.x = fmaf(v.x, w, o.x);
          o.y = fmaf(v.y, w, o.y);
          o.z = fmaf(v.z, w, o.z);
          o.w = fmaf(v.w, w, o.w);
        }
      }
    }
    for (int x0 = 16; x0; x0 >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x0);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    if (d < a.D)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + s.b * a.o_stride[0] + static_cast<long long>(i) * a.o_stride[1] +
                                static_cast<long long>(h) * a.o_stride[2] + d) =
          make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  }
}

// --------------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 tiled_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// Map over [B, rows, heads, D] with boxes of 64 dims.  order_rows: box rows run
// over positions (K, V; dims D, row, head, batch), else over heads, then
// positions (Q; dims D, head, row, batch).
bool encode(CUtensorMap* map, const yb_attn_args& a, const void* base, const long long* st, int rows, int heads,
            bool order_rows, int box1, int box2, bool one_batch) {
  const auto enc = tiled_encoder();
  if (!enc) return false;
  auto bytes = [](long long s, int n) { return static_cast<cuuint64_t>(n > 1 ? s * 2 : 16); };
  const cuuint64_t nr = rows > 0 ? rows : 1, nh = heads, nb = one_batch ? 1 : a.B;
  const cuuint64_t sr = bytes(st[1], rows), sh = bytes(st[2], heads), sb = bytes(st[0], static_cast<int>(nb));
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.D), order_rows ? nr : nh, order_rows ? nh : nr, nb};
  cuuint64_t strides[3] = {order_rows ? sr : sh, order_rows ? sh : sr, sb};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box1), static_cast<cuuint32_t>(box2), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, a.dtype == YB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Calls f with the kernel for these options.
template <typename T, int HDP, bool CAP, bool BIAS, typename F>
cudaError_t pick_mode(bool split, F f) {
  if (split) return f(attn_tc_kernel<T, HDP, CAP, BIAS, true>, smem_bytes<HDP, true>());
  return f(attn_tc_kernel<T, HDP, CAP, BIAS, false>, smem_bytes<HDP, false>());
}
template <typename T, int HDP, typename F>
cudaError_t pick_score(bool cap, bool bias, bool split, F f) {
  if (cap && bias) return pick_mode<T, HDP, true, true>(split, f);
  if (cap) return pick_mode<T, HDP, true, false>(split, f);
  if (bias) return pick_mode<T, HDP, false, true>(split, f);
  return pick_mode<T, HDP, false, false>(split, f);
}
template <typename F>
cudaError_t pick(int dtype, int hdp, bool cap, bool bias, bool split, F f) {
  if (dtype == YB_F16)
    return hdp == 64 ? pick_score<__half, 64>(cap, bias, split, f) : pick_score<__half, 128>(cap, bias, split, f);
  return hdp == 64 ? pick_score<__nv_bfloat16, 64>(cap, bias, split, f)
                   : pick_score<__nv_bfloat16, 128>(cap, bias, split, f);
}

}  // namespace

AttnPlan plan_attn(const yb_attn_args& a, int num_sms) {
  AttnPlan p;
  p.a = a;
  const int share = a.Hq / a.Hkv;
  p.gp = share <= kB ? share : 1;
  p.np = kB / p.gp;
  p.groups = a.Hq / p.gp;
  p.tiles = (a.Sq + p.np - 1) / p.np;
  p.rows = p.gp * (p.np < a.Sq ? p.np : a.Sq);
  p.q_bmul = a.B > 1 && a.q_stride[0] == 0 ? 0 : 1;
  p.k_bmul = a.B > 1 && a.k_stride[0] == 0 ? 0 : 1;
  p.v_bmul = a.B > 1 && a.v_stride[0] == 0 ? 0 : 1;
  p.fd_gp = FastDiv(static_cast<uint32_t>(p.gp));
  const long long segs = static_cast<long long>(a.B) * p.tiles * p.groups;
  const int blocks = (a.Sk + kB - 1) / kB;
  // A CTA per row tile, both pipelines on its blocks, where there is one tile a
  // sequence or no more tiles than SMs; beyond that row mode, whose pipelines
  // share each block (16 heads on 4, D 128, causal prompts of 152 / 200 / 296
  // tiles: 29 / 35 / 47 us in row mode, 60 / 82 / 141 cut over the SMs; of 148
  // tiles 44 in row mode, 41 with a CTA per tile).
  p.split = p.tiles == 1 || segs <= num_sms;
  if (p.split) {
    // Tiles stay whole, without a join, while cutting them would not pay: the
    // fewer SMs the tiles leave idle, the longer.  Steps of 16 heads on 4 at D
    // 128, us cut / whole: 1 tile of 700 keys 21 / 21, of 1,300 21 / 28; 32
    // tiles of 700 29 / 21, of 1,800 29 / 33; 64 of 1,800 36 / 33, of 4,000
    // 52 / 62; 96 of 2,500 53 / 44, of 8,000 96 / 109; 148 of 4,000 80 / 66;
    // prompts of 136 tiles over 5,000 keys 98 / 86, of 64 over 5,000 64 / 78.
    // More tiles than SMs run in uneven waves when whole: 200 of 1,300 65 / 55,
    // of 4,000 104 / 120.
    const long long most_blocks = segs > num_sms ? 16 : 7 + 54 * segs * segs / (num_sms * num_sms);
    p.whole = blocks <= most_blocks;
    // A CTA's least share: with 8 blocks instead of 4 one sequence of 2,000 keys
    // takes 26 us instead of 21, with 2 as long.
    p.unit_min = 4;
    const long long most = p.whole ? segs : segs * blocks;
    p.grid = static_cast<int>(most < num_sms ? most : num_sms);
  } else {
    p.grid = static_cast<int>(static_cast<long long>(a.B) * p.groups * ((p.tiles + 1) / 2));
  }
  return p;
}

size_t attn_workspace_bytes(const AttnPlan& p) {
  if (!p.split || p.whole) return 0;
  return static_cast<size_t>(p.grid) * 2 * p.rows * (p.a.D + 4) * sizeof(float);
}

cudaError_t prepare_attn() {
  for (int dt : {YB_F16, YB_BF16})
    for (int hdp : {64, 128})
      for (int o = 0; o < 8; ++o) {
        const cudaError_t e = pick(dt, hdp, o & 1, o & 2, o & 4, [](auto kernel, int smem) {
          return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        });
        if (e != cudaSuccess) return e;
      }
  cudaFuncAttributes fa;
  cudaError_t e = cudaFuncGetAttributes(&fa, attn_join_kernel<__half>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, attn_join_kernel<__nv_bfloat16>);
  return e;
}

cudaError_t launch_attn(const AttnPlan& p, cudaStream_t s) {
  const yb_attn_args& a = p.a;
  CUtensorMap tmq, tmk, tmv;
  const void* k = a.Sk ? a.k : a.q;
  const void* v = a.Sk ? a.v : a.q;
  if (!encode(&tmq, a, a.q, a.q_stride, a.Sq, a.Hq, false, p.gp, p.np, !p.q_bmul) ||
      !encode(&tmk, a, k, a.k_stride, a.Sk, a.Hkv, true, kB, 1, !p.k_bmul) ||
      !encode(&tmv, a, v, a.v_stride, a.Sk, a.Hkv, true, kB, 1, !p.v_bmul))
    return cudaErrorInvalidValue;
  cudaError_t e = pick(a.dtype, a.D <= 64 ? 64 : 128, a.cap > 0.f, a.slopes != nullptr, p.split,
                       [&](auto kernel, int smem) {
                         kernel<<<p.grid, kThreads, smem, s>>>(p, tmq, tmk, tmv);
                         return cudaGetLastError();
                       });
  if (e != cudaSuccess || !p.split || p.whole) return e;
  const dim3 grid(static_cast<unsigned>(p.grid)), block(static_cast<unsigned>(32 * (p.rows < 32 ? p.rows : 32)));
  if (a.dtype == YB_F16) return launch_pdl(attn_join_kernel<__half>, grid, block, 0, s, p);
  return launch_pdl(attn_join_kernel<__nv_bfloat16>, grid, block, 0, s, p);
}

}  // namespace yb
