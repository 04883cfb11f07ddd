// Attention of the text-decoder operators (yb_lm.h): the launch plan shared by
// the host entry (attn_lm_api.cu) and the kernels (attn_lm.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "fastdiv.h"
#include "yb_lm.h"

namespace yb {

constexpr int kAttnMaxD = 128;
constexpr int kAttnBlock = 128;  // keys per block, and rows per tile (UMMA M)

struct AttnPlan {
  yb_attn_args a;
  int gp = 1, np = 1;     // query heads of one key head and positions in a tile: row = position * gp + head
  int groups = 1;         // Hq / gp
  int tiles = 1;          // row tiles of a sequence
  int rows = 1;           // rows of a tile that any sequence can use
  bool split = false;     // one row tile per CTA, keys cut over CTAs and the CTA's two pipelines
  bool whole = false;     // split: no tile is cut over CTAs, no scratch
  int grid = 1;
  int unit_min = 1;       // split: key blocks per CTA at least
  int q_bmul = 1, k_bmul = 1, v_bmul = 1;  // 0: batch stride 0
  float* ws = nullptr;
  int* err = nullptr;
  uint64_t wait_ns = 0;
  int withhold = 0;  // test hook: no loads are issued
  FastDiv fd_gp;
};

// Sizes, modes and grid for these arguments on a device of num_sms SMs.
AttnPlan plan_attn(const yb_attn_args& a, int num_sms);
size_t attn_workspace_bytes(const AttnPlan& p);
cudaError_t prepare_attn();  // shared-memory limits of every kernel on the current device
cudaError_t launch_attn(const AttnPlan& p, cudaStream_t s);

}  // namespace yb
