// Attention of the text-decoder operators (yb_lm.h): launch arguments shared by
// the host entry (attn_lm_api.cu) and the kernels.
#pragma once
#include <cuda_runtime.h>

#include "yb_lm.h"

namespace yb {

constexpr int kAttnMaxD = 128;

cudaError_t launch_attn_rows(const yb_attn_args& a, cudaStream_t s);

}  // namespace yb
