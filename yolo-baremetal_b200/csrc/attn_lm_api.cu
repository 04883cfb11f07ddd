// Host entry of the text-decoder attention (yb_lm.h): argument checks, the
// handle with the kernels' error word, and the launch.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <new>
#include <string>

#include "attn_lm.h"
#include "lm.h"
#include "sm100.cuh"

namespace yb {
namespace {

struct Attn {
  int device = 0, num_sms = 148;
  int* err = nullptr;
  std::atomic<bool> withhold_next{false};  // test hook armed by yb_attn_debug_withhold
};

status_t bad(const char* msg) {
  set_error(std::string("attn: ") + msg);
  return ERROR_INVALID_DIMS;
}

bool operand_ok(const void* p, const long long* s, bool zero_batch) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8 || s[i] > (1LL << 38)) return false;
  return zero_batch || s[0] > 0;
}

// Sizes and values; pointers are checked by the run.
status_t check_sizes(const yb_attn_args& a) {
  if (a.B < 0 || a.Sq < 0 || a.Sk < 0 || a.Hq < 1 || a.Hkv < 1) return bad("sizes must not be negative, heads >= 1");
  if (a.Hq % a.Hkv) return bad("Hq must be a multiple of Hkv");
  if (a.D < 8 || a.D > kAttnMaxD || a.D % 8) return bad("D must be a multiple of 8 in [8, 128]");
  if (a.dtype != YB_F16 && a.dtype != YB_BF16) return bad("dtype must be YB_F16 or YB_BF16");
  // Rows first: the product of all three may pass 64 bits.
  const long long rows = static_cast<long long>(a.B) * a.Sq;
  if (a.Sk > (1 << 30) || a.Sq > (1 << 30) || rows > INT_MAX || rows * a.Hq > INT_MAX ||
      static_cast<long long>(a.B) * a.Hkv > (1 << 30))
    return bad("at most 2^30 keys and 2^31 - 1 rows times heads");
  if (!std::isfinite(a.scale) || !(a.scale > 0.f)) return bad("scale must be finite and > 0");
  if (!std::isfinite(a.cap) || a.cap < 0.f) return bad("cap must be finite and >= 0");
  if (!std::isfinite(a.scale * 1.5f) || !std::isfinite(a.cap * 1.5f) ||
      (a.cap > 0.f && (!std::isfinite(a.scale / a.cap) || a.scale / a.cap == 0.f)))
    return bad("scale, cap or scale / cap leaves the range of fp32");
  if (a.causal != 0 && a.causal != 1) return bad("causal must be 0 or 1");
  if (a.prefix && !a.causal) return bad("prefix needs causal");
  return SUCCESS;
}

}  // namespace
}  // namespace yb

using namespace yb;

extern "C" status_t yb_attn_create(int device, void** attn) {
  if (!attn) return ERROR_NULL_POINTER;
  *attn = nullptr;
  DeviceScope scope(device);
  if (scope.error() != cudaSuccess) return cuda_status(scope.error(), "cudaSetDevice");
  auto* h = new (std::nothrow) Attn();
  if (!h) return ERROR_OUT_OF_MEMORY;
  h->device = device;
  cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, device);
  cudaError_t e = prepare_attn();
  if (e == cudaSuccess) e = cudaMalloc(&h->err, sizeof(int));
  if (e == cudaSuccess) e = cudaMemset(h->err, 0, sizeof(int));
  if (e != cudaSuccess) {
    if (h->err) cudaFree(h->err);
    delete h;
    return cuda_status(e, "attn create");
  }
  *attn = h;
  return SUCCESS;
}

extern "C" status_t yb_attn_workspace(void* attn, const yb_attn_args* a, size_t* bytes) {
  if (!a || !bytes) return ERROR_NULL_POINTER;
  *bytes = 0;
  const status_t st = check_sizes(*a);
  if (st != SUCCESS) return st;
  if (!attn) return ERROR_NULL_POINTER;
  if (a->B && a->Sq) *bytes = attn_workspace_bytes(plan_attn(*a, static_cast<Attn*>(attn)->num_sms));
  return SUCCESS;
}

extern "C" status_t yb_attn_run(void* attn, const yb_attn_args* p, void* workspace, size_t workspace_bytes,
                                void* stream) {
  auto* h = static_cast<Attn*>(attn);
  if (!p) return ERROR_NULL_POINTER;
  const yb_attn_args a = *p;
  const status_t st = check_sizes(a);
  if (st != SUCCESS) return st;
  if (a.B == 0 || a.Sq == 0) return h ? SUCCESS : ERROR_NULL_POINTER;
  if (!a.q || !a.o || (a.Sk > 0 && (!a.k || !a.v))) return ERROR_NULL_POINTER;
  if (a.o == a.q || a.o == a.k || a.o == a.v) return bad("o must not be an input");
  // A stride of a dimension of size one is never used.
  auto ok = [&](const void* ptr, const long long* s, int rows, int heads, bool out) {
    const long long t[3] = {a.B > 1 ? s[0] : 8, rows > 1 ? s[1] : 8, heads > 1 ? s[2] : 8};
    return operand_ok(ptr, t, !out) && t[1] > 0 && t[2] > 0;
  };
  if (!ok(a.q, a.q_stride, a.Sq, a.Hq, false) || !ok(a.o, a.o_stride, a.Sq, a.Hq, true) ||
      (a.Sk > 0 && (!ok(a.k, a.k_stride, a.Sk, a.Hkv, false) || !ok(a.v, a.v_stride, a.Sk, a.Hkv, false))))
    return bad("q, k, v, o: 16-byte aligned, strides multiples of 8 elements; only batch strides of inputs may be 0");
  if (!on_boundary(8, a.key_range)) return bad("key_range must be 8-byte aligned");
  if (!on_boundary(4, a.q_len, a.k_len, a.prefix, a.slopes)) return bad("lengths, prefix and slopes: 4-byte aligned");
  if (!h) return ERROR_NULL_POINTER;
  DeviceScope scope(h->device);
  if (scope.error() != cudaSuccess) return cuda_status(scope.error(), "cudaSetDevice");
  AttnPlan plan = plan_attn(a, h->num_sms);
  const size_t need = attn_workspace_bytes(plan);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return bad("workspace must be 16-byte aligned and hold yb_attn_workspace bytes");
  plan.ws = static_cast<float*>(workspace);
  plan.err = h->err;
  // In split mode other roles wait while a warp computes up to 32 rows again
  // (a value that is not finite): 0.15 us a row and key at D = 128, 1 us allowed
  // for, up to a minute in all.  (A bound that begins anew while such a warp makes
  // progress took 62 instead of 57 us for 50 sequences of 2,500 keys.)
  plan.wait_ns = kWaitNs + std::min<uint64_t>(32000ull * static_cast<uint64_t>(a.Sk), 58000000000ull);
  if (h->withhold_next.exchange(false)) {
    plan.withhold = 1;
    plan.wait_ns = 1000000;  // 1 ms
  }
  return cuda_status(launch_attn(plan, static_cast<cudaStream_t>(stream)), "attn");
}

extern "C" status_t yb_attn_debug_withhold(void* attn) {
  if (!attn) return ERROR_NULL_POINTER;
  static_cast<Attn*>(attn)->withhold_next = true;
  return SUCCESS;
}

extern "C" status_t yb_attn_check(void* attn) {
  auto* h = static_cast<Attn*>(attn);
  if (!h) return ERROR_NULL_POINTER;
  DeviceScope scope(h->device);
  cudaError_t e = scope.error();
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  int k = 0;
  if (e == cudaSuccess) e = cudaMemcpy(&k, h->err, sizeof(int), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return cuda_status(e, "attn check");
  if (k) {
    cudaMemset(h->err, 0, sizeof(int));
    set_error("attn kernel reported error code " + std::to_string(k));
    return ERROR_DEVICE;
  }
  return SUCCESS;
}

extern "C" status_t yb_attn_destroy(void* attn) {
  if (!attn) return ERROR_NULL_POINTER;
  const status_t st = yb_attn_check(attn);
  auto* h = static_cast<Attn*>(attn);
  DeviceScope scope(h->device);
  cudaFree(h->err);
  delete h;
  return st;
}
