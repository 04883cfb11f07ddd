// Shared by the text-decoder operators (yb_lm.h): element types in registers,
// and a scope that runs an entry point on a device and puts the caller's
// current device back.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "runtime.h"
#include "yb_lm.h"

namespace yb {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Every pointer (null ones included) lies on a boundary of `bytes`: a device
// load off its element's boundary is a fault.
template <typename... P>
bool on_boundary(size_t bytes, const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) % bytes == 0) && ...);
}

class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if ((err_ = cudaGetDevice(&old_)) != cudaSuccess) return;
    if (old_ != device && (err_ = cudaSetDevice(device)) == cudaSuccess) changed_ = true;
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(old_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t error() const { return err_; }

 private:
  int old_ = 0;
  bool changed_ = false;
  cudaError_t err_ = cudaSuccess;
};

}  // namespace yb
