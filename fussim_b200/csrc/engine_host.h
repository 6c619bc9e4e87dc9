// Host-side pieces shared by the library's translation units: the calling thread's last
// error, NVTX ranges, and the device's SM count.
#pragma once

#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <cstdint>
#include <mutex>
#include <string>

#include "fussim_b200.h"

namespace fssim_host {

inline thread_local std::string g_last_error;

// NVTX range over an entry point's host-side work (argument checks and launches), so a
// timeline tool shows the forward, backward and cross-GPU exchange by name. Without a tool
// attached a push/pop costs a few nanoseconds.
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

inline int fail(int code, const std::string& msg) {
  g_last_error = msg;
  return code;
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

inline int device_sms(int* sms) {
  static std::mutex mu;
  static int cached[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail(FSSIM_ERR_CUDA, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
  if (dev < 0 || dev >= 64) return fail(FSSIM_ERR_CUDA, "device ordinal out of range");
  std::lock_guard<std::mutex> lock(mu);
  if (cached[dev] == 0) {
    int v = 0;
    e = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess)
      return fail(FSSIM_ERR_CUDA, std::string("cudaDeviceGetAttribute: ") + cudaGetErrorString(e));
    cached[dev] = v;
  }
  *sms = cached[dev];
  return FSSIM_OK;
}

}  // namespace fssim_host
