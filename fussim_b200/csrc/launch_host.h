// Launches and entry points of the training-step operators, host side.
#pragma once

#include <cuda_runtime.h>

#include <exception>
#include <string>

#include "engine_host.h"

namespace fssim_host {

// A launch that may begin while the kernel before it on the stream is finishing (the kernels wait
// for that one's end before they touch memory).
template <typename... KA, typename... A>
int launch(void (*k)(KA...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, const char* what,
           const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, args...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(FSSIM_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e) + " (" + std::to_string(grid) +
                                    " CTAs of " + std::to_string(block) + " threads, " + std::to_string(smem) +
                                    " bytes of shared memory)");
  }
  return FSSIM_OK;
}

// No exception crosses the C boundary.
template <typename F>
int guarded(F f) {
  try {
    g_last_error.clear();
    return f();
  } catch (const std::exception&) {
    g_last_error = "host exception";  // short: no allocation
    return FSSIM_ERR_CUDA;
  }
}

}  // namespace fssim_host
