// Launches of the block norms' row kernels: one source file for each pair of types.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "block_norm.cuh"
#include "engine_host.h"
#include "launch_host.h"

namespace fssim_host {

struct BlockLaunch {
  int groups;   // of eight numbers, of a thread
  bool vec;     // whole 16-byte vectors
  bool warp;    // a row within a warp
  bool staged;  // the arrays in shared memory
  int mode;     // fssim::BlockMode
  unsigned grid, block;
  size_t memory;
};

int block_norm_f32(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream);
int block_norm_f16(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream);
int block_norm_bf16(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream);
int block_norm_f32_f16(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream);
int block_norm_f32_bf16(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream);

constexpr int64_t kBlockMemory = 208 << 10;  // dynamic shared memory of a CTA at most

// Opts a kernel in to that, once for each device. `done` belongs to one kernel.
template <typename Kernel>
int block_allow(Kernel kernel, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64)) return fail(FSSIM_ERR_CUDA, "device ordinal out of range");
  if (e == cudaSuccess && !done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kBlockMemory));
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  }
  return e == cudaSuccess ? FSSIM_OK : fail(FSSIM_ERR_CUDA, cudaGetErrorString(e));
}

// Columns that go to a thread together.
template <typename X>
constexpr int block_unit(bool vec) { return !vec ? 1 : sizeof(X) == 4 ? 4 : 8; }

template <typename X, typename Y, int V, bool VEC, bool WARP, int MODE, bool STAGED = true>
int block_forward(const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  static std::atomic<bool> done[64];
  const auto kernel = fssim::block_norm_forward_kernel<X, Y, V, block_unit<X>(VEC), WARP, MODE, STAGED>;
  const int st = block_allow(kernel, done);
  return st ? st : launch(kernel, l.grid, l.block, l.memory, stream, "block norm forward launch", p);
}
template <typename X, typename Y, int V, bool VEC, bool WARP, int MODE, bool STAGED = true>
int block_backward(const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  static std::atomic<bool> done[64];
  const auto kernel = fssim::block_norm_backward_kernel<X, Y, V, block_unit<X>(VEC), WARP, MODE, STAGED>;
  const int st = block_allow(kernel, done);
  return st ? st : launch(kernel, l.grid, l.block, l.memory, stream, "block norm backward launch", p);
}

// Which kernels there are: see layout() in block_norm.cu. Kernels of one mode alone, and one for all
// modes for the longest rows. Against the latter for all rows: 8x1500x1001 FP16 without a branch forward 25
// us (29) and backward 43 (47), 8x4000x99 FP32 10 (12) and 19 (23), 8x3000x2003 FP32 to BF16 with a plain
// branch backward 254 (282), 8x1024x1152 BF16 without a branch backward 30 (40), 16x1024x1024 with a plain
// branch and an FP32 residual 68 (70). Some lose without a branch: 8x16384x96 FP32 forward 19 (16),
// 16x400x1843 FP32 backward 65 (60), 16384x4096 BF16 backward 170 (140).
template <typename X, typename Y, int V, bool WARP, bool VEC = true>
int block_forward_mode(const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  using namespace fssim;
  if (l.mode == kBlockBefore) return block_forward<X, Y, V, VEC, WARP, kBlockBefore>(l, p, stream);
  if (l.mode == kBlockPlain) return block_forward<X, Y, V, VEC, WARP, kBlockPlain>(l, p, stream);
  return block_forward<X, Y, V, VEC, WARP, kBlockAfter>(l, p, stream);
}
template <typename X, typename Y, int V, bool WARP, bool VEC = true>
int block_backward_mode(const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  using namespace fssim;
  if (l.mode == kBlockBefore) return block_backward<X, Y, V, VEC, WARP, kBlockBefore>(l, p, stream);
  if (l.mode == kBlockPlain) return block_backward<X, Y, V, VEC, WARP, kBlockPlain>(l, p, stream);
  return block_backward<X, Y, V, VEC, WARP, kBlockAfter>(l, p, stream);
}

template <typename X, typename Y>
int block_norm_types(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  using fssim::kBlockAfter;
  if (backward) {
    if (!l.vec)
      return l.warp          ? block_backward_mode<X, Y, 1, true, false>(l, p, stream)
             : l.groups == 1 ? block_backward_mode<X, Y, 1, false, false>(l, p, stream)
             : l.groups == 2 ? block_backward_mode<X, Y, 2, false, false>(l, p, stream)
                             : block_backward<X, Y, 4, false, false, kBlockAfter, false>(l, p, stream);
    if (l.groups == 4)
      return l.staged ? block_backward<X, Y, 4, true, false, kBlockAfter>(l, p, stream)
                      : block_backward<X, Y, 4, true, false, kBlockAfter, false>(l, p, stream);
    if (l.warp)
      return l.groups == 1 ? block_backward_mode<X, Y, 1, true>(l, p, stream)
                           : block_backward_mode<X, Y, 2, true>(l, p, stream);
    return l.groups == 1 ? block_backward_mode<X, Y, 1, false>(l, p, stream)
                         : block_backward_mode<X, Y, 2, false>(l, p, stream);
  }
  if (!l.vec)
    return l.warp          ? block_forward_mode<X, Y, 1, true, false>(l, p, stream)
           : l.groups == 1 ? block_forward_mode<X, Y, 1, false, false>(l, p, stream)
           : l.groups == 2 ? block_forward<X, Y, 2, false, false, kBlockAfter>(l, p, stream)
                           : block_forward<X, Y, 4, false, false, kBlockAfter, false>(l, p, stream);
  if (!l.staged) return block_forward<X, Y, 4, true, false, kBlockAfter, false>(l, p, stream);
  if (l.warp) {
    switch (l.groups) {
      case 1: return block_forward_mode<X, Y, 1, true>(l, p, stream);
      case 3: return block_forward_mode<X, Y, 3, true>(l, p, stream);
      case 4: return block_forward_mode<X, Y, 4, true>(l, p, stream);
      default: return block_forward_mode<X, Y, 5, true>(l, p, stream);
    }
  }
  switch (l.groups) {
    case 1: return block_forward_mode<X, Y, 1, false>(l, p, stream);
    case 3: return block_forward_mode<X, Y, 3, false>(l, p, stream);
    default: return block_forward_mode<X, Y, 4, false>(l, p, stream);
  }
}

}  // namespace fssim_host
