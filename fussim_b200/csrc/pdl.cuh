#pragma once

namespace fssim {

// Programmatic dependent launch. The kernels are launched so that they may start while the
// previous kernel on the stream is finishing; their set-up (barrier init, step cursor)
// overlaps that tail, and griddepcontrol.wait, before the first access to global memory,
// waits for the previous kernel to complete and its writes to be visible. (Both are no-ops
// for a regular launch.) A kernel then allows its own dependent to launch.
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

}  // namespace fssim
