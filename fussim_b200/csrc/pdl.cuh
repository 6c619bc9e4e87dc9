#pragma once

namespace fssim {

// Programmatic dependent launch. The kernels are launched so that they may start while the
// previous kernel on the stream is finishing; their set-up (barrier init, step cursor)
// overlaps that tail, and griddepcontrol.wait waits for the previous kernel to complete and
// its writes to be visible. (Both are no-ops for a regular launch.) A kernel then allows its own
// dependent to launch.
//
// The rule for accesses to global memory: none before the wait, but for reads of what was complete
// before the preceding launch passed its own wait. So a kernel that reads ahead of its wait (the
// applying passes of the group norm) is never the first of a call, and every kernel waits
// before it allows its dependent to launch, whatever the dependent may be.
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

}  // namespace fssim
