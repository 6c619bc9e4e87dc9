// Many tensors in one launch, shared by gradient clipping and the AdamW step: flat runs of memory
// named by a table in the kernel's parameters, cut into units of kRunUnit numbers, which are dealt out
// to the CTAs in equal contiguous ranges. A table has size[], unit0[] (the first unit of each
// run, and at the end the number of units) and count.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fssim {

constexpr int kRunUnit = 2048;  // numbers: eight for each of 256 threads

__device__ __forceinline__ float run_widen(float v) { return v; }
__device__ __forceinline__ float run_widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float run_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T run_narrow(float v);
template <> __device__ __forceinline__ float run_narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half run_narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 run_narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Sums of pairs, rounded by themselves: a packed product and a packed sum become one fused multiply-add
// (whatever rounding they name), which two single sums do not.
__device__ __forceinline__ float2 pair_add(float2 a, float2 b) {
  return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}

// The unit range of a CTA.
__device__ __forceinline__ int64_t run_range(int64_t units, int64_t b, int64_t grid) {
  return units / grid * b + (units % grid) * b / grid;
}

// Calls f(run, first number, one past the last) for each piece of a run in the units [u0, u1), from
// the last piece to the first when BACKWARDS.
template <bool BACKWARDS, typename Table, typename F>
__device__ __forceinline__ void run_walk(const Table& t, int64_t u0, int64_t u1, F f) {
  if (u0 >= u1) return;
  const int64_t key = BACKWARDS ? u1 - 1 : u0;
  int lo = 0, hi = t.count - 1;  // the last run whose first unit is at most key
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.unit0[mid] <= key) lo = mid;
    else hi = mid - 1;
  }
  for (int r = lo; BACKWARDS ? (r >= 0 && t.unit0[r + 1] > u0) : (r < t.count && t.unit0[r] < u1);
       r += BACKWARDS ? -1 : 1) {
    const int64_t first = t.unit0[r];
    const int64_t b = max(u0 - first, int64_t{0}) * kRunUnit;
    const int64_t e = min((u1 - first) * kRunUnit, t.size[r]);
    if (b < e) f(r, b, e);
  }
}

}  // namespace fssim
