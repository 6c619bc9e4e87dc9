// Global gradient norm over many tensors, and clipping: kernels for sm_100a (B200).
//
//   norm = sqrt(sum over all tensors of g^2),  coef = min(1, max_norm / (norm + 1e-6)),
//   out = coef * g
//
// The tensors are flat runs of memory, named by a table in the kernel's parameters (so a
// captured launch carries its own copy, and no device memory or copy is needed for it). Each
// run is cut into units of kClipUnit numbers; the units of all runs, end to end, are split
// over the grid in equal contiguous ranges, so every CTA streams the same number of bytes
// whatever the tensors' sizes. A CTA finds its first run by bisection and walks on from there.
//
// Norm: squares are summed in FP32 over the eight numbers of one step of a thread and in FP64
// from there on; a step whose FP32 sum leaves the range where squares are exact enough is
// summed again in FP64, where the square of an FP32 number neither overflows nor vanishes. One
// FP64 partial per CTA, summed in a fixed order by whoever needs the norm: results repeat bit
// for bit, and the workspace needs no initial value.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"

namespace fssim {

constexpr int kClipThreads = 256;
constexpr int kClipUnit = 2048;     // numbers: eight for each thread
constexpr int kClipMaxCtas = 148 * 8;

// Runs of one launch. Two capacities: launches copy the whole table, and most models need few.
template <int K>
struct ClipTable {
  const void* src[K];
  void* dst[K];
  int64_t size[K];
  int64_t unit0[K + 1];   // first unit of each run; unit0[count] is their number
  unsigned char src_dtype[K];
  unsigned char dst_dtype[K];
  int count;
  double* partials;       // of the whole call
  int num_partials;       // of the whole call
  int first_partial;      // of this launch's CTAs
  float* norm;            // written by the launch that has it set
  float max_norm;
};

template <typename T> struct ClipVec;
template <> struct ClipVec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void load(const float* p, float* f) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void store8(float* p, const float* f) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  static __device__ __forceinline__ void put(float* p, float f) { *p = f; }
};
template <> struct ClipVec<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void load(const __half* p, float* f) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store8(__half* p, const float* f) {
    uint4 v;
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
  static __device__ __forceinline__ void put(__half* p, float f) { *p = __float2half_rn(f); }
};
template <> struct ClipVec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* f) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __bfloat1622float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store8(__nv_bfloat16* p, const float* f) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float f) { *p = __float2bfloat16_rn(f); }
};

// Eight consecutive numbers at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void clip_load8(const T* p, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += ClipVec<T>::n) ClipVec<T>::load(p + i, f + i);
}

// Squares of eight numbers, added up. Between 2^-80 and 2^100 the FP32 sum is right to a few
// of its roundings: no term overflowed, and what underflowed is below 2^-46 of the sum.
__device__ __forceinline__ double sum_squares8(const float (&f)[8]) {
  float a = fmaf(f[1], f[1], f[0] * f[0]), b = fmaf(f[3], f[3], f[2] * f[2]);
  float c = fmaf(f[5], f[5], f[4] * f[4]), d = fmaf(f[7], f[7], f[6] * f[6]);
  const float s = (a + b) + (c + d);
  if (s < 0x1p-80f || s > 0x1p100f) {
    double w = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w = fma(static_cast<double>(f[i]), static_cast<double>(f[i]), w);
    return w;
  }
  return s;  // NaN too
}

// The unit range of a CTA.
__device__ __forceinline__ int64_t clip_range(int64_t units, int64_t b, int64_t grid) {
  return units / grid * b + (units % grid) * b / grid;
}

// Calls f(run, first number, one past the last) for each piece of a run in this CTA's range,
// from the last piece to the first when BACKWARDS.
template <bool BACKWARDS, int K, typename F>
__device__ __forceinline__ void clip_walk(const ClipTable<K>& t, F f) {
  const int64_t units = t.unit0[t.count];
  const int64_t u0 = clip_range(units, blockIdx.x, gridDim.x);
  const int64_t u1 = clip_range(units, blockIdx.x + 1, gridDim.x);
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
    const int64_t b = max(u0 - first, int64_t{0}) * kClipUnit;
    const int64_t e = min((u1 - first) * kClipUnit, t.size[r]);
    if (b < e) f(r, b, e);
  }
}

// Numbers before the first 16-byte boundary of p + b, at most e - b.
template <typename T>
__device__ __forceinline__ int64_t clip_head(const T* p, int64_t b, int64_t e) {
  const int64_t off = static_cast<int64_t>((reinterpret_cast<uintptr_t>(p + b) % 16) / sizeof(T));
  const int64_t head = off ? 16 / static_cast<int64_t>(sizeof(T)) - off : 0;
  return min(head, e - b);
}

template <typename T>
__device__ __forceinline__ double clip_piece_squares(const T* src, int64_t b, int64_t e) {
  double acc = 0.0;
  const int64_t head = clip_head(src, b, e);
  const int64_t body = b + head;
  const int64_t n8 = (e - body) / 8;
  const int64_t tail = body + n8 * 8;
  constexpr int U = 4;
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * kClipThreads < n8; i += U * kClipThreads) {
    float f[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) clip_load8(src + body + (i + u * kClipThreads) * 8, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) acc += sum_squares8(f[u]);
  }
  for (; i < n8; i += kClipThreads) {
    float f[8];
    clip_load8(src + body + i * 8, f);
    acc += sum_squares8(f);
  }
  // what is left at the two ends: fewer than 8 numbers each
  const int64_t ends = head + (e - tail);
  if (threadIdx.x < ends) {
    const int64_t at = threadIdx.x < head ? b + threadIdx.x : tail + (threadIdx.x - head);
    const double v = ClipVec<T>::one(src + at);
    acc = fma(v, v, acc);
  }
  return acc;
}

// The factor, as two that are multiplied in turn: one below 2^-120 (a norm near or beyond
// FP32's largest number) is carried as 2^64 times itself and 2^-64, so that it keeps its bits.
struct ClipFactor {
  float a, b;
  __device__ __forceinline__ explicit ClipFactor(double c)
      : a(static_cast<float>(c < 0x1p-120 ? c * 0x1p64 : c)), b(c < 0x1p-120 ? 0x1p-64f : 1.f) {}
  __device__ __forceinline__ float operator*(float v) const { return v * a * b; }
};

template <typename S, typename D>
__device__ __forceinline__ void clip_piece_scale(const S* src, D* dst, int64_t b, int64_t e, ClipFactor coef) {
  const int64_t head = clip_head(src, b, e);
  const int64_t body = b + head;
  if (reinterpret_cast<uintptr_t>(dst + body) % 16 != 0) {
    // the two sides' boundaries differ: number by number, still in whole rows of a warp
    for (int64_t i = b + threadIdx.x; i < e; i += kClipThreads)
      ClipVec<D>::put(dst + i, coef * ClipVec<S>::one(src + i));
    return;
  }
  const int64_t n8 = (e - body) / 8;
  const int64_t tail = body + n8 * 8;
  constexpr int U = 2;
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * kClipThreads < n8; i += U * kClipThreads) {
    float f[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) clip_load8(src + body + (i + u * kClipThreads) * 8, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[u][k] = coef * f[u][k];
      ClipVec<D>::store8(dst + body + (i + u * kClipThreads) * 8, f[u]);
    }
  }
  for (; i < n8; i += kClipThreads) {
    float f[8];
    clip_load8(src + body + i * 8, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = coef * f[k];
    ClipVec<D>::store8(dst + body + i * 8, f);
  }
  const int64_t ends = head + (e - tail);
  if (threadIdx.x < ends) {
    const int64_t at = threadIdx.x < head ? b + threadIdx.x : tail + (threadIdx.x - head);
    ClipVec<D>::put(dst + at, coef * ClipVec<S>::one(src + at));
  }
}

// Sum of a double over the block, in every thread.
__device__ __forceinline__ double clip_block_sum(double v) {
  __shared__ double sm[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kClipThreads / 32; ++i) s += sm[i];
  return s;
}

template <int K>
__global__ void __launch_bounds__(kClipThreads) grad_squares_kernel(const __grid_constant__ ClipTable<K> t) {
  grid_dependency_wait();
  grid_launch_dependents();
  double acc = 0.0;
  clip_walk<false>(t, [&](int r, int64_t b, int64_t e) {
    if (t.src_dtype[r] == 0) acc += clip_piece_squares(static_cast<const float*>(t.src[r]), b, e);
    else if (t.src_dtype[r] == 1) acc += clip_piece_squares(static_cast<const __half*>(t.src[r]), b, e);
    else acc += clip_piece_squares(static_cast<const __nv_bfloat16*>(t.src[r]), b, e);
  });
  acc = clip_block_sum(acc);
  if (threadIdx.x == 0) t.partials[t.first_partial + blockIdx.x] = acc;
}

__device__ __forceinline__ double grad_norm_of(const double* partials, int n) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kClipThreads) v += partials[i];
  return sqrt(clip_block_sum(v));
}

__global__ void __launch_bounds__(kClipThreads) grad_norm_kernel(const double* partials, int n, float* norm) {
  grid_dependency_wait();
  grid_launch_dependents();
  const double v = grad_norm_of(partials, n);
  if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

// The second read goes through the CTA's range from its end, which the norm's pass read last
// and L2 still holds.
template <int K>
__global__ void __launch_bounds__(kClipThreads) grad_clip_kernel(const __grid_constant__ ClipTable<K> t) {
  grid_dependency_wait();
  grid_launch_dependents();
  const double norm = grad_norm_of(t.partials, t.num_partials);
  if (t.norm && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = static_cast<float>(norm);
  const double ratio = static_cast<double>(t.max_norm) / (norm + 1e-6);
  const ClipFactor coef(ratio >= 1.0 ? 1.0 : ratio);  // a NaN norm gives NaN
  clip_walk<true>(t, [&](int r, int64_t b, int64_t e) {
    const int kind = t.src_dtype[r] * 3 + t.dst_dtype[r];
    if (ratio >= 1.0 && t.src[r] == t.dst[r]) return;  // in place and below the limit: as it was
    const void* s = t.src[r];
    void* d = t.dst[r];
    switch (kind) {
      case 0: clip_piece_scale(static_cast<const float*>(s), static_cast<float*>(d), b, e, coef); break;
      case 3: clip_piece_scale(static_cast<const __half*>(s), static_cast<float*>(d), b, e, coef); break;
      case 4: clip_piece_scale(static_cast<const __half*>(s), static_cast<__half*>(d), b, e, coef); break;
      case 6: clip_piece_scale(static_cast<const __nv_bfloat16*>(s), static_cast<float*>(d), b, e, coef); break;
      case 8:
        clip_piece_scale(static_cast<const __nv_bfloat16*>(s), static_cast<__nv_bfloat16*>(d), b, e, coef);
        break;
      default: break;  // refused by the host
    }
  });
}

}  // namespace fssim
