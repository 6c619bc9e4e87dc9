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

// Eight consecutive numbers at a 16-byte boundary: as they lie in memory (16 or 32 bytes, so that
// several such loads can be in flight before the first is converted), and as FP32.
template <typename T> struct ClipVec;
template <> struct ClipVec<float> {
  struct Raw { float4 a, b; };
  static __device__ __forceinline__ Raw load8(const float* p) {
    return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
    f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void store8(float* p, const float* f) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  static __device__ __forceinline__ void put(float* p, float f) { *p = f; }
};
__device__ __forceinline__ float2 clip_widen(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 clip_widen(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ void clip_narrow(__half2& v, float a, float b) { v = __floats2half2_rn(a, b); }
__device__ __forceinline__ void clip_narrow(__nv_bfloat162& v, float a, float b) {
  v = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void clip_narrow(__half& v, float a) { v = __float2half_rn(a); }
__device__ __forceinline__ void clip_narrow(__nv_bfloat16& v, float a) { v = __float2bfloat16_rn(a); }
template <typename T, typename T2>
struct ClipVec16 {
  using Raw = uint4;
  static __device__ __forceinline__ Raw load8(const T* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) {
    const T2* h = reinterpret_cast<const T2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = clip_widen(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ float one(const T* p) { return static_cast<float>(*p); }
  static __device__ __forceinline__ void store8(T* p, const float* f) {
    uint4 v;
    T2* h = reinterpret_cast<T2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) clip_narrow(h[i], f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
  static __device__ __forceinline__ void put(T* p, float f) { clip_narrow(*p, f); }
};
template <>
struct ClipVec<__half> : ClipVec16<__half, __half2> {};
template <>
struct ClipVec<__nv_bfloat16> : ClipVec16<__nv_bfloat16, __nv_bfloat162> {};

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
  using IO = ClipVec<T>;
  constexpr int U = 128 / sizeof(typename IO::Raw);  // 128 bytes of a thread in flight
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * kClipThreads < n8; i += U * kClipThreads) {
    typename IO::Raw raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = IO::load8(src + body + (i + u * kClipThreads) * 8);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      IO::unpack(raw[u], f);
      acc += sum_squares8(f);
    }
  }
  for (; i < n8; i += kClipThreads) {
    float f[8];
    IO::unpack(IO::load8(src + body + i * 8), f);
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
  using IO = ClipVec<S>;
  constexpr int U = 64 / sizeof(typename IO::Raw);
  const auto emit = [&](const typename IO::Raw& raw, int64_t at) {
    float f[8];
    IO::unpack(raw, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = coef * f[k];
    ClipVec<D>::store8(dst + body + at * 8, f);
  };
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * kClipThreads < n8; i += U * kClipThreads) {
    typename IO::Raw raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = IO::load8(src + body + (i + u * kClipThreads) * 8);
#pragma unroll
    for (int u = 0; u < U; ++u) emit(raw[u], i + u * kClipThreads);
  }
  for (; i < n8; i += kClipThreads) emit(IO::load8(src + body + i * 8), i);
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
