// Global gradient norm over many tensors, and clipping: kernels for sm_100a (B200).
//
//   norm = sqrt(sum over all tensors of g^2),  coef = min(1, max_norm / (norm + 1e-6)),
//   out = coef * g
//
// The tensors are flat runs of memory, named by a table in the kernel's parameters (so a
// captured launch carries its own copy, and no device memory or copy is needed for it). Each
// run is cut into units of kRunUnit numbers; the units of all runs, end to end, are split
// over the grid in equal contiguous ranges, so every CTA streams the same number of bytes
// whatever the tensors' sizes. A CTA finds its first run by bisection and walks on from there.
//
// Norm: squares are summed in FP32 over the numbers of a thread's batch of vectors (16 or 32) and in
// FP64 from there on; a batch whose FP32 sum leaves the range where squares are exact enough is
// summed again in FP64, where the square of an FP32 number neither overflows nor vanishes. One
// FP64 partial per CTA, summed in a fixed order by whoever needs the norm: results repeat bit
// for bit, and the workspace needs no initial value.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"
#include "runs.cuh"

namespace fssim {

constexpr int kClipThreads = 256;
constexpr int kClipResident = 3;    // CTAs on one SM
constexpr int kClipMaxCtas = 148 * kClipResident;
// The clipping copies vectors asynchronously into a ring of kClipRing batches of kClipBatch vectors
// for each thread in shared memory (slots of its own: no barrier), ahead of their use.
constexpr int kClipBatch = 4;
constexpr int kClipRing = 4;
constexpr int kClipRingBytes = kClipThreads * 16 * kClipBatch * kClipRing;

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
  double* partials;       // of the whole call, or their sum
  int num_partials;       // of the whole call
  int first_partial;      // of this launch's CTAs
  float* norm;            // written by the launch that has it set
  float max_norm;
  int ranges;             // CTAs of the norm's pass, each with a range of units
  int cuts;               // CTAs of the clipping for each range
  float keep;             // share of the gradients that may stay in L2 from the norm to the clipping
};

// N consecutive numbers in one access of up to 16 bytes.
template <int BYTES> struct ClipRaw;
template <> struct ClipRaw<16> { using type = uint4; };
template <> struct ClipRaw<8> { using type = uint2; };

template <typename T, int N>
struct ClipVec {
  using Raw = typename ClipRaw<sizeof(T) * N>::type;
  static __device__ __forceinline__ Raw load(const T* p, uint64_t policy) {
    static_assert(sizeof(Raw) == 16, "whole vectors");
    Raw r;
    asm volatile("ld.global.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p), "l"(policy));
    return r;
  }
  static __device__ __forceinline__ void copy(unsigned slot, const T* p, uint64_t policy) {
    if constexpr (sizeof(Raw) == 16)
      asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(slot), "l"(p),
                   "l"(policy) : "memory");
    else
      asm volatile("cp.async.ca.shared.global.L2::cache_hint [%0], [%1], 8, %2;" ::"r"(slot), "l"(p),
                   "l"(policy) : "memory");
  }
  static __device__ __forceinline__ Raw take(unsigned slot) {
    Raw r;
    if constexpr (sizeof(Raw) == 16)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(slot) : "memory");
    else
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(slot) : "memory");
    return r;
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = run_widen(e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[N], uint64_t policy) {
    Raw r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = run_narrow<T>(f[i]);
    if constexpr (sizeof(Raw) == 16)
      asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(p), "r"(r.x),
                   "r"(r.y), "r"(r.z), "r"(r.w), "l"(policy) : "memory");
    else
      asm volatile("st.global.L2::cache_hint.v2.u32 [%0], {%1, %2}, %3;" ::"l"(p), "r"(r.x), "r"(r.y),
                   "l"(policy) : "memory");
  }
};

// L2 priorities, for gradients that are larger than it (keep < 1): the last `keep` of what a CTA
// reads for the norm is to stay for the clipping, which reads it first; all else, and what is
// written, goes past it.
struct ClipPolicy {
  uint64_t stay, pass;
  __device__ __forceinline__ explicit ClipPolicy(bool large) {
    asm("createpolicy.fractional.L2::evict_normal.b64 %0;" : "=l"(stay));
    asm("createpolicy.fractional.L2::evict_first.b64 %0;" : "=l"(pass));
    if (!large) pass = stay;
  }
};

// Squares of a batch's numbers (missing vectors are zero), added up with the packed FP32
// instructions, as a tree: at most six roundings on the way of any term. Between 2^-80 and 2^100
// that is right: no term overflowed, and what underflowed is below 2^-46 of the sum.
template <typename T, int N>
__device__ __forceinline__ double sum_squares(const typename ClipVec<T, N>::Raw (&raw)[kClipBatch]) {
  static_assert(kClipBatch == 4, "summed as a tree");
  float2 sum[kClipBatch];
#pragma unroll
  for (int u = 0; u < kClipBatch; ++u) {
    float f[N];
    ClipVec<T, N>::unpack(raw[u], f);
    float2 part[2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 v = make_float2(f[2 * i], f[2 * i + 1]);
      part[i & 1] = i < 2 ? __fmul2_rn(v, v) : __ffma2_rn(v, v, part[i & 1]);
    }
    sum[u] = __fadd2_rn(part[0], part[1]);
  }
  const float2 pair = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
  const float s = pair.x + pair.y;
  if (s < 0x1p-80f || s > 0x1p100f) {
    double w = 0.0;
#pragma unroll
    for (int u = 0; u < kClipBatch; ++u) {
      float f[N];
      ClipVec<T, N>::unpack(raw[u], f);
      unsigned bits = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) bits |= __float_as_uint(f[i]) << 1;
      if (bits == 0) continue;  // all zero, as gradients of what was not seen are
#pragma unroll
      for (int i = 0; i < N; ++i) w = fma(static_cast<double>(f[i]), static_cast<double>(f[i]), w);
    }
    return w;
  }
  return s;  // NaN too
}

// Numbers before the first 16-byte boundary of p + b, at most e - b.
template <typename T>
__device__ __forceinline__ int64_t clip_head(const T* p, int64_t b, int64_t e) {
  const int64_t off = static_cast<int64_t>((reinterpret_cast<uintptr_t>(p + b) % 16) / sizeof(T));
  const int64_t head = off ? 16 / static_cast<int64_t>(sizeof(T)) - off : 0;
  return min(head, e - b);
}

// Clipping: use(batch, vector, k) for the vectors of N numbers [0, n) of a piece at `src`, those of a
// thread kClipThreads apart, from the last to the first. A batch begins at that vector and has
// k of them (more than kClipBatch stands for all).
template <int N, typename T, typename Use>
__device__ __forceinline__ void clip_vectors(const T* src, int64_t n, uint64_t policy, Use use) {
  using IO = ClipVec<T, N>;
  constexpr int U = kClipBatch, B = kClipRing;
  extern __shared__ __align__(16) unsigned char clip_ring[];
  const unsigned ring = static_cast<unsigned>(__cvta_generic_to_shared(clip_ring)) + threadIdx.x * 16;
  const int64_t count = threadIdx.x < n ? (n - threadIdx.x - 1) / kClipThreads + 1 : 0;
  const int64_t first = threadIdx.x + (count - 1) * kClipThreads;
  constexpr int64_t step = -static_cast<int64_t>(kClipThreads);
  const T* next = src + first * N;
  int64_t todo = count, left = count, at = first;
  const auto start = [&](int slot) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < todo) IO::copy(ring + (slot * U + u) * kClipThreads * 16, next + u * step * N, policy);
    asm volatile("cp.async.commit_group;" ::: "memory");
    next += U * step * N;
    todo -= U;
  };
#pragma unroll
  for (int b = 0; b < B - 1; ++b) start(b);
  while (left > 0) {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      start((b + B - 1) % B);
      asm volatile("cp.async.wait_group %0;" ::"n"(B - 1) : "memory");
      typename IO::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) raw[u] = IO::take(ring + (b * U + u) * kClipThreads * 16);
        else raw[u] = typename IO::Raw{};
      use(raw, at, left);
      left -= U;
      at += U * step;
      if (left <= 0) break;
    }
  }
}

template <typename T>
__device__ __noinline__ double clip_piece_squares(const T* src, int64_t b, int64_t e, uint64_t policy) {
  constexpr int N = 16 / sizeof(T);
  const int64_t head = clip_head(src, b, e);
  const int64_t body = b + head;
  const int64_t n = (e - body) / N;
  const int64_t tail = body + n * N;
  double acc = 0.0;
  // what is left at the two ends: fewer than N numbers each
  const int64_t ends = head + (e - tail);
  if (threadIdx.x < ends) {
    const int64_t at = threadIdx.x < head ? b + threadIdx.x : tail + (threadIdx.x - head);
    const double v = run_widen(src[at]);
    acc = v * v;
  }
  // Read straight into registers: this pass writes nothing, and on its way through shared memory the
  // same data would cross the SM's load path twice (236 MB: 40 against 45 us on a B200).
  using IO = ClipVec<T, N>;
  const T* at = src + body + threadIdx.x * N;
  constexpr int kStep = kClipBatch * kClipThreads;
  int64_t left = n - threadIdx.x;
#pragma unroll 1
  for (; left > kStep - kClipThreads + kStep; left -= 2 * kStep, at += 2 * kStep * N) {
    typename IO::Raw a[kClipBatch], b[kClipBatch];
#pragma unroll
    for (int u = 0; u < kClipBatch; ++u) a[u] = IO::load(at + u * kClipThreads * N, policy);
#pragma unroll
    for (int u = 0; u < kClipBatch; ++u) b[u] = IO::load(at + (kStep + u * kClipThreads) * N, policy);
    acc += sum_squares<T, N>(a);
    acc += sum_squares<T, N>(b);
  }
#pragma unroll 1
  for (; left > 0; left -= kStep, at += kStep * N) {
    typename IO::Raw a[kClipBatch];
#pragma unroll
    for (int u = 0; u < kClipBatch; ++u) {
      a[u] = typename IO::Raw{};
      if (u * kClipThreads < left) a[u] = IO::load(at + u * kClipThreads * N, policy);
    }
    acc += sum_squares<T, N>(a);
  }
  return acc;
}

// The factor, as an FP32 number and what its rounding lost, so that a scaled number is rounded once:
// with the rounded factor alone it would be off by up to two halves of a step. One below 2^-96
// (a norm near or beyond FP32's largest number) is carried as 2^64 times itself, so that both
// keep their bits, and the product times 2^-64.
struct ClipFactor {
  float high, low, back;
  __device__ __forceinline__ explicit ClipFactor(double c) {
    const bool tiny = c < 0x1p-96;
    if (tiny) c *= 0x1p64;
    high = static_cast<float>(c);
    low = static_cast<float>(c - high);
    back = tiny ? 0x1p-64f : 1.f;
  }
  __device__ __forceinline__ float operator*(float v) const { return fmaf(v, high, v * low) * back; }
};

template <typename S, typename D>
__device__ __noinline__ void clip_piece_scale(const S* src, D* dst, int64_t b, int64_t e, ClipFactor coef,
                                                 uint64_t policy) {
  // 16 bytes of the wider type, so that the lanes of a warp write one run of memory
  constexpr int N = 16 / (sizeof(S) > sizeof(D) ? sizeof(S) : sizeof(D));
  const int64_t head = clip_head(src, b, e);
  const int64_t body = b + head;
  if (reinterpret_cast<uintptr_t>(dst + body) % 16 != 0) {
    // The two sides' boundaries differ: number by number, still in whole rows of a warp (420 BF16
    // tensors of their own memory into a gap-free FP32 buffer: 691 us, 217 where both are packed
    // alike).
#pragma unroll 8
    for (int64_t i = b + threadIdx.x; i < e; i += kClipThreads)
      dst[i] = run_narrow<D>(coef * run_widen(src[i]));
    return;
  }
  const int64_t n = (e - body) / N;
  const int64_t tail = body + n * N;
  clip_vectors<N>(src + body, n, policy, [&](const auto& raw, int64_t i, int64_t k) {
#pragma unroll
    for (int u = 0; u < kClipBatch; ++u)
      if (u < k) {
        float f[N];
        ClipVec<S, N>::unpack(raw[u], f);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = coef * f[j];
        ClipVec<D, N>::store(dst + body + (i - u * kClipThreads) * N, f, policy);
      }
  });
  const int64_t ends = head + (e - tail);
  if (threadIdx.x < ends) {
    const int64_t at = threadIdx.x < head ? b + threadIdx.x : tail + (threadIdx.x - head);
    dst[at] = run_narrow<D>(coef * run_widen(src[at]));
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

// Bound by DRAM: 59 million FP32 in six tensors (236 MB) 40 us, 5.9 TB/s; 160 million BF16 in 420
// tensors (320 MB) 60 us, 5.4 TB/s, less for the start of each piece of a tensor.
template <int K>
__global__ void __launch_bounds__(kClipThreads, kClipResident)
    grad_squares_kernel(const __grid_constant__ ClipTable<K> t) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t units = t.unit0[t.count];
  const int64_t u0 = run_range(units, blockIdx.x, gridDim.x), u1 = run_range(units, blockIdx.x + 1, gridDim.x);
  const ClipPolicy policies(t.keep < 1.f);
  const int64_t split = u1 - static_cast<int64_t>(static_cast<float>(u1 - u0) * min(t.keep, 1.f));
  double acc = 0.0;
  for (int part = 0; part < 2; ++part) {  // what goes past L2, then what stays
    const uint64_t policy = part ? policies.stay : policies.pass;
    run_walk<false>(t, part ? split : u0, part ? u1 : split, [&](int r, int64_t b, int64_t e) {
      if (t.src_dtype[r] == 0) acc += clip_piece_squares(static_cast<const float*>(t.src[r]), b, e, policy);
      else if (t.src_dtype[r] == 1) acc += clip_piece_squares(static_cast<const __half*>(t.src[r]), b, e, policy);
      else acc += clip_piece_squares(static_cast<const __nv_bfloat16*>(t.src[r]), b, e, policy);
    });
  }
  acc = clip_block_sum(acc);
  if (threadIdx.x == 0) t.partials[t.first_partial + blockIdx.x] = acc;
}

__device__ __forceinline__ double grad_sum_of(const double* partials, int n) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kClipThreads) v += partials[i];
  return clip_block_sum(v);
}

// The partial sums' sum, in `total` (if given), and its root.
__global__ void __launch_bounds__(kClipThreads) grad_norm_kernel(const double* partials, int n, double* total,
                                                                 float* norm) {
  grid_dependency_wait();
  grid_launch_dependents();
  const double v = grad_sum_of(partials, n);
  if (threadIdx.x == 0) {
    if (total) *total = v;
    *norm = static_cast<float>(sqrt(v));
  }
}

// The second read begins at the ends of the norm's pass's ranges, which that pass read last and L2
// still holds: a range is cut into `cuts` pieces, and the CTAs take the last piece of every range
// first. Bound by DRAM: 59 million FP32 (236 MB in and out) 80 us, 5.2 TB/s; 160 million BF16
// into FP32 (320 MB in, 640 out) 162 us, 5.6 TB/s.
template <int K>
__global__ void __launch_bounds__(kClipThreads, kClipResident)
    grad_clip_kernel(const __grid_constant__ ClipTable<K> t) {
  grid_dependency_wait();
  grid_launch_dependents();
  const double norm = sqrt(grad_sum_of(t.partials, t.num_partials));
  if (t.norm && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = static_cast<float>(norm);
  const double ratio = static_cast<double>(t.max_norm) / (norm + 1e-6);
  const ClipFactor coef(ratio >= 1.0 ? 1.0 : ratio);  // a NaN norm gives NaN
  const uint64_t policy = ClipPolicy(t.keep < 1.f).pass;
  const int64_t units = t.unit0[t.count];
  const int cut = t.cuts - 1 - blockIdx.x / t.ranges, range = blockIdx.x % t.ranges;
  const int64_t u0 = run_range(units, range, t.ranges), n = run_range(units, range + 1, t.ranges) - u0;
  run_walk<true>(t, u0 + run_range(n, cut, t.cuts), u0 + run_range(n, cut + 1, t.cuts),
                  [&](int r, int64_t b, int64_t e) {
    if (ratio >= 1.0 && t.src[r] == t.dst[r]) return;  // in place and below the limit: as it was
    const void* s = t.src[r];
    void* d = t.dst[r];
    const auto scale = [&](auto* src, auto* dst) { clip_piece_scale(src, dst, b, e, coef, policy); };
    switch (t.src_dtype[r] * 3 + t.dst_dtype[r]) {
      case 0: scale(static_cast<const float*>(s), static_cast<float*>(d)); break;
      case 3: scale(static_cast<const __half*>(s), static_cast<float*>(d)); break;
      case 4: scale(static_cast<const __half*>(s), static_cast<__half*>(d)); break;
      case 6: scale(static_cast<const __nv_bfloat16*>(s), static_cast<float*>(d)); break;
      case 8: scale(static_cast<const __nv_bfloat16*>(s), static_cast<__nv_bfloat16*>(d)); break;
      default: break;  // refused by the host
    }
  });
}

}  // namespace fssim
