// The AdamW step over many tensors at once: kernels for sm_100a (B200).
//
//   m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2,
//   p' = (1 - lr wd) p - lr / (1 - b1^t) * m' / (sqrt(v' / (1 - b2^t)) + eps)
//
// with g multiplied by min(1, max_norm / (norm + 1e-6)) on its way in, where a norm is given. Moments
// are FP32, or e4m3 codes of m and of sqrt(v) with an FP32 scale for each block of 256 numbers.
// Everything between a load and the one rounding to the stored type is FP32, each product and sum
// rounded by itself (no fused multiply-add): codes are drawn from these numbers' bits, and so do not
// depend on how a compiler pairs operations.
//
// A warp has a block of 256 numbers, eight to a lane, of which it holds all inputs in registers; the
// largest moment of a block is one redux instruction. The tensors are flat runs of memory named by
// a table in the kernel's parameters and dealt out to the grid in equal ranges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"
#include "runs.cuh"

namespace fssim {

constexpr int kAdamwThreads = 256;
constexpr int kAdamwBlock = 256;     // numbers that share a scale
constexpr int kAdamwResident = 3;    // CTAs on one SM
constexpr int kAdamwMaxCtas = 148 * kAdamwResident;
static_assert(kRunUnit == kAdamwThreads / 32 * kAdamwBlock, "a unit is one block for each warp");

// What a step's arithmetic takes besides the tensors.
struct AdamwStep {
  double beta1, beta2, eps, lr, weight_decay, max_norm;
  int64_t step;
  const float* step_at;  // device memory, or null: `step` holds
  const float* lr_at;    // device memory, or null: `lr` holds
  const float* norm;     // device memory, or null: no clipping
  uint32_t seed;
  int maximize;
};

// Runs of one launch.
template <int K>
struct AdamwTable {
  void* param[K];
  const void* grad[K];
  void* first[K];
  void* second[K];
  float* scales[K];
  void* copy[K];
  int64_t size[K];
  int64_t unit0[K + 1];
  uint32_t index[K];        // the tensor's position in the call
  unsigned char kind[K];    // adamw_kind
  unsigned char copy_dtype[K];
  int count;
  AdamwStep step;
};

// Types of a parameter and its gradient: 3 * param + grad.
__host__ __device__ constexpr int adamw_kind(int param, int grad) { return 3 * param + grad; }

struct AdamwScalars {
  float beta1, rest1, beta2, rest2, eps, lift, rate, decay, coef;
  uint32_t key;
};

// A one-to-one scrambling of 32-bit numbers: odd factors (from the digits of square roots) carry
// low bits up, shifts bring high bits down.
__device__ __forceinline__ uint32_t adamw_mix(uint32_t v) {
  v = (v ^ (v >> 15)) * 0xBB67AE85u;
  v = (v ^ (v >> 13)) * 0x3C6EF373u;
  return v ^ (v >> 16);
}
// 32 random bits for a number of a block: steps of 2^32 / golden ratio from the block's key, with
// half of the scrambling. The low 20 bits round the first moment, the high 20 the second's root;
// each is decided by its upper bits, which are the word's low and high halves.
__device__ __forceinline__ uint32_t adamw_random(uint32_t block_key, uint32_t at) {
  uint32_t v = block_key + at * 0x9E3779B1u;
  v = (v ^ (v >> 15)) * 0xBB67AE85u;
  return v ^ (v >> 15);
}

__device__ __forceinline__ AdamwScalars adamw_scalars(const AdamwStep& a) {
  AdamwScalars s;
  const double t = a.step_at ? static_cast<double>(*a.step_at) : static_cast<double>(a.step);
  const double lr = a.lr_at ? static_cast<double>(*a.lr_at) : a.lr;
  s.beta1 = static_cast<float>(a.beta1);
  s.rest1 = static_cast<float>(1.0 - a.beta1);
  s.beta2 = static_cast<float>(a.beta2);
  s.rest2 = static_cast<float>(1.0 - a.beta2);
  s.eps = static_cast<float>(a.eps);
  s.lift = static_cast<float>(1.0 / sqrt(1.0 - pow(a.beta2, t)));
  s.rate = static_cast<float>(lr / (1.0 - pow(a.beta1, t)));
  s.decay = static_cast<float>(1.0 - lr * a.weight_decay);
  double coef = 1.0;
  if (a.norm) {
    const double ratio = a.max_norm / (static_cast<double>(*a.norm) + 1e-6);
    coef = ratio >= 1.0 ? 1.0 : ratio;  // a NaN norm gives NaN
  }
  s.coef = static_cast<float>(a.maximize ? -coef : coef);
  s.key = adamw_mix(adamw_mix(a.seed) + static_cast<uint32_t>(static_cast<int64_t>(t)));
  return s;
}

// Eight numbers of a lane: consecutive ones (VEC), or 32 apart where the memory begins at no
// vector's boundary or ends within the block.
template <bool VEC>
__device__ __forceinline__ int adamw_place(int i) {
  const int lane = threadIdx.x % 32;
  return VEC ? lane * 8 + i : lane + 32 * i;
}

template <bool VEC, typename T>
__device__ __forceinline__ void adamw_load(const T* p, int valid, float (&f)[8]) {
  if constexpr (VEC) {
    constexpr int N = 16 / sizeof(T);
    const uint4* at = reinterpret_cast<const uint4*>(p) + threadIdx.x % 32 * (8 / N);
    uint4 raw[8 / N];
#pragma unroll
    for (int k = 0; k < 8 / N; ++k) raw[k] = __ldcs(at + k);
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = run_widen(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = adamw_place<false>(i);
      f[i] = at < valid ? run_widen(p[at]) : 0.f;
    }
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void adamw_store(T* p, int valid, const float (&f)[8]) {
  if constexpr (VEC) {
    constexpr int N = 16 / sizeof(T);
    uint4 raw[8 / N];
    T* e = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = run_narrow<T>(f[i]);
    uint4* at = reinterpret_cast<uint4*>(p) + threadIdx.x % 32 * (8 / N);
#pragma unroll
    for (int k = 0; k < 8 / N; ++k) __stcs(at + k, raw[k]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = adamw_place<false>(i);
      if (at < valid) p[at] = run_narrow<T>(f[i]);
    }
  }
}

// Eight e4m3 codes, as the numbers that they stand for times `scale`.
template <bool VEC>
__device__ __forceinline__ void adamw_load_codes(const unsigned char* p, int valid, float scale, float (&f)[8]) {
  unsigned char c[8];
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(c) = __ldcs(reinterpret_cast<const uint2*>(p) + threadIdx.x % 32);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = adamw_place<false>(i);
      c[i] = at < valid ? p[at] : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(c[2 * i] | c[2 * i + 1] << 8), __NV_E4M3);
    const float2 pair = __half22float2(__half2(h));
    f[2 * i] = __fmul_rn(pair.x, scale);
    f[2 * i + 1] = __fmul_rn(pair.y, scale);
  }
}

template <bool VEC>
__device__ __forceinline__ void adamw_store_codes(unsigned char* p, int valid, const float (&f)[8]) {
  unsigned char c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp8x2_storage_t pair =
        __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    c[2 * i] = static_cast<unsigned char>(pair & 0xFF);
    c[2 * i + 1] = static_cast<unsigned char>(pair >> 8);
  }
  if constexpr (VEC) {
    __stcs(reinterpret_cast<uint2*>(p) + threadIdx.x % 32, *reinterpret_cast<const uint2*>(c));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = adamw_place<false>(i);
      if (at < valid) p[at] = c[i];
    }
  }
}

constexpr uint32_t kInfBits = 0x7F800000u;

// The largest magnitude of a block that is finite (and at least 2^-100, so that its reciprocal is
// too), from the lanes' eight numbers; `odd` tells whether one is not.
__device__ __forceinline__ float adamw_top(const float (&f)[8], bool& odd) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  uint32_t top = __reduce_max_sync(0xffffffffu, most);
  odd = top >= kInfBits;
  if (odd) {
    most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(f[i]) & 0x7FFFFFFFu;
      if (bits < kInfBits) most = max(most, bits);
    }
    top = __reduce_max_sync(0xffffffffu, most);
  }
  return fmaxf(__uint_as_float(top), 0x1p-100f);
}

// Rounds |x| times `up` to three bits behind the first, upwards in as many of the 2^20 cases of `rnd`
// as its distance from the lower neighbour asks for: on average a code stands for x itself, and a
// slow change of a moment is not lost in the codes' steps (6 to 12 %), as it is when each step
// rounds to the nearest. Numbers below 2^-6 lie between codes of even distance and go to the nearest.
template <bool ROOT>
__device__ __forceinline__ float adamw_draw(float x, float up, uint32_t rnd) {
  float y = __fmul_rn(fabsf(x), up);
  if (ROOT && x > 0.f) y = fmaxf(y, 0x1p-6f);  // a root that is not zero stays so: it divides
  y = __uint_as_float((__float_as_uint(y) + rnd) & 0xFFF00000u);
  return ROOT ? y : copysignf(y, x);
}

struct AdamwRun {
  void* param;
  const void* grad;
  void* first;
  void* second;
  float* scales;
  void* copy;
  int copy_dtype;
  uint32_t key;
};

template <typename P, typename G, int BITS, bool VEC>
__device__ __forceinline__ void adamw_block(const AdamwRun& r, const AdamwScalars& s, int64_t b, int valid) {
  float p[8], g[8], m[8], v[8];
  adamw_load<VEC>(static_cast<const P*>(r.param) + b, valid, p);
  adamw_load<VEC>(static_cast<const G*>(r.grad) + b, valid, g);
  const int64_t block = b / kAdamwBlock;
  if constexpr (BITS == 32) {
    adamw_load<VEC>(static_cast<const float*>(r.first) + b, valid, m);
    adamw_load<VEC>(static_cast<const float*>(r.second) + b, valid, v);
  } else {
    const float scale1 = r.scales[2 * block], scale2 = r.scales[2 * block + 1];
    adamw_load_codes<VEC>(static_cast<const unsigned char*>(r.first) + b, valid, scale1, m);
    adamw_load_codes<VEC>(static_cast<const unsigned char*>(r.second) + b, valid, scale2, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], v[i]);
  }
  float root[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float gi = __fmul_rn(g[i], s.coef);
    m[i] = __fadd_rn(__fmul_rn(m[i], s.beta1), __fmul_rn(gi, s.rest1));
    v[i] = __fadd_rn(__fmul_rn(v[i], s.beta2), __fmul_rn(__fmul_rn(gi, gi), s.rest2));
    root[i] = __fsqrt_rn(v[i]);
    const float change = __fdiv_rn(m[i], __fadd_rn(__fmul_rn(root[i], s.lift), s.eps));
    p[i] = __fsub_rn(__fmul_rn(p[i], s.decay), __fmul_rn(change, s.rate));
  }
  adamw_store<VEC>(static_cast<P*>(r.param) + b, valid, p);
  if (sizeof(P) == 4 && r.copy) {
    if (r.copy_dtype == 1) adamw_store<VEC>(static_cast<__half*>(r.copy) + b, valid, p);
    else adamw_store<VEC>(static_cast<__nv_bfloat16*>(r.copy) + b, valid, p);
  }
  if constexpr (BITS == 32) {
    adamw_store<VEC>(static_cast<float*>(r.first) + b, valid, m);
    adamw_store<VEC>(static_cast<float*>(r.second) + b, valid, v);
  } else {
    bool odd1, odd2;
    const float top1 = adamw_top(m, odd1), top2 = adamw_top(root, odd2);
    const float up1 = __fmul_rn(__frcp_rn(top1), 448.f), up2 = __fmul_rn(__frcp_rn(top2), 448.f);
    if (threadIdx.x % 32 < 2)
      r.scales[2 * block + threadIdx.x % 32] = __fmul_rn(threadIdx.x % 32 ? top2 : top1, 1.f / 448.f);
    const uint32_t key = adamw_mix(r.key + static_cast<uint32_t>(block));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t rnd = adamw_random(key, adamw_place<VEC>(i));
      const bool bad1 = odd1 && !isfinite(m[i]), bad2 = odd2 && !isfinite(root[i]);
      m[i] = bad1 ? NAN : adamw_draw<false>(m[i], up1, rnd & 0xFFFFFu);
      root[i] = bad2 ? NAN : adamw_draw<true>(root[i], up2, rnd >> 12);
    }
    adamw_store_codes<VEC>(static_cast<unsigned char*>(r.first) + b, valid, m);
    adamw_store_codes<VEC>(static_cast<unsigned char*>(r.second) + b, valid, root);
  }
}

// The numbers [b, e) of a run, b a multiple of a unit.
template <typename P, typename G, int BITS>
__device__ __noinline__ void adamw_piece(const AdamwRun& r, const AdamwScalars& s, int64_t b, int64_t e) {
  const uintptr_t ends = reinterpret_cast<uintptr_t>(r.param) | reinterpret_cast<uintptr_t>(r.grad) |
                         reinterpret_cast<uintptr_t>(r.copy);
  const uintptr_t state = reinterpret_cast<uintptr_t>(r.first) | reinterpret_cast<uintptr_t>(r.second);
  const bool vectors = ends % 16 == 0 && state % (BITS == 32 ? 16 : 8) == 0;
  for (int64_t at = b + threadIdx.x / 32 * kAdamwBlock; at < e; at += kRunUnit) {
    if (vectors && at + kAdamwBlock <= e) adamw_block<P, G, BITS, true>(r, s, at, kAdamwBlock);
    else adamw_block<P, G, BITS, false>(r, s, at, static_cast<int>(min(e - at, int64_t{kAdamwBlock})));
  }
}

template <int BITS, int K>
__global__ void __launch_bounds__(kAdamwThreads, kAdamwResident)
    adamw_kernel(const __grid_constant__ AdamwTable<K> t) {
  __shared__ AdamwScalars s;
  grid_dependency_wait();
  grid_launch_dependents();
  if (threadIdx.x == 0) s = adamw_scalars(t.step);
  __syncthreads();
  const int64_t units = t.unit0[t.count];
  run_walk<false>(t, run_range(units, blockIdx.x, gridDim.x), run_range(units, blockIdx.x + 1, gridDim.x),
                   [&](int i, int64_t b, int64_t e) {
    const AdamwRun r{t.param[i], t.grad[i], t.first[i], t.second[i], t.scales[i], t.copy[i], t.copy_dtype[i],
                     adamw_mix(s.key + t.index[i])};
    switch (t.kind[i]) {
      case adamw_kind(0, 0): adamw_piece<float, float, BITS>(r, s, b, e); break;
      case adamw_kind(0, 1): adamw_piece<float, __half, BITS>(r, s, b, e); break;
      case adamw_kind(0, 2): adamw_piece<float, __nv_bfloat16, BITS>(r, s, b, e); break;
      case adamw_kind(1, 0): adamw_piece<__half, float, BITS>(r, s, b, e); break;
      case adamw_kind(1, 1): adamw_piece<__half, __half, BITS>(r, s, b, e); break;
      case adamw_kind(2, 0): adamw_piece<__nv_bfloat16, float, BITS>(r, s, b, e); break;
      case adamw_kind(2, 2): adamw_piece<__nv_bfloat16, __nv_bfloat16, BITS>(r, s, b, e); break;
      default: break;  // refused by the host
    }
  });
}

}  // namespace fssim
