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

#include <type_traits>

#include "pdl.cuh"
#include "runs.cuh"

namespace fssim {

constexpr int kAdamwThreads = 256;
constexpr int kAdamwBlock = 256;     // numbers that share a scale
// CTAs on one SM: with moments of 32 bits fewer streams at a time (59 million numbers 272 us, three 273; 100
// million in mixed precision 525 and 532), with those of 8 more warps for the arithmetic, of which unaligned
// tensors have most (20 million without gaps 112 us, two 113; whole units are as fast with two: 160
// million 429 and 425).
__host__ __device__ constexpr int adamw_resident(int bits) { return bits == 32 ? 2 : 3; }
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

// How a lane's eight numbers lie in a block: units of four or eight consecutive ones (16 bytes of the
// widest tensor, so that the lanes' accesses lie side by side), or 32 apart where the memory begins
// at no vector's boundary, or (the same, counted) where it ends within the block.
enum AdamwLie { kAdamwApart = 1, kAdamwFours = 4, kAdamwEights = 8, kAdamwEnd = 0 };
template <int LIE>
__device__ __forceinline__ int adamw_place(int i) {
  const int lane = threadIdx.x % 32;
  return LIE > 1 ? (i / LIE * 32 + lane) * LIE + i % LIE : lane + 32 * i;
}

// Eight numbers, as the packed FP32 instructions take them (each half rounded as by itself).
struct AdamwEight {
  float2 p[4];
  __device__ __forceinline__ float& operator[](int i) { return i & 1 ? p[i / 2].y : p[i / 2].x; }
  __device__ __forceinline__ float operator[](int i) const { return i & 1 ? p[i / 2].y : p[i / 2].x; }
};
__device__ __forceinline__ float2 adamw_twice(float v) { return make_float2(v, v); }

template <int BYTES> struct AdamwUnit;
template <> struct AdamwUnit<16> { using type = uint4; };
template <> struct AdamwUnit<8> { using type = uint2; };
template <> struct AdamwUnit<4> { using type = unsigned; };

// Eight numbers of a lane, as they are in memory.
template <typename T, int LIE>
struct alignas(16) AdamwRaw {
  T e[8];
  __device__ __forceinline__ void load(const void* from, int64_t b, int valid) {
    const T* p = static_cast<const T*>(from) + b;
    if constexpr (LIE > 1 && LIE * sizeof(T) <= 16) {
      using Unit = typename AdamwUnit<LIE * sizeof(T)>::type;
#pragma unroll
      for (int k = 0; k < 8 / LIE; ++k)
        reinterpret_cast<Unit*>(e)[k] = __ldcs(reinterpret_cast<const Unit*>(p) + k * 32 + threadIdx.x % 32);
    } else if constexpr (LIE > 1) {  // (32-bit gradients beside 16-bit parameters)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        reinterpret_cast<uint4*>(e)[k] = __ldcs(reinterpret_cast<const uint4*>(p) + threadIdx.x % 32 * 2 + k);
    } else {
      p += threadIdx.x % 32;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = LIE == kAdamwApart || adamw_place<LIE>(i) < valid ? p[32 * i] : T{};
    }
  }
  __device__ __forceinline__ void store(void* to, int64_t b, int valid) const {
    T* p = static_cast<T*>(to) + b;
    if constexpr (LIE > 1) {
      using Unit = typename AdamwUnit<LIE * sizeof(T)>::type;
#pragma unroll
      for (int k = 0; k < 8 / LIE; ++k)
        __stcs(reinterpret_cast<Unit*>(p) + k * 32 + threadIdx.x % 32, reinterpret_cast<const Unit*>(e)[k]);
    } else {
      p += threadIdx.x % 32;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (LIE == kAdamwApart || adamw_place<LIE>(i) < valid) p[32 * i] = e[i];
    }
  }
  __device__ __forceinline__ AdamwEight widen() const {
    AdamwEight f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = run_widen(e[i]);
    return f;
  }
  __device__ __forceinline__ void narrow(const AdamwEight& f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = run_narrow<T>(f[i]);
  }
};
template <int LIE, typename T>
__device__ __forceinline__ void adamw_store(void* to, int64_t b, int valid, const AdamwEight& f) {
  AdamwRaw<T, LIE> raw;
  raw.narrow(f);
  raw.store(to, b, valid);
}

// Eight e4m3 codes, as the numbers that they stand for times `scale`.
template <int LIE>
__device__ __forceinline__ AdamwEight adamw_decode(const AdamwRaw<unsigned char, LIE>& c, float scale) {
  AdamwEight f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(c.e[2 * i] | c.e[2 * i + 1] << 8), __NV_E4M3);
    f.p[i] = __fmul2_rn(__half22float2(__half2(h)), adamw_twice(scale));
  }
  return f;
}
template <int LIE>
__device__ __forceinline__ void adamw_store_codes(void* to, int64_t b, int valid, const AdamwEight& f) {
  AdamwRaw<unsigned char, LIE> raw;
  unsigned pair[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) pair[i] = __nv_cvt_float2_to_fp8x2(f.p[i], __NV_SATFINITE, __NV_E4M3);
  if constexpr (LIE > 1) {
    reinterpret_cast<unsigned*>(raw.e)[0] = __byte_perm(pair[0], pair[1], 0x5410);
    reinterpret_cast<unsigned*>(raw.e)[1] = __byte_perm(pair[2], pair[3], 0x5410);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.e[i] = static_cast<unsigned char>(i & 1 ? pair[i / 2] >> 8 : pair[i / 2]);
  }
  raw.store(to, b, valid);
}

constexpr uint32_t kInfBits = 0x7F800000u;

// The largest of two magnitudes; NaN where one is.
__device__ __forceinline__ float adamw_most(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
  return m;
}

// The largest magnitude of a block that is finite, from the lanes' eight numbers; `odd` tells whether one
// is not.
__device__ __forceinline__ float adamw_top(const AdamwEight& f, bool& odd) {
  float most = adamw_most(f[0], f[1]);
#pragma unroll
  for (int i = 2; i < 8; ++i) most = adamw_most(most, f[i]);
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7FFFFFFFu);
  odd = top >= kInfBits;
  if (odd) {
    uint32_t finite = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(f[i]) & 0x7FFFFFFFu;
      if (bits < kInfBits) finite = max(finite, bits);
    }
    top = __reduce_max_sync(0xffffffffu, finite);
  }
  return __uint_as_float(top);
}

// Rounds x times `up` to three bits behind the first, away from zero in as many of the 2^20 cases of
// `rnd` as its distance from the lower neighbour asks for: on average a code stands for x itself, and a
// slow change of a moment is not lost in the codes' steps (6 to 12 %), as it is when each step
// rounds to the nearest. Numbers below 2^-6 lie between codes of even distance and go to the nearest.
template <bool ROOT>
__device__ __forceinline__ float adamw_draw(float y, bool floor, uint32_t rnd) {
  if (ROOT) y = floor ? fmaxf(y, 0x1p-6f) : y;  // a root that is not zero stays so: it divides
  return __uint_as_float((__float_as_uint(y) + rnd) & 0xFFF00000u);
}

// Roots and quotients after P. Markstein (Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990): an approximation, and a correction by its exact remainder, which a
// fused multiply-add gives; without the branches that CUDA's functions have for each number. They
// are the correctly rounded ones where adamw_ordinary holds: compared are all 2^24 roots of two binades, and
// for each divisor's mantissa all quotients near enough to a border between two results to miss it.
__device__ __forceinline__ float2 adamw_root(float2 v) {
  float2 y;  // (of zero any that is finite)
  const float2 up = __fadd2_rn(v, adamw_twice(0x1p-120f));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(up.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(up.y));
  const float2 g = __fmul2_rn(v, y), h = __fmul2_rn(y, adamw_twice(0.5f));
  const float2 rest = __ffma2_rn(__fmul2_rn(g, adamw_twice(-1.f)), g, v);
  return __ffma2_rn(rest, h, g);
}
__device__ __forceinline__ float2 adamw_quotient(float2 m, float2 d) {
  float2 y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(d.y));
  const float2 minus = __fmul2_rn(d, adamw_twice(-1.f));
  y = __ffma2_rn(y, __ffma2_rn(minus, y, adamw_twice(1.f)), y);
  const float2 q = __fmul2_rn(m, y);
  return __ffma2_rn(__ffma2_rn(minus, q, m), y, q);
}
// Every second moment is zero or within 2^-80 and 2^80, and every first at most that (`most` is the
// largest). (The quotient of a first moment below 2^-80 may be off in its last place: it is nothing
// beside a parameter.)
__device__ __forceinline__ bool adamw_ordinary(const AdamwEight& v, float most) {
  uint32_t least = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < 8; ++i) least = min(least, __float_as_uint(v[i]) - 1u);  // (zero is the largest)
  return least >= 0x17800000u - 1u && most <= 0x1p80f;
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

// What a lane reads of a block.
template <typename P, typename G, int BITS, int LIE>
struct AdamwBlock {
  AdamwRaw<P, LIE> p;
  AdamwRaw<G, LIE> g;
  AdamwRaw<std::conditional_t<BITS == 32, float, unsigned char>, LIE> m, v;
  float scale1, scale2;
  __device__ __forceinline__ void load(const AdamwRun& r, int64_t b, int valid) {
    p.load(r.param, b, valid);
    g.load(r.grad, b, valid);
    m.load(r.first, b, valid);
    v.load(r.second, b, valid);
    if constexpr (BITS == 8) {
      const float* scales = r.scales + b / kAdamwBlock * 2;
      scale1 = scales[0];
      scale2 = scales[1];
    }
  }
};

template <typename P, typename G, int BITS, int LIE>
__device__ __forceinline__ void adamw_block(const AdamwRun& r, const AdamwScalars& s,
                                            const AdamwBlock<P, G, BITS, LIE>& in, int64_t b, int valid) {
  AdamwEight p = in.p.widen(), m, v, root;
  const AdamwEight g = in.g.widen();
  if constexpr (BITS == 32) {
    m = in.m.widen();
    v = in.v.widen();
  } else {
    m = adamw_decode(in.m, in.scale1);
    v = adamw_decode(in.v, in.scale2);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.p[i] = __fmul2_rn(v.p[i], v.p[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 gi = __fmul2_rn(g.p[i], adamw_twice(s.coef));
    m.p[i] = pair_add(__fmul2_rn(m.p[i], adamw_twice(s.beta1)), __fmul2_rn(gi, adamw_twice(s.rest1)));
    v.p[i] = pair_add(__fmul2_rn(v.p[i], adamw_twice(s.beta2)), __fmul2_rn(__fmul2_rn(gi, gi), adamw_twice(s.rest2)));
  }
  // the largest moments of the block (8 bits), or of the lane
  bool odd1 = false, odd2 = false;
  float top1, top2, most;
  if constexpr (BITS == 8) {
    top1 = adamw_top(m, odd1);
    top2 = adamw_top(v, odd2);
    most = odd1 || odd2 ? __uint_as_float(kInfBits) : fmaxf(top1, top2);
  } else {
    most = adamw_most(m[0], v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) most = adamw_most(most, adamw_most(m[i], v[i]));
  }
  const bool ordinary = s.eps >= 0x1p-60f && adamw_ordinary(v, most);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto den = [&] { return pair_add(__fmul2_rn(root.p[i], adamw_twice(s.lift)), adamw_twice(s.eps)); };
    float2 change;
    if (ordinary) {
      root.p[i] = adamw_root(v.p[i]);
      change = adamw_quotient(m.p[i], den());
    } else {
      root.p[i] = make_float2(__fsqrt_rn(v.p[i].x), __fsqrt_rn(v.p[i].y));
      const float2 d = den();
      change = make_float2(__fdiv_rn(m.p[i].x, d.x), __fdiv_rn(m.p[i].y, d.y));
    }
    p.p[i] = pair_add(__fmul2_rn(p.p[i], adamw_twice(s.decay)), __fmul2_rn(change, adamw_twice(-s.rate)));
  }
  adamw_store<LIE, P>(r.param, b, valid, p);
  if (sizeof(P) == 4 && r.copy) {
    if (r.copy_dtype == 1) adamw_store<LIE, __half>(r.copy, b, valid, p);
    else adamw_store<LIE, __nv_bfloat16>(r.copy, b, valid, p);
  }
  if constexpr (BITS == 32) {
    adamw_store<LIE, float>(r.first, b, valid, m);
    adamw_store<LIE, float>(r.second, b, valid, v);
  } else {
    const int64_t block = b / kAdamwBlock;
    // (the largest root is the largest v's; both are at least 2^-100, so that their reciprocals are finite)
    top1 = fmaxf(top1, 0x1p-100f);
    top2 = fmaxf(__fsqrt_rn(top2), 0x1p-100f);
    const float up1 = __fmul_rn(__frcp_rn(top1), 448.f), up2 = __fmul_rn(__frcp_rn(top2), 448.f);
    if (threadIdx.x % 32 < 2)
      r.scales[2 * block + threadIdx.x % 32] = __fmul_rn(threadIdx.x % 32 ? top2 : top1, 1.f / 448.f);
    const uint32_t key = adamw_mix(r.key + static_cast<uint32_t>(block));
    AdamwEight code1, code2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      code1.p[i] = __fmul2_rn(m.p[i], adamw_twice(up1));
      code2.p[i] = __fmul2_rn(root.p[i], adamw_twice(up2));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t rnd = adamw_random(key, adamw_place<LIE>(i));
      code1[i] = adamw_draw<false>(code1[i], false, rnd & 0xFFFFFu);
      code2[i] = adamw_draw<true>(code2[i], root[i] > 0.f, rnd >> 12);
    }
    if (odd1 || odd2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!isfinite(m[i])) code1[i] = NAN;
        if (!isfinite(root[i])) code2[i] = NAN;
      }
    }
    adamw_store_codes<LIE>(r.first, b, valid, code1);
    adamw_store_codes<LIE>(r.second, b, valid, code2);
  }
}

// The numbers [b, e) of a run, b a multiple of a unit.
template <typename P, typename G, int BITS>
__device__ __noinline__ void adamw_piece(const AdamwRun run, const AdamwScalars* scalars, int64_t b, int64_t e) {
  const AdamwRun r = run;
  const AdamwScalars s = *scalars;
  constexpr int kUnits = BITS == 32 || sizeof(P) == 4 ? kAdamwFours : kAdamwEights;
  const uintptr_t ends = reinterpret_cast<uintptr_t>(r.param) | reinterpret_cast<uintptr_t>(r.grad) |
                         reinterpret_cast<uintptr_t>(r.copy);
  const uintptr_t state = reinterpret_cast<uintptr_t>(r.first) | reinterpret_cast<uintptr_t>(r.second);
  const bool vectors = ends % 16 == 0 && state % (BITS == 32 ? 16 : 8) == 0;
  int64_t at = b + threadIdx.x / 32 * kAdamwBlock;
  // Moments of 8 bits in whole units: the next block is on its way while one is worked on (few bytes for
  // much arithmetic); elsewhere the other warps' are enough.
  const auto whole = [&](auto lie) {
    constexpr bool kAhead = BITS == 8 && decltype(lie)::value > 1;
    using Block = AdamwBlock<P, G, BITS, decltype(lie)::value>;
    if (at + kAdamwBlock > e) return;
    Block next;
    if (kAhead) next.load(r, at, kAdamwBlock);
    for (; at + kAdamwBlock <= e; at += kRunUnit) {
      Block now;
      if (kAhead) {
        now = next;
        if (at + kRunUnit + kAdamwBlock <= e) next.load(r, at + kRunUnit, kAdamwBlock);
      } else {
        now.load(r, at, kAdamwBlock);
      }
      adamw_block(r, s, now, at, kAdamwBlock);
    }
  };
  if (vectors) whole(std::integral_constant<int, kUnits>{});
  else whole(std::integral_constant<int, kAdamwApart>{});
  if (at < e) {
    AdamwBlock<P, G, BITS, kAdamwEnd> last;
    last.load(r, at, static_cast<int>(e - at));
    adamw_block(r, s, last, at, static_cast<int>(e - at));
  }
}

// Moments of 32 bits: bound by DRAM (59 million FP32, 28 bytes a number, 271 us, 6.1 TB/s; 100 million in
// mixed precision, 300 tensors, 490 us, 5.7 TB/s). Of 8 bits: by arithmetic, some 70 instructions a number
// for 10 bytes (160 million BF16 428 us, 3.8 TB/s).
template <int BITS, int K>
__global__ void __launch_bounds__(kAdamwThreads, adamw_resident(BITS))
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
      case adamw_kind(0, 0): adamw_piece<float, float, BITS>(r, &s, b, e); break;
      case adamw_kind(0, 1): adamw_piece<float, __half, BITS>(r, &s, b, e); break;
      case adamw_kind(0, 2): adamw_piece<float, __nv_bfloat16, BITS>(r, &s, b, e); break;
      case adamw_kind(1, 0): adamw_piece<__half, float, BITS>(r, &s, b, e); break;
      case adamw_kind(1, 1): adamw_piece<__half, __half, BITS>(r, &s, b, e); break;
      case adamw_kind(2, 0): adamw_piece<__nv_bfloat16, float, BITS>(r, &s, b, e); break;
      case adamw_kind(2, 2): adamw_piece<__nv_bfloat16, __nv_bfloat16, BITS>(r, &s, b, e); break;
      default: break;  // refused by the host
    }
  });
}

}  // namespace fssim
