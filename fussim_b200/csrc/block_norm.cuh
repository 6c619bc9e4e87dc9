// Norms before and after a residual block, with its gate and modulation: kernels for sm_100a (B200).
//
//   r = x + s * gate * (after(y) * after_weight + after_bias)        rounded to x's type
//   z = (before(r) * weight + bias) * (1 + scale) + shift            of y's type
//
// A norm takes a row of C numbers to (v - mean) * rstd with rstd = 1 / sqrt(<(v - mean)^2> + eps); the
// "rms" kind has mean = 0. Each of the vectors of C numbers may be missing, and gate, scale and shift may have
// one for each of B samples of T rows. Backwards, with a = weight * (1 + scale), rhat and yhat the
// normalised rows, <> a row's mean (the first of the two only in the "layer" kind):
//
//   dR = dr + rstd_r * (a dz - <a dz> - rhat <a dz rhat>),   dx = dR
//   e  = s * gate * after_weight * dR,   dy = rstd_y * (e - <e> - yhat <e yhat>)
//
// and every gradient of a vector follows from four sums over a sample's rows, of dz, dz rhat, dR and
// dR yhat: dshift = sum dz, dscale = weight sum dz rhat + bias sum dz, and so on.
//
// A row belongs to part of a warp, a warp, or a CTA of up to 512 threads; a thread has V groups of eight
// of its numbers, the same columns from row to row of its CTA's rows. Rows come ahead of their use
// through a ring in shared memory, in which a thread copies and reads slots of its own (no barrier); the
// vectors, combined as the arithmetic takes them, are laid there once by each CTA; the four sums stay
// in registers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "pdl.cuh"
#include "runs.cuh"

namespace fssim {

constexpr int kBlockMaxThreads = 512;  // of a row
constexpr int kBlockMaxC = kBlockMaxThreads * 8 * 4;

enum BlockKind { kBlockNone = 0, kBlockRms = 1, kBlockLayer = 2 };

// What a kernel is compiled for: no block's output, one that is added as it is, and one with a norm
// (which also does for the other two, where there are no kernels of one mode alone).
enum BlockMode { kBlockBefore = 0, kBlockPlain = 1, kBlockAfter = 2 };

// C numbers, or C for each sample.
struct BlockChannels {
  const void* data;  // or null
  int dtype;
  int per_sample;
  int wide;          // whole 16-byte vectors at every multiple of eight columns
};

// The vectors as the kernels take them: s * gate (forward; of 16-bit rows whose branch has a norm, gate
// alone), weight * (1 + scale), bias * (1 + scale) + shift, after_weight, after_bias; backward, the first
// is s * gate * after_weight.
enum BlockArray { kArrayGate, kArrayFactor, kArrayOffset, kArrayAfterWeight, kArrayAfterBias, kArrays };

struct BlockParams {
  int64_t T;              // rows of a sample
  int64_t chunk;          // rows of a CTA
  int64_t chunks;         // CTAs of a sample
  int C;
  int threads;            // of a row
  int kind, after_kind;   // BlockKind
  float eps;
  double s, inv;          // inv: 1 / C
  int stages;             // of the ring of rows
  int arrays;             // bit k: array k is not all ones or zeros
  const void* x;          // forward
  const void* y;
  void* r;
  void* z;
  float2* stats;          // (mean, rstd) of each row of r; or null
  float2* after_stats;
  BlockChannels gate, weight, bias, scale, shift, after_weight, after_bias;
  // backward: r is read, and
  const void* dr;
  const void* dz;
  void* dx;
  void* dy;
  float* partials;        // (CTA, sum, C); null: no vector's gradient is asked for
  int sums;               // 2 (dz's alone) to 4
};

// Eight numbers, as the packed FP32 instructions take them.
struct Eight {
  float2 p[4];
  __device__ __forceinline__ float& operator[](int i) { return i & 1 ? p[i / 2].y : p[i / 2].x; }
  __device__ __forceinline__ float operator[](int i) const { return i & 1 ? p[i / 2].y : p[i / 2].x; }
};
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
__device__ __forceinline__ Eight eight(float v) { return {twice(v), twice(v), twice(v), twice(v)}; }
// f(pair of a, pair of b, ...) of all pairs.
template <typename F, typename... A>
__device__ __forceinline__ Eight pairs(F f, const A&... a) {
  Eight r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = f(a.p[i]...);
  return r;
}

__device__ __forceinline__ float2 block_widen2(float2 v) { return v; }
__device__ __forceinline__ float2 block_widen2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 block_widen2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
template <typename T> struct BlockPair { using type = float2; };
template <> struct BlockPair<__half> { using type = __half2; };
template <> struct BlockPair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <typename T> __device__ __forceinline__ typename BlockPair<T>::type block_narrow2(float2 v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float22half2_rn(v);
  else return __float22bfloat162_rn(v);
}
// Eight numbers in a type's memory form.
template <typename T>
struct alignas(16) BlockPacked {
  typename BlockPair<T>::type p[4];
  __device__ __forceinline__ Eight widen() const {
    return {block_widen2(p[0]), block_widen2(p[1]), block_widen2(p[2]), block_widen2(p[3])};
  }
  static __device__ __forceinline__ BlockPacked of(const Eight& f) {
    return {block_narrow2<T>(f.p[0]), block_narrow2<T>(f.p[1]), block_narrow2<T>(f.p[2]), block_narrow2<T>(f.p[3])};
  }
};

// A thread's place in a row: number i of its group v is in column at(v, i). Columns go out to the row's
// threads in turn by units that are 16 bytes of x: eight numbers of 16 bits, four of 32 (so that
// the threads' accesses lie side by side); single numbers where rows begin at no vector's boundary.
// The last of the V groups alone may lack some.
template <int UNIT, int V>
struct BlockColumns {
  int threads, tid, C;
  bool full;  // the last group has all its numbers, too
  __device__ __forceinline__ int at(int v, int i) const {
    return ((v * 8 + i) / UNIT * threads + tid) * UNIT + i % UNIT;
  }
  __device__ __forceinline__ bool inside(int v, int i) const {
    return v < V - 1 || full || at(v, i / UNIT * UNIT) < C;
  }
  // Zeros in place of what is past the row's end.
  __device__ __forceinline__ Eight keep(Eight f, int v) const {
    if (v == V - 1 && !full)
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = inside(v, i) ? f[i] : 0.f;
    return f;
  }
};

// ---- rows ----
// The ring: stages x warps x units x lanes: a warp copies whole runs of memory, at offsets that are
// known when compiled. Copies of one row are a group; the last stages - 1 groups are on their way
// while a row is worked on. What has no number, past a row's end or the last row, is filled with zeros.
constexpr int kBlockStages = 2;  // at most
struct BlockRing {
  unsigned char* memory;  // this warp's part of the first stage
  unsigned bytes;         // of a stage
  int stages, put = 0, get = 0;
  // `warp`: bytes of a warp's part of a stage
  __device__ __forceinline__ BlockRing(unsigned char* ring, int warp, int stages)
      : memory(ring + threadIdx.x / 32 * warp), bytes(warp * (blockDim.x / 32)), stages(stages) {}
  __device__ __forceinline__ unsigned char* next(int& at) const {
    unsigned char* slot = memory + at * bytes;
    at = at + 1 == stages ? 0 : at + 1;
    return slot;
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ void wait() const {
    // (the number is part of the instruction)
    if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // The last turns' copies, of zeros: they have to be over before the memory is anything else's (a barrier
  // orders no copy that is on its way).
  static __device__ __forceinline__ void drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }
};

// A thread's numbers of one tensor's row: through the ring, or (single numbers) loaded into registers.
// Offsets are of the row's first number.
template <typename T, int V, int UNIT>
struct BlockRow {
  static constexpr bool kVec = UNIT > 1;
  static constexpr int kPiece = UNIT * sizeof(T), kPieces = V * 8 / UNIT;  // bytes of a unit, units of a thread
  static constexpr int kBytes = kVec ? kPieces * kPiece * 32 : 0;          // of a warp's part of a stage
  using Bits = std::conditional_t<sizeof(T) == 4, unsigned, unsigned short>;
  // Of single numbers, eight are held (a register for each, also of 16 bits: to pack two the loads would
  // have to be waited for). Of longer rows only the place is, and they are read where they are used, for
  // each turn again, which caches serve (2 x 700 x 7001 FP32 to BF16 forward 51 us; held, they spilled: 287).
  static constexpr bool kHeld = !kVec && V == 1;
  unsigned one[kHeld ? 8 : 1];
  const Bits* place;

  static __device__ __forceinline__ void copy(unsigned char* slot, const void* from, int64_t offset,
                                              const BlockColumns<UNIT, V>& c, bool active) {
    const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(slot)) + threadIdx.x % 32 * kPiece;
    const T* row = static_cast<const T*>(from) + offset;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int at = c.at(0, k * UNIT);
      const bool ok = active && c.inside(k * UNIT / 8, k * UNIT % 8);
      const T* src = ok ? row + at : static_cast<const T*>(from);
      if constexpr (kPiece == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k * 512), "l"(src), "r"(ok ? 16 : 0)
                     : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to + k * 256), "l"(src), "r"(ok ? 8 : 0)
                     : "memory");
    }
  }
  // (without conditions, at places that are in the tensor: a load behind a branch is waited for there)
  __device__ __forceinline__ void load(const void* from, int64_t offset, const BlockColumns<UNIT, V>& c) {
    place = static_cast<const Bits*>(from) + offset;
    if constexpr (kHeld)
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = place[min(c.at(0, i), c.C - 1)];
  }
  // Group v; zeros where there are no numbers.
  __device__ __forceinline__ Eight get(const unsigned char* slot, int v, const BlockColumns<UNIT, V>& c, bool active) const {
    if constexpr (kVec) {
      using Piece = std::conditional_t<kPiece == 16, uint4, uint2>;
      constexpr int per = 8 / UNIT;
      alignas(16) Piece raw[per];
      const Piece* at = reinterpret_cast<const Piece*>(slot) + threadIdx.x % 32;
#pragma unroll
      for (int k = 0; k < per; ++k) raw[k] = at[(v * per + k) * 32];
      return reinterpret_cast<const BlockPacked<T>&>(raw).widen();
    } else {
      unsigned raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i] = kHeld ? one[kHeld ? i : 0] : place[min(c.at(v, i), c.C - 1)];
      Eight f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned bits = raw[i];
        float value;
        if constexpr (sizeof(T) == 4) value = __uint_as_float(bits);
        else if constexpr (std::is_same_v<T, __half>) value = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
        else value = __uint_as_float(bits << 16);
        f[i] = active && c.inside(v, i) ? value : 0.f;
      }
      return f;
    }
  }
};

// Group v to a row.
template <typename T, int UNIT, int V>
__device__ __forceinline__ void block_store(void* to, int64_t offset, const BlockColumns<UNIT, V>& c, int v,
                                            const BlockPacked<T>& e) {
  T* row = static_cast<T*>(to) + offset;
#pragma unroll
  for (int i = 0; i < 8; i += UNIT) {
    const int at = c.at(v, i);
    if (!c.inside(v, i)) continue;
    if constexpr (UNIT * sizeof(T) == 32) {  // (FP32 sums of eight columns)
      reinterpret_cast<uint4*>(row + at)[0] = reinterpret_cast<const uint4*>(&e)[0];
      reinterpret_cast<uint4*>(row + at)[1] = reinterpret_cast<const uint4*>(&e)[1];
    } else if constexpr (UNIT * sizeof(T) == 16) {
      *reinterpret_cast<uint4*>(row + at) = reinterpret_cast<const uint4*>(&e)[i / UNIT];
    } else if constexpr (UNIT > 1) {
      *reinterpret_cast<uint2*>(row + at) = reinterpret_cast<const uint2*>(&e)[i / UNIT];
    } else {
      row[at] = i & 1 ? e.p[i / 2].y : e.p[i / 2].x;
    }
  }
}

// ---- vectors ----
__device__ __forceinline__ float block_channel(const void* data, int dtype, int64_t at) {
  if (dtype == 0) return static_cast<const float*>(data)[at];
  if (dtype == 1) return run_widen(static_cast<const __half*>(data)[at]);
  return run_widen(static_cast<const __nv_bfloat16*>(data)[at]);
}

// Where eight numbers of a vector are: four `step` apart, and four `jump` behind these.
struct BlockSpan {
  int column, step, jump;
};

// Those numbers; `missing` stands for one that is not given.
template <bool VEC>
__device__ __forceinline__ void block_channels(const BlockChannels& ch, int64_t sample, int C, BlockSpan at,
                                               float missing, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = missing;
  if (!ch.data) return;
  const int64_t base = ch.per_sample ? sample * C : 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int column = at.column + h * at.jump;
    if (VEC && ch.wide) {
      if (column >= C) continue;
      if (ch.dtype == 0) {
        const float4 raw = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(ch.data) + base + column));
        f[h * 4] = raw.x, f[h * 4 + 1] = raw.y, f[h * 4 + 2] = raw.z, f[h * 4 + 3] = raw.w;
      } else {
        const uint2 raw = __ldg(reinterpret_cast<const uint2*>(static_cast<const __half*>(ch.data) + base + column));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[h * 4 + i] = ch.dtype == 1 ? run_widen(reinterpret_cast<const __half*>(&raw)[i])
                                       : run_widen(reinterpret_cast<const __nv_bfloat16*>(&raw)[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (column + i * at.step < C) f[h * 4 + i] = block_channel(ch.data, ch.dtype, base + column + i * at.step);
    }
  }
}

// Eight numbers of an array. WIDE: the gate is multiplied by s later, in FP64.
template <bool VEC, bool WIDE, bool BACKWARD>
__device__ __noinline__ void block_array(const BlockParams& p, int64_t sample, int array, BlockSpan at,
                                         float (&f)[8]) {
  float w[8], t[8];
  const int C = p.C;
  switch (array) {
    case kArrayGate:
      block_channels<VEC>(p.gate, sample, C, at, 1.f, f);
      if (WIDE) return;
      if (BACKWARD) {
        block_channels<VEC>(p.after_weight, sample, C, at, 1.f, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(p.s) * f[i] * w[i];
        return;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= static_cast<float>(p.s);
      return;
    case kArrayFactor:
      block_channels<VEC>(p.weight, sample, C, at, 1.f, w);
      block_channels<VEC>(p.scale, sample, C, at, 0.f, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = w[i] * (1.f + f[i]);
      return;
    case kArrayOffset:
      block_channels<VEC>(p.bias, sample, C, at, 0.f, w);
      block_channels<VEC>(p.scale, sample, C, at, 0.f, t);
      block_channels<VEC>(p.shift, sample, C, at, 0.f, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = fmaf(w[i], 1.f + t[i], f[i]);
      return;
    case kArrayAfterWeight: block_channels<VEC>(p.after_weight, sample, C, at, 1.f, f); return;
    default: block_channels<VEC>(p.after_bias, sample, C, at, 0.f, f); return;
  }
}

// The arrays of a sample lie in shared memory (those that are not constant, one behind the other;
// STAGED), or are made again for each row where that is too small. Of units of eight numbers the first
// halves lie before all second halves: lanes read consecutive vectors.
__device__ __forceinline__ float* block_place_of(const BlockParams& p, float* memory, int array) {
  return memory + __popc(p.arrays & ((1 << array) - 1)) * p.C;
}

// Lays the arrays there. All of a group's vectors are asked for before any is used: a CTA waits for
// memory once for each of its threads' groups, not for each vector.
template <int UNIT, bool WIDE, bool BACKWARD>
__device__ __noinline__ void block_stage(const BlockParams& p, int64_t sample, float* memory) {
  const int C = p.C, groups = (C + 7) / 8;
  const auto put = [&](int array, int g, const float(&f)[8]) {
    if (!(p.arrays >> array & 1)) return;
    float* at = block_place_of(p, memory, array);
    if constexpr (UNIT > 1) {
      const int first = UNIT == 8 ? g : 2 * g, second = UNIT == 8 ? groups + g : 2 * g + 1;
      reinterpret_cast<float4*>(at)[first] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(at)[second] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (g * 8 + i < C) at[g * 8 + i] = f[i];
    }
  };
  constexpr bool VEC = UNIT > 1;
  for (int g = threadIdx.x; g < groups; g += blockDim.x) {
    const BlockSpan at{g * 8, 1, 4};
    float gate[8], weight[8], bias[8], scale[8], shift[8], after_weight[8], after_bias[8];
    block_channels<VEC>(p.gate, sample, C, at, 1.f, gate);
    block_channels<VEC>(p.weight, sample, C, at, 1.f, weight);
    block_channels<VEC>(p.scale, sample, C, at, 0.f, scale);
    block_channels<VEC>(p.after_weight, sample, C, at, 1.f, after_weight);
    if constexpr (!BACKWARD) {
      block_channels<VEC>(p.bias, sample, C, at, 0.f, bias);
      block_channels<VEC>(p.shift, sample, C, at, 0.f, shift);
      block_channels<VEC>(p.after_bias, sample, C, at, 0.f, after_bias);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!WIDE) gate[i] *= static_cast<float>(p.s);
      if (BACKWARD) gate[i] *= after_weight[i];
      scale[i] += 1.f;
      weight[i] *= scale[i];
      if (!BACKWARD) shift[i] = fmaf(bias[i], scale[i], shift[i]);
    }
    put(kArrayGate, g, gate);
    put(kArrayFactor, g, weight);
    if constexpr (!BACKWARD) {
      put(kArrayOffset, g, shift);
      put(kArrayAfterWeight, g, after_weight);
      put(kArrayAfterBias, g, after_bias);
    }
  }
  __syncthreads();
}

template <int UNIT, int V, bool WIDE, bool BACKWARD, bool STAGED>
struct BlockArrays {
  const BlockParams& p;
  float* memory;
  int64_t sample;

  __device__ __forceinline__ void stage() const {
    if constexpr (STAGED) block_stage<UNIT, WIDE, BACKWARD>(p, sample, memory);
  }
  // Group v of a thread.
  __device__ __forceinline__ Eight get(int array, const BlockColumns<UNIT, V>& c, int v, float constant) const {
    if (!(p.arrays >> array & 1)) return eight(constant);
    Eight f;
    if constexpr (STAGED) {
      const float* at = block_place_of(p, memory, array);
      if constexpr (UNIT > 1) {
        // (a thread without numbers there reads others' and has no use for them)
        const float4* q = reinterpret_cast<const float4*>(at);
        const int first = UNIT == 8 ? v * c.threads + c.tid : 2 * v * c.threads + c.tid, second = first + c.threads;
        const int last = c.C / UNIT - 1;
        const auto in = [&](int g) { return v < V - 1 ? g : min(g, last); };
        const float4 a = q[in(first)], b = UNIT == 8 ? q[c.C / 8 + in(first)] : q[in(second)];
        f.p[0] = make_float2(a.x, a.y), f.p[1] = make_float2(a.z, a.w);
        f.p[2] = make_float2(b.x, b.y), f.p[3] = make_float2(b.z, b.w);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = at[min(c.at(v, i), c.C - 1)];
      }
    } else {
      float t[8];  // (of its own: what is passed to a function lies in local memory)
      block_array<(UNIT > 1), WIDE, BACKWARD>(
          p, sample, array, {c.at(v, 0), UNIT > 1 ? 1 : c.threads, c.at(v, 4) - c.at(v, 0)}, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = t[i];
    }
    return f;
  }
};

// ---- sums over a row's threads ----
// These are a power of two within a warp (WARP), or all of the CTA's warps. Results are the same in
// every thread. Two buffers in turn: one barrier for each sum.
template <bool WARP>
struct BlockTeam {
  int threads;
  int warps, span;  // span: the power of two that warps fit into
  double2* slots;   // 2 x 16
  float count, inv;  // this warp's numbers of the row (all, with WARP), and 1 / these
  int turn = 0;

  template <typename T>
  __device__ __forceinline__ void across(T& a, int from) const {
    for (int o = from; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  template <typename T2>
  __device__ __forceinline__ T2* next() {
    turn ^= 1;
    return reinterpret_cast<T2*>(slots + turn * 16);
  }
  // Pairs of FP32 or of FP64.
  template <bool BOTH, typename T2>
  __device__ __forceinline__ T2 sum(T2 v) {
    if constexpr (WARP) {
      across(v.x, threads >> 1);
      if (BOTH) across(v.y, threads >> 1);
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        if (BOTH) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      }
      T2* at = next<T2>();
      const int lane = threadIdx.x % 32;
      if (lane == 0) at[threadIdx.x / 32] = v;
      __syncthreads();
      v = lane < warps ? at[lane] : T2{};
      across(v.x, span >> 1);
      if (BOTH) across(v.y, span >> 1);
      // (lanes beyond the span have sums of zeros)
      v.x = __shfl_sync(0xffffffffu, v.x, 0);
      if (BOTH) v.y = __shfl_sync(0xffffffffu, v.y, 0);
    }
    return v;
  }
};

// (mean, sum of squares) of a row times `by` (1 unless SCALED), of which a thread has the groups f (zero
// past its end). The mean is taken of the distances from a number of the row, and the squares of those
// from the mean, warp by warp and then between the warps' means: rows of equal numbers have exactly
// their own mean.
template <bool SCALED, int V, int UNIT, bool WARP>
__device__ __forceinline__ float2 block_moments(BlockTeam<WARP>& team, const Eight (&f)[V], int kind, float by,
                                                const BlockColumns<UNIT, V>& c) {
  const auto at = [&](int v, int i) { return SCALED ? __fmul2_rn(f[v].p[i], twice(by)) : f[v].p[i]; };
  if (kind == kBlockRms) {
    float2 q[2] = {};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i & 1] = __ffma2_rn(at(v, i), at(v, i), q[i & 1]);
    q[0] = __fadd2_rn(q[0], q[1]);
    return make_float2(0.f, team.template sum<false>(make_float2(q[0].x + q[0].y, 0.f)).x);
  }
  const int lane = threadIdx.x % 32;
  const float pivot = __shfl_sync(0xffffffffu, at(0, 0).x, WARP ? lane & ~(team.threads - 1) : 0);
  float2 a = {}, q = {};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Eight d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d.p[i] = __fadd2_rn(at(v, i), twice(-pivot));
    d = c.keep(d, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) a = __fadd2_rn(a, d.p[i]);
  }
  float sum = a.x + a.y;
  team.across(sum, WARP ? team.threads >> 1 : 16);
  const float shift = sum * team.inv;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Eight d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d.p[i] = __fadd2_rn(__fadd2_rn(at(v, i), twice(-pivot)), twice(-shift));
    d = c.keep(d, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) q = __ffma2_rn(d.p[i], d.p[i], q);
  }
  float squares = q.x + q.y;
  team.across(squares, WARP ? team.threads >> 1 : 16);
  float mean = pivot + shift;
  if constexpr (!WARP) {
    // the warps' (mean, sum of squares, numbers)
    float4* slots = team.template next<float4>();
    if (lane == 0) slots[threadIdx.x / 32] = make_float4(mean, squares, team.count, 0.f);
    __syncthreads();
    const float first = slots[0].x;
    const float4 mine = lane < team.warps ? slots[lane] : make_float4(first, 0.f, 0.f, 0.f);
    float away = mine.z * (mine.x - first);
    team.across(away, team.span >> 1);
    mean = first + __shfl_sync(0xffffffffu, away, 0) / c.C;
    const float d = mine.x - mean;
    squares = fmaf(mine.z * d, d, mine.y);
    team.across(squares, team.span >> 1);
    squares = __shfl_sync(0xffffffffu, squares, 0);
  }
  return make_float2(mean, squares);
}

// (mean, rstd) of a row. FP32's range is that of the numbers, not of their squares or distances: where
// the squares' sum leaves it (or its accurate part, and eps does not cover that; NaN, as of two
// infinite distances, counts as left), it is taken again of numbers scaled by a power of two.
template <int V, int UNIT, bool WARP>
__device__ __forceinline__ float2 block_stats(BlockTeam<WARP>& team, const Eight (&f)[V], int kind, float eps,
                                              const BlockColumns<UNIT, V>& c) {
  const float2 m = block_moments<false, V, UNIT, WARP>(team, f, kind, 1.f, c);
  const bool large = !(m.y <= 0x1p120f), again = large || (m.y < 0x1p-80f && eps < 0x1p-90f);
  const float inv = 1.f / c.C;
  if (WARP ? __any_sync(0xffffffffu, again) : again) {
    // (16384 squares of 2^129 have to fit)
    const float by = !again ? 1.f : large ? 0x1p-80f : 0x1p70f;
    const float2 scaled = block_moments<true, V, UNIT, WARP>(team, f, kind, by, c);
    // (rows beside one that needs this keep their own)
    if (again) return make_float2(scaled.x / by, by * rsqrtf(scaled.y * inv + eps * by * by));
  }
  return make_float2(m.x, rsqrtf(m.y * inv + eps));
}

// The same in FP64, in one pass over the distances from a number of the row (from zero in the "rms"
// kind): these and their squares are exact, or nearly so, of 16-bit numbers.
template <int V, int UNIT, bool WARP>
__device__ __forceinline__ double2 block_stats_wide(BlockTeam<WARP>& team, const Eight (&f)[V], int kind, float eps,
                                                    double inv, const BlockColumns<UNIT, V>& c) {
  const int lane = threadIdx.x % 32;
  double pivot = 0.0;
  if (kind == kBlockLayer) {
    float first = __shfl_sync(0xffffffffu, f[0][0], WARP ? lane & ~(team.threads - 1) : 0);
    if constexpr (!WARP) {
      float2* at = team.template next<float2>();
      if (threadIdx.x == 0) at[0].x = first;
      __syncthreads();
      first = at[0].x;
    }
    pivot = first;
  }
  double2 sums = make_double2(0.0, 0.0);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c.inside(v, i)) {
        const double d = static_cast<double>(f[v][i]) - pivot;
        sums.x += d;
        sums.y = fma(d, d, sums.y);
      }
  sums = team.template sum<true>(sums);
  const double shift = kind == kBlockLayer ? sums.x * inv : 0.0;
  const double variance = sums.y * inv - shift * shift;  // (NaN stays)
  return make_double2(pivot + shift, rsqrt((variance < 0.0 ? 0.0 : variance) + static_cast<double>(eps)));
}

// (v - mean) * rstd of pairs. Distances of 2^128 and more are nothing that FP32 holds, so those of rows that
// reach so far (their rstd is at most sqrt(C) / 2^128, 2^-121) are taken halved; of all others in
// the bits of a difference.
struct BlockHat {
  float2 by, shift, rise;
  __device__ __forceinline__ explicit BlockHat(float2 stats) {
    const bool far = stats.y < 0x1p-120f;
    by = twice(far ? 0.5f : 1.f);
    shift = __fmul2_rn(by, twice(-stats.x));
    rise = twice(far ? stats.y * 2.f : stats.y);
  }
  __device__ __forceinline__ float2 operator()(float2 v) const { return __fmul2_rn(__ffma2_rn(v, by, shift), rise); }
};

// ---- the kernels ----
struct BlockPlace {
  int64_t sample, row0, row1;
  int tid, part, parts;  // place in the row; which of the CTA's rows at a time
};

template <bool WARP>
__device__ __forceinline__ BlockPlace block_place(const BlockParams& p) {
  BlockPlace b;
  b.sample = blockIdx.x / p.chunks;
  const int64_t k = blockIdx.x % p.chunks;
  b.row0 = b.sample * p.T + k * p.chunk;
  b.row1 = b.sample * p.T + min((k + 1) * p.chunk, p.T);
  b.tid = WARP ? threadIdx.x & (p.threads - 1) : threadIdx.x;
  b.part = WARP ? threadIdx.x / p.threads : 0;
  b.parts = WARP ? blockDim.x / p.threads : 1;
  return b;
}

template <int V, int UNIT, bool WARP>
__device__ __forceinline__ BlockTeam<WARP> block_team(const BlockParams& p, const BlockColumns<UNIT, V>& c, double2* slots) {
  BlockTeam<WARP> team{p.threads, p.threads / 32, 1, slots, static_cast<float>(p.C), 1.f / p.C};
  if constexpr (!WARP) {
    while (team.span < team.warps) team.span *= 2;
    float n = 0.f;
#pragma unroll
    for (int i = 0; i < V * 8; ++i) n += c.inside(i / 8, i % 8) ? 1.f : 0.f;
    team.across(n, 16);
    team.count = n;
    team.inv = 1.f / n;
  }
  return team;
}

// Registers, and with them how many threads an SM holds.
constexpr int block_forward_registers(int v, int mode, bool vec) {
  return mode == kBlockAfter || v > 4 || !vec ? 128 : v > 3 ? 104 : 88;
}
// (two groups, number by number: 16 warps hide the loads' way better than 12 with all in registers;
// 2 x 700 x 7001 FP32 to BF16 training pass 144 us against 400 with four groups of too few warps, but
// 1 x 1700 x 5003 FP16 214 against 197)
constexpr int block_backward_registers(int v, bool vec) { return v > 2 || (v == 2 && !vec) ? 128 : 168; }
constexpr int block_resident(int registers) { return 65536 / registers / 32 * 32; }

// Bound by DRAM where rows are many: 16384 x 4096 BF16 (RMS alone, 268 MB) 50 us, 5.4 TB/s; 16 x 1024 rows
// of 1024 with a 32-bit residual (201 MB) 40 us; 8 x 1024 x 1152 BF16 (76 MB, four rows a warp) 20 us, of
// which the arrays' and the first rows' way from memory takes a quarter. A single row of 2048: 6 us, latency.
template <typename X, typename Y, int V, int UNIT, bool WARP, int MODE, bool STAGED>
__global__ void __maxnreg__(block_forward_registers(V, MODE, UNIT > 1)) block_norm_forward_kernel(const __grid_constant__ BlockParams p) {
  extern __shared__ __align__(16) unsigned char block_memory[];
  __shared__ double2 slots[2 * 16];
  grid_dependency_wait();
  grid_launch_dependents();
  // 16-bit sums with a normalised branch are formed in FP64: FP32 steps would bring some of them (one in
  // 2^16 for each) to the other side of a border of their type. They go through FP32, as
  // torch's casts of FP64 do, so that the same sum cast there is the same number; one in 2^17 (BF16) or
  // 2^14 (FP16) is brought onto a border by that and goes to its other neighbour, half a step and 2^-24 off.
  constexpr bool kWide = MODE == kBlockAfter && sizeof(X) == 2;
  const BlockPlace b = block_place<WARP>(p);
  constexpr bool kVec = UNIT > 1;
  const BlockColumns<UNIT, V> c{p.threads, b.tid, p.C, V * 8 * p.threads == p.C};
  const int C = p.C;
  BlockTeam<WARP> team = block_team<V, UNIT, WARP>(p, c, slots);
  const bool branch = MODE == kBlockPlain || (MODE == kBlockAfter && p.y);
  const bool after_norm = MODE == kBlockAfter && p.after_kind;
  using RowX = BlockRow<X, V, UNIT>;
  using RowY = BlockRow<Y, V, UNIT>;
  // (number by number: a row is held, and the next on its way, in registers, where a thread has eight of it)
  RowX row_x, next_x;
  RowY row_y, next_y;
  constexpr int at_y = RowX::kBytes;
  BlockRing ring(block_memory, RowX::kBytes + (branch ? RowY::kBytes : 0), p.stages);
  int64_t ahead = b.row0 + b.part;
  const auto fetch = [&] {
    const bool active = ahead < b.row1;
    if constexpr (kVec) {
      unsigned char* slot = ring.next(ring.put);
      if (WARP || active) {
        RowX::copy(slot, p.x, ahead * C, c, active);
        if (branch) RowY::copy(slot + at_y, p.y, ahead * C, c, active);
      }
      ring.commit();
    } else {
      const int64_t offset = (active ? ahead : b.row0) * C;
      next_x.load(p.x, offset, c);
      if (branch) next_y.load(p.y, offset, c);
    }
    ahead += b.parts;
  };
  for (int k = kVec ? 1 : 0; k < (kVec ? p.stages : 1); ++k) fetch();
  const BlockArrays<UNIT, V, kWide, false, STAGED> arrays{p, reinterpret_cast<float*>(block_memory + (kVec ? p.stages * ring.bytes : 0)),
                                              b.sample};
  arrays.stage();
  const float s = static_cast<float>(p.s);
  for (int64_t first = b.row0; first < b.row1; first += b.parts) {
    const int64_t row = first + b.part, offset = row * C;
    const bool active = !WARP || row < b.row1;
    const unsigned char* slot = nullptr;
    if constexpr (kVec) {
      fetch();
      ring.wait();
      slot = ring.next(ring.get);
    } else {
      row_x = next_x;
      if (branch) row_y = next_y;
      fetch();
    }
    Eight r[V];
    float2 after = make_float2(0.f, 1.f);
    double2 wide = make_double2(0.0, 1.0);
    if (after_norm) {
#pragma unroll
      for (int v = 0; v < V; ++v) r[v] = row_y.get(slot + at_y, v, c, active);
      if constexpr (kWide) {
        wide = block_stats_wide<V, UNIT, WARP>(team, r, p.after_kind, p.eps, p.inv, c);
        after = make_float2(static_cast<float>(wide.x), static_cast<float>(wide.y));
      } else {
        after = block_stats<V, UNIT, WARP>(team, r, p.after_kind, p.eps, c);
      }
      if (p.after_stats && active && c.tid == 0) p.after_stats[row] = after;
    }
    const BlockHat after_hat(after);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      r[v] = row_x.get(slot, v, c, active);
      if (!branch) continue;
      Eight u = row_y.get(slot + at_y, v, c, active);
      Eight g = arrays.get(kArrayGate, c, v, kWide ? 1.f : s);
      BlockPacked<X> e;
      if (kWide && after_norm) {
        const auto one = [&](int i) -> X& { return i & 1 ? e.p[i / 2].y : e.p[i / 2].x; };
        const Eight w = arrays.get(kArrayAfterWeight, c, v, 1.f), o = arrays.get(kArrayAfterBias, c, v, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double t = fma((u[i] - wide.x) * wide.y, static_cast<double>(w[i]), static_cast<double>(o[i]));
          one(i) = run_narrow<X>(static_cast<float>(fma(t, p.s * g[i], static_cast<double>(r[v][i]))));
        }
      } else {
        if (after_norm) {
          const Eight w = arrays.get(kArrayAfterWeight, c, v, 1.f), o = arrays.get(kArrayAfterBias, c, v, 0.f);
          u = pairs([&](float2 a, float2 w2, float2 o2) { return __ffma2_rn(after_hat(a), w2, o2); }, u, w, o);
        }
        if (kWide) g = pairs([&](float2 a) { return __fmul2_rn(a, twice(s)); }, g);
        // (two roundings, as of a product and a sum one after the other)
        e = BlockPacked<X>::of(pairs([](float2 a, float2 g2, float2 x) { return pair_add(x, __fmul2_rn(g2, a)); }, u, g, r[v]));
      }
      if (active) block_store<X>(p.r, offset, c, v, e);
      r[v] = c.keep(e.widen(), v);  // z is the norm of r as it is held
    }
    if (MODE != kBlockBefore && !p.z) continue;
    const float2 stats = block_stats<V, UNIT, WARP>(team, r, p.kind, p.eps, c);
    if (p.stats && active && c.tid == 0) p.stats[row] = stats;
    const BlockHat hat(stats);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Eight a = arrays.get(kArrayFactor, c, v, 1.f), o = arrays.get(kArrayOffset, c, v, 0.f);
      const Eight z = pairs([&](float2 b, float2 a2, float2 o2) { return __ffma2_rn(hat(b), a2, o2); }, r[v], a, o);
      if (active) block_store<Y>(p.z, offset, c, v, BlockPacked<Y>::of(z));
    }
  }
  if constexpr (kVec) ring.drain();
}

// Bound by DRAM: 16 x 1024 rows of 1024 with a 32-bit residual (302 MB) 51 us, 8 x 16384 x 96 FP32 (as
// much) 50 us, 6.0 TB/s. The numbers are read from the ring for each of up to three turns (sums, dR, dy),
// so that the four sums can stay in registers.
template <typename X, typename Y, int V, int UNIT, bool WARP, int MODE, bool STAGED>
__global__ void __maxnreg__(block_backward_registers(V, UNIT > 1)) block_norm_backward_kernel(const __grid_constant__ BlockParams p) {
  extern __shared__ __align__(16) unsigned char block_memory[];
  __shared__ double2 slots[2 * 16];
  grid_dependency_wait();
  grid_launch_dependents();
  const BlockPlace b = block_place<WARP>(p);
  constexpr bool kVec = UNIT > 1;
  const BlockColumns<UNIT, V> c{p.threads, b.tid, p.C, V * 8 * p.threads == p.C};
  const int C = p.C;
  BlockTeam<WARP> team = block_team<V, UNIT, WARP>(p, c, slots);
  const bool branch = MODE == kBlockPlain || (MODE == kBlockAfter && p.y);
  const bool after_norm = MODE == kBlockAfter && p.after_kind;
  const bool has_dr = MODE != kBlockBefore && p.dr, has_dz = MODE == kBlockBefore || p.dz;
  using RowX = BlockRow<X, V, UNIT>;
  using RowY = BlockRow<Y, V, UNIT>;
  RowX row_r, row_dr, next_r, next_dr;
  RowY row_y, row_dz, next_y, next_dz;
  // places in a warp's part of a stage: r, dz, dr, y
  constexpr int at_dz = RowX::kBytes, at_dr = at_dz + RowY::kBytes, at_y = at_dr + (MODE == kBlockBefore ? 0 : RowX::kBytes);
  BlockRing ring(block_memory, at_y + (MODE == kBlockBefore ? 0 : RowY::kBytes), p.stages);
  int64_t ahead = b.row0 + b.part;
  // (number by number: the next row into registers where a thread has eight numbers of it)
  constexpr bool kAhead = kVec || V == 1;
  const auto fetch = [&] {
    const bool active = ahead < b.row1;
    const int64_t offset = (kVec || active ? ahead : b.row0) * C;
    if constexpr (kVec) {
      unsigned char* slot = ring.next(ring.put);
      if (WARP || active) {
        if (has_dz) {
          RowX::copy(slot, p.r, offset, c, active);
          RowY::copy(slot + at_dz, p.dz, offset, c, active);
        }
        if (has_dr) RowX::copy(slot + at_dr, p.dr, offset, c, active);
        if (branch) RowY::copy(slot + at_y, p.y, offset, c, active);
      }
      ring.commit();
    } else {
      if (has_dz) {
        next_r.load(p.r, offset, c);
        next_dz.load(p.dz, offset, c);
      }
      if (has_dr) next_dr.load(p.dr, offset, c);
      if (branch) next_y.load(p.y, offset, c);
    }
    ahead += b.parts;
  };
  if constexpr (kAhead)
    for (int k = kVec ? 1 : 0; k < (kVec ? p.stages : 1); ++k) fetch();
  const BlockArrays<UNIT, V, false, true, STAGED> arrays{p, reinterpret_cast<float*>(block_memory + (kVec ? p.stages * ring.bytes : 0)),
                                             b.sample};
  arrays.stage();
  constexpr int kSums = MODE == kBlockBefore ? 2 : MODE == kBlockPlain ? 3 : 4;
  Eight sums[kSums][V];  // over rows: dz, dz rhat, dR yhat, dR
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) sums[k][v] = eight(0.f);
  const float inv = 1.f / C, s = static_cast<float>(p.s);
  float2 next1, next2;
  const auto stats_of = [&](int64_t row) {
    const bool active = row < b.row1;
    next1 = active && has_dz ? p.stats[row] : float2{};
    next2 = active && after_norm ? p.after_stats[row] : make_float2(0.f, 1.f);
  };
  stats_of(b.row0 + b.part);
  for (int64_t first = b.row0; first < b.row1; first += b.parts) {
    const int64_t row = first + b.part, offset = row * C;
    const bool active = !WARP || row < b.row1;
    const float2 s1 = next1, s2 = next2;
    stats_of(row + b.parts);
    const unsigned char* slot = nullptr;
    if constexpr (kVec) {
      fetch();
      ring.wait();
      slot = ring.next(ring.get);
    } else {
      if constexpr (!kAhead) fetch();
      row_r = next_r;
      row_dz = next_dz;
      row_dr = next_dr;
      row_y = next_y;
      if constexpr (kAhead) fetch();
    }
    const BlockHat hat1(s1), hat2(s2);
    const auto get_rhat = [&](int v) {
      return pairs(hat1, row_r.get(slot, v, c, active));
    };
    const auto get_yhat = [&](int v) {
      const Eight y = row_y.get(slot + at_y, v, c, active);
      return after_norm ? pairs(hat2, y) : y;
    };
    const auto times = [](float2 a, float2 b2) { return __fmul2_rn(a, b2); };
    float m1 = 0.f, m2 = 0.f;
    if (has_dz) {
      float2 mean[2] = {};
#pragma unroll
      for (int v = 0; v < V; ++v) {
        // (past the row's end dz is zero, and so are its products)
        const Eight h = get_rhat(v), dz = row_dz.get(slot + at_dz, v, c, active);
        const Eight a = pairs(times, dz, arrays.get(kArrayFactor, c, v, 1.f));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sums[0][v].p[i] = __fadd2_rn(sums[0][v].p[i], dz.p[i]);
          sums[1][v].p[i] = __ffma2_rn(dz.p[i], h.p[i], sums[1][v].p[i]);
          mean[0] = __fadd2_rn(mean[0], a.p[i]);
          mean[1] = __ffma2_rn(a.p[i], h.p[i], mean[1]);
        }
      }
      const float2 m = team.template sum<true>(make_float2(mean[0].x + mean[0].y, mean[1].x + mean[1].y));
      m1 = p.kind == kBlockLayer ? m.x * inv : 0.f;
      m2 = m.y * inv;
    }
    Eight e[MODE == kBlockAfter ? V : 1];  // the gradient of yhat
    float2 mean[2] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Eight d = has_dr ? row_dr.get(slot + at_dr, v, c, active) : eight(0.f);
      if (has_dz) {
        const Eight h = get_rhat(v);
        const Eight a = pairs(times, row_dz.get(slot + at_dz, v, c, active), arrays.get(kArrayFactor, c, v, 1.f));
        d = pairs([&](float2 d2, float2 a2, float2 h2) {
          return __ffma2_rn(twice(s1.y), __ffma2_rn(h2, twice(-m2), __fadd2_rn(a2, twice(-m1))), d2);
        }, d, a, h);
      }
      if (p.dx && active) block_store<X>(p.dx, offset, c, v, BlockPacked<X>::of(d));
      if (!branch) continue;
      d = c.keep(d, v);
      const Eight y = get_yhat(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kSums > 2) sums[2][v].p[i] = __ffma2_rn(d.p[i], y.p[i], sums[2][v].p[i]);
        if constexpr (kSums > 3) sums[3][v].p[i] = __fadd2_rn(sums[3][v].p[i], d.p[i]);
      }
      d = pairs(times, d, arrays.get(kArrayGate, c, v, s));
      if (after_norm) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mean[0] = __fadd2_rn(mean[0], d.p[i]);
          mean[1] = __ffma2_rn(d.p[i], y.p[i], mean[1]);
        }
        if constexpr (MODE == kBlockAfter) e[v] = d;
      } else if (p.dy && active) {
        block_store<Y>(p.dy, offset, c, v, BlockPacked<Y>::of(d));
      }
    }
    if constexpr (MODE == kBlockAfter) {
      if (!p.dy || !after_norm) continue;
      const float2 m = team.template sum<true>(make_float2(mean[0].x + mean[0].y, mean[1].x + mean[1].y));
      m1 = p.after_kind == kBlockLayer ? m.x * inv : 0.f;
      m2 = m.y * inv;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Eight dy = pairs([&](float2 e2, float2 y2) {
          return __fmul2_rn(twice(s2.y), __ffma2_rn(y2, twice(-m2), __fadd2_rn(e2, twice(-m1))));
        }, e[v], get_yhat(v));
        if (active) block_store<Y>(p.dy, offset, c, v, BlockPacked<Y>::of(dy));
      }
    }
  }
  if constexpr (kVec) ring.drain();
  if (!p.partials) return;
  float* mine = p.partials + static_cast<int64_t>(blockIdx.x) * p.sums * C;
  if constexpr (!WARP) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
      if (k < p.sums)
#pragma unroll
        for (int v = 0; v < V; ++v) block_store<float>(mine, k * C, c, v, BlockPacked<float>::of(sums[k][v]));
  } else {
    // rows side by side: their sums are added up over the warp's parts and the warps
    float* all = reinterpret_cast<float*>(block_memory);
    const int warps = blockDim.x / 32;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (k >= p.sums) break;
      __syncthreads();  // (the ring's last rows, or the sums before, are read)
#pragma unroll
      for (int i = 0; i < V * 8; ++i) {
        float v = sums[k][i / 8][i % 8];
        for (int o = 16; o >= p.threads; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        const int at = c.at(i / 8, i % 8);
        if (threadIdx.x % 32 < p.threads && at < C) all[threadIdx.x / 32 * C + at] = v;
      }
      __syncthreads();
      for (int at = threadIdx.x; at < C; at += blockDim.x) {
        float v = 0.f;
        for (int w = 0; w < warps; ++w) v += all[w * C + at];
        mine[k * C + at] = v;
      }
    }
  }
}

}  // namespace fssim
