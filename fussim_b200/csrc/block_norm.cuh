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
// A row lies in the registers of up to 512 threads, eight numbers at a time to each (or of part of a
// warp); a thread keeps its columns from row to row of its CTA's rows, and so the vectors' numbers and
// its share of the four sums in registers, while the next row is on its way.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"
#include "runs.cuh"

namespace fssim {

constexpr int kBlockMaxThreads = 512;    // of a row
constexpr int kBlockSmallThreads = 256;  // of a CTA whose rows take a warp at most
constexpr int kBlockMaxVectors = 4;      // of eight numbers, of a thread
constexpr int kBlockMaxC = kBlockMaxThreads * 8 * kBlockMaxVectors;

enum BlockKind { kBlockNone = 0, kBlockRms = 1, kBlockLayer = 2 };

// C numbers, or C for each sample.
struct BlockChannels {
  const void* data;  // or null
  int dtype;
  int per_sample;
  int wide;          // whole 16-byte vectors at every multiple of eight columns
};

struct BlockParams {
  int64_t T;              // rows of a sample
  int64_t chunk;          // rows of a CTA
  int64_t chunks;         // CTAs of a sample
  int C;
  int threads;            // of a row
  int kind, after_kind;   // BlockKind
  float eps, s;
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
  int sums;               // 2 (dz's alone) or 4
};

template <bool VEC>
__device__ __forceinline__ int block_column(int threads, int tid, int v, int i) {
  return VEC ? (v * threads + tid) * 8 + i : tid + threads * (v * 8 + i);
}

// A row's numbers of a thread, as they are in memory.
template <typename T, int V, bool VEC>
struct BlockRaw {
  static constexpr int kVecs = VEC ? V * 8 * sizeof(T) / 16 : 1;
  uint4 vec[kVecs];
  T one[VEC ? 1 : V * 8];

  __device__ __forceinline__ void load(const T* row, int C, int threads, int tid, bool active) {
    if constexpr (VEC) {
      constexpr int per = 8 * sizeof(T) / 16;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int at = block_column<true>(threads, tid, v, 0);
#pragma unroll
        for (int k = 0; k < per; ++k)
          vec[v * per + k] = active && at < C ? __ldcs(reinterpret_cast<const uint4*>(row + at) + k) : uint4{};
      }
    } else {
#pragma unroll
      for (int i = 0; i < V * 8; ++i) {
        const int at = block_column<false>(threads, tid, 0, i);
        one[i] = active && at < C ? row[at] : run_narrow<T>(0.f);
      }
    }
  }
  __device__ __forceinline__ void widen(float (&f)[V * 8]) const {
    const T* e = VEC ? reinterpret_cast<const T*>(vec) : one;
#pragma unroll
    for (int i = 0; i < V * 8; ++i) f[i] = run_widen(e[i]);
  }
  __device__ __forceinline__ void narrow(const float (&f)[V * 8]) {
    T* e = VEC ? reinterpret_cast<T*>(vec) : one;
#pragma unroll
    for (int i = 0; i < V * 8; ++i) e[i] = run_narrow<T>(f[i]);
  }
  __device__ __forceinline__ void store(T* row, int C, int threads, int tid) const {
    if constexpr (VEC) {
      constexpr int per = 8 * sizeof(T) / 16;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int at = block_column<true>(threads, tid, v, 0);
#pragma unroll
        for (int k = 0; k < per; ++k)
          if (at < C) reinterpret_cast<uint4*>(row + at)[k] = vec[v * per + k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V * 8; ++i) {
        const int at = block_column<false>(threads, tid, 0, i);
        if (at < C) row[at] = one[i];
      }
    }
  }
};

__device__ __forceinline__ float block_channel(const void* data, int dtype, int64_t at) {
  if (dtype == 0) return static_cast<const float*>(data)[at];
  if (dtype == 1) return run_widen(static_cast<const __half*>(data)[at]);
  return run_widen(static_cast<const __nv_bfloat16*>(data)[at]);
}

// A thread's eight numbers (group v) of a vector; `missing` stands for one that is not given.
template <bool VEC>
__device__ __forceinline__ void block_channels(const BlockChannels& ch, int64_t sample, int C, int threads, int tid,
                                               int v, float missing, float (&f)[8]) {
  if (!ch.data) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = missing;
    return;
  }
  const int64_t base = ch.per_sample ? sample * C : 0;
  const int at = block_column<VEC>(threads, tid, v, 0);
  if (VEC && ch.wide) {
    if (at >= C) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = missing;
      return;
    }
    uint4 raw[2];
    if (ch.dtype == 0) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(ch.data) + base + at);
      raw[0] = __ldg(p);
      raw[1] = __ldg(p + 1);
      const float* e = reinterpret_cast<const float*>(raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = e[i];
    } else {
      raw[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(ch.data) + base + at));
      if (ch.dtype == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = run_widen(reinterpret_cast<const __half*>(raw)[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = run_widen(reinterpret_cast<const __nv_bfloat16*>(raw)[i]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = block_column<VEC>(threads, tid, v, i);
    f[i] = c < C ? block_channel(ch.data, ch.dtype, base + c) : missing;
  }
}

// Sums over a row's threads, which are a power of two within a warp, or all of the CTA's warps.
// Results are the same in every thread. Two buffers in turn: one barrier for each sum.
struct BlockTeam {
  int threads, warps;
  float2* slots;    // 2 x 32
  float* counts;    // a row's numbers of each warp
  float warp_inv;   // 1 / those of this one
  int turn = 0;

  // The buffer of the next exchange.
  __device__ __forceinline__ float2* next() {
    turn ^= 1;
    return slots + turn * 32;
  }

  __device__ __forceinline__ void warp_sum(float& a) const {
    const int from = warps > 1 ? 16 : threads / 2;
    for (int o = from; o > 0; o /= 2) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  __device__ __forceinline__ float2 sum(float a, float b) {
    if (warps > 1) {
#pragma unroll
      for (int o = 16; o > 0; o /= 2) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
      float2* at = next();
      if (threadIdx.x % 32 == 0) at[threadIdx.x / 32] = make_float2(a, b);
      __syncthreads();
      a = b = 0.f;
      for (int w = 0; w < warps; ++w) {
        a += at[w].x;
        b += at[w].y;
      }
    } else {
      for (int o = threads / 2; o > 0; o /= 2) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
    }
    return make_float2(a, b);
  }
};

// (mean, rstd) of a row, of which a thread has `f` (zero past the end). The mean is taken of the
// distances from a number of the row, and the squares of those from the mean, warp by warp and then
// between the warps' means: rows of equal numbers have exactly their own mean.
// FP32's range is that of the numbers, not of their squares: where their sum leaves it (or its
// accurate part, and eps does not cover that), it is taken again of numbers scaled by a power of two.
template <int V, bool VEC>
__device__ __forceinline__ float2 block_stats(BlockTeam& team, const float (&f)[V * 8], int kind, float eps, int C,
                                              int tid) {
  const int lane = threadIdx.x % 32;
  float by = 1.f;
  for (;;) {
    float mean = 0.f, squares = 0.f;
    if (kind == kBlockRms) {
#pragma unroll
      for (int i = 0; i < V * 8; ++i) squares = fmaf(f[i] * by, f[i] * by, squares);
      squares = team.sum(squares, 0.f).x;
    } else {
      const auto valid = [&](int i) { return block_column<VEC>(team.threads, tid, i / 8, i % 8) < C; };
      const float pivot = by * __shfl_sync(0xffffffffu, f[0], team.warps > 1 ? 0 : lane / team.threads * team.threads);
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < V * 8; ++i) a += valid(i) ? fmaf(f[i], by, -pivot) : 0.f;
      team.warp_sum(a);
      const float shift = a * team.warp_inv;
#pragma unroll
      for (int i = 0; i < V * 8; ++i) {
        const float d = valid(i) ? fmaf(f[i], by, -pivot) - shift : 0.f;
        squares = fmaf(d, d, squares);
      }
      team.warp_sum(squares);
      mean = pivot + shift;
      if (team.warps > 1) {
        float2* at = team.next();
        if (lane == 0) at[threadIdx.x / 32] = make_float2(mean, squares);
        __syncthreads();
        const float first = at[0].x;
        float away = 0.f;
        for (int w = 0; w < team.warps; ++w) away = fmaf(team.counts[w], at[w].x - first, away);
        mean = first + away / C;
        squares = 0.f;
        for (int w = 0; w < team.warps; ++w) {
          const float d = at[w].x - mean;
          squares += fmaf(team.counts[w] * d, d, at[w].y);
        }
      }
    }
    const bool large = squares > 0x1p120f, small = squares < 0x1p-80f && eps < 0x1p-90f;
    const bool again = by == 1.f && (large || small);
    if (team.warps > 1 ? !again : !__any_sync(0xffffffffu, again))
      return make_float2(mean / by, by / sqrtf(squares / C + eps * by * by));
    by = large ? 0x1p-70f : small ? 0x1p70f : by;
  }
}

struct BlockPlace {
  int64_t sample, row0, row1;
  int tid, part, parts;  // place in the row; which of the CTA's rows at a time
};

__device__ __forceinline__ BlockPlace block_place(const BlockParams& p) {
  BlockPlace b;
  b.sample = blockIdx.x / p.chunks;
  const int64_t k = blockIdx.x % p.chunks;
  b.row0 = b.sample * p.T + k * p.chunk;
  b.row1 = b.sample * p.T + min((k + 1) * p.chunk, p.T);
  b.tid = threadIdx.x % p.threads;
  b.part = threadIdx.x / p.threads;
  b.parts = blockDim.x / p.threads;
  return b;
}

template <int V, bool VEC>
__device__ __forceinline__ BlockTeam block_team(const BlockParams& p, int tid, float2* slots, float* counts) {
  BlockTeam team{p.threads, p.threads > 32 ? p.threads / 32 : 1, slots, counts, 0.f};
  float n = 0.f;
#pragma unroll
  for (int i = 0; i < V * 8; ++i) n += block_column<VEC>(p.threads, tid, i / 8, i % 8) < p.C ? 1.f : 0.f;
  team.warp_sum(n);
  team.warp_inv = n > 0.f ? 1.f / n : 0.f;
  if (threadIdx.x % 32 == 0) counts[threadIdx.x / 32] = n;  // (read behind a barrier)
  return team;
}

// The vectors of a thread's columns: kept in registers where it has eight of them.
template <int V, bool VEC>
struct BlockVectors {
  float keep[V == 1 ? 8 : 1];
  template <typename F>
  __device__ __forceinline__ void first(F make) {
    if constexpr (V == 1) make(0, keep);
  }
  template <typename F>
  __device__ __forceinline__ void get(int v, float (&f)[8], F make) const {
    if constexpr (V == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = keep[i];
    } else {
      make(v, f);
    }
  }
};

template <typename X, typename Y, int V, bool VEC>
__global__ void __launch_bounds__(kBlockMaxThreads, 2)
    block_norm_forward_kernel(const __grid_constant__ BlockParams p) {
  __shared__ float2 slots[2 * 32];
  __shared__ float counts[kBlockMaxThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const BlockPlace b = block_place(p);
  const int C = p.C, tid = b.tid;
  BlockTeam team = block_team<V, VEC>(p, tid, slots, counts);
  const auto channels = [&](const BlockChannels& ch, int v, float missing, float (&f)[8]) {
    block_channels<VEC>(ch, b.sample, C, p.threads, tid, v, missing, f);
  };
  // s * gate; z = rhat * factor + offset
  const auto make_gate = [&](int v, float (&f)[8]) {
    channels(p.gate, v, 1.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= p.s;
  };
  const auto make_factor = [&](int v, float (&f)[8]) {
    float w[8];
    channels(p.weight, v, 1.f, w);
    channels(p.scale, v, 0.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = w[i] * (1.f + f[i]);
  };
  const auto make_offset = [&](int v, float (&f)[8]) {
    float w[8], t[8];
    channels(p.bias, v, 0.f, w);
    channels(p.scale, v, 0.f, t);
    channels(p.shift, v, 0.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fmaf(w[i], 1.f + t[i], f[i]);
  };
  const auto make_after_weight = [&](int v, float (&f)[8]) { channels(p.after_weight, v, 1.f, f); };
  const auto make_after_bias = [&](int v, float (&f)[8]) { channels(p.after_bias, v, 0.f, f); };
  BlockVectors<V, VEC> gate, factor, offset, after_weight, after_bias;
  if (p.y) {
    gate.first(make_gate);
    after_weight.first(make_after_weight);
    after_bias.first(make_after_bias);
  }
  if (p.z) {
    factor.first(make_factor);
    offset.first(make_offset);
  }
  BlockRaw<X, V, VEC> x;
  BlockRaw<Y, V, VEC> y;
  const auto fetch = [&](int64_t row) {
    const bool active = row < b.row1;
    x.load(static_cast<const X*>(p.x) + row * C, C, p.threads, tid, active);
    if (p.y) y.load(static_cast<const Y*>(p.y) + row * C, C, p.threads, tid, active);
  };
  fetch(b.row0 + b.part);
  for (int64_t first = b.row0; first < b.row1; first += b.parts) {
    const int64_t row = first + b.part;
    const bool active = row < b.row1;
    float r[V * 8], t[V * 8];
    x.widen(r);
    if (p.y) y.widen(t);
    fetch(row + b.parts);
    if (p.y) {
      float2 after = make_float2(0.f, 1.f);
      if (p.after_kind) after = block_stats<V, VEC>(team, t, p.after_kind, p.eps, C, tid);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float g[8], w[8], o[8];
        gate.get(v, g, make_gate);
        if (p.after_kind) {
          after_weight.get(v, w, make_after_weight);
          after_bias.get(v, o, make_after_bias);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float u = t[v * 8 + i];
          if (p.after_kind) u = fmaf((u - after.x) * after.y, w[i], o[i]);
          r[v * 8 + i] = __fadd_rn(r[v * 8 + i], __fmul_rn(g[i], u));
        }
      }
      if (p.after_stats && active && tid == 0) p.after_stats[row] = after;
      BlockRaw<X, V, VEC> out;
      out.narrow(r);
      if (active) out.store(static_cast<X*>(p.r) + row * C, C, p.threads, tid);
      out.widen(r);  // z is the norm of r as it is held
      if (!VEC || V * 8 * p.threads != C) {
#pragma unroll
        for (int i = 0; i < V * 8; ++i)
          if (block_column<VEC>(p.threads, tid, i / 8, i % 8) >= C) r[i] = 0.f;
      }
    }
    if (!p.z) continue;
    const float2 stats = block_stats<V, VEC>(team, r, p.kind, p.eps, C, tid);
    if (p.stats && active && tid == 0) p.stats[row] = stats;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a[8], o[8];
      factor.get(v, a, make_factor);
      offset.get(v, o, make_offset);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[v * 8 + i] = fmaf((r[v * 8 + i] - stats.x) * stats.y, a[i], o[i]);
    }
    BlockRaw<Y, V, VEC> out;
    out.narrow(t);
    if (active) out.store(static_cast<Y*>(p.z) + row * C, C, p.threads, tid);
  }
}

template <typename X, typename Y, int V, bool VEC>
__global__ void __launch_bounds__(kBlockMaxThreads, 1)
    block_norm_backward_kernel(const __grid_constant__ BlockParams p) {
  __shared__ float2 slots[2 * 32];
  __shared__ float counts[kBlockMaxThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const BlockPlace b = block_place(p);
  const int C = p.C, tid = b.tid;
  BlockTeam team = block_team<V, VEC>(p, tid, slots, counts);
  const auto channels = [&](const BlockChannels& ch, int v, float missing, float (&f)[8]) {
    block_channels<VEC>(ch, b.sample, C, p.threads, tid, v, missing, f);
  };
  const auto make_gate = [&](int v, float (&f)[8]) {
    channels(p.gate, v, 1.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= p.s;
  };
  const auto make_factor = [&](int v, float (&f)[8]) {
    float w[8];
    channels(p.weight, v, 1.f, w);
    channels(p.scale, v, 0.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = w[i] * (1.f + f[i]);
  };
  const auto make_after_weight = [&](int v, float (&f)[8]) { channels(p.after_weight, v, 1.f, f); };
  BlockVectors<V, VEC> gate, factor, after_weight;
  if (p.y) {
    gate.first(make_gate);
    after_weight.first(make_after_weight);
  }
  if (p.dz) factor.first(make_factor);
  float sums[4][V * 8];  // over rows: dz, dz rhat, dR, dR yhat
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < V * 8; ++i) sums[k][i] = 0.f;
  BlockRaw<X, V, VEC> raw_r, raw_dr;
  BlockRaw<Y, V, VEC> raw_y, raw_dz;
  float2 stats{}, after{};
  const auto fetch = [&](int64_t row) {
    const bool active = row < b.row1;
    if (p.dz) {
      raw_r.load(static_cast<const X*>(p.r) + row * C, C, p.threads, tid, active);
      raw_dz.load(static_cast<const Y*>(p.dz) + row * C, C, p.threads, tid, active);
      stats = active ? p.stats[row] : float2{};
    }
    if (p.dr) raw_dr.load(static_cast<const X*>(p.dr) + row * C, C, p.threads, tid, active);
    if (p.y) {
      raw_y.load(static_cast<const Y*>(p.y) + row * C, C, p.threads, tid, active);
      after = active && p.after_kind ? p.after_stats[row] : make_float2(0.f, 1.f);
    }
  };
  const float inv = 1.f / C;
  fetch(b.row0 + b.part);
  for (int64_t first = b.row0; first < b.row1; first += b.parts) {
    const int64_t row = first + b.part;
    const bool active = row < b.row1;
    float d[V * 8], h[V * 8], y[V * 8];  // dR; rhat and then e; yhat
    const float2 s1 = stats, s2 = after;
#pragma unroll
    for (int i = 0; i < V * 8; ++i) d[i] = 0.f;
    if (p.dr) raw_dr.widen(d);
    if (p.y) {
      raw_y.widen(y);
#pragma unroll
      for (int i = 0; i < V * 8; ++i) y[i] = (y[i] - s2.x) * s2.y;
    }
    if (p.dz) {
      float dz[V * 8];
      raw_r.widen(h);
      raw_dz.widen(dz);
      fetch(row + b.parts);
      float a1 = 0.f, a2 = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f[8];
        factor.get(v, f, make_factor);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = v * 8 + i;
          h[j] = (h[j] - s1.x) * s1.y;
          sums[0][j] += dz[j];
          sums[1][j] = fmaf(dz[j], h[j], sums[1][j]);
          dz[j] *= f[i];
          a1 += dz[j];
          a2 = fmaf(dz[j], h[j], a2);
        }
      }
      const float2 a = team.sum(a1, a2);
      const float m1 = p.kind == kBlockLayer ? a.x * inv : 0.f, m2 = a.y * inv;
#pragma unroll
      for (int i = 0; i < V * 8; ++i) d[i] = fmaf(s1.y, (dz[i] - m1) - h[i] * m2, d[i]);
    } else {
      fetch(row + b.parts);
    }
    if (p.dx) {
      BlockRaw<X, V, VEC> out;
      out.narrow(d);
      if (active) out.store(static_cast<X*>(p.dx) + row * C, C, p.threads, tid);
    }
    if (!p.y) continue;
    float a1 = 0.f, a2 = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float g[8], w[8];
      gate.get(v, g, make_gate);
      after_weight.get(v, w, make_after_weight);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = v * 8 + i;
        if (block_column<VEC>(p.threads, tid, v, i) >= C || !active) d[j] = 0.f;
        sums[2][j] += d[j];
        sums[3][j] = fmaf(d[j], y[j], sums[3][j]);
        h[j] = d[j] * g[i];
        if (p.after_kind) h[j] *= w[i];
        a1 += h[j];
        a2 = fmaf(h[j], y[j], a2);
      }
    }
    if (!p.dy) continue;
    if (p.after_kind) {
      const float2 a = team.sum(a1, a2);
      const float m1 = p.after_kind == kBlockLayer ? a.x * inv : 0.f, m2 = a.y * inv;
#pragma unroll
      for (int i = 0; i < V * 8; ++i) h[i] = s2.y * ((h[i] - m1) - y[i] * m2);
    }
    BlockRaw<Y, V, VEC> out;
    out.narrow(h);
    if (active) out.store(static_cast<Y*>(p.dy) + row * C, C, p.threads, tid);
  }
  if (!p.partials) return;
  float* mine = p.partials + static_cast<int64_t>(blockIdx.x) * p.sums * C;
  if (p.threads > 32) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < p.sums)
#pragma unroll
        for (int i = 0; i < V * 8; ++i) {
          const int c = block_column<VEC>(p.threads, tid, i / 8, i % 8);
          if (c < C) mine[k * C + c] = sums[k][i];
        }
    return;
  }
  // rows side by side: their sums are added up over the warp's parts and the warps
  __shared__ float all[kBlockSmallThreads / 32][8 * 32];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= p.sums) break;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = sums[k][i];
      for (int o = 16; o >= p.threads; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
      const int c = block_column<VEC>(p.threads, tid, 0, i);
      if (threadIdx.x % 32 < p.threads && c < C) all[threadIdx.x / 32][c] = v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      float v = 0.f;
      for (int w = 0; w < blockDim.x / 32; ++w) v += all[w][c];
      mine[k * C + c] = v;
    }
    __syncthreads();
  }
}

constexpr int kBlockMergeColumns = 32, kBlockMergeTeams = 8;

// Adds the CTAs' sums up: to (sample, segment, sum, C) in FP64, over the segment's share of a sample's CTAs.
__global__ void __launch_bounds__(kBlockMergeColumns * kBlockMergeTeams)
    block_norm_merge_kernel(const float* partials, double* merged, int C, int sums, int64_t chunks, int segments) {
  __shared__ double sm[kBlockMergeTeams][kBlockMergeColumns];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % kBlockMergeColumns, team = threadIdx.x / kBlockMergeColumns;
  const int columns = (C + kBlockMergeColumns - 1) / kBlockMergeColumns;
  const int c = blockIdx.x % columns * kBlockMergeColumns + lane;
  const int64_t place = blockIdx.x / columns, sample = place / segments, segment = place % segments;
  const int64_t k0 = chunks * segment / segments, k1 = chunks * (segment + 1) / segments;
  for (int k = 0; k < sums; ++k) {
    double v = 0.0;
    if (c < C)
      for (int64_t j = k0 + team; j < k1; j += kBlockMergeTeams)
        v += static_cast<double>(partials[((sample * chunks + j) * sums + k) * C + c]);
    sm[team][lane] = v;
    __syncthreads();
    if (team == 0) {
      for (int t = 1; t < kBlockMergeTeams; ++t) v += sm[t][lane];
      if (c < C) merged[(place * sums + k) * C + c] = v;
    }
    __syncthreads();
  }
}

// A gradient's place: a vector's type and form (C, or C for each sample).
struct BlockGrad {
  void* data;
  int dtype;
  int per_sample;
};

struct BlockGradParams {
  const double* merged;   // or, of one CTA for each sample, its own sums:
  const float* partials;
  int64_t B;
  int segments, sums, C;
  float s;
  BlockChannels gate, weight, bias, scale, after_weight, after_bias;
  BlockGrad dgate, dweight, dbias, dscale, dshift, dafter_weight, dafter_bias;
};

__device__ __forceinline__ void block_put(const BlockGrad& g, int64_t at, double v) {
  if (g.dtype == 0) static_cast<float*>(g.data)[at] = static_cast<float>(v);
  else if (g.dtype == 1) static_cast<__half*>(g.data)[at] = run_narrow<__half>(static_cast<float>(v));
  else static_cast<__nv_bfloat16*>(g.data)[at] = run_narrow<__nv_bfloat16>(static_cast<float>(v));
}

// The vectors' gradients from a column's sums: those with one for each sample directly, others
// summed over the samples.
__global__ void __launch_bounds__(kBlockMergeColumns * kBlockMergeTeams)
    block_norm_grads_kernel(const __grid_constant__ BlockGradParams p) {
  __shared__ double sm[7][kBlockMergeTeams][kBlockMergeColumns];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % kBlockMergeColumns, team = threadIdx.x / kBlockMergeColumns;
  const int c = blockIdx.x * kBlockMergeColumns + lane, C = p.C;
  const BlockGrad* grads[7] = {&p.dshift, &p.dscale, &p.dweight, &p.dbias, &p.dgate, &p.dafter_weight, &p.dafter_bias};
  double all[7] = {};
  const auto of = [&](const BlockChannels& ch, int64_t sample, double missing) {
    return ch.data ? static_cast<double>(block_channel(ch.data, ch.dtype, ch.per_sample ? sample * C + c : c)) : missing;
  };
  if (c < C)
    for (int64_t b = team; b < p.B; b += kBlockMergeTeams) {
      double sum[4] = {};
      for (int g = 0; g < p.segments; ++g)
        for (int k = 0; k < p.sums; ++k) {
          const int64_t at = ((b * p.segments + g) * p.sums + k) * C + c;
          sum[k] += p.merged ? p.merged[at] : static_cast<double>(p.partials[at]);
        }
      const double lift = 1.0 + of(p.scale, b, 0.0), gate = p.s * of(p.gate, b, 1.0);
      const double v[7] = {sum[0],
                           of(p.weight, b, 1.0) * sum[1] + of(p.bias, b, 0.0) * sum[0],
                           lift * sum[1],
                           lift * sum[0],
                           p.s * (of(p.after_weight, b, 1.0) * sum[3] + of(p.after_bias, b, 0.0) * sum[2]),
                           gate * sum[3],
                           gate * sum[2]};
#pragma unroll
      for (int k = 0; k < 7; ++k) {
        if (grads[k]->data && grads[k]->per_sample) block_put(*grads[k], b * C + c, v[k]);
        all[k] += v[k];
      }
    }
#pragma unroll
  for (int k = 0; k < 7; ++k) sm[k][team][lane] = all[k];
  __syncthreads();
  if (team < 7 && c < C && grads[team]->data && !grads[team]->per_sample) {
    double v = 0.0;
    for (int t = 0; t < kBlockMergeTeams; ++t) v += sm[team][t][lane];
    block_put(*grads[team], c, v);
  }
}

}  // namespace fssim
