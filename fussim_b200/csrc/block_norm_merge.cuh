// The gradients of the block norms' vectors from the sums that each CTA of the backward pass left.
// Sums go on in FP64 (of eight CTAs' sums at a time), in a fixed order.
#pragma once

#include "block_norm.cuh"

namespace fssim {

constexpr int kBlockMergeColumns = 8, kBlockMergeTeams = 32;

// A gradient's place: a vector's type and form (C, or C for each sample).
struct BlockGrad {
  void* data;
  int dtype;
  int per_sample;
};

enum BlockVector { kVectorShift, kVectorScale, kVectorWeight, kVectorBias, kVectorGate, kVectorAfterWeight, kVectorAfterBias, kVectors };

struct BlockGradParams {
  const float* partials;  // (sample, CTA, sum, C)
  double* totals;         // (split, vector, C): of the samples' splits, where there are several; or null
  int B, chunks;          // chunks: CTAs of a sample
  int splits, split_samples, C;
  int shared;             // whether a gradient is a sum over samples
  double s;
  BlockChannels gate, weight, bias, scale, after_weight, after_bias;
  BlockGrad grads[kVectors];
};

__device__ __forceinline__ void block_put(const BlockGrad& g, int64_t at, double v) {
  if (g.dtype == 0) static_cast<float*>(g.data)[at] = static_cast<float>(v);
  else if (g.dtype == 1) static_cast<__half*>(g.data)[at] = run_narrow<__half>(static_cast<float>(v));
  else static_cast<__nv_bfloat16*>(g.data)[at] = run_narrow<__nv_bfloat16>(static_cast<float>(v));
}

// A CTA has eight columns (a sector of 32 bytes) of a split's samples. Its 32 teams of a thread for each
// column share the samples: several a team, or a power of two of teams a sample, which have its CTAs'
// sums in turn. Latency is all there is to it: several CTAs' sums are asked for before any is added, and
// few threads go through the rest (444 sums of 3 x 96 that lie in L2: 7.1 us; 12.7 with 64 teams of 16
// columns in 32 warps; 864 of 3 x 1024: 8.7 us).
template <int SUMS>
__global__ void __launch_bounds__(kBlockMergeColumns * kBlockMergeTeams)
    block_norm_grads_kernel(const __grid_constant__ BlockGradParams p) {
  constexpr int kWarps = kBlockMergeTeams / 4, kAtOnce = 8;
  static_assert(kBlockMergeColumns == 8, "a quarter of a warp");
  __shared__ double sm[kVectors][kWarps][kBlockMergeColumns];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % kBlockMergeColumns, team = threadIdx.x / kBlockMergeColumns, warp = team / 4;
  const int columns = (p.C + kBlockMergeColumns - 1) / kBlockMergeColumns, C = p.C;
  const int split = blockIdx.x / columns, c = (blockIdx.x - split * columns) * kBlockMergeColumns + lane;
  const int b0 = split * p.split_samples, b1 = min(b0 + p.split_samples, p.B);
  int shares = 1, log = 0;  // teams of a sample
  while (shares * 2 * (b1 - b0) <= kBlockMergeTeams) shares *= 2, ++log;
  const int part = team & (shares - 1), lead = team >> log;
  double all[kVectors] = {};
  // (every team goes round as often as the first)
  for (int first = b0; first < b1; first += kBlockMergeTeams >> log) {
    const int sample = first + lead;
    const bool active = c < C && sample < b1, mine = active && part == 0;
    const auto of = [&](const BlockChannels& ch, float missing) {
      if (!ch.data || !mine) return missing;
      return block_channel(ch.data, ch.dtype, ch.per_sample ? static_cast<int64_t>(sample) * C + c : c);
    };
    const float scale = of(p.scale, 0.f), gate = of(p.gate, 1.f), weight = of(p.weight, 1.f), bias = of(p.bias, 0.f);
    const float after_weight = of(p.after_weight, 1.f), after_bias = of(p.after_bias, 0.f);
    double sum[4] = {};
    if (active) {
      const float* from = p.partials + (static_cast<int64_t>(sample) * p.chunks + part) * SUMS * C + c;
      const int64_t step = static_cast<int64_t>(shares) * SUMS * C;
      int left = p.chunks - part;
      const auto add = [&](auto whole) {
        float f[SUMS][kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u, from += step)
#pragma unroll
          for (int k = 0; k < SUMS; ++k) f[k][u] = decltype(whole)::value || u * shares < left ? __ldcg(from + k * C) : 0.f;
        // (a batch in FP32, as a tree: three more roundings)
#pragma unroll
        for (int k = 0; k < SUMS; ++k)
          sum[k] += static_cast<double>(((f[k][0] + f[k][1]) + (f[k][2] + f[k][3])) + ((f[k][4] + f[k][5]) + (f[k][6] + f[k][7])));
        left -= kAtOnce * shares;
      };
      while (left > (kAtOnce - 1) * shares) add(std::true_type{});
      if (left > 0) add(std::false_type{});
    }
    if (shares > 1) {
#pragma unroll
      for (int k = 0; k < SUMS; ++k) {
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 8);
        if (shares > 2) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 16);
      }
      if (shares > 4) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < SUMS; ++k)
          if (team % 4 == 0) sm[k][warp][lane] = sum[k];
        __syncthreads();
        if (mine)
#pragma unroll
          for (int k = 0; k < SUMS; ++k)
            for (int w = 1; w < shares / 4; ++w) sum[k] += sm[k][warp + w][lane];
      }
    }
    if (mine) {
      const double lift = 1.0 + scale, sg = p.s * gate;
      const double v[kVectors] = {sum[0],        weight * sum[1] + bias * sum[0], lift * sum[1],
                                  lift * sum[0], p.s * (after_weight * sum[2] + after_bias * sum[3]), sg * sum[2],
                                  sg * sum[3]};
#pragma unroll
      for (int k = 0; k < kVectors; ++k) {
        if (!p.grads[k].data) continue;
        if (p.grads[k].per_sample) block_put(p.grads[k], static_cast<int64_t>(sample) * C + c, v[k]);
        else all[k] += v[k];
      }
    }
  }
  if (!p.shared) return;
  const bool alone = b1 - b0 == 1;  // one sample: it is the sum
  if (!alone) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      if (!p.grads[k].data || p.grads[k].per_sample) continue;
      all[k] += __shfl_xor_sync(0xffffffffu, all[k], 8);
      all[k] += __shfl_xor_sync(0xffffffffu, all[k], 16);
      if (team % 4 == 0) sm[k][warp][lane] = all[k];
    }
    __syncthreads();
  }
  if (team > 0 || c >= C) return;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    if (!p.grads[k].data || p.grads[k].per_sample) continue;
    double v = all[k];
    if (!alone)
      for (int w = 1; w < kWarps; ++w) v += sm[k][w][lane];
    if (p.totals) p.totals[(static_cast<int64_t>(split) * kVectors + k) * C + c] = v;
    else block_put(p.grads[k], c, v);
  }
}

// Gradients that are sums over all samples, from those of the splits.
__global__ void __launch_bounds__(256) block_norm_totals_kernel(const __grid_constant__ BlockGradParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.C) return;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    if (!p.grads[k].data || p.grads[k].per_sample) continue;
    double v = 0.0;
    for (int t = 0; t < p.splits; ++t) v += p.totals[(static_cast<int64_t>(t) * kVectors + k) * p.C + c];
    block_put(p.grads[k], c, v);
  }
}

}  // namespace fssim
