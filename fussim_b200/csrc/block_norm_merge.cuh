// The gradients of the block norms' vectors from the sums that each CTA of the backward pass left.
// Sums go on in FP64, in a fixed order.
#pragma once

#include "block_norm.cuh"

namespace fssim {

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
  double s;
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
                           p.s * (of(p.after_weight, b, 1.0) * sum[2] + of(p.after_bias, b, 0.0) * sum[3]),
                           gate * sum[2],
                           gate * sum[3]};
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
