// Group normalisation with an activation, channels last: kernels for sm_100a (B200).
//
// x is N samples of P pixels of C channels, the channels innermost (NHWC). Group (n, g) is the
// M = P * C/G numbers of sample n in the channels [g*C/G, (g+1)*C/G):
//
//   forward   mean, var over the group, rstd = 1/sqrt(var + eps),
//             z = (x - mean) * rstd * w_c + b_c,  y = act(z)
//   backward  dz = dy * act'(z);  db_c = sum dz;  dw_c = sum dz * xhat  (over n and pixels)
//             dx = rstd * (w dz - <w dz> - xhat <w dz xhat>),  <> the mean over the group
//
// Work split: a sample's pixels are cut into S parts (equal to within one pixel) and its
// channels into slices of at most 256 vectors of V channels. A CTA takes one (sample, part,
// slice). A thread keeps one vector of channels for the whole part and steps over its pixels,
// so the per-channel constants and sums stay in registers and a warp reads whole rows of
// memory. The group's numbers must all be seen before its first output, so each direction is
// a reducing pass and an applying pass; the second read comes from L2 when the samples that
// are in flight fit it (the host cuts the batch accordingly).
//
// Statistics: a thread takes U pixels at a time, forms each channel's mean and sum of squared
// deviations of those U values (two passes over registers), and merges them into its running
// pair (the pairwise update of Chan, Golub and LeVeque, 1979). No sum of raw squares is ever
// formed, so a mean far from zero costs no digits. Threads, parts and slices are merged the
// same way, in a fixed order (results repeat bit for bit), across parts in FP64.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"

namespace fssim {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;

enum NormAct { kNormActNone = 0, kNormActSilu = 1, kNormActRelu = 2 };

struct NormGeometry {
  int64_t N;   // samples of this launch
  int64_t P;   // pixels per sample
  int C, G, Cg;
  int SC;      // channels per slice (a multiple of V)
  int slices;
  int lanes;   // SC / V
  int rows;    // pixels a CTA takes per step
  int S;       // parts of a sample's pixels
  int GS;      // most groups that touch one slice
  float eps;

  __host__ __device__ int64_t part_begin(int64_t s) const { return P / S * s + (P % S) * s / S; }
};

struct NormParams {
  NormGeometry g;
  const void* x;
  const void* dy;
  void* out;            // y or dx
  const void* weight;   // C values of weight_dtype, or nullptr (ones)
  const void* bias;     // C values of weight_dtype, or nullptr (zeros)
  int weight_dtype;
  float* mean;          // N * G
  float* rstd;          // N * G
  float2* partial;      // forward: (mean, M2) per (sample, part, slice, group of the slice)
                        // backward: (sum dz, sum dz (x - mean)) per (sample, part, channel)
  float2* chan;         // backward: (sum dz, sum dz xhat) per (sample, channel)
  float2* coef;         // backward: (rstd <w dz>, rstd^2 <w dz xhat>) per (sample, group)
  void* dweight;
  void* dbias;
};

// ---- element types ----
template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<4> { using type = unsigned; };
template <> struct RawVec<2> { using type = unsigned short; };

template <typename T, int V>
struct VecIO {
  using Raw = typename RawVec<sizeof(T) * V>::type;
  static __device__ __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void store(T* p, const Raw& r) { *reinterpret_cast<Raw*>(p) = r; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[V]);
  static __device__ __forceinline__ Raw pack(const float (&f)[V]);
};

__device__ __forceinline__ float norm_to_float(float v) { return v; }
__device__ __forceinline__ float norm_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float norm_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T norm_from_float(float v);
template <> __device__ __forceinline__ float norm_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half norm_from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 norm_from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, int V>
__device__ __forceinline__ void VecIO<T, V>::unpack(const Raw& r, float (&f)[V]) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = norm_to_float(e[i]);
}
template <typename T, int V>
__device__ __forceinline__ typename VecIO<T, V>::Raw VecIO<T, V>::pack(const float (&f)[V]) {
  Raw r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = norm_from_float<T>(f[i]);
  return r;
}

// Weights come in any of the three types, whatever x's is; read once per thread.
__device__ __forceinline__ float load_weight(const void* p, int dtype, int c) {
  if (dtype == 0) return static_cast<const float*>(p)[c];
  if (dtype == 1) return __half2float(static_cast<const __half*>(p)[c]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
}
__device__ __forceinline__ void store_weight(void* p, int dtype, int c, float v) {
  if (dtype == 0) static_cast<float*>(p)[c] = v;
  else if (dtype == 1) static_cast<__half*>(p)[c] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
}

// ---- activations ----
// The logistic function. For 16-bit tensors the hardware's approximate exponential and
// reciprocal do (relative errors near 2^-21, against a half step of 2^-9 or 2^-12 in the
// output); 32-bit tensors take the full-precision functions.
template <typename T>
__device__ __forceinline__ float logistic(float z) {
  if constexpr (sizeof(T) == 2) return __fdividef(1.f, 1.f + __expf(-z));
  else return 1.f / (1.f + expf(-z));
}
template <typename T, int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == kNormActSilu) return z * logistic<T>(z);
  else if constexpr (ACT == kNormActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  else return z;
}
// dy * act'(z)
template <typename T, int ACT>
__device__ __forceinline__ float activate_grad(float z, float dy) {
  if constexpr (ACT == kNormActSilu) {
    const float s = logistic<T>(z);
    return dy * (s * fmaf(z, 1.f - s, 1.f));
  } else if constexpr (ACT == kNormActRelu) {
    return z <= 0.f ? 0.f : dy;
  } else {
    return dy;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A CTA's place in the work split.
struct NormTile {
  int64_t n;         // sample
  int s;             // part
  int slice;
  int c0, c1;        // channels of the slice
  int g0, g1;        // groups that touch it
  int64_t p0, p1;    // pixels of the part
  int row, chan;     // this thread's first pixel (from p0) and first channel (from c0)
  bool active;

  __device__ __forceinline__ NormTile(const NormGeometry& g, int V) {
    const int64_t b = blockIdx.x;
    n = b / g.S;
    s = static_cast<int>(b - n * g.S);
    slice = blockIdx.y;
    c0 = slice * g.SC;
    c1 = min(c0 + g.SC, g.C);
    g0 = c0 / g.Cg;
    g1 = (c1 - 1) / g.Cg + 1;
    p0 = g.part_begin(s);
    p1 = g.part_begin(s + 1);
    row = threadIdx.x / g.lanes;
    chan = (threadIdx.x - row * g.lanes) * V;
    active = row < g.rows && c0 + chan < c1;
  }
};

// ---- forward: statistics ----
template <typename T, int V, int U>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sm_mean[kNormThreads * V];
  __shared__ float sm_m2[kNormThreads * V];
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  float mean[V], m2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.f;
  if (t.active) {
    const T* x = static_cast<const T*>(p.x) + t.n * g.P * g.C + t.c0 + t.chan;
    const int64_t step = static_cast<int64_t>(g.rows);
    float count = 0.f;
    int64_t px = t.p0 + t.row;
    for (; px + (U - 1) * step < t.p1; px += U * step) {
      typename IO::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = IO::load(x + (px + u * step) * g.C);
      float f[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) IO::unpack(raw[u], f[u]);
      const float total = count + U;
      const float share = U / total;          // weight of the new values in the mean
      const float cross = count * share;      // and of the squared distance of the two means
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) sum += f[u][v];
        const float m = sum * (1.f / U);
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) q = fmaf(f[u][v] - m, f[u][v] - m, q);
        const float d = m - mean[v];
        mean[v] = fmaf(d, share, mean[v]);
        m2[v] += fmaf(d * d, cross, q);
      }
      count = total;
    }
    for (; px < t.p1; px += step) {
      float f[V];
      IO::unpack(IO::load(x + px * g.C), f);
      count += 1.f;
      const float share = 1.f / count;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = f[v] - mean[v];
        mean[v] = fmaf(d, share, mean[v]);
        m2[v] = fmaf(d, f[v] - mean[v], m2[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sm_mean[t.row * g.SC + t.chan + v] = mean[v];
      sm_m2[t.row * g.SC + t.chan + v] = m2[v];
    }
  }
  __syncthreads();
  // one warp per group: the rows' and channels' pairs become one pair
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t pixels = t.p1 - t.p0;
  const int64_t full = pixels / g.rows;                      // pixels that every row took
  const int extra = static_cast<int>(pixels - full * g.rows);  // rows that took one more
  for (int grp = t.g0 + warp; grp < t.g1; grp += kNormWarps) {
    const int cb = max(grp * g.Cg, t.c0), width = min((grp + 1) * g.Cg, t.c1) - cb;
    const int entries = g.rows * width;
    // means are averaged as distances from one of them: equal values give that value exactly
    const float ref = sm_mean[cb - t.c0];
    float sum = 0.f;
    for (int i = lane; i < entries; i += 32) {
      const int r = i / width;
      const float cnt = static_cast<float>(full + (r < extra));
      sum += cnt > 0.f ? cnt * (sm_mean[r * g.SC + cb - t.c0 + i - r * width] - ref) : 0.f;
    }
    const float m = ref + warp_sum(sum) / (static_cast<float>(pixels) * width);
    float q = 0.f;
    for (int i = lane; i < entries; i += 32) {
      const int r = i / width, at = r * g.SC + cb - t.c0 + i - r * width;
      const float cnt = static_cast<float>(full + (r < extra));
      const float d = sm_mean[at] - m;
      q += cnt > 0.f ? fmaf(cnt * d, d, sm_m2[at]) : 0.f;
    }
    q = warp_sum(q);
    if (lane == 0)
      p.partial[((t.n * g.S + t.s) * g.slices + t.slice) * g.GS + grp - t.g0] = make_float2(m, q);
  }
}

// Merge the parts' pairs of the groups [g0, g1) of sample n: stats[grp - g0] = (mean, rstd).
__device__ __forceinline__ void merge_stats(const NormParams& p, int64_t n, int g0, int g1,
                                            float2* stats) {
  const NormGeometry& g = p.g;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int grp = g0 + warp; grp < g1; grp += kNormWarps) {
    const int first = grp * g.Cg / g.SC, last = ((grp + 1) * g.Cg - 1) / g.SC;
    const int pieces = last - first + 1;
    const int64_t total = static_cast<int64_t>(g.S) * pieces;
    double sum = 0.0, q = 0.0, inv = 1.0 / (static_cast<double>(g.P) * g.Cg), m = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
      for (int64_t i = lane; i < total; i += 32) {
        const int64_t s = i / pieces;
        const int k = first + static_cast<int>(i - s * pieces);
        const int c0 = k * g.SC, c1 = min(c0 + g.SC, g.C);
        const int width = min((grp + 1) * g.Cg, c1) - max(grp * g.Cg, c0);
        const double cnt = static_cast<double>(g.part_begin(s + 1) - g.part_begin(s)) * width;
        const float2 v = p.partial[((n * g.S + s) * g.slices + k) * g.GS + grp - c0 / g.Cg];
        if (pass == 0) sum += cnt * v.x;
        else q += v.y + cnt * (v.x - m) * (v.x - m);
      }
      if (pass == 0) m = warp_sum(sum) * inv;
    }
    const double var = warp_sum(q) * inv;
    if (lane == 0)
      stats[grp - g0] = make_float2(static_cast<float>(m),
                                    static_cast<float>(1.0 / sqrt(var + static_cast<double>(g.eps))));
  }
}

// ---- forward: y ----
template <typename T, int V, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 stats[kNormThreads * V];
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  merge_stats(p, t.n, t.g0, t.g1, stats);
  __syncthreads();
  if (p.mean && t.s == 0) {
    // the slice that holds a group's first channel writes its statistics
    for (int grp = t.g0 + threadIdx.x; grp < t.g1; grp += kNormThreads)
      if (grp * g.Cg >= t.c0) {
        p.mean[t.n * g.G + grp] = stats[grp - t.g0].x;
        p.rstd[t.n * g.G + grp] = stats[grp - t.g0].y;
      }
  }
  if (!t.active) return;
  float mean[V], a[V], b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = t.c0 + t.chan + v;
    const float2 st = stats[c / g.Cg - t.g0];
    mean[v] = st.x;
    a[v] = p.weight ? st.y * load_weight(p.weight, p.weight_dtype, c) : st.y;
    b[v] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
  }
  const int64_t base = t.n * g.P * g.C + t.c0 + t.chan;
  const T* x = static_cast<const T*>(p.x) + base;
  T* y = static_cast<T*>(p.out) + base;
  const int64_t step = g.rows;
  int64_t px = t.p0 + t.row;
  auto emit = [&](const typename IO::Raw& raw, int64_t at) {
    float f[V];
    IO::unpack(raw, f);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = activate<T, ACT>(fmaf(f[v] - mean[v], a[v], b[v]));
    IO::store(y + at * g.C, IO::pack(f));
  };
  for (; px + (U - 1) * step < t.p1; px += U * step) {
    typename IO::Raw raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = IO::load(x + (px + u * step) * g.C);
#pragma unroll
    for (int u = 0; u < U; ++u) emit(raw[u], px + u * step);
  }
  for (; px < t.p1; px += step) emit(IO::load(x + px * g.C), px);
}

// ---- backward: per-channel sums of one part ----
template <typename T, int V, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads) norm_grad_sums_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sm1[kNormThreads * V];
  __shared__ float sm2[kNormThreads * V];
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  if (t.active) {
    float mean[V], a[V], b[V], s1[V], s2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = t.c0 + t.chan + v;
      const int64_t at = t.n * g.G + c / g.Cg;
      mean[v] = p.mean[at];
      a[v] = p.weight ? p.rstd[at] * load_weight(p.weight, p.weight_dtype, c) : p.rstd[at];
      b[v] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
      s1[v] = s2[v] = 0.f;
    }
    const int64_t base = t.n * g.P * g.C + t.c0 + t.chan;
    const T* x = static_cast<const T*>(p.x) + base;
    const T* dy = static_cast<const T*>(p.dy) + base;
    const int64_t step = g.rows;
    int64_t px = t.p0 + t.row;
    auto take = [&](const typename IO::Raw& rx, const typename IO::Raw& rd) {
      float f[V], d[V];
      IO::unpack(rx, f);
      IO::unpack(rd, d);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xc = f[v] - mean[v];
        const float dz = activate_grad<T, ACT>(fmaf(xc, a[v], b[v]), d[v]);
        s1[v] += dz;
        s2[v] = fmaf(dz, xc, s2[v]);
      }
    };
    for (; px + (U - 1) * step < t.p1; px += U * step) {
      typename IO::Raw rx[U], rd[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        rx[u] = IO::load(x + (px + u * step) * g.C);
        rd[u] = IO::load(dy + (px + u * step) * g.C);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) take(rx[u], rd[u]);
    }
    for (; px < t.p1; px += step) take(IO::load(x + px * g.C), IO::load(dy + px * g.C));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sm1[t.row * g.SC + t.chan + v] = s1[v];
      sm2[t.row * g.SC + t.chan + v] = s2[v];
    }
  }
  __syncthreads();
  // L lanes (a power of two, at most a warp) sum the rows of one channel
  int L = 1;
  while (L < 32 && 2 * L <= g.rows) L *= 2;
  const int sub = threadIdx.x % L, width = t.c1 - t.c0;
  const int passes = (width + kNormThreads / L - 1) / (kNormThreads / L);
  for (int i = 0; i < passes; ++i) {
    const int c = i * (kNormThreads / L) + threadIdx.x / L;
    float v1 = 0.f, v2 = 0.f;
    if (c < width)
      for (int r = sub; r < g.rows; r += L) {
        v1 += sm1[r * g.SC + c];
        v2 += sm2[r * g.SC + c];
      }
    for (int o = L / 2; o > 0; o >>= 1) {
      v1 += __shfl_xor_sync(0xffffffffu, v1, o);
      v2 += __shfl_xor_sync(0xffffffffu, v2, o);
    }
    if (c < width && sub == 0)
      p.partial[(t.n * g.S + t.s) * g.C + t.c0 + c] = make_float2(v1, v2);
  }
}

// ---- backward: sums over the parts, and each group's two means. One CTA per (group, sample) ----
__global__ void __launch_bounds__(kNormThreads) norm_grad_coef_kernel(const __grid_constant__ NormParams p) {
  __shared__ double sm1[kNormThreads], sm2[kNormThreads];
  const NormGeometry& g = p.g;
  const int grp = blockIdx.x;
  const int64_t n = blockIdx.y + static_cast<int64_t>(gridDim.y) * blockIdx.z;
  if (n >= g.N) return;
  grid_dependency_wait();
  grid_launch_dependents();
  // cols channels at a time (a power of two, at most 32), kNormThreads / cols threads each
  int cols = 1;
  while (cols < 32 && cols < g.Cg) cols *= 2;
  const int col = threadIdx.x % cols, sub = threadIdx.x / cols, subs = kNormThreads / cols;
  const float rstd = p.rstd[n * g.G + grp];
  double w1 = 0.0, w2 = 0.0;  // sum of w dz and of w dz xhat, kept by the threads with sub == 0
  for (int cb = 0; cb < g.Cg; cb += cols) {
    const int c = cb + col;
    double v1 = 0.0, v2 = 0.0;
    if (c < g.Cg)
      for (int s = sub; s < g.S; s += subs) {
        const float2 v = p.partial[(n * g.S + s) * g.C + grp * g.Cg + c];
        v1 += v.x;
        v2 += v.y;
      }
    sm1[threadIdx.x] = v1;
    sm2[threadIdx.x] = v2;
    __syncthreads();
    for (int o = subs / 2; o > 0; o >>= 1) {
      if (sub < o) {
        sm1[threadIdx.x] += sm1[threadIdx.x + o * cols];
        sm2[threadIdx.x] += sm2[threadIdx.x + o * cols];
      }
      __syncthreads();
    }
    if (sub == 0 && c < g.Cg) {
      const int ch = grp * g.Cg + c;
      const double s1 = sm1[threadIdx.x], s2 = sm2[threadIdx.x] * rstd;
      p.chan[n * g.C + ch] = make_float2(static_cast<float>(s1), static_cast<float>(s2));
      const double w = p.weight ? load_weight(p.weight, p.weight_dtype, ch) : 1.0;
      w1 += w * s1;
      w2 += w * s2;
    }
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    w1 = warp_sum(sub == 0 ? w1 : 0.0);
    w2 = warp_sum(sub == 0 ? w2 : 0.0);
    if (threadIdx.x == 0) {
      const double m = static_cast<double>(g.P) * g.Cg;
      p.coef[n * g.G + grp] = make_float2(static_cast<float>(rstd * (w1 / m)),
                                          static_cast<float>(rstd * (rstd * (w2 / m))));
    }
  }
}

// ---- backward: dweight and dbias, sums over the samples in their order ----
__global__ void __launch_bounds__(kNormThreads) norm_param_grad_kernel(const __grid_constant__ NormParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int c = blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= p.g.C) return;
  double db = 0.0, dw = 0.0;
  for (int64_t n = 0; n < p.g.N; ++n) {
    const float2 v = p.chan[n * p.g.C + c];
    db += v.x;
    dw += v.y;
  }
  if (p.dweight) store_weight(p.dweight, p.weight_dtype, c, static_cast<float>(dw));
  if (p.dbias) store_weight(p.dbias, p.weight_dtype, c, static_cast<float>(db));
}

// ---- backward: dx ----
template <typename T, int V, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads) norm_grad_apply_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  if (!t.active) return;
  float mean[V], a[V], b[V], k1[V], k2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = t.c0 + t.chan + v;
    const int64_t at = t.n * g.G + c / g.Cg;
    mean[v] = p.mean[at];
    a[v] = p.weight ? p.rstd[at] * load_weight(p.weight, p.weight_dtype, c) : p.rstd[at];
    b[v] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
    const float2 k = p.coef[at];
    k1[v] = k.x;
    k2[v] = k.y;
  }
  const int64_t base = t.n * g.P * g.C + t.c0 + t.chan;
  const T* x = static_cast<const T*>(p.x) + base;
  const T* dy = static_cast<const T*>(p.dy) + base;
  T* dx = static_cast<T*>(p.out) + base;
  const int64_t step = g.rows;
  int64_t px = t.p0 + t.row;
  auto emit = [&](const typename IO::Raw& rx, const typename IO::Raw& rd, int64_t at) {
    float f[V], d[V];
    IO::unpack(rx, f);
    IO::unpack(rd, d);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float xc = f[v] - mean[v];
      const float dz = activate_grad<T, ACT>(fmaf(xc, a[v], b[v]), d[v]);
      f[v] = fmaf(-xc, k2[v], fmaf(a[v], dz, -k1[v]));
    }
    IO::store(dx + at * g.C, IO::pack(f));
  };
  for (; px + (U - 1) * step < t.p1; px += U * step) {
    typename IO::Raw rx[U], rd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rx[u] = IO::load(x + (px + u * step) * g.C);
      rd[u] = IO::load(dy + (px + u * step) * g.C);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) emit(rx[u], rd[u], px + u * step);
  }
  for (; px < t.p1; px += step) emit(IO::load(x + px * g.C), IO::load(dy + px * g.C), px);
}

}  // namespace fssim
