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
// a reducing pass, a small launch that merges the parts, and an applying pass; the second read
// comes from L2 where the samples in flight fit it (the host cuts the batch accordingly), from
// the end of each part backwards, because that is what the reducing pass read last.
//
// Statistics: a thread takes U pixels at a time, forms each channel's mean and sum of squared
// deviations of those U values (two passes over registers), and merges them into its running
// pair (the pairwise update of Chan, Golub and LeVeque, 1979). No sum of raw squares is ever
// formed, so a mean far from zero costs no digits. Threads, channels, parts and slices are
// merged likewise, in a fixed order (results repeat bit for bit), across parts in FP64.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

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

  int64_t base;  // pixels of a part; the first `extra` parts have one more
  int extra;

  __device__ __forceinline__ int64_t part_pixels(int s) const { return base + (s < extra); }
  __device__ __forceinline__ int64_t part_begin(int s) const { return base * s + min(s, extra); }
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
  float2* sums;         // backward: (sum dz, sum dz xhat) per (sample, channel)
  float* channel;       // what the applying pass needs, C values each, per sample: the mean, the
                        // factor a = rstd w and the shift b (kNormForwardRows rows); in the
                        // backward also rstd <w dz> and rstd^2 <w dz xhat> (kNormBackwardRows)
  int early;            // a reducing pass that need not wait for the launch before it to begin
  void* dweight;
  void* dbias;
};

constexpr int kNormForwardRows = 3;
constexpr int kNormBackwardRows = 5;

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

// V consecutive values of a row of `channel`, which starts at a multiple of V floats.
template <int V>
__device__ __forceinline__ void load_channels(const float* p, float (&f)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = p[i];
  }
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
  int n;             // sample
  int s;             // part
  int slice;
  int c0, c1;        // channels of the slice
  int g0, g1;        // groups that touch it
  int64_t p0, p1;    // pixels of the part
  int row, chan;     // this thread's first pixel (from p0) and first channel (from c0)
  bool active;

  __device__ __forceinline__ NormTile(const NormGeometry& g, int V) {
    n = blockIdx.x / g.S;
    s = blockIdx.x - n * g.S;
    slice = blockIdx.y;
    c0 = slice * g.SC;
    c1 = min(c0 + g.SC, g.C);
    g0 = c0 / g.Cg;
    g1 = (c1 - 1) / g.Cg + 1;
    p0 = g.part_begin(s);
    p1 = p0 + g.part_pixels(s);
    row = threadIdx.x / g.lanes;
    chan = (threadIdx.x - row * g.lanes) * V;
    active = row < g.rows && c0 + chan < c1;
  }
};

// First channel, from the slice's first, of the group that channel c of the slice is in.
__device__ __forceinline__ int group_begin(const NormGeometry& g, const NormTile& t, int c) {
  return max((t.c0 + c) / g.Cg * g.Cg - t.c0, 0);
}

// out[c] = sum over the rows r of f(r, c), for the `width` channels of a slice: L lanes (a power
// of two, at most a warp) for each channel. All threads take part.
template <typename F>
__device__ __forceinline__ void norm_sum_rows(int rows, int pitch, int width, float* out, F f) {
  const int L = rows >= 32 ? 32 : 1 << (31 - __clz(rows));
  const int sub = threadIdx.x & (L - 1), each = kNormThreads / L;
  for (int b = 0; b < width; b += each) {
    const int c = b + threadIdx.x / L;
    float v = 0.f;
    if (c < width)
      for (int r = sub; r < rows; r += L) v += f(r, c);
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (c < width && sub == 0) out[c] = v;
  }
}

// f(i, cb, w, sum of in[cb .. cb + w)) for the i-th group that touches the slice, its channels
// [cb, cb + w) of the slice: a thread for each narrow group, a warp for each wide one.
template <typename F>
__device__ __forceinline__ void norm_sum_groups(const NormGeometry& g, const NormTile& t, const float* in, F f) {
  const bool narrow = g.Cg <= 32;
  const int lane = narrow ? 0 : threadIdx.x % 32, lanes = narrow ? 1 : 32;
  for (int i = threadIdx.x / lanes; i < t.g1 - t.g0; i += kNormThreads / lanes) {
    const int cb = max((t.g0 + i) * g.Cg, t.c0) - t.c0;
    const int w = min((t.g0 + i + 1) * g.Cg, t.c1) - t.c0 - cb;
    float v = 0.f;
    for (int c = lane; c < w; c += lanes) v += in[cb + c];
    if (!narrow) v = warp_sum(v);
    if (lane == 0) f(i, cb, w, v);
  }
}

// The pixels of a thread in the applying passes: from the end of its part to the beginning (what
// the reducing pass read last is what L2 still holds), U at a time; the last step, at the
// beginning of the part, may be short.
template <int U>
struct NormSteps {
  int64_t at;      // first pixel of the current step
  int64_t left;    // pixels still to do, the current step's among them
  int rows;

  __device__ __forceinline__ NormSteps(const NormGeometry& g, const NormTile& t) : rows(g.rows) {
    const int64_t first = t.p0 + t.row;
    left = t.active && first < t.p1 ? (t.p1 - first - 1) / rows + 1 : 0;
    at = first + (left - U) * rows;
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  // the short step lacks its first pixels
  __device__ __forceinline__ bool has(int u) const { return left >= U || u >= U - left; }
  __device__ __forceinline__ int64_t pixel(int u) const { return at + static_cast<int64_t>(u) * rows; }
  __device__ __forceinline__ void next() {
    at -= static_cast<int64_t>(U) * rows;
    left -= U;
  }
};

// ---- forward: statistics ----
template <typename T, int V, int U>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sm_mean[kNormThreads * V];
  __shared__ float sm_m2[kNormThreads * V];
  __shared__ float column[kNormThreads * V];
  __shared__ float centre[kNormThreads * V];
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  if (!p.early) grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  float mean[V], m2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.f;
  if (t.active) {
    const T* x = static_cast<const T*>(p.x) + static_cast<int64_t>(t.n) * g.P * g.C + t.c0 + t.chan;
    const int64_t step = static_cast<int64_t>(g.rows);
    float count = 0.f;
    int64_t px = t.p0 + t.row;
    // U pixels, or the last k of them (k < U) with the missing ones left out
    auto take = [&](auto whole, int k) {
      constexpr bool kWhole = decltype(whole)::value;
      typename IO::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (kWhole || u < k) raw[u] = IO::load(x + (px + u * step) * g.C);
        else raw[u] = typename IO::Raw{};
      }
      float f[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) IO::unpack(raw[u], f[u]);
      const float taken = kWhole ? U : k;
      const float total = count + taken;
      const float each = kWhole ? 1.f / U : 1.f / taken;
      const float share = taken / total;   // weight of the new values in the mean
      const float cross = count * share;   // and of the squared distance of the means
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) sum += f[u][v];
        const float m = sum * each;
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float d = kWhole || u < k ? f[u][v] - m : 0.f;
          q = fmaf(d, d, q);
        }
        const float d = m - mean[v];
        mean[v] = fmaf(d, share, mean[v]);
        m2[v] += fmaf(d * d, cross, q);
      }
      count = total;
    };
    for (; px + (U - 1) * step < t.p1; px += U * step) take(std::true_type{}, U);
    if (px < t.p1) take(std::false_type{}, static_cast<int>((t.p1 - px - 1) / step) + 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sm_mean[t.row * g.SC + t.chan + v] = mean[v];
      sm_m2[t.row * g.SC + t.chan + v] = m2[v];
    }
  }
  __syncthreads();
  // The rows' and channels' pairs become one pair per group: first the mean (as distances from
  // one of the means, so that equal values give that value exactly), then the deviations.
  const int64_t pixels = t.p1 - t.p0;
  const int64_t full = pixels / g.rows;                        // pixels that every row took
  const int extra = static_cast<int>(pixels - full * g.rows);  // rows that took one more
  const int width = t.c1 - t.c0;
  const auto count_of = [&](int row) { return static_cast<float>(full + (row < extra)); };
  norm_sum_rows(g.rows, g.SC, width, column, [&](int r, int c) {
    const float cnt = count_of(r);
    return cnt > 0.f ? cnt * (sm_mean[r * g.SC + c] - sm_mean[group_begin(g, t, c)]) : 0.f;
  });
  __syncthreads();
  float2* partial = p.partial + ((static_cast<int64_t>(t.n) * g.S + t.s) * g.slices + t.slice) * g.GS;
  norm_sum_groups(g, t, column, [&](int i, int cb, int w, float sum) {
    centre[i] = sm_mean[cb] + sum / (static_cast<float>(pixels) * w);
  });
  __syncthreads();
  norm_sum_rows(g.rows, g.SC, width, column, [&](int r, int c) {
    const float cnt = count_of(r);
    const float d = sm_mean[r * g.SC + c] - centre[(t.c0 + c) / g.Cg - t.g0];
    return cnt > 0.f ? fmaf(cnt * d, d, sm_m2[r * g.SC + c]) : 0.f;
  });
  __syncthreads();
  norm_sum_groups(g, t, column, [&](int i, int cb, int w, float sum) {
    partial[i] = make_float2(centre[i], sum);
  });
  if (p.early) grid_dependency_wait();
}

// ---- forward: the parts' pairs become the groups' statistics. One warp per (sample, group) ----
__global__ void __launch_bounds__(kNormThreads) norm_merge_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kNormWarps + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  grid_dependency_wait();
  grid_launch_dependents();
  if (id >= g.N * g.G) return;
  const int64_t n = id / g.G;
  const int grp = static_cast<int>(id - n * g.G);
  const int c0 = grp * g.Cg, c1 = c0 + g.Cg;
  const int first = c0 / g.SC, last = (c1 - 1) / g.SC;
  const double inv = 1.0 / (static_cast<double>(g.P) * g.Cg);
  double ref = 0.0, sum = 0.0, q = 0.0;  // sums of distances from ref, and of squares around it
  for (int k = first; k <= last; ++k) {  // the slices that hold a piece of the group
    const int b = k * g.SC, width = min(c1, b + g.SC) - max(c0, b);
    const float2* pairs = p.partial + (n * g.S * g.slices + k) * g.GS + grp - b / g.Cg;
    if (k == first) ref = pairs[0].x;
    for (int s = lane; s < g.S; s += 32) {
      const float2 v = pairs[static_cast<int64_t>(s) * g.slices * g.GS];
      const double cnt = static_cast<double>(g.part_pixels(s)) * width;
      const double d = v.x - ref;
      sum = fma(cnt, d, sum);
      q += fma(cnt * d, d, static_cast<double>(v.y));
    }
  }
  sum = warp_sum(sum) * inv;
  double var = warp_sum(q) * inv - sum * sum;
  if (var < 0.0) var = 0.0;  // a NaN stays
  const float mean = static_cast<float>(ref + sum);
  const float rstd = static_cast<float>(1.0 / sqrt(var + static_cast<double>(g.eps)));
  if (p.mean && lane == 0) {
    p.mean[id] = mean;
    p.rstd[id] = rstd;
  }
  float* row = p.channel + n * kNormForwardRows * g.C;
  for (int c = c0 + lane; c < c1; c += 32) {
    row[c] = mean;
    row[g.C + c] = p.weight ? rstd * load_weight(p.weight, p.weight_dtype, c) : rstd;
    row[2 * static_cast<int64_t>(g.C) + c] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
  }
}

// ---- forward: y ----
template <typename T, int V, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  using IO = VecIO<T, V>;
  const int64_t base = static_cast<int64_t>(t.n) * g.P * g.C + t.c0 + t.chan;
  const T* x = static_cast<const T*>(p.x) + base;
  T* y = static_cast<T*>(p.out) + base;
  NormSteps<U> steps(g, t);
  // x was complete before the statistics' launch began its work, so the first reads need not
  // wait for that launch to end
  typename IO::Raw raw[U];
  auto fetch = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (steps.has(u)) raw[u] = IO::load(x + steps.pixel(u) * g.C);
  };
  if (steps.more()) fetch();
  grid_dependency_wait();
  float mean[V], a[V], b[V];
  if (t.active) {
    const float* row = p.channel + static_cast<int64_t>(t.n) * kNormForwardRows * g.C + t.c0 + t.chan;
    load_channels<V>(row, mean);
    load_channels<V>(row + g.C, a);
    load_channels<V>(row + 2 * static_cast<int64_t>(g.C), b);
  }
  grid_launch_dependents();  // the statistics have been read
  auto emit = [&](const typename IO::Raw& r, int64_t at) {
    float f[V];
    IO::unpack(r, f);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = activate<T, ACT>(fmaf(f[v] - mean[v], a[v], b[v]));
    IO::store(y + at * g.C, IO::pack(f));
  };
  while (steps.more()) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (steps.has(u)) emit(raw[u], steps.pixel(u));
    steps.next();
    if (steps.more()) fetch();
  }
}

// ---- backward: per-channel sums of one part ----
template <typename T, int V, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads) norm_grad_sums_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sm1[kNormThreads * V];
  __shared__ float sm2[kNormThreads * V];
  __shared__ float column1[kNormThreads * V];
  __shared__ float column2[kNormThreads * V];
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  if (!p.early) grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  if (t.active) {
    float mean[V], a[V], b[V], s1[V], s2[V];
    const int first = t.c0 + t.chan;
    int grp = first / g.Cg, end = (grp + 1) * g.Cg;  // one division; the next channels follow
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = first + v;
      if (c == end) {
        ++grp;
        end += g.Cg;
      }
      const int64_t at = static_cast<int64_t>(t.n) * g.G + grp;
      mean[v] = p.mean[at];
      a[v] = p.weight ? p.rstd[at] * load_weight(p.weight, p.weight_dtype, c) : p.rstd[at];
      b[v] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
      s1[v] = s2[v] = 0.f;
    }
    const int64_t base = static_cast<int64_t>(t.n) * g.P * g.C + t.c0 + t.chan;
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
    for (; px < t.p1; px += U * step) {
      typename IO::Raw rx[U], rd[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (px + u * step < t.p1) {
          rx[u] = IO::load(x + (px + u * step) * g.C);
          rd[u] = IO::load(dy + (px + u * step) * g.C);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (px + u * step < t.p1) take(rx[u], rd[u]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sm1[t.row * g.SC + t.chan + v] = s1[v];
      sm2[t.row * g.SC + t.chan + v] = s2[v];
    }
  }
  __syncthreads();
  const int width = t.c1 - t.c0;
  norm_sum_rows(g.rows, g.SC, width, column1, [&](int r, int c) { return sm1[r * g.SC + c]; });
  norm_sum_rows(g.rows, g.SC, width, column2, [&](int r, int c) { return sm2[r * g.SC + c]; });
  __syncthreads();
  float2* partial = p.partial + (static_cast<int64_t>(t.n) * g.S + t.s) * g.C + t.c0;
  for (int c = threadIdx.x; c < width; c += kNormThreads) partial[c] = make_float2(column1[c], column2[c]);
  if (p.early) grid_dependency_wait();
}

// ---- backward: sums over the parts, and each group's two means. One CTA per (group, sample) ----
__global__ void __launch_bounds__(kNormThreads) norm_grad_coef_kernel(const __grid_constant__ NormParams p) {
  __shared__ double sm1[kNormThreads], sm2[kNormThreads];
  __shared__ float means[2];
  const NormGeometry& g = p.g;
  const int64_t n = blockIdx.x / static_cast<unsigned>(g.G);
  const int grp = static_cast<int>(blockIdx.x - n * g.G);
  grid_dependency_wait();
  grid_launch_dependents();
  // cols channels at a time (a power of two, at most 32), kNormThreads / cols threads each
  int cols = 1;
  while (cols < 32 && cols < g.Cg) cols *= 2;
  const int col = threadIdx.x % cols, sub = threadIdx.x / cols, subs = kNormThreads / cols;
  const float mean = p.mean[n * g.G + grp], rstd = p.rstd[n * g.G + grp];
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
      p.sums[n * g.C + ch] = make_float2(static_cast<float>(s1), static_cast<float>(s2));
      const double w = p.weight ? load_weight(p.weight, p.weight_dtype, ch) : 1.0;
      w1 += w * s1;
      w2 += w * s2;
    }
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    w1 = warp_sum(sub == 0 ? w1 : 0.0);
    w2 = warp_sum(sub == 0 ? w2 : 0.0);
    const double m = static_cast<double>(g.P) * g.Cg;
    if (threadIdx.x == 0) {
      means[0] = static_cast<float>(rstd * (w1 / m));
      means[1] = static_cast<float>(rstd * (rstd * (w2 / m)));
    }
  }
  __syncthreads();
  float* row = p.channel + n * kNormBackwardRows * g.C;
  for (int c = grp * g.Cg + threadIdx.x; c < (grp + 1) * g.Cg; c += kNormThreads) {
    const int64_t C = g.C;
    row[c] = mean;
    row[C + c] = p.weight ? rstd * load_weight(p.weight, p.weight_dtype, c) : rstd;
    row[2 * C + c] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
    row[3 * C + c] = means[0];
    row[4 * C + c] = means[1];
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
    const float2 v = p.sums[n * p.g.C + c];
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
  using IO = VecIO<T, V>;
  const int64_t base = static_cast<int64_t>(t.n) * g.P * g.C + t.c0 + t.chan;
  const T* x = static_cast<const T*>(p.x) + base;
  const T* dy = static_cast<const T*>(p.dy) + base;
  T* dx = static_cast<T*>(p.out) + base;
  NormSteps<U> steps(g, t);
  // as in the forward, the first reads do not wait for the launch before
  typename IO::Raw rx[U], rd[U];
  auto fetch = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (steps.has(u)) {
        rx[u] = IO::load(x + steps.pixel(u) * g.C);
        rd[u] = IO::load(dy + steps.pixel(u) * g.C);
      }
    }
  };
  if (steps.more()) fetch();
  grid_dependency_wait();
  float mean[V], a[V], b[V], k1[V], k2[V];
  if (t.active) {
    const int64_t C = g.C;
    const float* row = p.channel + t.n * kNormBackwardRows * C + t.c0 + t.chan;
    load_channels<V>(row, mean);
    load_channels<V>(row + C, a);
    load_channels<V>(row + 2 * C, b);
    load_channels<V>(row + 3 * C, k1);
    load_channels<V>(row + 4 * C, k2);
  }
  grid_launch_dependents();  // the means have been read
  auto emit = [&](const typename IO::Raw& ra, const typename IO::Raw& rb, int64_t at) {
    float f[V], d[V];
    IO::unpack(ra, f);
    IO::unpack(rb, d);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float xc = f[v] - mean[v];
      const float dz = activate_grad<T, ACT>(fmaf(xc, a[v], b[v]), d[v]);
      f[v] = fmaf(-xc, k2[v], fmaf(a[v], dz, -k1[v]));
    }
    IO::store(dx + at * g.C, IO::pack(f));
  };
  while (steps.more()) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (steps.has(u)) emit(rx[u], rd[u], steps.pixel(u));
    steps.next();
    if (steps.more()) fetch();
  }
}

}  // namespace fssim
