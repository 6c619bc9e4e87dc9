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
// Work split: the group's numbers must all be seen before its first output, so each direction is a
// reducing pass, a small launch that merges its results, and an applying pass. The channels are
// cut into slices of at most 256 vectors of V channels. A thread keeps one vector of channels and
// steps over pixels, so the per-channel constants and sums stay in registers and a warp reads
// whole rows of memory. Where C is no multiple of the vector (three-channel images), the least
// number of pixels whose channels together are, `period` of them, is taken as one pixel of
// period * C channels: a span. Elsewhere a span is a pixel.
//   Reducing: a sample's pixels are cut into tiles and dealt out in turn to S parts, one CTA
//   each and one wave of CTAs in all: few results to merge, and the GPU reads memory as one
//   moving window.
//   Applying: S short contiguous parts, a CTA each, from the end of the samples to their
//   beginning: what the reducing pass read last is what L2 still holds.
//
// Statistics: a thread takes U spans at a time, forms each channel's mean and sum of squared
// deviations of those U values (from their distances to the first of them), and merges them into
// its running pair (the pairwise update of Chan, Golub and LeVeque, 1979). No sum of raw squares is
// ever formed, so a mean far from zero costs no digits. Threads, channels, parts and slices are
// merged likewise, in a fixed order (results repeat bit for bit), within a CTA in FP32, over a
// thread's long part and across parts in FP64.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "pdl.cuh"

namespace fssim {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;
constexpr int kNormResident = 2;       // CTAs of a reducing pass on one SM
constexpr int kNormApplyResident = 2;  // and of an applying pass

enum NormAct { kNormActNone = 0, kNormActSilu = 1, kNormActRelu = 2 };

struct NormGeometry {
  int64_t N;   // samples
  int64_t P;   // pixels per sample
  int C, G, Cg;
  int period;  // pixels of a span
  int Cv;      // channels of a span: period * C
  int SC;      // channels of a span per slice (a multiple of V); one slice has all where period > 1
  int slices;
  int lanes;   // SC / V
  int rows;    // spans a CTA takes per step
  int S;       // parts of a sample's spans
  int GS;      // most groups that touch one slice
  float eps;
  float keep;        // share of the input that may stay in L2 from pass to pass
  double inv_m;      // 1 / (P * Cg)
  // Reducing passes: part s has the tiles s, s + S, ... of `tile` spans; the last of all, which
  // `last_part` has, lacks `lacking` spans. Parts have `part_tiles` tiles, the first `extra_tiles`
  // one more. (A part's pixels fit 31 bits, and the kernels divide no 64-bit numbers: that
  // alone took microseconds of a launch.)
  int tile, part_tiles, extra_tiles, last_part, lacking;
  // Applying passes: contiguous parts of `base` spans; the first `extra` have one more.
  int base, extra;

  __device__ __forceinline__ int tiles_of(int s) const { return part_tiles + (s < extra_tiles); }
  __device__ __forceinline__ int part_spans(int s) const {
    return tiles_of(s) * tile - (s == last_part ? lacking : 0);
  }
  __device__ __forceinline__ int part_pixels(int s) const { return part_spans(s) * period; }
  __device__ __forceinline__ int run_spans(int s) const { return base + (s < extra); }
  // In a CTA's shared memory a thread row holds one value for each channel of a span: seen by
  // pixels, rows * period rows of the real channels.
  __device__ __forceinline__ int pixel_rows() const { return rows * period; }
  __device__ __forceinline__ int pitch() const { return period == 1 ? SC : C; }
};

struct NormParams {
  NormGeometry g;
  const void* x;
  const void* dy;
  void* out;            // y or dx
  const void* weight;   // C values of weight_dtype, or nullptr (ones)
  const void* bias;     // C values of weight_dtype, or nullptr (zeros)
  int weight_vectors;   // both start at a multiple of 16 bytes
  int merges;           // parts of a sample whose results the applying pass merges itself, or 0
  int weight_dtype;
  float* mean;          // N * G
  float* rstd;          // N * G
  float2* partial;      // forward: (mean, M2) per (sample, part, slice, group of the slice)
                        // backward: (sum dz, sum dz (x - mean)) per (sample, part, channel)
  float2* sums;         // backward: (sum dz, sum dz xhat) per (sample, channel)
  float* channel;       // what the applying pass needs, C values each, per sample: the mean, the
                        // factor a = rstd w and the shift b (kNormForwardRows rows); in the
                        // backward also rstd <w dz> and rstd^2 <w dz xhat> (kNormBackwardRows)
  void* dweight;
  void* dbias;
  int fold_params;      // the applying pass of the backward sums dweight and dbias too
};

constexpr int kNormForwardRows = 3;
constexpr int kNormBackwardRows = 5;

// ---- element types ----
template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<4> { using type = unsigned; };
template <> struct RawVec<2> { using type = unsigned short; };

// V elements in registers as pairs, for the packed FP32 instructions (one for two elements). A
// lone element has a pair to itself, whose second half is zero and never stored.
template <int V> constexpr int kPairs = (V + 1) / 2;

__device__ __forceinline__ float2 norm_pair(unsigned w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 norm_pair(unsigned w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ unsigned norm_word(float2 f, __half) {
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned norm_word(float2 f, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const unsigned*>(&h);
}

template <typename T, int V>
struct VecIO {
  using Raw = typename RawVec<sizeof(T) * V>::type;
  static constexpr int N = kPairs<V>;
  static __device__ __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void store(T* p, const Raw& r) { *reinterpret_cast<Raw*>(p) = r; }
  static __device__ __forceinline__ void unpack(const Raw& r, float2 (&f)[N]) {
    if constexpr (sizeof(T) == 4) {
      const float* e = reinterpret_cast<const float*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = make_float2(e[2 * i], V > 1 ? e[2 * i + 1] : 0.f);
    } else if constexpr (V == 1) {
      f[0] = norm_pair(static_cast<unsigned>(r), T());
    } else {
      const unsigned* w = reinterpret_cast<const unsigned*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = norm_pair(w[i], T());
    }
  }
  static __device__ __forceinline__ Raw pack(const float2 (&f)[N]) {
    Raw r;
    if constexpr (sizeof(T) == 4) {
      float* e = reinterpret_cast<float*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        e[2 * i] = f[i].x;
        if (V > 1) e[2 * i + 1] = f[i].y;
      }
    } else if constexpr (V == 1) {
      r = static_cast<Raw>(norm_word(f[0], T()));
    } else {
      unsigned* w = reinterpret_cast<unsigned*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = norm_word(f[i], T());
    }
    return r;
  }
};

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }
__device__ __forceinline__ float2 splat2(float a) { return make_float2(a, a); }

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
__device__ __forceinline__ void load_channels(const float* p, float2 (&f)[kPairs<V>]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      f[i / 2] = make_float2(v.x, v.y);
      f[i / 2 + 1] = make_float2(v.z, v.w);
    }
  } else if constexpr (V == 2) {
    f[0] = *reinterpret_cast<const float2*>(p);
  } else {
    f[0] = make_float2(*p, 0.f);
  }
}

// ---- activations, on pairs ----
// The logistic function s and 1 - s.
template <typename T>
__device__ __forceinline__ void logistic(float2 z, float2& s, float2& rest) {
  if constexpr (sizeof(T) == 2) {
    // The hardware's approximate power of two (2^-22 relative) and reciprocal (1 ulp), the latter of
    // 1 + exp(-z) in units of 2^24: it flushes subnormal results, and s is one below z = -87.3. With
    // the rounding of the power's exponent s is right to 2^-20 + |z| 2^-24, against a half step of
    // 2^-9 or 2^-12 in the output, down to z = -88.72, where exp(-z) leaves FP32 and s is 0. (The
    // whole of FP32's range, by half the exponent and a square, takes 0.5 to 2 % longer: 1080p
    // training pass 350 against 343 us.)
    constexpr float kLog = -1.44269504f;  // 2^(-z / ln 2) = exp(-z)
    const float2 unit = splat2(0x1p-24f);
    float2 e = mul2(z, splat2(kLog));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
    const float2 d = fma2(e, unit, unit);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(d.y));
    s = mul2(s, unit);
    rest = fma2(s, splat2(-1.f), splat2(1.f));
  } else {
    // With t = exp(-|z|), which does not overflow, they are r = 1 / (1 + t) and t r, in this order
    // for z >= 0 and the other way round below: nothing cancels, and s fades out through the
    // subnormal numbers near z = -104. r is the approximate reciprocal after one step of Newton's
    // iteration (1x48x517x999 training pass 129 us; 155 with the rounded reciprocal instead).
    const float2 t = make_float2(expf(-fabsf(z.x)), expf(-fabsf(z.y)));
    const float2 minus = fma2(t, splat2(-1.f), splat2(-1.f));
    float2 r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(-minus.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(-minus.y));
    r = fma2(r, fma2(minus, r, splat2(1.f)), r);
    const float2 q = mul2(t, r);
    s = make_float2(z.x < 0.f ? q.x : r.x, z.y < 0.f ? q.y : r.y);
    rest = make_float2(z.x < 0.f ? r.x : q.x, z.y < 0.f ? r.y : q.y);
  }
}
template <typename T, int ACT>
__device__ __forceinline__ float2 activate(float2 z) {
  if constexpr (ACT == kNormActSilu) {
    float2 s, rest;
    logistic<T>(z, s, rest);
    return mul2(z, s);
  } else if constexpr (ACT == kNormActRelu)
    return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y);  // NaN stays NaN
  else return z;
}
// dy * act'(z)
template <typename T, int ACT>
__device__ __forceinline__ float2 activate_grad(float2 z, float2 dy) {
  if constexpr (ACT == kNormActSilu) {
    float2 s, rest;
    logistic<T>(z, s, rest);
    return mul2(mul2(dy, s), fma2(z, rest, splat2(1.f)));
  } else if constexpr (ACT == kNormActRelu) {
    return make_float2(z.x <= 0.f ? 0.f : dy.x, z.y <= 0.f ? 0.f : dy.y);
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
  int row, chan;     // this thread's row, and its first channel (from c0)
  bool active;

  __device__ __forceinline__ NormTile(const NormGeometry& g, int V, bool applying) {
    if (applying) {
      s = blockIdx.x / static_cast<unsigned>(g.N);
      n = blockIdx.x - s * static_cast<unsigned>(g.N);
      s = g.S - 1 - s;
    } else {
      n = blockIdx.x / static_cast<unsigned>(g.S);
      s = blockIdx.x - n * g.S;
    }
    slice = blockIdx.y;
    place(g, V);
  }
  // the resident kernels: a cluster of S CTAs for each sample and slice
  __device__ __forceinline__ NormTile(const NormGeometry& g, int V) {
    const unsigned unit = blockIdx.x / static_cast<unsigned>(g.S);
    s = blockIdx.x - unit * g.S;
    n = unit / static_cast<unsigned>(g.slices);
    slice = unit - n * g.slices;
    place(g, V);
  }
  __device__ __forceinline__ void place(const NormGeometry& g, int V) {
    c0 = slice * g.SC;
    c1 = min(c0 + g.SC, g.C);
    g0 = c0 / g.Cg;
    g1 = (c1 - 1) / g.Cg + 1;
    row = threadIdx.x / g.lanes;
    chan = (threadIdx.x - row * g.lanes) * V;
    active = row < g.rows && c0 + chan < min(c0 + g.SC, g.Cv);
  }
};

// V values into shared memory.
template <int V>
__device__ __forceinline__ void norm_put(float* p, const float2 (&f)[kPairs<V>]) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    p[2 * i] = f[i].x;
    if (V > 1) p[2 * i + 1] = f[i].y;
  }
}

// Sums over a CTA's rows, then over a group's channels. The rows are shared out over T threads for
// each channel (all of the CTA's, where the slice has fewer channels than threads), which leave
// T subtotals of each channel in out[j * cols + c], T * cols of them in all where T is not 1 (a
// slice may be the last and narrow); f(c) gives the function of a row for channel c.
struct NormColumns {
  int cols, T, col, sub;
  __device__ __forceinline__ explicit NormColumns(int width) {
    const int shift = width > kNormThreads / 2 ? __ffs(kNormThreads) - 1 : width > 1 ? 32 - __clz(width - 1) : 0;
    cols = 1 << shift;
    T = kNormThreads >> shift;
    col = threadIdx.x & (cols - 1);
    sub = threadIdx.x >> shift;
  }
  template <typename F>
  __device__ __forceinline__ void sum_rows(const NormGeometry& g, int width, float* out, F f) const {
    for (int c = col; c < width; c += cols) {
      const auto value = f(c);
      float v = 0.f;
#pragma unroll 4
      for (int r = sub; r < g.pixel_rows(); r += T) v += value(r);
      out[sub * cols + c] = v;
    }
  }
  // f(i, cb, w, sum of the subtotals of [cb, cb + w)) for the i-th group that touches the slice,
  // its channels [cb, cb + w) of the slice: a thread for each where there is little to add, a
  // warp for each otherwise, whose lanes share out both the channels and the subtotals
  // (1x1x1080x1920 16-bit forward 13 us, and 47 with the subtotals added by one lane).
  template <typename F>
  __device__ __forceinline__ void sum_groups(const NormGeometry& g, const NormTile& t, const float* in, F f) const {
    const bool narrow = g.Cg * T <= 16;
    const int lane = narrow ? 0 : threadIdx.x % 32, team = narrow ? 0 : 5;
    const int step = narrow ? kNormThreads : kNormWarps;
    for (int i = narrow ? threadIdx.x : threadIdx.x / 32; i < t.g1 - t.g0; i += step) {
      const int cb = max((t.g0 + i) * g.Cg, t.c0) - t.c0;
      const int w = min((t.g0 + i + 1) * g.Cg, t.c1) - t.c0 - cb;
      const int shift = min(team, w > 1 ? 32 - __clz(w - 1) : 0), beside = 1 << shift;
      float v = 0.f;
      for (int j = lane >> shift; j < T; j += 1 << (team - shift))
        for (int c = lane & (beside - 1); c < w; c += beside) v += in[j * cols + cb + c];
      if (!narrow) v = warp_sum(v);
      if (lane == 0) f(i, cb, w, v);
    }
  }
};

// L2 priorities, for tensors that are larger than it (keep < 1): of what the reducing pass reads,
// the last `keep` is to stay for the applying pass, which reads it first; all else, and what is
// written, goes past it.
struct NormPolicy {
  uint64_t stay, pass;
  __device__ __forceinline__ explicit NormPolicy(bool large) {
    asm("createpolicy.fractional.L2::evict_normal.b64 %0;" : "=l"(stay));
    asm("createpolicy.fractional.L2::evict_first.b64 %0;" : "=l"(pass));
    if (!large) pass = stay;
  }
};

// The vectors of one thread in a pass: its row's spans of the part, in batches of U; the last batch
// may be short. A reducing pass goes from tile to tile (a batch of each, `rows` spans apart), an
// applying one from the part's last span to its first. Vectors of 16 bytes are copied
// asynchronously into a ring of B batches in shared memory, B - 1 batches ahead of their use
// (each thread into slots of its own, so that no barrier is needed): what a thread has in flight
// is bounded by shared memory instead of registers and does not pause while it computes.
// Narrower vectors are loaded when they are used.
template <typename T, int V, int U, int B, bool APPLYING, bool FOLDS = false>
struct NormWalk {
  using IO = VecIO<T, V>;
  using Raw = typename IO::Raw;
  static constexpr bool kAsync = sizeof(Raw) == 16;
  static constexpr int kU = U;
  static constexpr int kRingBytes = kAsync ? kNormThreads * 16 * U * B : 0;
  // Shared memory of a reducing pass over some tensors: their rings, where the merge that follows has
  // its scratch (four floats per thread and channel), and where it FOLDS, two FP64 sums per thread
  // and channel.
  static constexpr int kScratchBytes = 4 * kNormThreads * V * static_cast<int>(sizeof(float));
  static __host__ __device__ constexpr int wide_offset(int tensors) {
    return tensors * kRingBytes > kScratchBytes ? tensors * kRingBytes : kScratchBytes;
  }
  static __host__ __device__ constexpr int reducing_bytes(int tensors) {
    return wide_offset(tensors) + (FOLDS ? 2 * kNormThreads * V * static_cast<int>(sizeof(double)) : 0);
  }

  int count;       // vectors of this thread
  int64_t first;   // element offset of the first one
  int64_t stride;  // from one to the next in a batch
  int64_t jump;    // and besides that from batch to batch

  __device__ __forceinline__ NormWalk(const NormGeometry& g, const NormTile& t) {
    stride = static_cast<int64_t>(g.rows) * g.Cv;
    int64_t span;
    if (APPLYING) {
      const int spans = g.run_spans(t.s);
      count = t.row < spans ? (spans - t.row - 1) / g.rows + 1 : 0;
      span = static_cast<int64_t>(g.base) * t.s + min(t.s, g.extra) + t.row + static_cast<int64_t>(count - 1) * g.rows;
      stride = -stride;
      jump = 0;
    } else {
      const int missing = t.s == g.last_part ? g.lacking : 0;
      // spans of a full tile that this row lacks in the last one
      const int last = g.tile - missing;
      const int lost = missing == 0 ? 0 : U - (t.row < last ? (last - t.row - 1) / g.rows + 1 : 0);
      count = g.tiles_of(t.s) * U - lost;
      span = static_cast<int64_t>(t.s) * g.tile + t.row;
      jump = static_cast<int64_t>(g.S - 1) * g.tile * g.Cv;
    }
    if (!t.active) count = 0;
    first = t.n * g.P * g.C + span * g.Cv + t.c0 + t.chan;
  }
  // pixels of the reducing pass that come before those that are to stay in L2
  __device__ __forceinline__ int passing(float keep) const {
    return keep >= 1.f ? 0 : static_cast<int>(static_cast<float>(count) * (1.f - keep));
  }

  // start(slot, todo) begins copying the next batch, of which `todo` vectors are left, into that
  // batch of the ring; use(slot, whole, k) takes one of k vectors (k == U when whole). A walk that
  // FOLDS calls fold() after each kFoldSpans that others follow.
  static constexpr int kFoldSpans = 8 * B * U;
  template <typename Start, typename Use, typename Fold>
  __device__ __forceinline__ void run(int prefilled, Start start, Use use, Fold fold) const {
    int todo = count - prefilled * U, left = count;
    while (left > 0) {
      const int stop = FOLDS ? max(left - kFoldSpans, 0) : 0;
      do {
#pragma unroll
        for (int b = 0; b < B; ++b) {
          start((b + B - 1) % B, todo);
          todo -= U;
          if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(B - 1) : "memory");
          if (left >= U) use(b, std::true_type{}, U);
          else use(b, std::false_type{}, left);
          left -= U;
          if (left <= 0) break;
        }
      } while (left > stop);
      if (FOLDS && left > 0) fold();
    }
  }
  template <typename Start, typename Use>
  __device__ __forceinline__ void run(int prefilled, Start start, Use use) const {
    run(prefilled, start, use, [] {});
  }
};

// One tensor's side of a walk: where its next vector to copy lies, and its ring.
template <typename W, typename T>
struct NormSource {
  const T* next;   // to copy (or, for narrow vectors, to load)
  unsigned ring;

  __device__ __forceinline__ NormSource(const W& w, const void* x, int offset)
      : next(static_cast<const T*>(x) + w.first), ring(address() + offset + threadIdx.x * 16) {}
  static __device__ __forceinline__ unsigned address() {
    extern __shared__ __align__(16) unsigned char norm_ring[];
    return static_cast<unsigned>(__cvta_generic_to_shared(norm_ring));
  }
  __device__ __forceinline__ void start(const W& w, int slot, int todo, uint64_t policy) {
    if constexpr (W::kAsync) {
#pragma unroll
      for (int u = 0; u < W::kU; ++u) {
        if (u < todo)
          asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(
                           ring + (slot * W::kU + u) * kNormThreads * 16),
                       "l"(next), "l"(policy) : "memory");
        next += w.stride;
      }
      next += w.jump;
    }
  }
  static __device__ __forceinline__ void commit() {
    if constexpr (W::kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // vector u of a batch that has arrived; each is taken once, in order
  __device__ __forceinline__ typename W::Raw get(const W& w, int slot, int u) {
    if constexpr (W::kAsync) {
      typename W::Raw r;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                   : "r"(ring + (slot * W::kU + u) * kNormThreads * 16) : "memory");
      return r;
    } else {
      const typename W::Raw r = W::IO::load(next);
      next += u + 1 < W::kU ? w.stride : w.stride + w.jump;
      return r;
    }
  }
};

template <typename W, typename T>
struct NormSink {
  T* next;
  __device__ __forceinline__ NormSink(const W& w, void* y) : next(static_cast<T*>(y) + w.first) {}
  __device__ __forceinline__ void put(const W& w, const typename W::Raw& r, uint64_t policy) {
    if constexpr (W::kAsync)
      asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(next), "r"(r.x),
                   "r"(r.y), "r"(r.z), "r"(r.w), "l"(policy) : "memory");
    else W::IO::store(next, r);
    next += w.stride;
  }
};

// A pass's shared memory: the ring, and in the reducing passes the merge's scratch after it is used
// and the FP64 sums behind both.
extern __shared__ __align__(16) unsigned char norm_ring[];
// V weights (or `missing` for each) from channel c, a multiple of V.
template <int V>
__device__ __forceinline__ void load_weights(const NormParams& p, const void* w, float missing, int c,
                                             float2 (&f)[kPairs<V>]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) f[i] = splat2(missing);
    return;
  }
  if constexpr (V % 4 == 0) {
    if (p.weight_vectors) {
      if (p.weight_dtype == 0) {
        load_channels<V>(static_cast<const float*>(w) + c, f);
      } else {
        const unsigned* words = reinterpret_cast<const unsigned*>(static_cast<const __half*>(w) + c);
        unsigned r[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; i += 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(words + i);
          r[i] = v.x;
          r[i + 1] = v.y;
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
          f[i] = p.weight_dtype == 1 ? norm_pair(r[i], __half()) : norm_pair(r[i], __nv_bfloat16());
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    f[i].x = load_weight(w, p.weight_dtype, c + 2 * i);
    f[i].y = 2 * i + 1 < V ? load_weight(w, p.weight_dtype, c + 2 * i + 1) : 0.f;
  }
}

// V values of a row of the C real channels from channel c of a span.
template <int V>
__device__ __forceinline__ void load_span(const NormGeometry& g, const float* row, int c, float2 (&f)[kPairs<V>]) {
  if (g.period == 1) {
    load_channels<V>(row + c, f);
    return;
  }
  c %= g.C;
#pragma unroll
  for (int v = 0; v < 2 * kPairs<V>; ++v) {
    (v & 1 ? f[v / 2].y : f[v / 2].x) = v < V ? row[c] : 0.f;
    if (++c == g.C) c = 0;
  }
}

// f = value(group).x and .y for each of V channels from c.
template <int V, typename Value>
__device__ __forceinline__ void by_group(const NormGeometry& g, int c, Value value, float2 (&x)[kPairs<V>],
                                         float2 (&y)[kPairs<V>]) {
  int grp = c / g.Cg, end = (grp + 1) * g.Cg;  // one division; the next channels follow
  float2 now = value(grp);
  if (end - c >= V) {
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      x[i] = splat2(now.x);
      y[i] = splat2(now.y);
    }
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (c + v == end) {
      now = value(++grp);
      end += g.Cg;
    }
    (v & 1 ? x[v / 2].y : x[v / 2].x) = now.x;
    (v & 1 ? y[v / 2].y : y[v / 2].x) = now.y;
  }
}

// A thread's channel constants: -mean, the factor rstd w and the shift, from stats(group) = (mean,
// rstd).
template <int V, typename Stats>
__device__ __forceinline__ void norm_constants(const NormParams& p, const NormTile& t, Stats stats,
                                               float2 (&minus)[kPairs<V>], float2 (&a)[kPairs<V>],
                                               float2 (&b)[kPairs<V>]) {
  int c = t.c0 + t.chan;
  if (p.g.period > 1) {
    c %= p.g.C;
#pragma unroll
    for (int v = 0; v < 2 * kPairs<V>; ++v) {
      const float2 st = stats(c / p.g.Cg);
      const float w = p.weight ? load_weight(p.weight, p.weight_dtype, c) : 1.f;
      (v & 1 ? minus[v / 2].y : minus[v / 2].x) = -st.x;
      (v & 1 ? a[v / 2].y : a[v / 2].x) = st.y * w;
      (v & 1 ? b[v / 2].y : b[v / 2].x) = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
      if (++c == p.g.C) c = 0;
    }
    return;
  }
  float2 w[kPairs<V>];
  load_weights<V>(p, p.weight, 1.f, c, w);
  load_weights<V>(p, p.bias, 0.f, c, b);
  by_group<V>(p.g, c, stats, minus, a);
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    minus[i] = neg2(minus[i]);
    a[i] = mul2(a[i], w[i]);
  }
}

// A thread's running statistics of its channels.
template <typename T, int V, int U>
struct NormMoments {
  using IO = VecIO<T, V>;
  static constexpr int N = IO::N;
  float2 mean[N], m2[N];
  float before = 0.f;  // batches taken

  __device__ __forceinline__ NormMoments() {
#pragma unroll
    for (int v = 0; v < N; ++v) mean[v] = m2[v] = splat2(0.f);
  }
  // a batch of U spans, or the last one of k (k < U); get(u) gives the vector of span u
  template <typename Whole, typename Get>
  __device__ __forceinline__ void take(Whole, int k, Get get) {
    constexpr bool kWhole = Whole::value;
    float2 f[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      typename IO::Raw raw{};
      if (kWhole || u < k) raw = get(u);
      IO::unpack(raw, f[u]);
    }
    // the new values' weight in the mean, and that of the squared distance of the two means; the first
    // batch's mean is taken as it is
    const float taken = kWhole ? U : k;
    const float share = before == 0.f ? 1.f : kWhole ? __fdividef(1.f, before + 1.f) : taken / fmaf(before, U, taken);
    const float cross = before * U * share;
    const float2 each = splat2(kWhole ? 1.f / U : 1.f / taken);
#pragma unroll
    for (int v = 0; v < N; ++v) {
      // From the distances e to the batch's first value: a sum of equal values would round. They
      // are small wherever the spread is, whatever the mean, and that value being one of the
      // batch, sum e^2 is at most U times the sum of squares around the mean: few digits cancel.
      const float2 first = neg2(f[0][v]);
      float2 sum = splat2(0.f), q = splat2(0.f);
#pragma unroll
      for (int u = 1; u < U; ++u)
        if (kWhole || u < k) {
          const float2 e = add2(f[u][v], first);
          sum = add2(sum, e);
          q = fma2(e, e, q);
        }
      const float2 shift = mul2(sum, each), m = add2(f[0][v], shift);
      q = fma2(neg2(sum), shift, q);
      const float2 d = add2(m, neg2(mean[v]));
      mean[v] = fma2(d, splat2(share), mean[v]);
      // (in this order: the first batch's distance is its mean, whose square may be infinite, times 0)
      m2[v] = add2(m2[v], fma2(mul2(d, splat2(cross)), d, q));
    }
    before += 1.f;
  }
};

// What a thread adds up over its part of a sample would be one chain of FP32 roundings as long as the
// part (3,370 terms of 1x255x997x1001 FP32, where the dbias of equal gradients was off by 565 * 2^-24).
// So every kFoldSpans spans the sums, of at most 64 terms (or 16 batches' moments), go on
// into FP64 ones in shared memory, two for each of the thread's channels, its own slots. Where no
// part is that long, kernels without them run (FOLDS).
template <int V>
struct NormWide {
  double* own;
  int folded = 0;  // spans that are in them
  __device__ __forceinline__ explicit NormWide(int offset)
      : own(reinterpret_cast<double*>(norm_ring + offset) + threadIdx.x) {}

  // f(wide, wide, sum, sum) for each of the thread's channels
  template <typename F>
  __device__ __forceinline__ void each(float2 (&a)[kPairs<V>], float2 (&b)[kPairs<V>], F f) const {
#pragma unroll
    for (int v = 0; v < V; ++v)
      f(own[2 * v * kNormThreads], own[(2 * v + 1) * kNormThreads], v & 1 ? a[v / 2].y : a[v / 2].x,
        v & 1 ? b[v / 2].y : b[v / 2].x);
  }
  __device__ __forceinline__ void add_sums(int spans, float2 (&a)[kPairs<V>], float2 (&b)[kPairs<V>]) {
    const bool first = folded == 0;
    each(a, b, [&](double& wa, double& wb, float& fa, float& fb) {
      wa = first ? fa : wa + fa;
      wb = first ? fb : wb + fb;
      fa = fb = 0.f;
    });
    folded += spans;
  }
  // the moments of this many spans more, merged as those of a batch are
  __device__ __forceinline__ void add_moments(int spans, float2 (&mean)[kPairs<V>], float2 (&m2)[kPairs<V>]) {
    const bool first = folded == 0;
    const double share = first ? 1.0 : static_cast<double>(spans) / (static_cast<double>(folded) + spans);
    const double cross = folded * share;
    each(mean, m2, [&](double& wm, double& w2, float& fm, float& f2) {
      const double d = first ? 0.0 : fm - wm;
      wm = first ? fm : fma(d, share, wm);
      w2 = first ? f2 : w2 + fma(d * cross, d, static_cast<double>(f2));
      fm = f2 = 0.f;
    });
    folded += spans;
  }
  // the whole part's, back in a and b
  __device__ __forceinline__ void take(float2 (&a)[kPairs<V>], float2 (&b)[kPairs<V>]) const {
    each(a, b, [](double& wa, double& wb, float& fa, float& fb) {
      fa = static_cast<float>(wa);
      fb = static_cast<float>(wb);
    });
  }
};

// The threads' pairs of a CTA that has `spans` spans of its part become one pair per group: first
// the mean (as distances from one of the means, so that equal values give that value exactly),
// then the deviations. put(i, pair) takes the i-th group's. `scratch` has four floats for each
// thread and channel.
template <int V, typename Put>
__device__ __forceinline__ void norm_merge_rows(const NormGeometry& g, const NormTile& t, int spans,
                                                const float2 (&mean)[kPairs<V>], const float2 (&m2)[kPairs<V>],
                                                float* scratch, Put put) {
  float* sm_mean = scratch;
  float* sm_m2 = sm_mean + kNormThreads * V;
  float* column = sm_m2 + kNormThreads * V;
  float* centre = column + kNormThreads * V;
  if (t.active) {
    norm_put<V>(sm_mean + t.row * g.SC + t.chan, mean);
    norm_put<V>(sm_m2 + t.row * g.SC + t.chan, m2);
  }
  __syncthreads();
  const int full = spans / g.rows;                       // pixels that every row took
  const int extra = (spans - full * g.rows) * g.period;  // rows that took one more
  const float pixels = static_cast<float>(spans) * g.period;
  const int width = t.c1 - t.c0, pitch = g.pitch();
  const NormColumns columns(width);
  const auto count_of = [&](int row) { return static_cast<float>(full + (row < extra)); };
  columns.sum_rows(g, width, column, [&](int c) {
    const float ref = sm_mean[max((t.c0 + c) / g.Cg * g.Cg - t.c0, 0)];
    return [&, c, ref](int r) {
      const float cnt = count_of(r);
      return cnt > 0.f ? cnt * (sm_mean[r * pitch + c] - ref) : 0.f;
    };
  });
  __syncthreads();
  columns.sum_groups(g, t, column, [&](int i, int cb, int w, float sum) {
    centre[i] = sm_mean[cb] + sum / (pixels * w);
  });
  __syncthreads();
  columns.sum_rows(g, width, column, [&](int c) {
    const float m = centre[(t.c0 + c) / g.Cg - t.g0];
    return [&, c, m](int r) {
      const float cnt = count_of(r);
      const float d = sm_mean[r * pitch + c] - m;
      return cnt > 0.f ? fmaf(cnt * d, d, sm_m2[r * pitch + c]) : 0.f;
    };
  });
  __syncthreads();
  columns.sum_groups(g, t, column, [&](int i, int cb, int w, float sum) { put(i, make_float2(centre[i], sum)); });
}

// The threads' sums of a CTA become put(c, sums) for each channel of the slice.
template <int V, typename Put>
__device__ __forceinline__ void norm_merge_sums(const NormGeometry& g, const NormTile& t,
                                                const float2 (&s1)[kPairs<V>], const float2 (&s2)[kPairs<V>],
                                                float* scratch, Put put) {
  float* sm1 = scratch;
  float* sm2 = sm1 + kNormThreads * V;
  float* column1 = sm2 + kNormThreads * V;
  float* column2 = column1 + kNormThreads * V;
  if (t.active) {
    norm_put<V>(sm1 + t.row * g.SC + t.chan, s1);
    norm_put<V>(sm2 + t.row * g.SC + t.chan, s2);
  }
  __syncthreads();
  const int width = t.c1 - t.c0, pitch = g.pitch();
  const NormColumns columns(width);
  columns.sum_rows(g, width, column1, [&](int c) { return [&, c](int r) { return sm1[r * pitch + c]; }; });
  columns.sum_rows(g, width, column2, [&](int c) { return [&, c](int r) { return sm2[r * pitch + c]; }; });
  __syncthreads();
  if (columns.T >= 32) {  // at most eight channels, and many subtotals of each: a warp for each
    const int c = threadIdx.x / 32;
    if (c < width) {
      float v1 = 0.f, v2 = 0.f;
      for (int j = threadIdx.x % 32; j < columns.T; j += 32) {
        v1 += column1[j * columns.cols + c];
        v2 += column2[j * columns.cols + c];
      }
      v1 = warp_sum(v1);
      v2 = warp_sum(v2);
      if (threadIdx.x % 32 == 0) put(c, make_float2(v1, v2));
    }
    return;
  }
  for (int c = threadIdx.x; c < width; c += kNormThreads) {
    float v1 = 0.f, v2 = 0.f;
    for (int j = 0; j < columns.T; ++j) {
      v1 += column1[j * columns.cols + c];
      v2 += column2[j * columns.cols + c];
    }
    put(c, make_float2(v1, v2));
  }
}

// ---- forward: statistics ----
// Bound by DRAM: 8x128x512^2 16-bit (537 MB) 87 us, 6.2 TB/s; 1x64x1080x1920 (265 MB) 49 us. Two
// CTAs an SM and batches of 8: more CTAs or shorter batches ran up to 6 % slower.
template <typename T, int V, int U, int B, bool FOLDS>
__global__ void __launch_bounds__(kNormThreads, kNormResident) norm_stats_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const NormTile t(g, V, false);
  grid_dependency_wait();
  grid_launch_dependents();
  using Walk = NormWalk<T, V, U, B, false, FOLDS>;
  const Walk walk(g, t);
  NormSource<Walk, T> x(walk, p.x, 0);
  const NormPolicy policy(g.keep < 1.f);
  const int staying = walk.count - walk.passing(g.keep);
  const auto start = [&](int slot, int todo) {
    x.start(walk, slot, todo, todo > staying ? policy.pass : policy.stay);
    x.commit();
  };
#pragma unroll
  for (int b = 0; b < B - 1; ++b) start(b, walk.count - b * U);
  NormMoments<T, V, U> moments;
  NormWide<V> wide(Walk::wide_offset(1));
  walk.run(B - 1, start, [&](int slot, auto whole, int k) {
    moments.take(whole, k, [&](int u) { return x.get(walk, slot, u); });
  }, [&] {
    wide.add_moments(Walk::kFoldSpans, moments.mean, moments.m2);
    moments.before = 0.f;
  });
  if (wide.folded) {
    wide.add_moments(walk.count - wide.folded, moments.mean, moments.m2);
    wide.take(moments.mean, moments.m2);
  }
  __syncthreads();  // the ring is done with: its memory is the merge's scratch
  float2* partial = p.partial + ((static_cast<int64_t>(t.n) * g.S + t.s) * g.slices + t.slice) * g.GS;
  norm_merge_rows<V>(g, t, g.part_spans(t.s), moments.mean, moments.m2, reinterpret_cast<float*>(norm_ring),
                     [&](int i, float2 pair) { partial[i] = pair; });
}

// (mean, rstd) of a group from its sums of distances from ref and of squares around it.
__device__ __forceinline__ float2 norm_statistics(const NormGeometry& g, double ref, double sum, double q) {
  sum *= g.inv_m;
  double var = q * g.inv_m - sum * sum;
  if (var < 0.0) var = 0.0;  // a NaN stays
  return make_float2(static_cast<float>(ref + sum),
                     __frsqrt_rn(static_cast<float>(var + static_cast<double>(g.eps))));
}

// ---- the merging launches: a team of kNormThreads / teams threads for each (sample, group) ----
// Sums of two values over a team (a power of two of threads, a warp at least), in all its
// threads. Every thread of the block takes part.
__device__ __forceinline__ double2 team_sum(double a, double b, int team_shift, double2* sm) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (team_shift == 5) return make_double2(a, b);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = make_double2(a, b);
  __syncthreads();
  const int warps = 1 << (team_shift - 5), first = threadIdx.x / 32 & ~(warps - 1);
  double2 s = make_double2(0.0, 0.0);
  for (int i = 0; i < warps; ++i) {
    s.x += sm[first + i].x;
    s.y += sm[first + i].y;
  }
  return s;
}

// Forward: the parts' pairs become the group's statistics and its channels' constants. Bound by the
// latency of a few dependent reads: about 4 us of a chain of launches.
__global__ void __launch_bounds__(kNormThreads) norm_merge_kernel(const __grid_constant__ NormParams p,
                                                                  int team_shift) {
  __shared__ double2 sm[kNormWarps];
  const NormGeometry& g = p.g;
  const int team_threads = 1 << team_shift;
  const unsigned id = blockIdx.x * (kNormThreads >> team_shift) + (threadIdx.x >> team_shift);
  const int lane = threadIdx.x & (team_threads - 1);
  grid_dependency_wait();
  grid_launch_dependents();
  const bool real = id < g.N * g.G;
  const unsigned sample = id / static_cast<unsigned>(g.G);
  const int grp = static_cast<int>(id - sample * g.G);
  const int64_t n = sample;
  const int c0 = grp * g.Cg, c1 = c0 + g.Cg;
  double ref = 0.0, sum = 0.0, q = 0.0;  // sums of distances from ref, and of squares around it
  if (real) {
    const int first = c0 / g.SC, last = (c1 - 1) / g.SC;
    for (int k = first; k <= last; ++k) {  // the slices that hold a piece of the group
      const int b = k * g.SC, width = min(c1, b + g.SC) - max(c0, b);
      const float2* pairs = p.partial + (n * g.S * g.slices + k) * g.GS + grp - b / g.Cg;
      if (k == first) ref = pairs[0].x;
      for (int s = lane; s < g.S; s += team_threads) {
        const float2 v = pairs[static_cast<int64_t>(s) * g.slices * g.GS];
        const double cnt = static_cast<double>(g.part_pixels(s)) * width;
        const double d = v.x - ref;
        sum = fma(cnt, d, sum);
        q += fma(cnt * d, d, static_cast<double>(v.y));
      }
    }
  }
  const double2 total = team_sum(sum, q, team_shift, sm);
  if (!real) return;
  const float2 st = norm_statistics(g, ref, total.x, total.y);
  const float mean = st.x, rstd = st.y;
  if (p.mean && lane == 0) {
    p.mean[id] = mean;
    p.rstd[id] = rstd;
  }
  const int64_t C = g.C;
  float* row = p.channel + n * kNormForwardRows * C;
  for (int c = c0 + lane; c < c1; c += team_threads) {
    row[c] = -mean;
    row[C + c] = p.weight ? rstd * load_weight(p.weight, p.weight_dtype, c) : rstd;
    row[2 * C + c] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
  }
}

// In an applying pass that has no merging launch before it: the statistics of all groups of sample n
// from its p.merges parts, by a power of two of threads, at most a warp, for each group.
__device__ __forceinline__ void norm_merge_here(const NormParams& p, int n, float2* stats) {
  const NormGeometry& g = p.g;
  int shift = 5;
  while (shift > 0 && g.G << shift > kNormThreads) --shift;
  const int lane = threadIdx.x & ((1 << shift) - 1), step = kNormThreads >> shift;
  for (int b = 0; b < g.G; b += step) {
    const int grp = b + (threadIdx.x >> shift);
    double ref = 0.0, sum = 0.0, q = 0.0;
    if (grp < g.G) {
      const float2* pairs = p.partial + static_cast<int64_t>(n) * p.merges * g.G + grp;
      ref = pairs[0].x;
#pragma unroll 4
      for (int k = lane; k < p.merges; k += 1 << shift) {
        const float2 v = pairs[k * g.G];
        const double cnt = static_cast<double>(g.part_pixels(k)) * g.Cg;
        const double d = v.x - ref;
        sum = fma(cnt, d, sum);
        q += fma(cnt * d, d, static_cast<double>(v.y));
      }
    }
    for (int o = 1 << shift >> 1; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    if (grp < g.G && lane == 0) stats[grp] = norm_statistics(g, ref, sum, q);
  }
  __syncthreads();
}

// ---- forward: y ----
// Bound by DRAM on large tensors (8x128x512^2 16-bit, 537 MB in and out: 166 us, 6.1 TB/s), by the
// special-function unit where most of x comes from L2 (SiLU takes two of its operations an
// element; 8x128x256^2: 47 us, 4.6 TB/s).
constexpr int kNormMergeGroups = 256;  // groups that an applying pass merges itself, at most

template <typename T, int V, int ACT, int U, int B>
__global__ void __launch_bounds__(kNormThreads, kNormApplyResident) norm_apply_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const NormTile t(g, V, true);
  using IO = VecIO<T, V>;
  using Walk = NormWalk<T, V, U, B, true>;
  const Walk walk(g, t);
  NormSource<Walk, T> x(walk, p.x, 0);
  NormSink<Walk, T> y(walk, p.out);
  const NormPolicy policy(g.keep < 1.f);
  const auto start = [&](int slot, int todo) {
    x.start(walk, slot, todo, policy.pass);
    x.commit();
  };
  // x was complete before the statistics' launch passed its wait, so the first reads need not wait
  // for the launches in between to end (which rests on that launch being there, before this one)
#pragma unroll
  for (int j = 0; j < B - 1; ++j) start(j, walk.count - j * U);
  grid_dependency_wait();
  constexpr int N = IO::N;
  float2 minus[N], a[N], b[N];  // -mean, the factor and the shift
  if (p.merges) {
    __shared__ float2 stats[kNormMergeGroups];
    norm_merge_here(p, t.n, stats);
    if (t.active) norm_constants<V>(p, t, [&](int grp) { return stats[grp]; }, minus, a, b);
    if (p.mean && t.s == 0)
      for (int i = threadIdx.x; i < g.G; i += kNormThreads) {
        p.mean[static_cast<int64_t>(t.n) * g.G + i] = stats[i].x;
        p.rstd[static_cast<int64_t>(t.n) * g.G + i] = stats[i].y;
      }
  } else if (t.active) {
    const int64_t C = g.C;
    const float* row = p.channel + t.n * kNormForwardRows * C;
    const int c = t.c0 + t.chan;
    load_span<V>(g, row, c, minus);
    load_span<V>(g, row + C, c, a);
    load_span<V>(g, row + 2 * C, c, b);
  }
  grid_launch_dependents();  // the statistics have been read
  walk.run(B - 1, start, [&](int slot, auto whole, int k) {
    constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kWhole || u < k) {
        float2 f[N];
        IO::unpack(x.get(walk, slot, u), f);
#pragma unroll
        for (int v = 0; v < N; ++v) f[v] = activate<T, ACT>(fma2(add2(f[v], minus[v]), a[v], b[v]));
        y.put(walk, IO::pack(f), policy.pass);
      }
  });
}

// ---- backward: per-channel sums of one part ----
// Bound by DRAM: 8x128x512^2 16-bit (1,074 MB) 168 us, 6.4 TB/s; 1x48x517x999 FP32 (198 MB) 37 us.
template <typename T, int V, int ACT, int U, int B, bool FOLDS>
__global__ void __launch_bounds__(kNormThreads, kNormResident) norm_grad_sums_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const NormTile t(g, V, false);
  grid_dependency_wait();
  grid_launch_dependents();
  using IO = VecIO<T, V>;
  using Walk = NormWalk<T, V, U, B, false, FOLDS>;
  const Walk walk(g, t);
  NormSource<Walk, T> x(walk, p.x, 0), dy(walk, p.dy, Walk::kRingBytes);
  const NormPolicy policy(g.keep < 1.f);
  const int staying = walk.count - walk.passing(g.keep);
  const auto start = [&](int slot, int todo) {
    const uint64_t how = todo > staying ? policy.pass : policy.stay;
    x.start(walk, slot, todo, how);
    dy.start(walk, slot, todo, how);
    x.commit();
  };
#pragma unroll
  for (int j = 0; j < B - 1; ++j) start(j, walk.count - j * U);
  constexpr int N = IO::N;
  float2 s1[N], s2[N];
#pragma unroll
  for (int v = 0; v < N; ++v) s1[v] = s2[v] = splat2(0.f);
  if (t.active) {
    float2 minus[N], a[N], b[N];
    norm_constants<V>(p, t, [&](int grp) {
      const int64_t at = static_cast<int64_t>(t.n) * g.G + grp;
      return make_float2(p.mean[at], p.rstd[at]);
    }, minus, a, b);
    NormWide<V> wide(Walk::wide_offset(2));
    walk.run(B - 1, start, [&](int slot, auto whole, int k) {
      constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (kWhole || u < k) {
          float2 f[N], d[N];
          IO::unpack(x.get(walk, slot, u), f);
          IO::unpack(dy.get(walk, slot, u), d);
#pragma unroll
          for (int v = 0; v < N; ++v) {
            const float2 xc = add2(f[v], minus[v]);
            const float2 dz = activate_grad<T, ACT>(fma2(xc, a[v], b[v]), d[v]);
            s1[v] = add2(s1[v], dz);
            s2[v] = fma2(dz, xc, s2[v]);
          }
        }
    }, [&] { wide.add_sums(Walk::kFoldSpans, s1, s2); });
    if (wide.folded) {
      wide.add_sums(walk.count - wide.folded, s1, s2);
      wide.take(s1, s2);
    }
  }
  __syncthreads();
  float2* partial = p.partial + (static_cast<int64_t>(t.n) * g.S + t.s) * g.C + t.c0;
  norm_merge_sums<V>(g, t, s1, s2, reinterpret_cast<float*>(norm_ring),
                     [&](int c, float2 sums) { partial[c] = sums; });
}

// Backward: sums over the parts, and the group's two means. `cols` channels (at most 32) are summed
// at a time, by team_threads / cols threads each.
__global__ void __launch_bounds__(kNormThreads) norm_grad_merge_kernel(const __grid_constant__ NormParams p,
                                                                       int team_shift, int col_shift) {
  __shared__ double2 sm[kNormThreads];
  const NormGeometry& g = p.g;
  const int team_threads = 1 << team_shift;
  const unsigned id = blockIdx.x * (kNormThreads >> team_shift) + (threadIdx.x >> team_shift);
  const int lane = threadIdx.x & (team_threads - 1);
  grid_dependency_wait();
  grid_launch_dependents();
  const bool real = id < g.N * g.G;
  const unsigned sample = id / static_cast<unsigned>(g.G);
  const int grp = static_cast<int>(id - sample * g.G);
  const int64_t n = sample;
  const int cols = 1 << col_shift, col = lane & (cols - 1), sub = lane >> col_shift;
  const int subs = team_threads >> col_shift;
  const float mean = real ? p.mean[id] : 0.f, rstd = real ? p.rstd[id] : 0.f;
  double w1 = 0.0, w2 = 0.0;  // sum of w dz and of w dz xhat, kept by the threads with sub == 0
  for (int cb = 0; cb < g.Cg; cb += cols) {
    const int c = cb + col, ch = grp * g.Cg + c;
    const bool mine = real && c < g.Cg;
    double v1 = 0.0, v2 = 0.0;
    if (mine) {
      const float2* at = p.partial + n * g.S * g.C + ch;
#pragma unroll 4
      for (int s = sub; s < g.S; s += subs) {
        const float2 v = at[static_cast<int64_t>(s) * g.C];
        v1 += v.x;
        v2 += v.y;
      }
    }
    // within the warp first, then over the team's warps
    for (int o = 16; o >= cols; o >>= 1) {
      v1 += __shfl_xor_sync(0xffffffffu, v1, o);
      v2 += __shfl_xor_sync(0xffffffffu, v2, o);
    }
    if (team_threads > 32) {
      __syncthreads();
      if (threadIdx.x % 32 < cols) sm[threadIdx.x / 32 * 32 + col] = make_double2(v1, v2);
      __syncthreads();
      if (sub == 0) {
        v1 = v2 = 0.0;
        for (int i = 0; i < team_threads; i += 32) {
          v1 += sm[threadIdx.x + i].x;
          v2 += sm[threadIdx.x + i].y;
        }
      }
    }
    if (mine && sub == 0) {
      v2 *= rstd;
      // (rounded to FP32: 2^-24 of each sample's sum, and half the traffic of the last sum)
      p.sums[n * g.C + ch] = make_float2(static_cast<float>(v1), static_cast<float>(v2));
      const double w = p.weight ? load_weight(p.weight, p.weight_dtype, ch) : 1.0;
      w1 += w * v1;
      w2 += w * v2;
      if (g.N == 1) {  // one sample: its sums are the parameters' gradients
        if (p.dweight) store_weight(p.dweight, p.weight_dtype, ch, static_cast<float>(v2));
        if (p.dbias) store_weight(p.dbias, p.weight_dtype, ch, static_cast<float>(v1));
      }
    }
  }
  const double2 total = team_sum(w1, w2, team_shift, sm);
  if (!real) return;
  const float k1 = static_cast<float>(rstd * (total.x * g.inv_m));
  const float k2 = static_cast<float>(rstd * (rstd * (total.y * g.inv_m)));
  const int64_t C = g.C;
  float* row = p.channel + n * kNormBackwardRows * C;
  for (int c = grp * g.Cg + lane; c < (grp + 1) * g.Cg; c += team_threads) {
    row[c] = -mean;
    row[C + c] = p.weight ? rstd * load_weight(p.weight, p.weight_dtype, c) : rstd;
    row[2 * C + c] = p.bias ? load_weight(p.bias, p.weight_dtype, c) : 0.f;
    row[3 * C + c] = -k1;
    row[4 * C + c] = -k2;
  }
}

// ---- backward: dweight and dbias, sums over the samples: a warp for each channel, from the blocks'
// first on ----
__device__ __forceinline__ void norm_param_grads(const NormParams& p) {
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * kNormWarps + threadIdx.x / 32; c < p.g.C;
       c += static_cast<int64_t>(gridDim.x) * kNormWarps) {
    double db = 0.0, dw = 0.0;
#pragma unroll 4
    for (int64_t n = threadIdx.x % 32; n < p.g.N; n += 32) {
      const float2 v = p.sums[n * p.g.C + c];
      db += v.x;
      dw += v.y;
    }
    db = warp_sum(db);
    dw = warp_sum(dw);
    if (threadIdx.x % 32 == 0) {
      if (p.dweight) store_weight(p.dweight, p.weight_dtype, static_cast<int>(c), static_cast<float>(dw));
      if (p.dbias) store_weight(p.dbias, p.weight_dtype, static_cast<int>(c), static_cast<float>(db));
    }
  }
}

// (a launch of its own where there is no dx, or the resident kernel made it)
__global__ void __launch_bounds__(kNormThreads) norm_param_grad_kernel(const __grid_constant__ NormParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  norm_param_grads(p);
}

// ---- backward: dx ----
// Bound by DRAM: 8x128x512^2 16-bit (1,074 MB in, 537 out) 237 us, 6.6 TB/s; 8x128x256^2 63 us.
template <typename T, int V, int ACT, int U, int B>
__global__ void __launch_bounds__(kNormThreads, kNormApplyResident) norm_grad_apply_kernel(const __grid_constant__ NormParams p) {
  const NormGeometry& g = p.g;
  const NormTile t(g, V, true);
  using IO = VecIO<T, V>;
  using Walk = NormWalk<T, V, U, B, true>;
  const Walk walk(g, t);
  NormSource<Walk, T> x(walk, p.x, 0), dy(walk, p.dy, Walk::kRingBytes);
  NormSink<Walk, T> dx(walk, p.out);
  const NormPolicy policy(g.keep < 1.f);
  const auto start = [&](int slot, int todo) {
    x.start(walk, slot, todo, policy.pass);
    dy.start(walk, slot, todo, policy.pass);
    x.commit();
  };
  // as in the forward, the first reads do not wait for the launches before
#pragma unroll
  for (int j = 0; j < B - 1; ++j) start(j, walk.count - j * U);
  grid_dependency_wait();
  if (p.fold_params && blockIdx.y == 0) norm_param_grads(p);
  constexpr int N = IO::N;
  float2 minus[N], a[N], b[N], k1[N], k2[N];  // -mean, factor, shift, and the two means negated
  if (t.active) {
    const int64_t C = g.C;
    const float* row = p.channel + t.n * kNormBackwardRows * C;
    const int c = t.c0 + t.chan;
    load_span<V>(g, row, c, minus);
    load_span<V>(g, row + C, c, a);
    load_span<V>(g, row + 2 * C, c, b);
    load_span<V>(g, row + 3 * C, c, k1);
    load_span<V>(g, row + 4 * C, c, k2);
  }
  grid_launch_dependents();  // the means have been read
  walk.run(B - 1, start, [&](int slot, auto whole, int k) {
    constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kWhole || u < k) {
        float2 f[N], d[N];
        IO::unpack(x.get(walk, slot, u), f);
        IO::unpack(dy.get(walk, slot, u), d);
#pragma unroll
        for (int v = 0; v < N; ++v) {
          const float2 xc = add2(f[v], minus[v]);
          const float2 dz = activate_grad<T, ACT>(fma2(xc, a[v], b[v]), d[v]);
          f[v] = fma2(xc, k2[v], fma2(a[v], dz, k1[v]));
        }
        dx.put(walk, IO::pack(f), policy.pass);
      }
  });
}

// ---- small tensors: one launch for each direction ----
// A cluster of S CTAs takes one sample's slice of whole groups, each CTA a contiguous part of the
// pixels, which it keeps in shared memory: the statistics pass from CTA to CTA over distributed
// shared memory, and the input is read once. No workspace; what bounds these is latency: 1x64x16^2
// 6.7 us forward and 6.0 backward, 4x512x32^2 (4 MB) 10.3 and 9.7, one launch after another.
constexpr int kNormScratch = 6;  // floats of scratch for each thread and channel

// A resident part: vector i of a thread, in its own slots.
template <typename T, int V>
struct NormResidentPart {
  using Walk = NormWalk<T, V, 1, 1, true>;
  static_assert(Walk::kAsync, "16-byte vectors");
  unsigned base;
  __device__ __forceinline__ explicit NormResidentPart(int offset)
      : base(NormSource<Walk, T>::address() + offset + threadIdx.x * 16) {}
  __device__ __forceinline__ void start(const Walk& w, const void* x) const {
    const T* next = static_cast<const T*>(x) + w.first;
    for (int i = 0; i < w.count; ++i, next += w.stride)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + i * kNormThreads * 16), "l"(next)
                   : "memory");
  }
  __device__ __forceinline__ uint4 get(int i) const {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(base + i * kNormThreads * 16) : "memory");
    return r;
  }
};
__device__ __forceinline__ void norm_wait_resident() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_resident_kernel(const __grid_constant__ NormParams p) {
  namespace cg = cooperative_groups;
  constexpr int U = 4, N = kPairs<V>;
  using IO = VecIO<T, V>;
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  const typename NormResidentPart<T, V>::Walk walk(g, t);
  float* scratch = reinterpret_cast<float*>(norm_ring);
  const NormResidentPart<T, V> x(kNormScratch * kNormThreads * V * 4);
  grid_dependency_wait();
  grid_launch_dependents();
  x.start(walk, p.x);
  norm_wait_resident();
  NormMoments<T, V, U> moments;
  for (int i = 0; i < walk.count; i += U) {
    const auto get = [&](int u) { return x.get(i + u); };
    if (i + U <= walk.count) moments.take(std::true_type{}, U, get);
    else moments.take(std::false_type{}, walk.count - i, get);
  }
  // pairs: this CTA's, for the cluster to read; stats: the cluster's (mean, rstd) of each group
  float2* pairs = reinterpret_cast<float2*>(scratch + 4 * kNormThreads * V);
  float2* stats = reinterpret_cast<float2*>(scratch);
  norm_merge_rows<V>(g, t, g.run_spans(t.s), moments.mean, moments.m2, scratch,
                     [&](int i, float2 pair) { pairs[i] = pair; });
  const cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = threadIdx.x; i < t.g1 - t.g0; i += kNormThreads) {
    const double ref = cluster.map_shared_rank(pairs, 0)[i].x;
    double sum = 0.0, q = 0.0;
    for (int r = 0; r < g.S; ++r) {
      const float2 v = cluster.map_shared_rank(pairs, r)[i];
      const double cnt = static_cast<double>(g.run_spans(r)) * g.Cg;
      const double d = v.x - ref;
      sum = fma(cnt, d, sum);
      q += fma(cnt * d, d, static_cast<double>(v.y));
    }
    const float2 st = norm_statistics(g, ref, sum, q);
    stats[i] = st;
    if (p.mean && t.s == 0) {
      p.mean[static_cast<int64_t>(t.n) * g.G + t.g0 + i] = st.x;
      p.rstd[static_cast<int64_t>(t.n) * g.G + t.g0 + i] = st.y;
    }
  }
  cluster.sync();  // stats are written, and nobody reads another's pairs any more
  if (!t.active) return;
  float2 minus[N], a[N], b[N];
  norm_constants<V>(p, t, [&](int grp) { return stats[grp - t.g0]; }, minus, a, b);
  T* y = static_cast<T*>(p.out) + walk.first;
  for (int i = 0; i < walk.count; ++i, y += walk.stride) {
    float2 f[N];
    IO::unpack(x.get(i), f);
#pragma unroll
    for (int v = 0; v < N; ++v) f[v] = activate<T, ACT>(fma2(add2(f[v], minus[v]), a[v], b[v]));
    IO::store(y, IO::pack(f));
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_grad_resident_kernel(const __grid_constant__ NormParams p,
                                                                          int slots) {
  namespace cg = cooperative_groups;
  constexpr int N = kPairs<V>;
  using IO = VecIO<T, V>;
  const NormGeometry& g = p.g;
  const NormTile t(g, V);
  const typename NormResidentPart<T, V>::Walk walk(g, t);
  float* scratch = reinterpret_cast<float*>(norm_ring);
  constexpr int kArray = kNormThreads * V;
  const NormResidentPart<T, V> x(kNormScratch * kArray * 4), dy(kNormScratch * kArray * 4 + slots * kNormThreads * 16);
  grid_dependency_wait();
  grid_launch_dependents();
  x.start(walk, p.x);
  dy.start(walk, p.dy);
  float2 minus[N], a[N], b[N], s1[N], s2[N];
#pragma unroll
  for (int v = 0; v < N; ++v) minus[v] = a[v] = b[v] = s1[v] = s2[v] = splat2(0.f);
  if (t.active)
    norm_constants<V>(p, t, [&](int grp) {
      const int64_t at = static_cast<int64_t>(t.n) * g.G + grp;
      return make_float2(p.mean[at], p.rstd[at]);
    }, minus, a, b);
  norm_wait_resident();
  for (int i = 0; i < walk.count; ++i) {
    float2 f[N], d[N];
    IO::unpack(x.get(i), f);
    IO::unpack(dy.get(i), d);
#pragma unroll
    for (int v = 0; v < N; ++v) {
      const float2 xc = add2(f[v], minus[v]);
      const float2 dz = activate_grad<T, ACT>(fma2(xc, a[v], b[v]), d[v]);
      s1[v] = add2(s1[v], dz);
      s2[v] = fma2(dz, xc, s2[v]);
    }
  }
  // sums: this CTA's, for the cluster to read; weighted: the cluster's, times w, of each channel;
  // means: of each group
  float2* sums = reinterpret_cast<float2*>(scratch + 4 * kArray);
  float2* weighted = reinterpret_cast<float2*>(scratch);
  float2* means = reinterpret_cast<float2*>(scratch + 2 * kArray);
  norm_merge_sums<V>(g, t, s1, s2, scratch, [&](int c, float2 v) { sums[c] = v; });
  const cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = threadIdx.x; i < t.c1 - t.c0; i += kNormThreads) {
    const int c = t.c0 + i;
    double v1 = 0.0, v2 = 0.0;
    for (int r = 0; r < g.S; ++r) {
      const float2 v = cluster.map_shared_rank(sums, r)[i];
      v1 += v.x;
      v2 += v.y;
    }
    const float rstd = p.rstd[static_cast<int64_t>(t.n) * g.G + c / g.Cg];
    v2 *= rstd;
    const double w = p.weight ? load_weight(p.weight, p.weight_dtype, c) : 1.0;
    // (FP32 here and in `sums`: 2^-24 of a channel's own sum, against the FP32 terms' roundings)
    weighted[i] = make_float2(static_cast<float>(w * v1 * g.inv_m), static_cast<float>(w * v2 * g.inv_m));
    if (t.s == 0) {
      if (g.N == 1) {  // one sample: its sums are the parameters' gradients
        if (p.dweight) store_weight(p.dweight, p.weight_dtype, c, static_cast<float>(v2));
        if (p.dbias) store_weight(p.dbias, p.weight_dtype, c, static_cast<float>(v1));
      } else if (p.sums) {
        p.sums[static_cast<int64_t>(t.n) * g.C + c] = make_float2(static_cast<float>(v1), static_cast<float>(v2));
      }
    }
  }
  cluster.sync();  // nobody reads another's sums any more
  if (!p.out) return;
  const int lane = threadIdx.x % 32;
  for (int i = threadIdx.x / 32; i < t.g1 - t.g0; i += kNormWarps) {
    const int cb = (t.g0 + i) * g.Cg - t.c0;
    float v1 = 0.f, v2 = 0.f;
    for (int c = lane; c < g.Cg; c += 32) {
      v1 += weighted[cb + c].x;
      v2 += weighted[cb + c].y;
    }
    v1 = warp_sum(v1);
    v2 = warp_sum(v2);
    if (lane == 0) {
      const float rstd = p.rstd[static_cast<int64_t>(t.n) * g.G + t.g0 + i];
      means[i] = make_float2(-rstd * v1, -rstd * rstd * v2);
    }
  }
  __syncthreads();
  if (!t.active) return;
  float2 k1[N], k2[N];
  by_group<V>(g, t.c0 + t.chan, [&](int grp) { return means[grp - t.g0]; }, k1, k2);
  T* dx = static_cast<T*>(p.out) + walk.first;
  for (int i = 0; i < walk.count; ++i, dx += walk.stride) {
    float2 f[N], d[N];
    IO::unpack(x.get(i), f);
    IO::unpack(dy.get(i), d);
#pragma unroll
    for (int v = 0; v < N; ++v) {
      const float2 xc = add2(f[v], minus[v]);
      const float2 dz = activate_grad<T, ACT>(fma2(xc, a[v], b[v]), d[v]);
      f[v] = fma2(xc, k2[v], fma2(a[v], dz, k1[v]));
    }
    IO::store(dx, IO::pack(f));
  }
}

}  // namespace fssim
