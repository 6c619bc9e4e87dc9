// C entry points of the group normalisation with an activation: argument checks, the split of
// the work, and the launches. The kernels are in group_norm.cuh.
#include "group_norm.cuh"

#include <atomic>
#include <climits>
#include <cstdint>
#include <exception>
#include <numeric>
#include <string>

#include "engine_host.h"

namespace {

using fssim::NormGeometry;
using fssim::NormParams;
using fssim_host::aligned;
using fssim_host::fail;
using fssim_host::NvtxRange;

constexpr int64_t kMaxChannels = int64_t{1} << 23;  // 65535 slices of at least 256 vectors
constexpr int64_t kMaxSamples = int64_t{1} << 30;
constexpr unsigned kSms = 148;  // a B200's; grids of other sizes would be right too
// CTAs of one wave.
constexpr int64_t kWave = kSms * fssim::kNormResident;
// Bytes of input that are to stay in L2 from the reducing pass to the applying one, of larger
// tensors (1x64x1080x1920 16-bit forward 152 us without, 143 with; flat from 64 to 120 MB). Smaller
// tensors, and what a pass writes of them, keep the usual priority: read after 60 MB of other
// traffic, 33 and 67 MB outputs cost 2.5 and 1.4 us less so (by the very next norm 1.2 us more).
constexpr double kKeptBytes = 80 << 20;

// Vectors of a thread's batch and batches of its ring: 64 KB of ring for a CTA in every pass. The
// statistics merge once a batch, so theirs are long; a batch of the backward has two tensors'.
constexpr int kStatsU = 8, kStatsB = 2;
constexpr int kApplyU = 4, kApplyB = 4;
constexpr int kGradU = 2, kGradB = 4;
// The resident kernels: the largest input they take (x, in the backward x and dy), the most vectors
// of a thread, and their slices' bytes a pixel. On a B200 they are faster than the passes below
// these (16-bit, device time, fwd / bwd us: 1x64x16^2 6.7 / 6.0 against 7.9 / 7.2, 4x512x32^2
// 10.3 / 9.7 against 11.0 / 15.5) and slower above (1x128x128^2 with 32 vectors 16.1 against
// 10.9 forward, 16x64x64^2 of 16 MB 23.6 against 16.9 backward); one launch in place of three
// also saves 4 us of the host's time.
constexpr double kResidentBytes = 8 << 20;
constexpr int kResidentSlots = 8;
constexpr int64_t kSliceBytes = 64;
// An applying pass of one wave merges the statistics itself, without a launch between, where a
// sample has at most this many parts times groups: each CTA reads them all. On a B200, 128 channels
// in 16 bits, 128^2 and 256^2 pixels, 1 to 16 samples, 1 to 128 groups: without the launch 3 to 8 % less
// time up to 1,184 of them (8x128x256^2, 32 groups, 67.9 us against 70.3), between 3 % less and 5 % more
// near 2,368, as much to 18 % more from 4,736 on (1x128x256^2, 32 groups, 20.3 against 17.1).
constexpr int kMergeMost = 2048;
constexpr int64_t kApplySteps = 32, kApplyWaves = 6;

size_t elem_size(int dtype) { return dtype == FSSIM_F32 ? 4 : 2; }
bool known_dtype(int d) { return d == FSSIM_F32 || d == FSSIM_F16 || d == FSSIM_BF16; }
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Elements per vector: 16 bytes where every tensor's address is a multiple of that and either the
// channels are whole vectors, or the samples are whole spans of at most a CTA's vectors; else 4
// bytes by the same rule, else one element. On a B200 whole vectors against the narrow ones that
// the channel count alone allows (forward, us): 4x3x1080x1920 16-bit 33 against 161, 32-bit 51
// against 211; 1x30x1080x1920 72 against 258, 124 against 551.
int vector_width(int64_t C, int64_t P, size_t esize, const void* a, const void* b, const void* c) {
  for (size_t bytes : {size_t{16}, size_t{4}}) {
    const int64_t v = static_cast<int64_t>(bytes / esize);
    if (!aligned(a, bytes) || !aligned(b, bytes) || !aligned(c, bytes)) continue;
    if (C % v == 0) return static_cast<int>(v);
    if (P % (v / std::gcd(C, v)) == 0 && C / std::gcd(C, v) <= fssim::kNormThreads) return static_cast<int>(v);
  }
  return 1;
}

NormGeometry make_geometry(int64_t N, int64_t P, int64_t C, int64_t G, int V, int reduce_batch, float eps) {
  NormGeometry g{};
  g.N = N;
  g.P = P;
  g.C = static_cast<int>(C);
  g.G = static_cast<int>(G);
  g.Cg = static_cast<int>(C / G);
  g.eps = eps;
  g.inv_m = 1.0 / (static_cast<double>(P) * static_cast<double>(g.Cg));
  g.period = static_cast<int>(V / std::gcd(C, static_cast<int64_t>(V)));
  g.Cv = static_cast<int>(C * g.period);
  const int64_t spans = P / g.period, vectors = g.Cv / V;
  const int64_t slices = (vectors + fssim::kNormThreads - 1) / fssim::kNormThreads;
  g.lanes = static_cast<int>((vectors + slices - 1) / slices);
  g.slices = static_cast<int>((vectors + g.lanes - 1) / g.lanes);
  g.SC = g.lanes * V;
  g.rows = fssim::kNormThreads / g.lanes;
  g.GS = g.slices == 1 ? g.G : static_cast<int>((g.SC + g.Cg - 2) / g.Cg + 1);
  if (g.GS > g.G) g.GS = g.G;
  // Parts of the reducing pass: one wave of CTAs, or where the samples are more than that, enough
  // that the last wave's idle SMs weigh little; no more than there are tiles.
  g.tile = g.rows * reduce_batch;
  const int64_t tiles = (spans + g.tile - 1) / g.tile;
  const int64_t each = N * g.slices;
  const int64_t S = each <= kWave ? kWave / each : (4 * kWave + each - 1) / each;
  g.S = static_cast<int>(S < tiles ? S : tiles);
  g.part_tiles = static_cast<int>(tiles / g.S);
  g.extra_tiles = static_cast<int>(tiles % g.S);
  g.last_part = static_cast<int>((tiles - 1) % g.S);
  g.lacking = static_cast<int>(tiles * g.tile - spans);
  return g;
}

// The same for the applying pass: one wave of CTAs with equal parts, or for large tensors short
// parts of kApplySteps pixels for each thread, which the SMs take in their order. On a B200
// short parts are faster from about kApplyWaves waves of them (8x128x512^2 16-bit training
// pass 676 against 729 us), one wave below (8x128x256^2: 183 against 187 us), where the last
// wave's idle SMs weigh more than the order of the accesses.
NormGeometry apply_geometry(NormGeometry g) {
  const int64_t spans = g.P / g.period;
  const int64_t each = g.N * g.slices, most = (spans + g.rows - 1) / g.rows;
  const int64_t step = static_cast<int64_t>(g.rows) * kApplySteps;
  int64_t S = (spans + step - 1) / step;
  if (S * each < kApplyWaves * kWave) S = each <= kWave ? kWave / each : (4 * kWave + each - 1) / each;
  if (S > most) S = most;
  g.S = static_cast<int>(S);
  g.base = static_cast<int>(spans / S);
  g.extra = static_cast<int>(spans % S);
  return g;
}

// The resident kernels' split, where they take the call: slices of whole groups of at least
// kSliceBytes a pixel, and clusters large enough to spread the work, for `tensors` tensors held
// at a time. slots is 0 where they do not take it.
struct ResidentPlan {
  NormGeometry g;
  int slots;    // vectors of a thread
  size_t smem;
};

ResidentPlan plan_resident(int64_t N, int64_t P, int64_t C, int64_t G, int V, size_t esize, float eps, int tensors) {
  ResidentPlan r{};
  if (V * esize != 16 || C % V != 0 || static_cast<double>(N) * P * C * esize * tensors > kResidentBytes) return r;
  const int64_t Cg = C / G;
  const int64_t unit = std::lcm(static_cast<int64_t>(V), Cg);
  int64_t SC = unit * ((kSliceBytes / static_cast<int64_t>(esize) + unit - 1) / unit);
  if (SC > C) SC = C;
  if (SC / V > fssim::kNormThreads) return r;
  NormGeometry& g = r.g;
  g.N = N;
  g.P = P;
  g.C = static_cast<int>(C);
  g.G = static_cast<int>(G);
  g.Cg = static_cast<int>(Cg);
  g.eps = eps;
  g.keep = 1.f;
  g.inv_m = 1.0 / (static_cast<double>(P) * static_cast<double>(Cg));
  g.period = 1;
  g.Cv = g.C;
  g.SC = static_cast<int>(SC);
  g.lanes = static_cast<int>(SC / V);
  g.slices = static_cast<int>((C + SC - 1) / SC);
  g.rows = fssim::kNormThreads / g.lanes;
  g.GS = static_cast<int>(SC / Cg);
  const int64_t units = N * g.slices;
  const auto slots = [&](int K) { return ((P + K - 1) / K + g.rows - 1) / g.rows; };
  const size_t scratch = sizeof(float) * fssim::kNormScratch * fssim::kNormThreads * V;
  int K = 1;
  while (K < 8 && (slots(K) > kResidentSlots || (slots(K) > 2 && units * K * 2 <= kWave))) K *= 2;
  if (slots(K) > kResidentSlots) return r;
  g.S = K;
  g.base = static_cast<int>(P / K);
  g.extra = static_cast<int>(P % K);
  r.slots = static_cast<int>(slots(K));
  r.smem = scratch + static_cast<size_t>(r.slots) * 16 * fssim::kNormThreads * tensors;
  return r;
}

// Share of a launch's input that stays in L2 from the reducing pass to the applying one.
float kept_share(double bytes) {
  return bytes <= kKeptBytes ? 1.f : static_cast<float>(kKeptBytes / bytes);
}

template <typename Kernel, typename... Extra>
int launch(Kernel k, dim3 grid, int cluster, size_t smem, const NormParams& p, cudaStream_t stream,
           const char* what, Extra... extra) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(fssim::kNormThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  // Clusters that start while the kernel before still has its CTAs on the SMs go one to an SM, and
  // more of them than SMs then take a second wave (16x64x64^2 16-bit training pass 33 against
  // 28 us): such a launch waits for that kernel's end.
  if (cluster == 1 || grid.x <= kSms) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, p, extra...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(FSSIM_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  return FSSIM_OK;
}

// Opts a pass in to its ring of shared memory, once for each kernel and device. `done` belongs to
// one kernel instantiation.
template <typename Kernel>
int allow_ring(Kernel k, size_t smem, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64)) return fail(FSSIM_ERR_CUDA, "device ordinal out of range");
  if (e == cudaSuccess && !done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  }
  return e == cudaSuccess ? FSSIM_OK : fail(FSSIM_ERR_CUDA, cudaGetErrorString(e));
}

// A pass over the tiles of g.
template <auto K, size_t SMEM>
int launch_pass(const NormGeometry& g, const NormParams& p, cudaStream_t stream, const char* what) {
  if (g.N * g.S > INT_MAX) return fail(FSSIM_ERR_SHAPE, "more than 2^31 tiles");
  static std::atomic<bool> done[64];
  const int st = allow_ring(K, SMEM, done);
  if (st) return st;
  return launch(K, dim3(static_cast<unsigned>(g.N * g.S), static_cast<unsigned>(g.slices)), 1, SMEM, p, stream, what);
}

// Whether some thread of a reducing pass has more spans than it may add up in FP32. Kernels and
// memory for folded sums only then: where they are not needed they cost 1 to 4 % (1x128x256^2 16-bit
// forward 18.1 us against 17.8, 1x128x128^2 training pass 24.7 against 23.9).
template <typename Walk>
bool folds(const NormGeometry& g) {
  return (static_cast<int64_t>(g.part_tiles) + (g.extra_tiles > 0)) * Walk::kU > Walk::kFoldSpans;
}

int check_common(int dtype, int weight_dtype, int activation, int64_t N, int64_t P, int64_t C,
                 int64_t G, float eps) {
  if (!known_dtype(dtype)) return fail(FSSIM_ERR_DTYPE, "dtype must be F32, F16 or BF16");
  if (!known_dtype(weight_dtype)) return fail(FSSIM_ERR_DTYPE, "weight_dtype must be F32, F16 or BF16");
  if (activation < FSSIM_ACT_NONE || activation > FSSIM_ACT_RELU)
    return fail(FSSIM_ERR_ARGUMENT, "activation must be 0 (none), 1 (silu) or 2 (relu)");
  if (N < 0 || P < 0 || C < 0) return fail(FSSIM_ERR_SHAPE, "negative dimension");
  if (G < 1 || C < 1 || C % G != 0)
    return fail(FSSIM_ERR_SHAPE, "the channels must divide into the groups (C = " +
                                     std::to_string(C) + ", groups = " + std::to_string(G) + ")");
  if (C > kMaxChannels) return fail(FSSIM_ERR_SHAPE, "C must be at most 2^23");
  if (N > kMaxSamples) return fail(FSSIM_ERR_SHAPE, "N must be at most 2^30");
  if (N * G > INT_MAX) return fail(FSSIM_ERR_SHAPE, "N*groups must be < 2^31");
  if (static_cast<double>(N) * P * C > 1.0e18) return fail(FSSIM_ERR_SHAPE, "N*P*C overflows int64");
  if (P > (int64_t{1} << 38)) return fail(FSSIM_ERR_SHAPE, "P must be at most 2^38");
  if (!(eps >= 0.f)) return fail(FSSIM_ERR_ARGUMENT, "eps must not be negative");
  return FSSIM_OK;
}

struct ForwardPlan {
  int V;
  ResidentPlan resident;
  NormGeometry g, apply;
  int merges;  // of the applying pass, or 0
  size_t partial, bytes;
};

ForwardPlan plan_forward(const fssim_group_norm_forward_args& a) {
  ForwardPlan p{};
  const size_t E = elem_size(a.dtype);
  p.V = vector_width(a.C, a.P, E, a.x, a.y, nullptr);
  p.resident = plan_resident(a.N, a.P, a.C, a.groups, p.V, E, a.eps, 1);
  if (p.resident.slots) return p;
  p.g = make_geometry(a.N, a.P, a.C, a.groups, p.V, kStatsU, a.eps);
  p.apply = apply_geometry(p.g);
  const bool wave = static_cast<int64_t>(p.apply.S) * a.N <= kWave && p.g.slices == 1;
  if (wave && a.groups <= fssim::kNormMergeGroups && p.g.S * a.groups <= kMergeMost) p.merges = p.g.S;
  p.partial = round256(sizeof(float2) * static_cast<size_t>(a.N) * p.g.S * p.g.slices * p.g.GS);
  p.bytes = p.partial + sizeof(float) * fssim::kNormForwardRows * static_cast<size_t>(a.N) * a.C;
  return p;
}

struct BackwardPlan {
  int V;
  ResidentPlan resident;
  NormGeometry g;
  size_t partial, sums, bytes;
};

BackwardPlan plan_backward(const fssim_group_norm_backward_args& a) {
  BackwardPlan p{};
  const size_t E = elem_size(a.dtype);
  p.V = vector_width(a.C, a.P, E, a.x, a.dy, a.dx);
  p.resident = plan_resident(a.N, a.P, a.C, a.groups, p.V, E, 0.f, 2);
  if (p.resident.slots) {
    // the samples' sums of the parameters' gradients, where there are several
    if (a.N > 1 && (a.dweight || a.dbias)) p.bytes = sizeof(float2) * static_cast<size_t>(a.N) * a.C;
    return p;
  }
  p.g = make_geometry(a.N, a.P, a.C, a.groups, p.V, kGradU, 0.f);
  p.partial = round256(sizeof(float2) * static_cast<size_t>(a.N) * p.g.S * a.C);
  p.sums = round256(sizeof(float2) * static_cast<size_t>(a.N) * a.C);
  p.bytes = p.partial + p.sums + sizeof(float) * fssim::kNormBackwardRows * static_cast<size_t>(a.N) * a.C;
  return p;
}

// Threads that merge one group, for this many partial results, as a power of two: a warp at least, a
// CTA at most.
int team_shift(int64_t results) {
  int t = 5;
  while ((1 << t) < fssim::kNormThreads && (1 << t) < results) ++t;
  return t;
}
dim3 team_grid(const NormGeometry& g, int shift) {
  const int64_t teams = fssim::kNormThreads >> shift;
  return dim3(static_cast<unsigned>((g.N * g.G + teams - 1) / teams));
}

template <typename T, int V, int ACT>
int forward_kernels(const NormParams& p, const NormGeometry& apply, cudaStream_t s) {
  using Short = fssim::NormWalk<T, V, kStatsU, kStatsB, false>;
  using Long = fssim::NormWalk<T, V, kStatsU, kStatsB, false, true>;
  using Apply = fssim::NormWalk<T, V, kApplyU, kApplyB, true>;
  const char* what = "group norm statistics launch";
  int st = folds<Short>(p.g)
               ? launch_pass<fssim::norm_stats_kernel<T, V, kStatsU, kStatsB, true>, Long::reducing_bytes(1)>(p.g, p, s, what)
               : launch_pass<fssim::norm_stats_kernel<T, V, kStatsU, kStatsB, false>, Short::reducing_bytes(1)>(p.g, p, s, what);
  if (st) return st;
  if (!p.merges) {
    const int team = team_shift(p.g.S);
    st = launch(fssim::norm_merge_kernel, team_grid(p.g, team), 1, 0, p, s, "group norm merge launch", team);
    if (st) return st;
  }
  NormParams q = p;  // (the applying pass reads x ahead of its wait: never without a launch before)
  q.g = apply;
  return launch_pass<fssim::norm_apply_kernel<T, V, ACT, kApplyU, kApplyB>, Apply::kRingBytes>(
      q.g, q, s, "group norm launch");
}

template <typename T, int V, int ACT>
int backward_kernels(const NormParams& p, cudaStream_t s) {
  using Short = fssim::NormWalk<T, V, kGradU, kGradB, false>;
  using Long = fssim::NormWalk<T, V, kGradU, kGradB, false, true>;
  const char* what = "group norm gradient sums launch";
  int st =
      folds<Short>(p.g)
          ? launch_pass<fssim::norm_grad_sums_kernel<T, V, ACT, kGradU, kGradB, true>, Long::reducing_bytes(2)>(p.g, p, s, what)
          : launch_pass<fssim::norm_grad_sums_kernel<T, V, ACT, kGradU, kGradB, false>, Short::reducing_bytes(2)>(p.g, p, s, what);
  if (st) return st;
  int cols = 0;  // channels merged at a time, likewise
  while (cols < 5 && (1 << cols) < p.g.Cg) ++cols;
  const int team = team_shift(static_cast<int64_t>(p.g.S) << cols);
  st = launch(fssim::norm_grad_merge_kernel, team_grid(p.g, team), 1, 0, p, s,
              "group norm gradient merge launch", team, cols);
  if (st || !p.out) return st;
  NormParams q = p;  // (likewise, with dy)
  q.g = apply_geometry(p.g);
  q.fold_params = p.g.N > 1 && (p.dweight || p.dbias);
  return launch_pass<fssim::norm_grad_apply_kernel<T, V, ACT, kGradU, kGradB>, 2 * Short::kRingBytes>(
      q.g, q, s, "group norm gradient launch");
}

// One launch list per (element type, vector width, activation).
template <template <typename, int, int> class Run, typename T, int V, typename Plan>
int by_activation(int act, const NormParams& p, const Plan& r, cudaStream_t s) {
  switch (act) {
    case FSSIM_ACT_SILU: return Run<T, V, fssim::kNormActSilu>::run(p, r, s);
    case FSSIM_ACT_RELU: return Run<T, V, fssim::kNormActRelu>::run(p, r, s);
    default: return Run<T, V, fssim::kNormActNone>::run(p, r, s);
  }
}
template <template <typename, int, int> class Run, typename T, typename Plan>
int by_width(int V, int act, const NormParams& p, const Plan& r, cudaStream_t s) {
  constexpr int full = 16 / sizeof(T), mid = 4 / sizeof(T);
  if (V == full) return by_activation<Run, T, full>(act, p, r, s);
  if constexpr (mid > 1) {
    if (V == mid) return by_activation<Run, T, mid>(act, p, r, s);
  }
  return by_activation<Run, T, 1>(act, p, r, s);
}
template <template <typename, int, int> class Run, typename Plan>
int dispatch(int dtype, int V, int act, const NormParams& p, const Plan& r, cudaStream_t s) {
  switch (dtype) {
    case FSSIM_F32: return by_width<Run, float>(V, act, p, r, s);
    case FSSIM_F16: return by_width<Run, __half>(V, act, p, r, s);
    default: return by_width<Run, __nv_bfloat16>(V, act, p, r, s);
  }
}
template <typename T, int V, int ACT>
struct Forward {
  static int run(const NormParams& p, const NormGeometry& apply, cudaStream_t s) {
    return forward_kernels<T, V, ACT>(p, apply, s);
  }
};
template <typename T, int V, int ACT>
struct Backward {
  static int run(const NormParams& p, const ResidentPlan&, cudaStream_t s) { return backward_kernels<T, V, ACT>(p, s); }
};

template <auto K, typename... Extra>
int launch_resident(const NormParams& p, const ResidentPlan& r, cudaStream_t s, const char* what, Extra... extra) {
  static std::atomic<bool> done[64];
  // (attribute for the most that any call may ask for)
  constexpr size_t most = fssim::kNormThreads * 16 * (2 * kResidentSlots + 2 * fssim::kNormScratch);
  const int st = allow_ring(K, most, done);
  if (st) return st;
  const int64_t ctas = p.g.N * p.g.slices * p.g.S;
  return launch(K, dim3(static_cast<unsigned>(ctas)), p.g.S, r.smem, p, s, what, extra...);
}
template <typename T, int V, int ACT>
struct ForwardResident {
  static int run(const NormParams& p, const ResidentPlan& r, cudaStream_t s) {
    if constexpr (sizeof(T) * V == 16)
      return launch_resident<fssim::norm_resident_kernel<T, V, ACT>>(p, r, s, "group norm launch");
    else return fail(FSSIM_ERR_ARGUMENT, "resident kernels take 16-byte vectors");
  }
};
template <typename T, int V, int ACT>
struct BackwardResident {
  static int run(const NormParams& p, const ResidentPlan& r, cudaStream_t s) {
    if constexpr (sizeof(T) * V == 16)
      return launch_resident<fssim::norm_grad_resident_kernel<T, V, ACT>>(p, r, s, "group norm gradient launch", r.slots);
    else return fail(FSSIM_ERR_ARGUMENT, "resident kernels take 16-byte vectors");
  }
};

int forward_impl(const fssim_group_norm_forward_args* a, cudaStream_t stream) {
  if (!a) return fail(FSSIM_ERR_NULLPTR, "args is NULL");
  int st = check_common(a->dtype, a->weight_dtype, a->activation, a->N, a->P, a->C, a->groups, a->eps);
  if (st) return st;
  if ((a->mean == nullptr) != (a->rstd == nullptr))
    return fail(FSSIM_ERR_NULLPTR, "mean and rstd are written together: give both or neither");
  if (a->N == 0 || a->P == 0) return FSSIM_OK;
  if (!a->x || !a->y) return fail(FSSIM_ERR_NULLPTR, "x and y are required");
  const size_t E = elem_size(a->dtype);
  if (!aligned(a->x, E) || !aligned(a->y, E))
    return fail(FSSIM_ERR_ARGUMENT, "x and y must be aligned to their element size");
  ForwardPlan plan = plan_forward(*a);
  if (!plan.resident.slots && a->P / plan.g.S >= (int64_t{1} << 30))
    return fail(FSSIM_ERR_SHAPE, "a CTA's part has 2^30 pixels or more");
  if (plan.bytes && (!a->workspace || a->workspace_bytes < plan.bytes))
    return fail(FSSIM_ERR_WORKSPACE, "workspace smaller than fssim_group_norm_forward_workspace_bytes");
  if (!aligned(a->workspace, 16)) return fail(FSSIM_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  NormParams p{};
  p.x = a->x;
  p.out = a->y;
  p.weight = a->weight;
  p.bias = a->bias;
  p.weight_dtype = a->weight_dtype;
  p.weight_vectors = aligned(a->weight, 16) && aligned(a->bias, 16);
  p.mean = a->mean;
  p.rstd = a->rstd;
  if (plan.resident.slots) {
    p.g = plan.resident.g;
    return dispatch<ForwardResident>(a->dtype, plan.V, a->activation, p, plan.resident, stream);
  }
  p.g = plan.g;
  p.g.keep = plan.apply.keep = kept_share(static_cast<double>(a->N) * a->P * a->C * E);
  p.partial = static_cast<float2*>(a->workspace);
  p.channel = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + plan.partial);
  p.merges = plan.merges;
  return dispatch<Forward>(a->dtype, plan.V, a->activation, p, plan.apply, stream);
}

int backward_impl(const fssim_group_norm_backward_args* a, cudaStream_t stream) {
  if (!a) return fail(FSSIM_ERR_NULLPTR, "args is NULL");
  int st = check_common(a->dtype, a->weight_dtype, a->activation, a->N, a->P, a->C, a->groups, 0.f);
  if (st) return st;
  const size_t WE = elem_size(a->weight_dtype);
  if (a->N == 0 || a->P == 0) {
    // nothing was summed: the parameters' gradients are zero
    for (void* w : {a->dweight, a->dbias})
      if (w) {
        const cudaError_t e = cudaMemsetAsync(w, 0, WE * static_cast<size_t>(a->C), stream);
        if (e != cudaSuccess) return fail(FSSIM_ERR_CUDA, cudaGetErrorString(e));
      }
    return FSSIM_OK;
  }
  if (!a->dx && !a->dweight && !a->dbias) return FSSIM_OK;
  if (!a->x || !a->dy) return fail(FSSIM_ERR_NULLPTR, "x and dy are required");
  if (!a->mean || !a->rstd) return fail(FSSIM_ERR_NULLPTR, "the forward's mean and rstd are required");
  const size_t E = elem_size(a->dtype);
  if (!aligned(a->x, E) || !aligned(a->dy, E) || !aligned(a->dx, E))
    return fail(FSSIM_ERR_ARGUMENT, "x, dy and dx must be aligned to their element size");
  const BackwardPlan plan = plan_backward(*a);
  if (!plan.resident.slots && a->P / plan.g.S >= (int64_t{1} << 30))
    return fail(FSSIM_ERR_SHAPE, "a CTA's part has 2^30 pixels or more");
  if (plan.bytes && (!a->workspace || a->workspace_bytes < plan.bytes))
    return fail(FSSIM_ERR_WORKSPACE, "workspace smaller than fssim_group_norm_backward_workspace_bytes");
  if (!aligned(a->workspace, 16)) return fail(FSSIM_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(a->workspace);
  NormParams p{};
  p.x = a->x;
  p.dy = a->dy;
  p.out = a->dx;
  p.weight = a->weight;
  p.bias = a->bias;
  p.weight_dtype = a->weight_dtype;
  p.weight_vectors = aligned(a->weight, 16) && aligned(a->bias, 16);
  p.mean = const_cast<float*>(a->mean);
  p.rstd = const_cast<float*>(a->rstd);
  p.dweight = a->dweight;
  p.dbias = a->dbias;
  if (plan.resident.slots) {
    p.g = plan.resident.g;
    p.sums = plan.bytes ? reinterpret_cast<float2*>(ws) : nullptr;
    st = dispatch<BackwardResident>(a->dtype, plan.V, a->activation, p, plan.resident, stream);
  } else {
    p.g = plan.g;
    p.g.keep = kept_share(2.0 * a->N * a->P * a->C * E);
    p.partial = reinterpret_cast<float2*>(ws);
    p.sums = reinterpret_cast<float2*>(ws + plan.partial);
    p.channel = reinterpret_cast<float*>(ws + plan.partial + plan.sums);
    st = dispatch<Backward>(a->dtype, plan.V, a->activation, p, plan.resident, stream);
  }
  if (st) return st;
  // One sample's sums are the parameters' gradients, and have been written; of several, the applying
  // pass has added them up.
  if (a->N == 1 || (!a->dweight && !a->dbias) || (!plan.resident.slots && a->dx)) return FSSIM_OK;
  const unsigned blocks = static_cast<unsigned>((a->C + fssim::kNormWarps - 1) / fssim::kNormWarps);
  return launch(fssim::norm_param_grad_kernel, dim3(blocks), 1, 0, p, stream,
                "group norm parameter gradient launch");
}

// No exception crosses the C boundary.
template <typename F>
int guarded(F f) {
  try {
    fssim_host::g_last_error.clear();
    return f();
  } catch (const std::exception&) {
    fssim_host::g_last_error = "host exception";  // short: no allocation
    return FSSIM_ERR_CUDA;
  }
}

}  // namespace

extern "C" {

size_t fssim_group_norm_forward_workspace_bytes(const fssim_group_norm_forward_args* a) {
  if (!a || a->N <= 0 || a->P <= 0 || a->groups < 1 || a->C < 1 || a->C > kMaxChannels ||
      a->N > kMaxSamples || a->C % a->groups != 0)
    return 0;
  return plan_forward(*a).bytes;
}

size_t fssim_group_norm_backward_workspace_bytes(const fssim_group_norm_backward_args* a) {
  if (!a || a->N <= 0 || a->P <= 0 || a->groups < 1 || a->C < 1 || a->C > kMaxChannels ||
      a->N > kMaxSamples || a->C % a->groups != 0)
    return 0;
  return plan_backward(*a).bytes;
}

int fssim_group_norm_forward(const fssim_group_norm_forward_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_group_norm_forward");
  return guarded([&] { return forward_impl(a, stream); });
}

int fssim_group_norm_backward(const fssim_group_norm_backward_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_group_norm_backward");
  return guarded([&] { return backward_impl(a, stream); });
}

}  // extern "C"
