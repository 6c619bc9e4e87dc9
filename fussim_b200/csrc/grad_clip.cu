// C entry points of the global gradient norm and of clipping: argument checks, the tables of
// tensors and the launches. The kernels are in grad_clip.cuh.
#include "grad_clip.cuh"

#include <atomic>
#include <climits>
#include <cstdint>
#include <exception>
#include <memory>
#include <string>

#include "engine_host.h"

namespace {

using fssim::ClipTable;
using fssim::kClipMaxCtas;
using fssim::kClipThreads;
using fssim::kClipUnit;
using fssim_host::aligned;
using fssim_host::fail;
using fssim_host::NvtxRange;

// Runs per launch: a small table (3 KB of parameters) or a large one (29 KB, of the 32 KB that
// a launch may carry).
constexpr int kFew = 96;
constexpr int kMany = 832;
// Units of a CTA of the clipping, in large calls.
constexpr int64_t kCutUnits = 16;
// Bytes of the gradients that are to stay in L2 from the norm to the clipping, of larger ones.
constexpr double kKeptBytes = 80 << 20;
static_assert(sizeof(ClipTable<kMany>) <= 32764, "kernel parameters are limited to 32764 bytes");

size_t elem_size(int dtype) { return dtype == FSSIM_F32 ? 4 : 2; }
bool known_dtype(int d) { return d == FSSIM_F32 || d == FSSIM_F16 || d == FSSIM_BF16; }

template <typename... KA, typename... A>
int launch(void (*k)(KA...), unsigned grid, size_t smem, cudaStream_t stream, const char* what, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kClipThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, args...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(FSSIM_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  return FSSIM_OK;
}

unsigned grid_for(int64_t units) {
  return static_cast<unsigned>(units < kClipMaxCtas ? units : kClipMaxCtas);
}

// CTAs of the clipping for each range of the norm's pass.
int cuts_of(int64_t units) {
  const int64_t cuts = units / (grid_for(units) * kCutUnits);
  return static_cast<int>(cuts < 1 ? 1 : cuts < 4096 ? cuts : 4096);
}

int64_t units_of(int64_t size) { return (size + kClipUnit - 1) / kClipUnit; }

// Launches of a call: runs of at most kMany non-empty tensors each.
struct Cut {
  int64_t begin, end;  // tensors
  int64_t units;
  int runs;
};

Cut next_cut(const fssim_grad_clip_args& a, int64_t begin) {
  Cut c{begin, begin, 0, 0};
  while (c.end < a.count && c.runs < kMany) {
    if (a.sizes[c.end] > 0) {
      c.units += units_of(a.sizes[c.end]);
      ++c.runs;
    }
    ++c.end;
  }
  return c;
}

int total_partials(const fssim_grad_clip_args& a) {
  int64_t n = 0;
  for (int64_t i = 0; i < a.count;) {
    const Cut c = next_cut(a, i);
    n += grid_for(c.units);
    i = c.end;
  }
  return static_cast<int>(n < INT_MAX ? n : INT_MAX);
}

int check(const fssim_grad_clip_args* a, bool clip) {
  if (!a) return fail(FSSIM_ERR_NULLPTR, "args is NULL");
  if (a->count < 0) return fail(FSSIM_ERR_SHAPE, "negative number of tensors");
  if (!a->norm) return fail(FSSIM_ERR_NULLPTR, "norm is required");
  if (a->count > 0 && (!a->grads || !a->sizes || !a->dtypes))
    return fail(FSSIM_ERR_NULLPTR, "grads, sizes and dtypes are required");
  if (clip && a->count > 0 && (!a->outs || !a->out_dtypes))
    return fail(FSSIM_ERR_NULLPTR, "outs and out_dtypes are required");
  if (clip && !(a->max_norm >= 0.f)) return fail(FSSIM_ERR_ARGUMENT, "max_norm must not be negative");
  for (int64_t i = 0; i < a->count; ++i) {
    if (a->sizes[i] < 0 || a->sizes[i] > (int64_t{1} << 60))
      return fail(FSSIM_ERR_SHAPE, "a tensor's size is negative or too large");
    if (!known_dtype(a->dtypes[i])) return fail(FSSIM_ERR_DTYPE, "gradients must be F32, F16 or BF16");
    if (clip && a->out_dtypes[i] != a->dtypes[i] && a->out_dtypes[i] != FSSIM_F32)
      return fail(FSSIM_ERR_DTYPE, "an output has its gradient's type or F32");
    if (a->sizes[i] == 0) continue;
    if (!a->grads[i] || (clip && !a->outs[i])) return fail(FSSIM_ERR_NULLPTR, "a tensor's pointer is NULL");
    if (!aligned(a->grads[i], elem_size(a->dtypes[i])) ||
        (clip && !aligned(a->outs[i], elem_size(a->out_dtypes[i]))))
      return fail(FSSIM_ERR_ARGUMENT, "a tensor is not aligned to its element size");
    if (clip && a->outs[i] == a->grads[i] && a->out_dtypes[i] != a->dtypes[i])
      return fail(FSSIM_ERR_ARGUMENT, "an output in its gradient's place has the gradient's type");
  }
  const int64_t need = fssim_grad_clip_workspace_bytes(a);
  if (need > 0 && (!a->workspace || a->workspace_bytes < static_cast<size_t>(need)))
    return fail(FSSIM_ERR_WORKSPACE, "workspace smaller than fssim_grad_clip_workspace_bytes");
  if (!aligned(a->workspace, 8)) return fail(FSSIM_ERR_WORKSPACE, "workspace must be 8-byte aligned");
  return FSSIM_OK;
}

// Opts the clipping in to its ring of shared memory, once for each device.
template <int K>
int allow_ring() {
  static std::atomic<bool> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64)) return fail(FSSIM_ERR_CUDA, "device ordinal out of range");
  if (e == cudaSuccess && !done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(fssim::grad_clip_kernel<K>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             fssim::kClipRingBytes);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  }
  return e == cudaSuccess ? FSSIM_OK : fail(FSSIM_ERR_CUDA, cudaGetErrorString(e));
}

template <int K>
int launch_cut(const fssim_grad_clip_args& a, const Cut& c, bool clip, bool summed, int partials, int first,
               float keep, cudaStream_t stream) {
  const std::unique_ptr<ClipTable<K>> t(new ClipTable<K>);
  int r = 0;
  int64_t unit = 0;
  for (int64_t i = c.begin; i < c.end; ++i) {
    if (a.sizes[i] == 0) continue;
    t->src[r] = a.grads[i];
    t->dst[r] = clip ? a.outs[i] : nullptr;
    t->size[r] = a.sizes[i];
    t->unit0[r] = unit;
    t->src_dtype[r] = static_cast<unsigned char>(a.dtypes[i]);
    t->dst_dtype[r] = static_cast<unsigned char>(clip ? a.out_dtypes[i] : 0);
    unit += units_of(a.sizes[i]);
    ++r;
  }
  t->unit0[r] = unit;
  t->count = r;
  // (the sum of the partial sums follows them)
  t->partials = static_cast<double*>(a.workspace) + (clip && summed ? partials : 0);
  t->num_partials = clip && summed ? 1 : partials;
  t->first_partial = first;
  t->norm = clip && !summed && first == 0 ? a.norm : nullptr;
  t->max_norm = a.max_norm;
  t->keep = keep;
  const unsigned ranges = grid_for(c.units);
  t->ranges = static_cast<int>(ranges);
  t->cuts = summed ? cuts_of(c.units) : 1;
  const int st = allow_ring<K>();
  if (st) return st;
  if (!clip)
    return launch(fssim::grad_squares_kernel<K>, ranges, 0, stream, "gradient norm launch", *t);
  return launch(fssim::grad_clip_kernel<K>, ranges * static_cast<unsigned>(t->cuts), fssim::kClipRingBytes, stream,
                "gradient clipping launch", *t);
}

// One pass over all tensors: the partial sums (clip == false) or the scaling.
int pass(const fssim_grad_clip_args& a, bool clip, bool summed, int partials, cudaStream_t stream) {
  double bytes = 0.0;
  for (int64_t i = 0; i < a.count; ++i) bytes += static_cast<double>(a.sizes[i]) * elem_size(a.dtypes[i]);
  const float keep = bytes <= kKeptBytes ? 1.f : static_cast<float>(kKeptBytes / bytes);
  int first = 0;
  for (int64_t i = 0; i < a.count;) {
    const Cut c = next_cut(a, i);
    i = c.end;
    if (c.runs == 0) continue;
    const int st = c.runs <= kFew ? launch_cut<kFew>(a, c, clip, summed, partials, first, keep, stream)
                                  : launch_cut<kMany>(a, c, clip, summed, partials, first, keep, stream);
    if (st) return st;
    first += static_cast<int>(grid_for(c.units));
  }
  return FSSIM_OK;
}

int run(const fssim_grad_clip_args* a, bool clip, cudaStream_t stream) {
  int st = check(a, clip);
  if (st) return st;
  const int partials = total_partials(*a);
  if (partials == 0) {
    const cudaError_t e = cudaMemsetAsync(a->norm, 0, sizeof(float), stream);
    return e == cudaSuccess ? FSSIM_OK : fail(FSSIM_ERR_CUDA, cudaGetErrorString(e));
  }
  // Large calls add the partial sums up in a launch of their own, so that the clipping can come in
  // many short CTAs, which the SMs take in their order, without each adding them up again.
  // (Not in place, where the usual call finds the norm within the limit and has nothing to do.)
  bool summed = !clip, moves = false;
  for (int64_t i = 0; i < a->count && clip && !moves; ++i) moves = a->sizes[i] > 0 && a->outs[i] != a->grads[i];
  for (int64_t i = 0; i < a->count && moves && !summed;) {
    const Cut c = next_cut(*a, i);
    summed = cuts_of(c.units) > 1;
    i = c.end;
  }
  st = pass(*a, false, summed, partials, stream);
  if (st) return st;
  if (summed) {
    double* sums = static_cast<double*>(a->workspace);
    st = launch(fssim::grad_norm_kernel, 1u, 0, stream, "gradient norm sum launch",
                static_cast<const double*>(sums), partials, sums + partials, a->norm);
    if (st || !clip) return st;
  }
  return pass(*a, true, summed, partials, stream);
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

size_t fssim_grad_clip_workspace_bytes(const fssim_grad_clip_args* a) {
  if (!a || a->count <= 0 || !a->sizes) return 0;
  const size_t partials = static_cast<size_t>(total_partials(*a));
  return partials ? sizeof(double) * (partials + 1) : 0;
}

int fssim_grad_norm(const fssim_grad_clip_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_grad_norm");
  return guarded([&] { return run(a, false, stream); });
}

int fssim_grad_clip(const fssim_grad_clip_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_grad_clip");
  return guarded([&] { return run(a, true, stream); });
}

}  // extern "C"
