// C entry points of the residual-block norms: argument checks, the split of rows over CTAs, and the
// launches. The kernels are in block_norm.cuh and block_norm_merge.cuh.
#include "block_norm_merge.cuh"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "block_norm_launch.h"
#include "engine_host.h"
#include "launch_host.h"

namespace {

using namespace fssim;
using fssim_host::aligned;
using fssim_host::fail;
using fssim_host::guarded;
using fssim_host::launch;
using fssim_host::NvtxRange;

constexpr int64_t kSms = 148;
constexpr int64_t kMaxRows = int64_t{1} << 40;

bool known_dtype(int d) { return d == FSSIM_F32 || d == FSSIM_F16 || d == FSSIM_BF16; }
size_t elem_size(int dtype) { return dtype == FSSIM_F32 ? 4 : 2; }

struct Shape {
  int64_t B, T, C;
  int x_dtype, y_dtype;
};

int check_shape(const Shape& s) {
  if (!known_dtype(s.x_dtype) || !known_dtype(s.y_dtype) || (s.x_dtype != s.y_dtype && s.x_dtype != FSSIM_F32))
    return fail(FSSIM_ERR_DTYPE, "types must be F32, F16 or BF16, the residual's the branch's or F32");
  if (s.B < 0 || s.T < 0 || s.B > kMaxRows || s.T > kMaxRows || (s.T > 0 && s.B > kMaxRows / s.T))
    return fail(FSSIM_ERR_SHAPE, "numbers of samples and rows must not be negative, nor their product above 2^40");
  if (s.C < 1 || s.C > kBlockMaxC)
    return fail(FSSIM_ERR_SHAPE, "rows must have 1 to " + std::to_string(kBlockMaxC) + " numbers");
  return FSSIM_OK;
}

int check_vector(const char* name, const void* data, int dtype) {
  if (!data) return FSSIM_OK;
  if (!known_dtype(dtype)) return fail(FSSIM_ERR_DTYPE, std::string(name) + " must be F32, F16 or BF16");
  if (!aligned(data, elem_size(dtype)))
    return fail(FSSIM_ERR_ARGUMENT, std::string(name) + " is not aligned to its element size");
  return FSSIM_OK;
}

int check_kind(int kind, bool none) {
  return kind == FSSIM_NORM_RMS || kind == FSSIM_NORM_LAYER || (none && kind == FSSIM_NORM_NONE)
             ? FSSIM_OK
             : fail(FSSIM_ERR_ARGUMENT, "unknown kind of norm");
}

struct Named {
  const char* name;
  const void* p;
  int dtype;
  bool required;
};

template <size_t N>
int check_tensors(const Named (&all)[N]) {
  for (const Named& t : all) {
    if (t.required && !t.p) return fail(FSSIM_ERR_NULLPTR, std::string(t.name) + " is required");
    if (t.p && !aligned(t.p, elem_size(t.dtype)))
      return fail(FSSIM_ERR_ARGUMENT, std::string(t.name) + " is not aligned to its element size");
  }
  return FSSIM_OK;
}

// How rows are laid over threads and CTAs.
struct Layout {
  bool vec, warp;
  int groups;    // of eight numbers, of a thread
  int threads;   // of a row
  int block;     // of a CTA
  int64_t B, T;  // samples and rows: all rows are one sample's where no vector has one for each sample
  int64_t chunk, chunks;
  int stages;    // of the ring
  bool staged;   // the arrays are in shared memory
  size_t memory;
};

constexpr int64_t kSmMemory = 216 << 10;  // of an SM's shared memory: for rings and arrays

// `bytes`(groups): of a stage of the ring, for each number of a row. `arrays`: how many there are.
template <typename Bytes>
Layout layout(const Shape& s, bool backward, int mode, bool per_sample, bool vec, Bytes bytes, int arrays) {
  Layout l{};
  const int needed = static_cast<int>((s.C + 7) / 8);
  // Rows within a warp where a thread has at most five groups of eight numbers (forward; two
  // backward, whose sums are in registers) of it: the fewest threads that are idle at a row's end, and
  // of those the most groups, since what a row costs each thread (sums, addresses) is paid for more numbers.
  const auto best = [&](std::initializer_list<int> choices, bool warp) {
    int padded = INT_MAX;
    for (const int g : choices) {
      int t = (needed + g - 1) / g;
      if (warp) {
        int p = 1;
        while (p < t) p *= 2;
        t = p;
        if (t > 32) continue;
      } else {
        t = (t + 31) / 32 * 32;
        if (t > kBlockMaxThreads || (backward && t > block_resident(block_backward_registers(g, l.vec)))) continue;
      }
      // (the kernels count on whole groups but for a row's last)
      if ((g - 1) * t < needed && t * g <= padded) {
        padded = t * g;
        l.groups = g;
        l.threads = t;
      }
    }
    l.warp = warp;
    return padded < INT_MAX;
  };
  l.vec = vec;
  for (;;) {
    if (!l.vec) {
      if (!best({1}, true) && !best({1}, false) && !best({2}, false)) best({4}, false);
    } else if (backward) {
      if (!best({1, 2}, true) && !best({1, 2}, false)) best({4}, false);
    } else if (s.B * s.T <= 2 * kSms && needed <= kBlockMaxThreads) {
      if (!best({1}, true)) best({1}, false);  // few rows: the fastest for each
    } else if (!best({1, 3, 4, 5}, true)) {
      if (needed > kBlockMaxThreads || !best({3, 4}, false)) best({4}, false);
    }
    const int resident = block_resident(
        backward ? block_backward_registers(l.groups, l.vec)
                 : block_forward_registers(l.groups, l.vec || l.groups == 1 ? mode : kBlockAfter, l.vec));
    l.B = per_sample ? s.B : 1;
    l.T = per_sample ? s.T : s.B * s.T;
    const int64_t array_bytes = static_cast<int64_t>(arrays) * s.C * sizeof(float);
    // As many threads on an SM as its registers and shared memory hold, with the arrays in each CTA and a
    // row ahead of each thread's own; of these the largest CTAs, which lay arrays down for the most rows.
    // (8x1024x1152 16-bit forward: CTAs of 256 threads 21.8 us, of 128 27.7; 16x1024x1024 with a 32-bit
    // residual, where two of 256 do not fit: 70 and 41.)
    Layout found = l;
    int64_t most = 0;
    for (int block = l.warp ? 256 : l.threads; l.warp ? block >= 32 : most == 0; block /= 2) {
      const int64_t parts = block / l.threads;
      if (parts < 1) break;
      const int64_t stage = l.vec ? static_cast<int64_t>(block) * l.groups * 8 * bytes(l.groups) : 0;
      if (stage > fssim_host::kBlockMemory) {
        if (l.warp) continue;
        break;
      }
      // Few rows: smaller CTAs, so that all SMs have some; backward of at least four rows of a thread, for
      // which it leaves one set of sums.
      const int64_t fewest = backward ? 4 : 1;
      if (l.warp && block > 32 && l.B * ((l.T + parts * fewest - 1) / (parts * fewest)) < 2 * kSms) continue;
      for (int64_t on_sm = std::max(resident / block, 1); on_sm >= 1 && on_sm * block > most; --on_sm) {
        const int64_t wanted = (kSms * on_sm + l.B - 1) / l.B;
        // a thread adds at most 256 rows up in FP32
        const int64_t rounds = std::clamp<int64_t>((l.T + parts * wanted - 1) / (parts * wanted),
                                                   std::min(fewest, (l.T + parts - 1) / parts), 256);
        const int64_t chunk = rounds * parts, chunks = (l.T + chunk - 1) / chunk;
        const int64_t crowd = std::min(on_sm, (l.B * chunks + kSms - 1) / kSms);
        const int64_t room = std::min<int64_t>(kSmMemory / crowd - 2048, fssim_host::kBlockMemory);
        // (kernels that make the arrays again for each row: four groups of a CTA's rows alone)
        const bool choice = l.groups == 4 && !l.warp;
        const bool fits = array_bytes + kBlockStages * stage <= room && (l.vec || !choice);
        if (!fits && (on_sm > 1 || (l.warp && block > 32))) continue;
        found.block = block;
        found.chunk = chunk;
        found.chunks = chunks;
        found.staged = fits || !choice;
        const int64_t rest = room - (found.staged ? array_bytes : 0);
        found.stages = stage ? static_cast<int>(std::clamp<int64_t>(rest / stage, 1, kBlockStages)) : 1;
        found.memory = static_cast<size_t>(stage * found.stages + (found.staged ? array_bytes : 0));
        most = on_sm * block;
      }
    }
    if (most == 0) {  // rows are loaded number by number
      l.vec = false;
      continue;
    }
    l = found;
    // (the backward pass adds up in it what rows side by side left)
    if (backward && l.warp) l.memory = std::max<size_t>(l.memory, sizeof(float) * (l.block / 32) * s.C);
    return l;
  }
}

BlockChannels channels(const fssim_channels& v, int64_t C) {
  return {v.data, v.dtype, v.per_sample, v.data && aligned(v.data, 16) && (!v.per_sample || C % 8 == 0)};
}

int launch_rows(bool backward, const Shape& s, const Layout& l, const BlockParams& p, cudaStream_t stream) {
  const auto run = s.x_dtype == FSSIM_F32 ? (s.y_dtype == FSSIM_F32   ? fssim_host::block_norm_f32
                                             : s.y_dtype == FSSIM_F16 ? fssim_host::block_norm_f32_f16
                                                                      : fssim_host::block_norm_f32_bf16)
                   : s.x_dtype == FSSIM_F16 ? fssim_host::block_norm_f16
                                            : fssim_host::block_norm_bf16;
  const int mode = p.after_kind || (!p.y && (p.dr || (backward && !p.dz))) ? kBlockAfter : p.y ? kBlockPlain : kBlockBefore;
  return run(backward, {l.groups, l.vec, l.warp, l.staged, mode, static_cast<unsigned>(l.B * l.chunks),
                        static_cast<unsigned>(l.block), l.memory}, p, stream);
}

int count_of(int bits) { return __builtin_popcount(static_cast<unsigned>(bits)); }

BlockParams params(const Shape& s, const Layout& l) {
  BlockParams p{};
  p.T = l.T;
  p.chunk = l.chunk;
  p.chunks = l.chunks;
  p.C = static_cast<int>(s.C);
  p.inv = 1.0 / static_cast<double>(s.C);
  p.threads = l.threads;
  p.stages = l.stages;
  return p;
}

int check_grid(int64_t ctas) {
  return ctas <= 0x7FFFFFFF ? FSSIM_OK : fail(FSSIM_ERR_SHAPE, "too many samples");
}

// A branch without a norm has no weight and bias (its kernels leave three sums, none for their gradients).
template <typename Args>
int check_branch(const Args& a, bool vectors) {
  if (!a.branch) return FSSIM_OK;
  if (a.branch_kind == FSSIM_NORM_NONE && vectors)
    return fail(FSSIM_ERR_ARGUMENT, "branch_weight and branch_bias go with a branch_kind");
  return std::isfinite(static_cast<float>(a.residual_scale))
             ? FSSIM_OK
             : fail(FSSIM_ERR_ARGUMENT, "residual_scale must be finite in FP32");
}
int check_branch(const fssim_block_norm_forward_args& a) { return check_branch(a, a.branch_weight.data || a.branch_bias.data); }
int check_branch(const fssim_block_norm_backward_args& a) {
  return check_branch(a, a.branch_weight.data || a.branch_bias.data || a.dbranch_weight.data || a.dbranch_bias.data);
}

int forward(const fssim_block_norm_forward_args* a, cudaStream_t stream) {
  if (!a) return fail(FSSIM_ERR_NULLPTR, "args is NULL");
  const Shape s{a->B, a->T, a->C, a->x_dtype, a->y_dtype};
  int st = check_shape(s);
  if (st || (st = check_kind(a->kind, !a->z)) || (st = check_kind(a->branch_kind, true))) return st;
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(FSSIM_ERR_ARGUMENT, "eps must be finite and not negative");
  for (const auto& [name, v] : {std::pair<const char*, fssim_channels>{"gate", a->gate}, {"weight", a->weight},
                                {"bias", a->bias}, {"scale", a->scale}, {"shift", a->shift},
                                {"branch_weight", a->branch_weight}, {"branch_bias", a->branch_bias}})
    if ((st = check_vector(name, v.data, v.dtype))) return st;
  if ((st = check_branch(*a))) return st;
  if (s.B == 0 || s.T == 0) return FSSIM_OK;
  if (!a->z && !a->branch) return fail(FSSIM_ERR_NULLPTR, "z or branch is required");
  const Named all[] = {{"x", a->x, s.x_dtype, true},
                       {"branch", a->branch, s.y_dtype, false},
                       {"r", a->r, s.x_dtype, a->branch != nullptr},
                       {"z", a->z, s.y_dtype, false},
                       {"stats", a->stats, FSSIM_F32, false},
                       {"branch_stats", a->branch_stats, FSSIM_F32, false}};
  if ((st = check_tensors(all))) return st;
  for (const float* p : {a->stats, a->branch_stats})
    if (!aligned(p, 8)) return fail(FSSIM_ERR_ARGUMENT, "statistics must be aligned to 8 bytes");
  const bool per_sample = a->gate.per_sample || a->scale.per_sample || a->shift.per_sample || a->weight.per_sample ||
                          a->bias.per_sample || a->branch_weight.per_sample || a->branch_bias.per_sample;
  const bool vec = s.C % 8 == 0 && aligned(a->x, 16) && aligned(a->branch, 16) && aligned(a->r, 16) && aligned(a->z, 16);
  const int bytes = static_cast<int>(elem_size(s.x_dtype) + (a->branch ? elem_size(s.y_dtype) : 0));
  const bool after = a->branch && a->branch_kind != FSSIM_NORM_NONE;
  const int arrays = (a->branch && a->gate.data ? 1 << kArrayGate : 0) |
                     (a->z && (a->weight.data || a->scale.data) ? 1 << kArrayFactor : 0) |
                     (a->z && (a->bias.data || a->shift.data) ? 1 << kArrayOffset : 0) |
                     (after && a->branch_weight.data ? 1 << kArrayAfterWeight : 0) |
                     (after && a->branch_bias.data ? 1 << kArrayAfterBias : 0);
  const Layout l = layout(s, false, !a->branch ? kBlockBefore : after ? kBlockAfter : kBlockPlain, per_sample, vec,
                          [&](int) { return bytes; }, count_of(arrays));
  if ((st = check_grid(l.B * l.chunks))) return st;
  BlockParams p = params(s, l);
  p.arrays = arrays;
  p.kind = a->kind;
  p.after_kind = a->branch ? a->branch_kind : kBlockNone;
  p.eps = a->eps;
  p.s = a->residual_scale;
  p.x = a->x;
  p.y = a->branch;
  p.r = a->r;
  p.z = a->z;
  p.stats = reinterpret_cast<float2*>(a->stats);
  p.after_stats = reinterpret_cast<float2*>(a->branch_stats);
  p.gate = channels(a->gate, s.C);
  p.weight = channels(a->weight, s.C);
  p.bias = channels(a->bias, s.C);
  p.scale = channels(a->scale, s.C);
  p.shift = channels(a->shift, s.C);
  p.after_weight = channels(a->branch_weight, s.C);
  p.after_bias = channels(a->branch_bias, s.C);
  return launch_rows(false, s, l, p, stream);
}

// The backward pass's split of its sums.
struct Merge {
  int sums, splits, split_samples;
  int64_t columns;  // blocks of columns
  bool shared;      // a gradient is a sum over samples
  size_t partial_bytes, total_bytes;
  size_t bytes() const { return partial_bytes + total_bytes; }
};

bool wants_sums(const fssim_block_norm_backward_args& a, int* sums) {
  const bool after = a.dgate.data || a.dbranch_weight.data || a.dbranch_bias.data;
  *sums = !after ? 2 : a.branch_kind == FSSIM_NORM_NONE ? 3 : 4;
  return after || a.dweight.data || a.dbias.data || a.dscale.data || a.dshift.data;
}

int backward_arrays(const fssim_block_norm_backward_args& a) {
  return (a.branch && (a.gate.data || (a.branch_kind && a.branch_weight.data)) ? 1 << kArrayGate : 0) |
         (a.dz && (a.weight.data || a.scale.data) ? 1 << kArrayFactor : 0);
}

Layout backward_layout(const fssim_block_norm_backward_args& a) {
  const Shape s{a.B, a.T, a.C, a.x_dtype, a.y_dtype};
  const bool per_sample = a.gate.per_sample || a.scale.per_sample || a.weight.per_sample || a.bias.per_sample ||
                          a.branch_weight.per_sample || a.branch_bias.per_sample || a.dshift.per_sample;
  bool vec = s.C % 8 == 0;
  for (const void* p : {a.r, a.branch, a.dr, a.dz, static_cast<const void*>(a.dx), static_cast<const void*>(a.dbranch)})
    vec = vec && aligned(p, 16);
  const int x = static_cast<int>(elem_size(s.x_dtype)), y = static_cast<int>(elem_size(s.y_dtype));
  // as the kernels lay a stage out: r and dz, and except in those for one norm before a block dr and y
  const bool before = !a.branch && a.dz && !a.dr;
  const auto bytes = [&](int groups) { return before && groups < 4 ? x + y : 2 * (x + y); };
  const int mode = !a.branch ? kBlockBefore : a.branch_kind ? kBlockAfter : kBlockPlain;
  return layout(s, true, mode, per_sample, vec, bytes, count_of(backward_arrays(a)));
}

Merge merge_of(const fssim_block_norm_backward_args& a, const Layout& l) {
  Merge m{};
  if (!wants_sums(a, &m.sums)) return Merge{};
  m.columns = (a.C + kBlockMergeColumns - 1) / kBlockMergeColumns;
  // many samples: more CTAs for them, down to one for each team
  const int64_t splits = std::min((2 * kSms + m.columns - 1) / m.columns, l.B / kBlockMergeTeams);
  m.split_samples = static_cast<int>((l.B + std::max<int64_t>(splits, 1) - 1) / std::max<int64_t>(splits, 1));
  m.splits = static_cast<int>((l.B + m.split_samples - 1) / m.split_samples);
  for (const fssim_channels_grad* g : {&a.dgate, &a.dweight, &a.dbias, &a.dscale, &a.dshift, &a.dbranch_weight, &a.dbranch_bias})
    m.shared = m.shared || (g->data && !g->per_sample);
  m.partial_bytes = (static_cast<size_t>(l.B * l.chunks) * m.sums * a.C * sizeof(float) + 15) / 16 * 16;
  if (m.splits > 1 && m.shared) m.total_bytes = static_cast<size_t>(m.splits) * kVectors * a.C * sizeof(double);
  return m;
}

int backward(const fssim_block_norm_backward_args* a, cudaStream_t stream) {
  if (!a) return fail(FSSIM_ERR_NULLPTR, "args is NULL");
  const Shape s{a->B, a->T, a->C, a->x_dtype, a->y_dtype};
  int st = check_shape(s);
  if (st || (st = check_kind(a->kind, !a->dz)) || (st = check_kind(a->branch_kind, true))) return st;
  for (const auto& [name, v] : {std::pair<const char*, fssim_channels>{"gate", a->gate}, {"weight", a->weight},
                                {"bias", a->bias}, {"scale", a->scale}, {"branch_weight", a->branch_weight},
                                {"branch_bias", a->branch_bias}})
    if ((st = check_vector(name, v.data, v.dtype))) return st;
  for (const auto& [name, v] : {std::pair<const char*, fssim_channels_grad>{"dgate", a->dgate}, {"dweight", a->dweight},
                                {"dbias", a->dbias}, {"dscale", a->dscale}, {"dshift", a->dshift},
                                {"dbranch_weight", a->dbranch_weight}, {"dbranch_bias", a->dbranch_bias}})
    if ((st = check_vector(name, v.data, v.dtype))) return st;
  if ((st = check_branch(*a))) return st;
  if (s.B == 0 || s.T == 0) return FSSIM_OK;
  const bool branch = a->branch != nullptr;
  const Named all[] = {{"r", a->r, s.x_dtype, a->dz != nullptr},
                       {"branch", a->branch, s.y_dtype, a->dbranch != nullptr},
                       {"dr", a->dr, s.x_dtype, a->dz == nullptr},
                       {"dz", a->dz, s.y_dtype, false},
                       {"stats", a->stats, FSSIM_F32, a->dz != nullptr},
                       {"branch_stats", a->branch_stats, FSSIM_F32, branch && a->branch_kind != FSSIM_NORM_NONE},
                       {"dx", a->dx, s.x_dtype, false},
                       {"dbranch", a->dbranch, s.y_dtype, false}};
  if ((st = check_tensors(all))) return st;
  for (const float* p : {a->stats, a->branch_stats})
    if (!aligned(p, 8)) return fail(FSSIM_ERR_ARGUMENT, "statistics must be aligned to 8 bytes");
  if (!branch && (a->dgate.data || a->dbranch_weight.data || a->dbranch_bias.data))
    return fail(FSSIM_ERR_NULLPTR, "branch is required for its vectors' gradients");
  const Layout l = backward_layout(*a);
  if ((st = check_grid(l.B * l.chunks))) return st;
  const Merge m = merge_of(*a, l);
  const size_t need = m.bytes();
  if (need > 0 && (!a->workspace || a->workspace_bytes < need))
    return fail(FSSIM_ERR_WORKSPACE, "workspace smaller than fssim_block_norm_backward_workspace_bytes");
  if (!aligned(a->workspace, 16)) return fail(FSSIM_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  if (!m.sums && !a->dx && !a->dbranch) return FSSIM_OK;
  BlockParams p = params(s, l);
  p.arrays = backward_arrays(*a);
  p.kind = a->kind;
  p.after_kind = branch ? a->branch_kind : kBlockNone;
  p.s = a->residual_scale;
  p.r = const_cast<void*>(a->r);
  p.y = a->branch;
  p.dr = a->dr;
  p.dz = a->dz;
  p.dx = a->dx;
  p.dy = a->dbranch;
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(a->stats));
  p.after_stats = reinterpret_cast<float2*>(const_cast<float*>(a->branch_stats));
  p.gate = channels(a->gate, s.C);
  p.weight = channels(a->weight, s.C);
  p.scale = channels(a->scale, s.C);
  p.after_weight = channels(a->branch_weight, s.C);
  p.partials = m.sums ? static_cast<float*>(a->workspace) : nullptr;
  p.sums = m.sums;
  st = launch_rows(true, s, l, p, stream);
  if (st || !m.sums) return st;
  BlockGradParams g{};
  g.partials = p.partials;
  g.totals = m.total_bytes ? reinterpret_cast<double*>(static_cast<char*>(a->workspace) + m.partial_bytes) : nullptr;
  g.B = static_cast<int>(l.B);
  g.chunks = static_cast<int>(l.chunks);
  g.split_samples = m.split_samples;
  g.shared = m.shared;
  g.splits = m.splits;
  g.C = p.C;
  g.s = a->residual_scale;
  g.gate = p.gate;
  g.weight = p.weight;
  g.bias = channels(a->bias, s.C);
  g.scale = p.scale;
  g.after_weight = p.after_weight;
  g.after_bias = channels(a->branch_bias, s.C);
  const auto place = [](const fssim_channels_grad& v) { return BlockGrad{v.data, v.dtype, v.per_sample}; };
  g.grads[kVectorGate] = place(a->dgate);
  g.grads[kVectorWeight] = place(a->dweight);
  g.grads[kVectorBias] = place(a->dbias);
  g.grads[kVectorScale] = place(a->dscale);
  g.grads[kVectorShift] = place(a->dshift);
  g.grads[kVectorAfterWeight] = place(a->dbranch_weight);
  g.grads[kVectorAfterBias] = place(a->dbranch_bias);
  const auto kernel = m.sums == 2   ? block_norm_grads_kernel<2>
                      : m.sums == 3 ? block_norm_grads_kernel<3>
                                    : block_norm_grads_kernel<4>;
  st = launch(kernel, static_cast<unsigned>(m.columns * m.splits), kBlockMergeColumns * kBlockMergeTeams, 0, stream,
              "block norm gradients launch", g);
  if (st || !m.total_bytes) return st;
  return launch(block_norm_totals_kernel, static_cast<unsigned>((s.C + 255) / 256), 256, 0, stream,
                "block norm totals launch", g);
}

}  // namespace

extern "C" {

int fssim_block_norm_forward(const fssim_block_norm_forward_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_block_norm_forward");
  return guarded([&] { return forward(a, stream); });
}

size_t fssim_block_norm_backward_workspace_bytes(const fssim_block_norm_backward_args* a) {
  if (!a || a->B <= 0 || a->T <= 0 || check_shape({a->B, a->T, a->C, a->x_dtype, a->y_dtype}) || check_branch(*a))
    return 0;
  const Merge m = merge_of(*a, backward_layout(*a));
  return m.bytes();
}

int fssim_block_norm_backward(const fssim_block_norm_backward_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_block_norm_backward");
  return guarded([&] { return backward(a, stream); });
}

}  // extern "C"
