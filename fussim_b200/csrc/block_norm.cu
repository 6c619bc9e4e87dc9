// C entry points of the residual-block norms: argument checks, the split of rows over CTAs, and the
// launches. The kernels are in block_norm.cuh.
#include "block_norm.cuh"

#include <cmath>
#include <cstdint>
#include <string>

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
  bool vec;
  int vectors;   // of eight numbers, of a thread
  int threads;   // of a row
  int block;     // of a CTA
  int64_t B, T;  // samples and rows: all rows are one sample's where no vector has one for each sample
  int64_t chunk, chunks;
};

Layout layout(const Shape& s, bool per_sample, bool vec, int resident_threads) {
  Layout l{};
  l.vec = vec;
  const int groups = static_cast<int>((s.C + 7) / 8);
  if (groups <= 32) {
    l.vectors = 1;
    for (l.threads = 1; l.threads < groups;) l.threads *= 2;
    l.block = kBlockSmallThreads;
  } else {
    l.vectors = groups <= kBlockMaxThreads ? 1 : groups <= 2 * kBlockMaxThreads ? 2 : 4;
    l.threads = (groups + 32 * l.vectors - 1) / (32 * l.vectors) * 32;
    l.block = l.threads;
  }
  l.B = per_sample ? s.B : 1;
  l.T = per_sample ? s.T : s.B * s.T;
  const int64_t parts = l.block / l.threads;
  const int64_t ctas = kSms * (resident_threads / l.block > 0 ? resident_threads / l.block : 1);
  const int64_t wanted = (ctas + l.B - 1) / l.B;
  int64_t rounds = (l.T + parts * wanted - 1) / (parts * wanted);
  // a thread adds at most this many rows up in FP32
  if (rounds > 256) rounds = 256;
  l.chunk = rounds * parts;
  l.chunks = (l.T + l.chunk - 1) / l.chunk;
  return l;
}

BlockChannels channels(const fssim_channels& v, int64_t C) {
  return {v.data, v.dtype, v.per_sample, v.data && aligned(v.data, 16) && (!v.per_sample || C % 8 == 0)};
}

template <typename F>
int with_layout(const Layout& l, F f) {
  const auto vec = [&](auto v) {
    return l.vec ? f(v, std::true_type{}) : f(v, std::false_type{});
  };
  switch (l.vectors) {
    case 1: return vec(std::integral_constant<int, 1>{});
    case 2: return vec(std::integral_constant<int, 2>{});
    default: return vec(std::integral_constant<int, 4>{});
  }
}

template <typename F>
int with_types(int x, int y, F f) {
  if (x == FSSIM_F32 && y == FSSIM_F32) return f(float{}, float{});
  if (x == FSSIM_F32 && y == FSSIM_F16) return f(float{}, __half{});
  if (x == FSSIM_F32) return f(float{}, __nv_bfloat16{});
  if (x == FSSIM_F16) return f(__half{}, __half{});
  return f(__nv_bfloat16{}, __nv_bfloat16{});
}

BlockParams params(const Shape& s, const Layout& l) {
  BlockParams p{};
  p.T = l.T;
  p.chunk = l.chunk;
  p.chunks = l.chunks;
  p.C = static_cast<int>(s.C);
  p.threads = l.threads;
  return p;
}

int check_grid(int64_t ctas) {
  return ctas <= 0x7FFFFFFF ? FSSIM_OK : fail(FSSIM_ERR_SHAPE, "too many samples");
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
  const Layout l = layout(s, per_sample, vec, 1024);
  if ((st = check_grid(l.B * l.chunks))) return st;
  BlockParams p = params(s, l);
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
  return with_types(s.x_dtype, s.y_dtype, [&](auto x, auto y) {
    return with_layout(l, [&](auto v, auto wide) {
      return launch(block_norm_forward_kernel<decltype(x), decltype(y), v(), wide()>,
                    static_cast<unsigned>(l.B * l.chunks), l.block, 0, stream, "block norm forward launch", p);
    });
  });
}

// The backward pass's split of its sums.
struct Merge {
  int sums, segments;
  size_t partial_bytes, merged_bytes;
};

bool wants_sums(const fssim_block_norm_backward_args& a, int* sums) {
  const bool after = a.dgate.data || a.dbranch_weight.data || a.dbranch_bias.data;
  *sums = after ? 4 : 2;
  return after || a.dweight.data || a.dbias.data || a.dscale.data || a.dshift.data;
}

Layout backward_layout(const fssim_block_norm_backward_args& a) {
  const Shape s{a.B, a.T, a.C, a.x_dtype, a.y_dtype};
  const bool per_sample = a.gate.per_sample || a.scale.per_sample || a.weight.per_sample || a.bias.per_sample ||
                          a.branch_weight.per_sample || a.branch_bias.per_sample || a.dshift.per_sample;
  bool vec = s.C % 8 == 0;
  for (const void* p : {a.r, a.branch, a.dr, a.dz, static_cast<const void*>(a.dx), static_cast<const void*>(a.dbranch)})
    vec = vec && aligned(p, 16);
  return layout(s, per_sample, vec, 512);
}

Merge merge_of(const fssim_block_norm_backward_args& a, const Layout& l) {
  Merge m{};
  if (!wants_sums(a, &m.sums)) return Merge{};
  const int64_t columns = (a.C + kBlockMergeColumns - 1) / kBlockMergeColumns;
  int64_t segments = (2 * kSms + columns * l.B - 1) / (columns * l.B);
  const int64_t most = l.chunks / (4 * kBlockMergeTeams);
  segments = segments > most ? most : segments;
  m.segments = static_cast<int>(segments < 1 ? 1 : segments);
  m.partial_bytes = (static_cast<size_t>(l.B * l.chunks) * m.sums * a.C * sizeof(float) + 15) / 16 * 16;
  m.merged_bytes = l.chunks > 1 ? static_cast<size_t>(l.B) * m.segments * m.sums * a.C * sizeof(double) : 0;
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
  const size_t need = m.partial_bytes + m.merged_bytes;
  if (need > 0 && (!a->workspace || a->workspace_bytes < need))
    return fail(FSSIM_ERR_WORKSPACE, "workspace smaller than fssim_block_norm_backward_workspace_bytes");
  if (!aligned(a->workspace, 16)) return fail(FSSIM_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  if (!m.sums && !a->dx && !a->dbranch) return FSSIM_OK;
  BlockParams p = params(s, l);
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
  st = with_types(s.x_dtype, s.y_dtype, [&](auto x, auto y) {
    return with_layout(l, [&](auto v, auto wide) {
      return launch(block_norm_backward_kernel<decltype(x), decltype(y), v(), wide()>,
                    static_cast<unsigned>(l.B * l.chunks), l.block, 0, stream, "block norm backward launch", p);
    });
  });
  if (st || !m.sums) return st;
  const int64_t columns = (s.C + kBlockMergeColumns - 1) / kBlockMergeColumns;
  constexpr unsigned kMergeThreads = kBlockMergeColumns * kBlockMergeTeams;
  double* merged = m.merged_bytes ? reinterpret_cast<double*>(static_cast<char*>(a->workspace) + m.partial_bytes) : nullptr;
  if (merged) {
    if ((st = check_grid(columns * l.B * m.segments))) return st;
    st = launch(block_norm_merge_kernel, static_cast<unsigned>(columns * l.B * m.segments), kMergeThreads, 0, stream,
                "block norm merge launch", static_cast<const float*>(p.partials), merged, p.C, m.sums, l.chunks,
                m.segments);
    if (st) return st;
  }
  BlockGradParams g{};
  g.merged = merged;
  g.partials = p.partials;
  g.B = l.B;
  g.segments = m.segments;
  g.sums = m.sums;
  g.C = p.C;
  g.s = a->residual_scale;
  g.gate = p.gate;
  g.weight = p.weight;
  g.bias = channels(a->bias, s.C);
  g.scale = p.scale;
  g.after_weight = p.after_weight;
  g.after_bias = channels(a->branch_bias, s.C);
  const auto place = [](const fssim_channels_grad& v) { return BlockGrad{v.data, v.dtype, v.per_sample}; };
  g.dgate = place(a->dgate);
  g.dweight = place(a->dweight);
  g.dbias = place(a->dbias);
  g.dscale = place(a->dscale);
  g.dshift = place(a->dshift);
  g.dafter_weight = place(a->dbranch_weight);
  g.dafter_bias = place(a->dbranch_bias);
  return launch(block_norm_grads_kernel, static_cast<unsigned>(columns), kMergeThreads, 0, stream,
                "block norm gradients launch", g);
}

}  // namespace

extern "C" {

int fssim_block_norm_forward(const fssim_block_norm_forward_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_block_norm_forward");
  return guarded([&] { return forward(a, stream); });
}

size_t fssim_block_norm_backward_workspace_bytes(const fssim_block_norm_backward_args* a) {
  if (!a || a->B <= 0 || a->T <= 0 || check_shape({a->B, a->T, a->C, a->x_dtype, a->y_dtype})) return 0;
  const Merge m = merge_of(*a, backward_layout(*a));
  return m.partial_bytes + m.merged_bytes;
}

int fssim_block_norm_backward(const fssim_block_norm_backward_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_block_norm_backward");
  return guarded([&] { return backward(a, stream); });
}

}  // extern "C"
