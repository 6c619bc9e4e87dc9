// Torch binding of the training-step operators over the C ABI (include/fussim_b200.h, section
// 4): group normalisation with an activation as a C++ autograd function, and the gradient norm
// with clipping. Everything launches on torch's current CUDA stream of the tensors' device;
// workspaces are allocated by the call from torch's caching allocator (so calls on different
// streams, and captured graphs, never share one).
#include "torch_training.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/util/SmallVector.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <numeric>
#include <stdexcept>
#include <string>
#include <vector>

#include "fussim_b200.h"

namespace {

void check_status(int st) {
  if (st == FSSIM_OK) return;
  throw std::runtime_error(std::string("fussim_b200: ") + fssim_status_string(st) + ": " +
                           fssim_last_error());
}

fssim_stream_t current_stream() {
  return reinterpret_cast<fssim_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FSSIM_F32;
    case at::kHalf: return FSSIM_F16;
    case at::kBFloat16: return FSSIM_BF16;
    default: throw std::invalid_argument("unsupported dtype for fussim_b200");
  }
}

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

using OptTensor = std::optional<at::Tensor>;

// A lazily negated view (the imaginary part of a conjugate) holds its numbers with the other sign.
at::Tensor resolved(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
OptTensor resolved(const OptTensor& t) { return t.has_value() ? OptTensor(resolved(*t)) : t; }

// Weight and bias as the C ABI takes them: dense, of one type (group_norm_act has checked device,
// shape and type), and with memory of their own, since no pointer stands for no weight there.
struct Affine {
  at::Tensor weight, bias;
  int dtype = FSSIM_F32;
  Affine(const OptTensor& w, const OptTensor& b) {
    if (w.has_value() && w->defined()) weight = w->contiguous();
    if (b.has_value() && b->defined()) bias = b->contiguous();
    for (const at::Tensor* t : {&weight, &bias})
      if (t->defined() && !t->const_data_ptr())
        throw std::runtime_error("weight and bias must be tensors with memory (not fake ones)");
    if (weight.defined()) dtype = dtype_code(weight.scalar_type());
    else if (bias.defined()) dtype = dtype_code(bias.scalar_type());
  }
  const void* w() const { return weight.defined() ? weight.data_ptr() : nullptr; }
  const void* b() const { return bias.defined() ? bias.data_ptr() : nullptr; }
};

struct NormResult {
  at::Tensor y, mean, rstd;
};

// x: dense channels-last.
NormResult norm_forward(const at::Tensor& x, int64_t groups, const Affine& affine, double eps,
                        int64_t activation, bool with_stats) {
  const at::cuda::OptionalCUDAGuard guard(x.device());
  NormResult r;
  r.y = at::empty(x.sizes(), x.options(), at::MemoryFormat::ChannelsLast);
  fssim_group_norm_forward_args a{};
  a.dtype = dtype_code(x.scalar_type());
  a.weight_dtype = affine.dtype;
  a.activation = static_cast<int32_t>(activation);
  a.N = x.size(0);
  a.C = x.size(1);
  a.P = x.size(2) * x.size(3);
  a.groups = groups;
  a.eps = static_cast<float>(eps);
  a.x = x.data_ptr();
  a.weight = affine.w();
  a.bias = affine.b();
  a.y = r.y.data_ptr();
  if (with_stats) {
    r.mean = at::empty({a.N, groups}, x.options().dtype(at::kFloat));
    r.rstd = at::empty({a.N, groups}, x.options().dtype(at::kFloat));
    a.mean = r.mean.data_ptr<float>();
    a.rstd = r.rstd.data_ptr<float>();
  }
  a.workspace_bytes = fssim_group_norm_forward_workspace_bytes(&a);
  at::Tensor ws;
  if (a.workspace_bytes) {
    ws = workspace(a.workspace_bytes, x);
    a.workspace = ws.data_ptr();
  }
  check_status(fssim_group_norm_forward(&a, current_stream()));
  return r;
}

struct GroupNormFn : public torch::autograd::Function<GroupNormFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, at::Tensor x, OptTensor weight,
                            OptTensor bias, int64_t groups, double eps, int64_t activation) {
    const at::Tensor dense = x.contiguous(at::MemoryFormat::ChannelsLast);
    const Affine affine(weight, bias);
    const NormResult r = norm_forward(dense, groups, affine, eps, activation, true);
    ctx->save_for_backward({dense, affine.weight, affine.bias, r.mean, r.rstd});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = activation;
    return r.y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "group_norm_act is differentiable once: its backward cannot be recorded "
                "(create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &bias = saved[2];
    const Affine affine(weight, bias);
    // the gradient slots of the inputs that are tensors, in their order
    size_t slot = 0;
    const bool need_x = ctx->needs_input_grad(slot++);
    const bool need_w = weight.defined() && ctx->needs_input_grad(slot);
    slot += weight.defined();
    const bool need_b = bias.defined() && ctx->needs_input_grad(slot);
    const at::cuda::OptionalCUDAGuard guard(x.device());
    const at::Tensor dy = resolved(grads[0]).to(x.scalar_type()).contiguous(at::MemoryFormat::ChannelsLast);
    at::Tensor dx, dw, db;
    if (need_x) dx = at::empty(x.sizes(), x.options(), at::MemoryFormat::ChannelsLast);
    if (need_w) dw = at::empty_like(weight);
    if (need_b) db = at::empty_like(bias);
    fssim_group_norm_backward_args a{};
    a.dtype = dtype_code(x.scalar_type());
    a.weight_dtype = affine.dtype;
    a.activation = static_cast<int32_t>(ctx->saved_data["act"].toInt());
    a.N = x.size(0);
    a.C = x.size(1);
    a.P = x.size(2) * x.size(3);
    a.groups = ctx->saved_data["groups"].toInt();
    a.x = x.data_ptr();
    a.dy = dy.data_ptr();
    a.weight = affine.w();
    a.bias = affine.b();
    a.mean = saved[3].data_ptr<float>();
    a.rstd = saved[4].data_ptr<float>();
    a.dx = need_x ? dx.data_ptr() : nullptr;
    a.dweight = need_w ? dw.data_ptr() : nullptr;
    a.dbias = need_b ? db.data_ptr() : nullptr;
    a.workspace_bytes = fssim_group_norm_backward_workspace_bytes(&a);
    at::Tensor ws;
    if (a.workspace_bytes) {
      ws = workspace(a.workspace_bytes, x);
      a.workspace = ws.data_ptr();
    }
    check_status(fssim_group_norm_backward(&a, current_stream()));
    return {dx, dw, db, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

[[noreturn]] void value_error(const std::string& msg) { throw std::invalid_argument(msg); }
[[noreturn]] void runtime_error(const std::string& msg) { throw std::runtime_error(msg); }

std::string shape_text(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}
std::string type_text(at::ScalarType t) { return std::string(c10::toString(t)); }
bool known_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

void require_cuda(const char* what) {
  if (!at::hasCUDA() || at::cuda::device_count() == 0)
    runtime_error(std::string("CUDA is not available. ") + what + " requires a CUDA-capable GPU.");
}

// A tracer records the operators that torch dispatches: of a call here it would keep the allocation
// of the result and not the launches.
void refuse_tracing(const char* what) {
  using Key = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(Key::PROXY).has_value())
    runtime_error(std::string(what) + " cannot be traced (torch.jit.trace, make_fx, torch.export): its kernels "
                  "are launched outside torch's dispatcher");
}

// Nor is there a forward-mode derivative: a result without a tangent would stand for a zero one.
void refuse_tangent(const at::Tensor& t, const char* name, const char* what) {
  if (t._fw_grad(/*level=*/0).defined())
    runtime_error(std::string(what) + " has no forward-mode derivative, but " + name + " carries a tangent");
}

int64_t activation_code(const std::optional<std::string>& name) {
  if (!name.has_value()) return FSSIM_ACT_NONE;
  if (*name == "silu") return FSSIM_ACT_SILU;
  if (*name == "relu") return FSSIM_ACT_RELU;
  value_error("activation must be one of (None, 'silu', 'relu'), got '" + *name + "'");
}

void check_norm_settings(int64_t groups, int64_t channels, double eps,
                         const std::optional<std::string>& activation) {
  activation_code(activation);
  if (groups < 1 || channels < 1 || channels % groups != 0)
    value_error("the channels must divide into the groups, got " + std::to_string(channels) +
                " channels and " + std::to_string(groups) + " groups");
  if (!(eps >= 0.0 && std::isfinite(eps)))
    value_error("eps must be finite and not negative, got " + std::to_string(eps));
}

// Checks, then the operator: recorded for autograd where a gradient may be asked for.
at::Tensor group_norm_act(const at::Tensor& given, int64_t groups, const OptTensor& given_weight,
                          const OptTensor& given_bias, double eps,
                          const std::optional<std::string>& activation) {
  const at::Tensor x = resolved(given);
  const OptTensor weight = resolved(given_weight), bias = resolved(given_bias);
  if (x.dim() != 4)
    value_error("Expected 4D tensor (B, C, H, W), but got " + std::to_string(x.dim()) +
                "D tensor with shape " + shape_text(x));
  const int64_t channels = x.size(1);
  check_norm_settings(groups, channels, eps, activation);
  if (!known_type(x.scalar_type()))
    value_error("x must be float32, float16 or bfloat16, got " + type_text(x.scalar_type()));
  refuse_tracing("group_norm_act");
  refuse_tangent(x, "x", "group_norm_act");
  bool train = x.requires_grad();
  for (const OptTensor* o : {&weight, &bias}) {
    if (!o->has_value()) continue;
    const at::Tensor& t = **o;
    const std::string name = o == &weight ? "weight" : "bias";
    if (t.dim() != 1 || t.size(0) != channels)
      value_error(name + " must have shape (" + std::to_string(channels) + ",), got " + shape_text(t));
    if (!known_type(t.scalar_type()))
      value_error(name + " must be float32, float16 or bfloat16, got " + type_text(t.scalar_type()));
    if (t.device() != x.device())
      runtime_error(name + " must be on x's device.\nx: " + x.device().str() + ", " + name + ": " +
                    t.device().str());
    refuse_tangent(t, name.c_str(), "group_norm_act");
    train = train || t.requires_grad();
  }
  if (weight.has_value() && bias.has_value() && weight->scalar_type() != bias->scalar_type())
    value_error("weight and bias must have the same dtype, got " + type_text(weight->scalar_type()) +
                " and " + type_text(bias->scalar_type()));
  require_cuda("group_norm_act");
  if (!x.is_cuda())
    runtime_error("x must be on a CUDA device, but got device: " + x.device().str());
  const int64_t act = activation_code(activation);
  if (train && at::GradMode::is_enabled())
    return GroupNormFn::apply(x, weight, bias, groups, eps, act);
  const at::NoGradGuard no_grad;
  return norm_forward(x.contiguous(at::MemoryFormat::ChannelsLast), groups, Affine(weight, bias),
                      eps, act, false)
      .y;
}

// ---- gradient norm and clipping ----
// Models have hundreds of gradients and a call's device time is tens of microseconds, so the
// tensors are read where the caller's list holds them (no copies of their handles) and in one pass.
using Refs = std::vector<const at::Tensor*>;

const at::Tensor& tensor_of(py::handle h, const char* what, size_t index) {
  if (!THPVariable_Check(h.ptr()))
    throw py::type_error(std::string(what) + " must be tensors, but that at index " + std::to_string(index) +
                         " is not");
  return THPVariable_Unpack(h.ptr());
}

Refs refs_of(const py::list& list, const char* what) {
  Refs refs;
  refs.reserve(list.size());
  for (size_t i = 0; i < list.size(); ++i) refs.push_back(&tensor_of(PyList_GET_ITEM(list.ptr(), i), what, i));
  return refs;
}

void check_grads(const Refs& grads, const char* what) {
  refuse_tracing(what);
  for (size_t i = 0; i < grads.size(); ++i) {
    const at::Tensor& g = *grads[i];
    const auto at = [&] { return " at index " + std::to_string(i) + " "; };
    if (g.layout() != at::kStrided) value_error("gradients must be dense tensors, but that" + at() + "is not");
    if (!known_type(g.scalar_type()))
      value_error("gradients must be float32, float16 or bfloat16, but that" + at() + "is " +
                  type_text(g.scalar_type()));
    if (g.device() != grads[0]->device())
      runtime_error("gradients must be on one device.\nfirst: " + grads[0]->device().str() + "," + at() +
                    g.device().str());
  }
  require_cuda(what);
  if (!grads.empty() && !grads[0]->is_cuda())
    runtime_error("gradients must be on a CUDA device, but got device: " + grads[0]->device().str());
}

// The memory of a tensor, and where the tensor stands in the call.
struct Span {
  uintptr_t begin, end;
  int64_t index;
  bool out;
};

// The ways to write a number as a sum of terms c * x, 0 <= x <= most, each c at least 1: depth first
// from the largest c, whose x the rest leaves little choice for where strides are nested, as those
// of slices are. Gives up after some hundred thousand steps, and then reports what was sought.
class SumSearch {
 public:
  void add(int64_t c, int64_t most) {
    if (most < 1) return;
    for (Term& t : terms_)
      if (merge_ && t.c == c) {
        t.most += most;
        return;
      }
    terms_.push_back({c, most, 0, 0});
  }
  explicit SumSearch(bool merge) : merge_(merge) {}  // equal c count as one term
  int ways(int64_t target, int sought) {
    std::sort(terms_.begin(), terms_.end(), [](const Term& a, const Term& b) { return a.c > b.c; });
    int64_t rest = 0, gcd = 0;
    for (size_t k = terms_.size(); k-- > 0;) {
      terms_[k].after = rest;
      rest += terms_[k].c * terms_[k].most;
      terms_[k].gcd = gcd = std::gcd(gcd, terms_[k].c);
    }
    if (target < 0 || target > rest) return 0;
    return search(0, target, sought);
  }

 private:
  struct Term {
    int64_t c, most, after, gcd;  // after: the most that the terms behind add; gcd: of these and c
  };
  int search(size_t k, int64_t target, int sought) {
    if (k == terms_.size()) return target == 0;
    const Term& t = terms_[k];
    if (target % t.gcd != 0) return 0;
    int found = 0;
    const int64_t least = target > t.after ? (target - t.after + t.c - 1) / t.c : 0;
    for (int64_t x = std::min(t.most, target / t.c); x >= least && found < sought; --x) {
      if (++steps_ > kSteps) return sought;
      found += search(k + 1, target - x * t.c, sought - found);
    }
    return found;
  }
  static constexpr int kSteps = 300000;
  c10::SmallVector<Term, 12> terms_;
  bool merge_;
  int steps_ = 0;
};

// An output and the bytes that it reaches over; it fills them where no tensor is given. Its numbers
// begin at multiples of `grid` bytes from the first.
struct Reach {
  uintptr_t begin, end;
  int64_t index;
  const at::Tensor* tensor;
  uintptr_t grid;
};
Reach reach_of(const at::Tensor& t, int64_t index) {
  int64_t last = 0, grid = 0;
  for (int64_t d = 0; d < t.dim(); ++d) {
    last += (t.size(d) - 1) * t.stride(d);
    if (t.size(d) > 1) grid = std::gcd(grid, t.stride(d));
  }
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {begin, begin + (last + 1) * t.element_size(), index, &t, grid * t.element_size()};
}

// Whether a number of the tensor has two indices.
bool overlaps_itself(const at::Tensor& t) {
  SumSearch differences(/*merge=*/false);  // of two indices in each dimension, from -(size - 1) up
  int64_t none = 0;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) > 1 && t.stride(d) == 0) return true;
    differences.add(t.stride(d), 2 * (t.size(d) - 1));
    none += (t.size(d) - 1) * t.stride(d);
  }
  return differences.ways(none, 2) > 1;  // other than all differences zero
}

bool share_memory(const Reach& a, const Reach& b) {
  if (a.end <= b.begin || b.end <= a.begin) return false;
  // columns of one buffer: numbers of both lie on the same grid, these between those
  if (a.tensor && b.tensor && a.grid == b.grid && a.grid > 0 && a.begin <= b.begin) {
    const uintptr_t beside = (b.begin - a.begin) % a.grid;
    if (beside >= a.tensor->element_size() && beside + b.tensor->element_size() <= a.grid) return false;
  }
  SumSearch bytes(/*merge=*/true);  // of a from its first on, and of b from its last down
  for (const Reach* r : {&a, &b}) {
    if (!r->tensor) {
      bytes.add(1, static_cast<int64_t>(r->end - r->begin) - 1);
      continue;
    }
    const int64_t size = static_cast<int64_t>(r->tensor->element_size());
    bytes.add(1, size - 1);
    for (int64_t d = 0; d < r->tensor->dim(); ++d)
      bytes.add(r->tensor->stride(d) * size, r->tensor->size(d) - 1);
  }
  return bytes.ways(static_cast<int64_t>(b.end - 1 - a.begin), 1) > 0;
}

// Refuses outputs that overlap each other or a gradient (but for outs[i] being grads[i]): two
// CTAs would write the same numbers, or read what another has already scaled. Tensors that do
// not fill their memory are copied before and after the kernels, which touch the copies alone; of
// those it is enough that no such output (they come in `outs`) overlaps itself or any other.
void check_overlap(std::vector<Span>& spans, std::vector<Reach>& outs) {
  const auto by_begin = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  const auto refuse = [](int64_t index) {
    value_error("tensors that are written must not overlap themselves, each other or another gradient "
                "(the same tensor twice, or views of the same memory; at index " +
                std::to_string(index) + ")");
  };
  if (!std::is_sorted(spans.begin(), spans.end(), by_begin)) std::sort(spans.begin(), spans.end(), by_begin);
  uintptr_t any_end = 0, out_end = 0;  // how far the spans so far reach
  for (const Span& s : spans) {
    if (s.begin < (s.out ? any_end : out_end)) refuse(s.index);
    any_end = std::max(any_end, s.end);
    if (s.out) out_end = std::max(out_end, s.end);
  }
  if (outs.empty()) return;
  for (const Reach& r : outs)
    if (overlaps_itself(*r.tensor)) refuse(r.index);
  for (const Span& s : spans)
    if (s.out) outs.push_back({s.begin, s.end, s.index, nullptr, 0});
  std::sort(outs.begin(), outs.end(), [](const Reach& a, const Reach& b) { return a.begin < b.begin; });
  for (size_t i = 0; i < outs.size(); ++i)
    for (size_t j = i + 1; j < outs.size() && outs[j].begin < outs[i].end; ++j)
      if ((outs[i].tensor || outs[j].tensor) && share_memory(outs[i], outs[j])) refuse(outs[j].index);
}

struct ClipArrays {
  std::vector<const void*> grads;
  std::vector<void*> outs;
  std::vector<int64_t> sizes;
  std::vector<int32_t> dtypes, out_dtypes;
  fssim_grad_clip_args args{};

  explicit ClipArrays(size_t n) {
    grads.reserve(n);
    outs.reserve(n);
    sizes.reserve(n);
    dtypes.reserve(n);
    out_dtypes.reserve(n);
  }
  void add(const void* g, void* o, int64_t size, int32_t dtype, int32_t out_dtype) {
    grads.push_back(g);
    outs.push_back(o);
    sizes.push_back(size);
    dtypes.push_back(dtype);
    out_dtypes.push_back(out_dtype);
  }
  fssim_grad_clip_args& fill(float max_norm, float* norm) {
    args.count = static_cast<int64_t>(grads.size());
    args.grads = grads.data();
    args.sizes = sizes.data();
    args.dtypes = dtypes.data();
    args.outs = outs.data();
    args.out_dtypes = out_dtypes.data();
    args.max_norm = max_norm;
    args.norm = norm;
    args.workspace_bytes = fssim_grad_clip_workspace_bytes(&args);
    return args;
  }
};

at::Tensor zero_norm() {
  return at::zeros({}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA));
}

// Tensors whose numbers fill their memory are taken as they lie; others, and lazily negated views, go
// through a dense copy.
bool as_it_lies(const at::Tensor& t) { return t.is_non_overlapping_and_dense() && !t.is_neg(); }
at::Tensor dense_copy(const at::Tensor& t) { return resolved(t).contiguous(); }

at::Tensor norm_of(const Refs& grads) {
  const at::NoGradGuard no_grad;
  const at::cuda::OptionalCUDAGuard guard(grads[0]->device());
  at::Tensor norm = at::empty({}, grads[0]->options().dtype(at::kFloat));
  ClipArrays arrays(grads.size());
  std::vector<at::Tensor> held;
  for (const at::Tensor* g : grads) {
    const bool dense = as_it_lies(*g);
    if (!dense) held.push_back(dense_copy(*g));
    void* data = (dense ? *g : held.back()).data_ptr();
    const int32_t dtype = dtype_code(g->scalar_type());
    arrays.add(data, data, g->numel(), dtype, dtype);
  }
  fssim_grad_clip_args& a = arrays.fill(0.f, norm.data_ptr<float>());
  at::Tensor ws = workspace(a.workspace_bytes, *grads[0]);
  a.workspace = ws.data_ptr();
  check_status(fssim_grad_norm(&a, current_stream()));
  return norm;
}

at::Tensor clip_into(const Refs& grads, const Refs& outs, double max_norm, bool error_if_nonfinite) {
  const at::NoGradGuard no_grad;
  const at::cuda::OptionalCUDAGuard guard(grads[0]->device());
  const size_t n = grads.size();
  ClipArrays arrays(n);
  std::vector<Span> spans;
  std::vector<Reach> scattered;  // outputs that are not written as they lie
  spans.reserve(n);
  std::vector<at::Tensor> held;                         // dense stand-ins of gradients
  std::vector<std::pair<size_t, at::Tensor>> copy_back;  // (index of an output, its stand-in)
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &g = *grads[i], &o = *outs[i];
    const int64_t size = g.numel(), index = static_cast<int64_t>(i);
    const int32_t dtype = dtype_code(g.scalar_type());
    void* const gp = g.data_ptr();
    const bool g_dense = as_it_lies(g);
    const bool same = &g == &o || (o.data_ptr() == gp && o.dtype() == g.dtype() && o.strides() == g.strides() &&
                                   o.is_neg() == g.is_neg());
    void* const op = same ? gp : o.data_ptr();
    const int32_t out_dtype = same ? dtype : dtype_code(o.scalar_type());
    const bool o_dense = same ? g_dense : as_it_lies(o);
    if (size) {
      const uintptr_t gb = reinterpret_cast<uintptr_t>(gp), ob = reinterpret_cast<uintptr_t>(op);
      if (o_dense) spans.push_back({ob, ob + size * o.element_size(), index, true});
      else scattered.push_back(reach_of(o, index));
      if (!same && g_dense) spans.push_back({gb, gb + size * g.element_size(), index, false});
    }
    if (g_dense && o_dense && ((g.is_contiguous() && o.is_contiguous()) || g.strides() == o.strides())) {
      arrays.add(gp, op, size, dtype, out_dtype);
    } else {
      arrays.add(nullptr, nullptr, size, dtype, out_dtype);
      copy_back.emplace_back(i, at::Tensor());
    }
  }
  check_overlap(spans, scattered);
  if (error_if_nonfinite) {
    const at::Tensor probe = norm_of(grads);
    double norm = 0.0;
    {
      const py::gil_scoped_release other_threads_run;  // while this one waits for the device
      norm = probe.item<double>();
    }
    if (!std::isfinite(norm))
      runtime_error("the gradients' norm is " + std::to_string(norm) +
                    "; nothing was clipped. Pass error_if_nonfinite=False to clip all the same");
  }
  for (auto& [i, d] : copy_back) {
    held.push_back(dense_copy(*grads[i]));
    d = at::empty(outs[i]->sizes(), outs[i]->options(), at::MemoryFormat::Contiguous);
    arrays.grads[i] = held.back().data_ptr();
    arrays.outs[i] = d.data_ptr();
  }
  at::Tensor norm = at::empty({}, grads[0]->options().dtype(at::kFloat));
  fssim_grad_clip_args& a = arrays.fill(static_cast<float>(max_norm), norm.data_ptr<float>());
  at::Tensor ws = workspace(a.workspace_bytes, *grads[0]);
  a.workspace = ws.data_ptr();
  // the kernels write past autograd's sight: a graph that saved an output has to notice
  for (const at::Tensor* o : outs) o->unsafeGetTensorImpl()->bump_version();
  check_status(fssim_grad_clip(&a, current_stream()));
  for (auto& [i, d] : copy_back) outs[i]->copy_(d);
  return norm;
}

void check_max_norm(double max_norm) {
  if (!(max_norm >= 0.0)) value_error("max_norm must not be negative, got " + std::to_string(max_norm));
}

at::Tensor grad_norm(const py::list& list) {
  const Refs grads = refs_of(list, "gradients");
  check_grads(grads, "grad_norm");
  return grads.empty() ? zero_norm() : norm_of(grads);
}

std::tuple<py::list, at::Tensor> clip_grad_norm(const py::list& list, double max_norm,
                                                const std::optional<py::list>& out, bool error_if_nonfinite) {
  check_max_norm(max_norm);
  if (out.has_value() && out->size() != list.size())
    value_error("out must have a tensor for each gradient, got " + std::to_string(out->size()) + " for " +
                std::to_string(list.size()));
  const Refs grads = refs_of(list, "gradients");
  check_grads(grads, "clip_grad_norm");
  if (grads.empty()) return {py::list(), zero_norm()};
  py::list result;
  if (out.has_value()) {
    result = *out;
  } else {
    for (const at::Tensor* g : grads)
      result.append(py::cast(at::empty_like(*g, g->options().requires_grad(false))));
  }
  const Refs outs = refs_of(result, "outputs");
  for (size_t i = 0; i < outs.size() && out.has_value(); ++i) {
    const at::Tensor &g = *grads[i], &o = *outs[i];
    const auto name = [&] { return "out[" + std::to_string(i) + "]"; };
    if (o.sizes() != g.sizes()) value_error(name() + " must have shape " + shape_text(g) + ", got " + shape_text(o));
    if (o.scalar_type() != g.scalar_type() && o.scalar_type() != at::kFloat)
      value_error(name() + " must be " + type_text(g.scalar_type()) + " or float32, got " +
                  type_text(o.scalar_type()));
    if (o.device() != g.device() || o.layout() != at::kStrided)
      runtime_error(name() + " must be a dense tensor on " + g.device().str());
  }
  at::Tensor norm = clip_into(grads, outs, max_norm, error_if_nonfinite);
  return {std::move(result), norm};
}

at::Tensor clip_grad_norm_(const py::list& parameters, double max_norm, bool error_if_nonfinite) {
  check_max_norm(max_norm);
  Refs grads;
  std::vector<at::Tensor> held;  // another thread may drop a parameter's gradient during the wait
  grads.reserve(parameters.size());
  if (error_if_nonfinite) held.reserve(parameters.size());
  for (size_t i = 0; i < parameters.size(); ++i) {
    const at::Tensor& g = tensor_of(PyList_GET_ITEM(parameters.ptr(), i), "parameters", i).grad();
    if (!g.defined()) continue;
    if (error_if_nonfinite) held.push_back(g);
    grads.push_back(error_if_nonfinite ? &held.back() : &g);
  }
  check_grads(grads, "clip_grad_norm_");
  return grads.empty() ? zero_norm() : clip_into(grads, grads, max_norm, error_if_nonfinite);
}

}  // namespace

void bind_training(py::module& m) {
  m.def("group_norm_act", &group_norm_act, py::arg("x"), py::arg("num_groups"), py::arg("weight"),
        py::arg("bias"), py::arg("eps"), py::arg("activation"));
  m.def("check_norm_settings", &check_norm_settings, py::arg("num_groups"), py::arg("num_channels"),
        py::arg("eps"), py::arg("activation"));
  m.def("grad_norm", &grad_norm, py::arg("grads"));
  m.def("clip_grad_norm", &clip_grad_norm, py::arg("grads"), py::arg("max_norm"), py::arg("out"),
        py::arg("error_if_nonfinite"));
  m.def("clip_grad_norm_", &clip_grad_norm_, py::arg("parameters"), py::arg("max_norm"),
        py::arg("error_if_nonfinite"));
}
