// Torch binding of the residual-block norms over the C ABI, as a C++ autograd function. Everything
// launches on torch's current CUDA stream of the tensors' device; workspaces are allocated by the
// call from torch's caching allocator.
#include "torch_training.h"

#include <c10/cuda/CUDAGuard.h>

#include <array>
#include <cmath>
#include <string>

using namespace fssim_torch;

namespace {

// The vectors of C numbers, in the order in which the autograd function takes them.
enum Vector { kGate, kWeight, kBias, kScale, kShift, kBranchWeight, kBranchBias, kVectors };
constexpr const char* kNames[kVectors] = {"gate", "weight", "bias", "scale", "shift", "branch_weight", "branch_bias"};
using Vectors = std::array<at::Tensor, kVectors>;  // undefined where there is none

struct Settings {
  int64_t kind, branch_kind;
  double residual_scale, eps;
  bool norm;                 // z is wanted
  at::ScalarType out_dtype;  // z's
};

int64_t kind_code(const std::optional<std::string>& name, const char* what, bool none) {
  if (!name.has_value() && none) return FSSIM_NORM_NONE;
  if (name.has_value() && *name == "rms") return FSSIM_NORM_RMS;
  if (name.has_value() && *name == "layer") return FSSIM_NORM_LAYER;
  value_error(std::string(what) + " must be " + (none ? "None, " : "") + "'rms' or 'layer', got " +
              (name.has_value() ? "'" + *name + "'" : "None"));
}

bool per_sample(const at::Tensor& t) { return t.defined() && t.dim() == 2; }
fssim_channels channels(const at::Tensor& t) {
  fssim_channels c{};
  if (!t.defined()) return c;
  c.data = t.const_data_ptr();
  if (!c.data && t.numel()) runtime_error("vectors must be tensors with memory (not fake ones)");
  c.dtype = dtype_code(t.scalar_type());
  c.per_sample = per_sample(t);
  return c;
}
fssim_channels_grad channels_grad(const at::Tensor& t) {
  fssim_channels_grad c{};
  if (!t.defined()) return c;
  c.data = t.data_ptr();
  c.dtype = dtype_code(t.scalar_type());
  c.per_sample = per_sample(t);
  return c;
}

// B samples of T rows: the first dimension, and those between it and the last.
template <typename Args>
void set_shape(Args& a, const at::Tensor& x, at::ScalarType x_type, at::ScalarType y) {
  a.x_dtype = dtype_code(x_type);
  a.y_dtype = dtype_code(y);
  a.C = x.size(-1);
  a.B = x.dim() > 1 ? x.size(0) : 1;
  a.T = a.B > 0 ? x.numel() / a.C / a.B : 0;
}

struct Result {
  at::Tensor r, z, stats, branch_stats;
};

// x, branch (undefined where there is none) and the vectors: dense.
Result run_forward(const at::Tensor& x, const at::Tensor& branch, const Vectors& v, const Settings& set, bool train) {
  const at::cuda::OptionalCUDAGuard guard(x.device());
  Result out;
  fssim_block_norm_forward_args a{};
  set_shape(a, x, x.scalar_type(), set.out_dtype);
  a.kind = static_cast<int32_t>(set.norm ? set.kind : FSSIM_NORM_NONE);
  a.branch_kind = static_cast<int32_t>(set.branch_kind);
  a.eps = static_cast<float>(set.eps);
  a.residual_scale = set.residual_scale;
  a.x = x.data_ptr();
  const std::array<int64_t, 3> rows = {a.B, a.T, 2};
  if (branch.defined()) {
    out.r = at::empty(x.sizes(), x.options());
    a.branch = branch.data_ptr();
    a.r = out.r.data_ptr();
    if (train && set.branch_kind != FSSIM_NORM_NONE) {
      out.branch_stats = at::empty(rows, x.options().dtype(at::kFloat));
      a.branch_stats = out.branch_stats.data_ptr<float>();
    }
  }
  if (set.norm) {
    out.z = at::empty(x.sizes(), x.options().dtype(set.out_dtype));
    a.z = out.z.data_ptr();
    if (train) {
      out.stats = at::empty(rows, x.options().dtype(at::kFloat));
      a.stats = out.stats.data_ptr<float>();
    }
  }
  a.gate = channels(v[kGate]);
  a.weight = channels(v[kWeight]);
  a.bias = channels(v[kBias]);
  a.scale = channels(v[kScale]);
  a.shift = channels(v[kShift]);
  a.branch_weight = channels(v[kBranchWeight]);
  a.branch_bias = channels(v[kBranchBias]);
  check_status(fssim_block_norm_forward(&a, current_stream()));
  return out;
}

at::Tensor dense(const OptTensor& t) { return t.has_value() && t->defined() ? t->contiguous() : at::Tensor(); }

struct BlockNormFn : public torch::autograd::Function<BlockNormFn> {
  // Results: r where there is a branch, then z where it is wanted.
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, at::Tensor x, OptTensor branch,
                                                OptTensor gate, OptTensor weight, OptTensor bias, OptTensor scale,
                                                OptTensor shift, OptTensor branch_weight, OptTensor branch_bias,
                                                const Settings& set) {
    const at::Tensor rows = x.contiguous(), y = dense(branch);
    const Vectors v = {dense(gate),  dense(weight),        dense(bias),       dense(scale),
                       dense(shift), dense(branch_weight), dense(branch_bias)};
    const Result out = run_forward(rows, y, v, set, true);
    // without a branch r is x itself; without a norm of it the backward has no use for it
    torch::autograd::variable_list saved = {!set.norm ? at::Tensor() : y.defined() ? out.r : rows, y, out.stats,
                                            out.branch_stats};
    saved.insert(saved.end(), v.begin(), v.end());
    ctx->save_for_backward(std::move(saved));
    ctx->set_materialize_grads(false);
    if (!set.norm) ctx->saved_data["x_dtype"] = static_cast<int64_t>(rows.scalar_type());
    ctx->saved_data["kind"] = set.kind;
    ctx->saved_data["branch_kind"] = set.branch_kind;
    ctx->saved_data["residual_scale"] = set.residual_scale;
    ctx->saved_data["out_dtype"] = static_cast<int64_t>(set.out_dtype);
    ctx->saved_data["norm"] = set.norm;
    torch::autograd::variable_list results;
    if (y.defined()) results.push_back(out.r);
    if (set.norm) results.push_back(out.z);
    return results;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the block norms are differentiable once: their backward cannot be recorded (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &r = saved[0], &y = saved[1], &stats = saved[2], &branch_stats = saved[3];
    Vectors v;
    std::copy(saved.begin() + 4, saved.end(), v.begin());
    const auto x_dtype = r.defined() ? r.scalar_type() : static_cast<at::ScalarType>(ctx->saved_data["x_dtype"].toInt());
    const auto out_dtype = static_cast<at::ScalarType>(ctx->saved_data["out_dtype"].toInt());
    const at::Tensor& like = r.defined() ? r : y;  // of x's shape
    // the gradient slots of the inputs that are tensors, in their order
    size_t slot = 0;
    const auto needed = [&](const at::Tensor& t) { return t.defined() && ctx->needs_input_grad(slot++); };
    const bool need_x = needed(like), need_y = needed(y);
    std::array<bool, kVectors> need;
    for (int i = 0; i < kVectors; ++i) need[i] = needed(v[i]);
    const at::cuda::OptionalCUDAGuard guard(like.device());
    const auto rows_of = [&](size_t i, at::ScalarType type) {
      return grads[i].defined() ? resolved(grads[i]).to(type).contiguous() : at::Tensor();
    };
    at::Tensor dr, dz;
    size_t output = 0;
    if (y.defined()) dr = rows_of(output++, x_dtype);
    if (ctx->saved_data["norm"].toBool()) dz = rows_of(output++, out_dtype);
    torch::autograd::variable_list result(10);  // the settings have none
    if (!dr.defined() && !dz.defined()) return result;
    at::Tensor& dx = result[0];
    at::Tensor& dy = result[1];
    // with no row, or no gradient that reaches a vector, its sums are zero
    const auto make = [&](const at::Tensor& t, at::ScalarType type, bool reached) {
      const auto options = t.options().dtype(type);
      return like.numel() && reached ? at::empty(t.sizes(), options) : at::zeros(t.sizes(), options);
    };
    if (need_x) dx = make(like, x_dtype, true);
    if (need_y) dy = make(y, out_dtype, true);
    for (int i = 0; i < kVectors; ++i)
      if (need[i]) result[2 + i] = make(v[i], v[i].scalar_type(), dz.defined() || i == kGate || i == kBranchWeight || i == kBranchBias);
    fssim_block_norm_backward_args a{};
    set_shape(a, like, x_dtype, out_dtype);
    a.kind = static_cast<int32_t>(ctx->saved_data["kind"].toInt());
    a.branch_kind = static_cast<int32_t>(ctx->saved_data["branch_kind"].toInt());
    a.residual_scale = ctx->saved_data["residual_scale"].toDouble();
    const auto at = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    a.r = at(r);
    a.branch = at(y);
    a.dr = at(dr);
    a.dz = at(dz);
    a.stats = static_cast<const float*>(at(stats));
    a.branch_stats = static_cast<const float*>(at(branch_stats));
    a.gate = channels(v[kGate]);
    a.weight = channels(v[kWeight]);
    a.bias = channels(v[kBias]);
    a.scale = channels(v[kScale]);
    a.branch_weight = channels(v[kBranchWeight]);
    a.branch_bias = channels(v[kBranchBias]);
    a.dx = at(dx);
    a.dbranch = at(dy);
    a.dgate = channels_grad(result[2 + kGate]);
    a.dbranch_weight = channels_grad(result[2 + kBranchWeight]);
    a.dbranch_bias = channels_grad(result[2 + kBranchBias]);
    if (dz.defined()) {
      a.dweight = channels_grad(result[2 + kWeight]);
      a.dbias = channels_grad(result[2 + kBias]);
      a.dscale = channels_grad(result[2 + kScale]);
      a.dshift = channels_grad(result[2 + kShift]);
    }
    a.workspace_bytes = fssim_block_norm_backward_workspace_bytes(&a);
    at::Tensor ws;
    if (a.workspace_bytes) {
      ws = workspace(a.workspace_bytes, like);
      a.workspace = ws.data_ptr();
    }
    check_status(fssim_block_norm_backward(&a, current_stream()));
    return result;
  }
};

// Checks, then the operator: recorded for autograd where a gradient may be asked for.
torch::autograd::variable_list block_norm(const char* what, const at::Tensor& given_x, const OptTensor& given_branch,
                                          std::array<OptTensor, kVectors> v, Settings set,
                                          const std::optional<at::ScalarType>& out_dtype) {
  const at::Tensor x = resolved(given_x);
  const OptTensor branch = resolved(given_branch);
  for (OptTensor& t : v) t = resolved(t);
  if (x.layout() != at::kStrided) value_error("x must be a dense tensor");
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 16384)
    value_error("x must have at least one dimension, and 1 to 16384 numbers in its last, got shape " + shape_text(x));
  if (!known_type(x.scalar_type()))
    value_error("x must be float32, float16 or bfloat16, got " + type_text(x.scalar_type()));
  if (!(set.eps >= 0.0 && std::isfinite(set.eps)))
    value_error("eps must be finite and not negative, got " + std::to_string(set.eps));
  if (!std::isfinite(static_cast<float>(set.residual_scale)))
    value_error("residual_scale must be finite in float32, got " + std::to_string(set.residual_scale));
  refuse_tracing(what);
  refuse_tangent(x, "x", what);
  bool train = x.requires_grad();
  set.out_dtype = out_dtype.value_or(x.scalar_type());
  if (branch.has_value()) {
    if (branch->sizes() != x.sizes())
      value_error("branch must have x's shape " + shape_text(x) + ", got " + shape_text(*branch));
    if (branch->layout() != at::kStrided) value_error("branch must be a dense tensor");
    if (branch->device() != x.device())
      runtime_error("branch must be on x's device.\nx: " + x.device().str() + ", branch: " + branch->device().str());
    refuse_tangent(*branch, "branch", what);
    set.out_dtype = branch->scalar_type();
    train = train || branch->requires_grad();
  }
  if (!known_type(set.out_dtype) || (x.scalar_type() != at::kFloat && set.out_dtype != x.scalar_type()))
    value_error(std::string(branch.has_value() ? "branch" : "out_dtype") + " must be of x's type" +
                (x.scalar_type() == at::kFloat ? ", float16 or bfloat16" : "") + ", got " + type_text(set.out_dtype));
  const int64_t C = x.size(-1);
  for (int i = 0; i < kVectors; ++i) {
    if (!v[i].has_value()) continue;
    const at::Tensor& t = *v[i];
    const std::string name = kNames[i];
    const bool samples = i == kGate || i == kScale || i == kShift;
    if (!(t.dim() == 1 && t.size(0) == C) &&
        !(samples && t.dim() == 2 && x.dim() > 1 && t.size(0) == x.size(0) && t.size(1) == C))
      value_error(name + " must have shape (" + std::to_string(C) + ",)" +
                  (samples && x.dim() > 1 ? " or (" + std::to_string(x.size(0)) + ", " + std::to_string(C) + ")" : "") +
                  ", got " + shape_text(t));
    if (!known_type(t.scalar_type()))
      value_error(name + " must be float32, float16 or bfloat16, got " + type_text(t.scalar_type()));
    if (t.layout() != at::kStrided) value_error(name + " must be a dense tensor");
    if (t.device() != x.device())
      runtime_error(name + " must be on x's device.\nx: " + x.device().str() + ", " + name + ": " + t.device().str());
    refuse_tangent(t, kNames[i], what);
    train = train || t.requires_grad();
  }
  if (branch.has_value() && set.branch_kind == FSSIM_NORM_NONE && (v[kBranchWeight].has_value() || v[kBranchBias].has_value()))
    value_error("branch_weight and branch_bias go with branch_kind");
  require_cuda(what);
  if (!x.is_cuda()) runtime_error("x must be on a CUDA device, but got device: " + x.device().str());
  if (train && at::GradMode::is_enabled())
    return BlockNormFn::apply(x, branch, v[kGate], v[kWeight], v[kBias], v[kScale], v[kShift], v[kBranchWeight],
                              v[kBranchBias], set);
  const at::NoGradGuard no_grad;
  Vectors d;
  for (int i = 0; i < kVectors; ++i) d[i] = dense(v[i]);
  const Result out = run_forward(x.contiguous(), dense(branch), d, set, false);
  torch::autograd::variable_list results;
  if (branch.has_value()) results.push_back(out.r);
  if (set.norm) results.push_back(out.z);
  return results;
}

at::Tensor block_norm_(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& scale,
                       const OptTensor& shift, const std::optional<std::string>& kind, double eps,
                       const std::optional<at::ScalarType>& out_dtype) {
  const Settings set{kind_code(kind, "kind", false), FSSIM_NORM_NONE, 1.0, eps, true, at::kFloat};
  return block_norm("block_norm", x, std::nullopt, {std::nullopt, weight, bias, scale, shift, std::nullopt, std::nullopt},
                    set, out_dtype)[0];
}

at::Tensor gated_residual(const at::Tensor& x, const at::Tensor& branch, const OptTensor& gate, double residual_scale,
                          const std::optional<std::string>& branch_kind, const OptTensor& branch_weight,
                          const OptTensor& branch_bias, double eps) {
  const Settings set{FSSIM_NORM_NONE, kind_code(branch_kind, "branch_kind", true), residual_scale, eps, false, at::kFloat};
  return block_norm("gated_residual", x, branch,
                    {gate, std::nullopt, std::nullopt, std::nullopt, std::nullopt, branch_weight, branch_bias}, set,
                    std::nullopt)[0];
}

std::tuple<at::Tensor, at::Tensor> gated_residual_norm(
    const at::Tensor& x, const at::Tensor& branch, const OptTensor& gate, const OptTensor& weight, const OptTensor& bias,
    const OptTensor& scale, const OptTensor& shift, const std::optional<std::string>& kind, double residual_scale,
    const std::optional<std::string>& branch_kind, const OptTensor& branch_weight, const OptTensor& branch_bias,
    double eps) {
  const Settings set{kind_code(kind, "kind", false), kind_code(branch_kind, "branch_kind", true), residual_scale, eps,
                     true, at::kFloat};
  const auto out = block_norm("gated_residual_norm", x, branch,
                              {gate, weight, bias, scale, shift, branch_weight, branch_bias}, set, std::nullopt);
  return {out[0], out[1]};
}

}  // namespace

void bind_block_norm(py::module& m) {
  m.def("block_norm", &block_norm_, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("scale"),
        py::arg("shift"), py::arg("kind"), py::arg("eps"), py::arg("out_dtype"));
  m.def("gated_residual", &gated_residual, py::arg("x"), py::arg("branch"), py::arg("gate"),
        py::arg("residual_scale"), py::arg("branch_kind"), py::arg("branch_weight"), py::arg("branch_bias"),
        py::arg("eps"));
  m.def("gated_residual_norm", &gated_residual_norm, py::arg("x"), py::arg("branch"), py::arg("gate"),
        py::arg("weight"), py::arg("bias"), py::arg("scale"), py::arg("shift"), py::arg("kind"),
        py::arg("residual_scale"), py::arg("branch_kind"), py::arg("branch_weight"), py::arg("branch_bias"),
        py::arg("eps"));
}
