// Torch binding of the AdamW step over the C ABI. It launches on torch's current CUDA stream of the
// tensors' device; what it allocates (the gradients' norm, copies of gradients of other strides)
// comes from torch's caching allocator.
#include "torch_training.h"

#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <variant>
#include <vector>

using namespace fssim_torch;

namespace {

constexpr int64_t kBlock = 256;  // numbers of an 8-bit moment that share a scale
using Number = std::variant<double, at::Tensor>;
using OptList = std::optional<py::list>;

bool same_order(const at::Tensor& a, const at::Tensor& b) {
  return (a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides();
}

// A device-side number: one FP32.
const float* number_at(const at::Tensor& t, const char* name, const at::Device& device) {
  if (t.numel() != 1 || t.scalar_type() != at::kFloat)
    value_error(std::string(name) + " must be one float32 number, got shape " + shape_text(t) + " of " +
                type_text(t.scalar_type()));
  if (t.device() != device || t.layout() != at::kStrided || t.is_neg())
    runtime_error(std::string(name) + " must be a dense tensor on the parameters' device.\nparameters: " +
                  device.str() + ", " + name + ": " + t.device().str());
  return t.data_ptr<float>();
}

struct Lists {
  Refs params, grads, firsts, seconds, scales, copies;
};

[[noreturn]] void wrong(const char* what, size_t i, const std::string& why) {
  value_error(std::string(what) + " at index " + std::to_string(i) + " " + why);
}

void check_lists(const Lists& l, bool has_scales, bool has_copies) {
  refuse_tracing("adamw_step_");
  const bool coded = !l.firsts.empty() && l.firsts[0]->scalar_type() == at::kFloat8_e4m3fn;
  if (coded != has_scales && !l.firsts.empty())
    value_error(coded ? "8-bit moments need their scales" : "scales go with moments of float8_e4m3fn, got " +
                                                                type_text(l.firsts[0]->scalar_type()));
  const at::ScalarType moment = coded ? at::kFloat8_e4m3fn : at::kFloat;
  for (size_t i = 0; i < l.params.size(); ++i) {
    const at::Tensor &p = *l.params[i], &g = *l.grads[i];
    const auto type = p.scalar_type();
    if (!known_type(type)) wrong("the parameter", i, "must be float32, float16 or bfloat16, got " + type_text(type));
    if (p.layout() != at::kStrided || !as_it_lies(p)) wrong("the parameter", i, "must fill its memory (dense, no view with gaps)");
    if (g.layout() != at::kStrided) wrong("the gradient", i, "must be a dense tensor");
    const auto gtype = g.scalar_type();
    if (!known_type(gtype) || (type != at::kFloat && gtype != type && gtype != at::kFloat))
      wrong("the gradient", i, "must be of the parameter's type or float32 (float16 or bfloat16 beside a float32 "
            "parameter, too), got " + type_text(gtype) + " beside " + type_text(type));
    const auto like = [&](const at::Tensor& t, const char* what, bool ordered) {
      if (t.sizes() != p.sizes()) wrong(what, i, "must have shape " + shape_text(p) + ", got " + shape_text(t));
      if (t.device() != l.params[0]->device())
        runtime_error(std::string(what) + " at index " + std::to_string(i) + " must be on the first parameter's "
                      "device.\nfirst: " + l.params[0]->device().str() + ", " + what + ": " + t.device().str());
      if (ordered && (t.layout() != at::kStrided || !as_it_lies(t) || !same_order(t, p)))
        wrong(what, i, "must be dense, with the parameter's strides");
    };
    like(p, "the parameter", false);
    like(g, "the gradient", false);
    for (const at::Tensor* t : {l.firsts[i], l.seconds[i]}) {
      const char* what = t == l.firsts[i] ? "exp_avg" : "exp_avg_sq";
      if (t->scalar_type() != moment)
        wrong(what, i, "must be " + std::string(coded ? "float8_e4m3fn, as the first" : "float32 (or all moments "
              "float8_e4m3fn)") + ", got " + type_text(t->scalar_type()));
      like(*t, what, true);
    }
    if (has_copies) {
      const at::Tensor& c = *l.copies[i];
      if (type != at::kFloat || (c.scalar_type() != at::kHalf && c.scalar_type() != at::kBFloat16))
        wrong("the copy", i, "must be float16 or bfloat16, of a float32 parameter, got " +
              type_text(c.scalar_type()) + " of " + type_text(type));
      like(c, "the copy", true);
    }
    if (coded) {
      const at::Tensor& s = *l.scales[i];
      const int64_t blocks = (p.numel() + kBlock - 1) / kBlock;
      if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != blocks || s.size(1) != 2 ||
          s.layout() != at::kStrided || !s.is_contiguous() || s.is_neg())
        wrong("scales", i, "must be contiguous float32 of shape (" + std::to_string(blocks) + ", 2), got " +
              shape_text(s) + " of " + type_text(s.scalar_type()));
      if (s.device() != l.params[0]->device()) runtime_error("scales must be on the parameters' device");
    }
  }
  require_cuda("adamw_step_");
  if (!l.params.empty() && !l.params[0]->is_cuda())
    runtime_error("parameters must be on a CUDA device, but got device: " + l.params[0]->device().str());
}

double host_number(const Number& n) { return std::holds_alternative<double>(n) ? std::get<double>(n) : 0.0; }

// A step that is ready: checked, the norm and the copies of gradients on their way, and no tensor of the
// caller's written. The lists keep the tensors alive.
struct Step {
  std::vector<py::list> lists;
  Lists l;
  std::vector<at::Tensor> held;  // numbers on the device; gradients in their parameter's order
  std::vector<const void*> g_at;
  std::vector<void*> p_at, m_at, v_at, c_at;
  std::vector<float*> s_at;
  std::vector<int64_t> sizes;
  std::vector<int32_t> dtypes, g_dtypes, c_dtypes;
  fssim_adamw_args a{};
  std::optional<at::Tensor> norm;
  std::optional<at::Device> device;

  Step(const py::list& params, const py::list& grads, const py::list& exp_avgs, const py::list& exp_avg_sqs,
       const OptList& scales, const Number& step, const Number& lr, double beta1, double beta2, double eps,
       double weight_decay, bool maximize, std::optional<double> max_norm, const OptTensor& norm_in,
       const OptList& copies, int64_t seed);
  Step(const Step&) = delete;  // (the arguments point into it)
  // Once: writes the tensors.
  std::optional<at::Tensor> run();
};

Step::Step(const py::list& params, const py::list& grads, const py::list& exp_avgs, const py::list& exp_avg_sqs,
           const OptList& scales, const Number& step, const Number& lr, double beta1, double beta2, double eps,
           double weight_decay, bool maximize, std::optional<double> max_norm, const OptTensor& norm_in,
           const OptList& copies, int64_t seed) {
  const size_t n = params.size();
  const auto sized = [&](const py::list& list, const char* name) {
    if (list.size() != n)
      value_error(std::string(name) + " must have a tensor for each parameter, got " + std::to_string(list.size()) +
                  " for " + std::to_string(n));
  };
  sized(grads, "grads");
  sized(exp_avgs, "exp_avgs");
  sized(exp_avg_sqs, "exp_avg_sqs");
  if (scales.has_value()) sized(*scales, "scales");
  if (copies.has_value()) sized(*copies, "copies");
  const auto finite = [](double v, const char* name) {
    if (!(v >= 0.0 && std::isfinite(v)))
      value_error(std::string(name) + " must be finite and not negative, got " + std::to_string(v));
  };
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
    value_error("betas must be at least 0 and below 1, got (" + std::to_string(beta1) + ", " + std::to_string(beta2) + ")");
  finite(eps, "eps");
  finite(weight_decay, "weight_decay");
  finite(host_number(lr), "lr");
  const double t = host_number(step);
  if (std::holds_alternative<double>(step) && !(t >= 1.0 && t == std::floor(t) && t < 0x1p53))
    value_error("step must be a whole number from 1 up, got " + std::to_string(t));
  if (max_norm.has_value() && !(*max_norm >= 0.0))
    value_error("max_norm must not be negative, got " + std::to_string(*max_norm));
  if (norm_in.has_value() && !max_norm.has_value()) value_error("norm goes with max_norm");
  if (seed < 0 || seed > 0xFFFFFFFF) value_error("seed must be from 0 to 2^32 - 1, got " + std::to_string(seed));
  l = {refs_of(params, "parameters"), refs_of(grads, "gradients"), refs_of(exp_avgs, "exp_avgs"),
       refs_of(exp_avg_sqs, "exp_avg_sqs"), scales.has_value() ? refs_of(*scales, "scales") : Refs(),
       copies.has_value() ? refs_of(*copies, "copies") : Refs()};
  check_lists(l, scales.has_value(), copies.has_value());
  if (n == 0) {
    if (max_norm.has_value()) norm = norm_in.has_value() ? *norm_in : zero_norm();
    return;
  }
  lists = {params, grads, exp_avgs, exp_avg_sqs};
  if (scales.has_value()) lists.push_back(*scales);
  if (copies.has_value()) lists.push_back(*copies);

  const at::NoGradGuard no_grad;
  device = l.params[0]->device();
  const at::cuda::OptionalCUDAGuard guard(device);
  a.count = static_cast<int64_t>(n);
  a.state_bits = scales.has_value() ? 8 : 32;
  a.maximize = maximize;
  a.seed = static_cast<uint32_t>(seed);
  a.step = static_cast<int64_t>(t);
  a.lr = host_number(lr);
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.max_norm = max_norm.value_or(0.0);
  std::vector<Span> spans;
  spans.reserve(6 * n + 3);
  const auto span = [&](const void* p, int64_t bytes, size_t i, bool out) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(p);
    if (bytes) spans.push_back({b, b + bytes, static_cast<int64_t>(i), out});
  };
  const auto number = [&](const at::Tensor& v, const char* name) {
    const float* p = number_at(v, name, *device);
    span(p, 4, 0, false);
    held.push_back(v);
    return p;
  };
  if (std::holds_alternative<at::Tensor>(step)) a.step_at = number(std::get<at::Tensor>(step), "step");
  if (std::holds_alternative<at::Tensor>(lr)) a.lr_at = number(std::get<at::Tensor>(lr), "lr");
  if (norm_in.has_value()) a.norm = number(*norm_in, "norm");

  // Each list's tensors, in the order in which they commonly lie in memory.
  g_at.resize(n);
  for (auto* at : {&p_at, &m_at, &v_at, &c_at}) at->resize(n);
  s_at.resize(n);
  sizes.resize(n);
  for (auto* codes : {&dtypes, &g_dtypes, &c_dtypes}) codes->resize(n);
  const auto pointers = [&](const Refs& refs, auto& at) {
    for (size_t i = 0; i < refs.size(); ++i) {
      at[i] = static_cast<std::decay_t<decltype(at[i])>>(refs[i]->data_ptr());
      span(at[i], refs[i]->numel() * refs[i]->element_size(), i, true);
    }
  };
  pointers(l.params, p_at);
  pointers(l.firsts, m_at);
  pointers(l.seconds, v_at);
  pointers(l.scales, s_at);
  pointers(l.copies, c_at);
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = *l.params[i], &g = *l.grads[i];
    sizes[i] = p.numel();
    dtypes[i] = dtype_code(p.scalar_type());
    g_dtypes[i] = dtype_code(g.scalar_type());
    if (copies.has_value()) c_dtypes[i] = dtype_code(l.copies[i]->scalar_type());
    if (as_it_lies(g) && same_order(g, p)) {
      g_at[i] = g.data_ptr();
      span(g_at[i], g.numel() * g.element_size(), i, false);
    } else {
      g_at[i] = nullptr;
    }
  }
  check_spans(spans);
  if (max_norm.has_value()) {
    norm = norm_in.has_value() ? *norm_in : norm_of(l.grads);
    a.norm = norm->data_ptr<float>();
  }
  for (size_t i = 0; i < n; ++i)
    if (!g_at[i]) {
      held.push_back(at::empty_strided(l.params[i]->sizes(), l.params[i]->strides(), l.grads[i]->options()).copy_(*l.grads[i]));
      g_at[i] = held.back().data_ptr();
    }
  a.params = p_at.data();
  a.grads = g_at.data();
  a.exp_avgs = m_at.data();
  a.exp_avg_sqs = v_at.data();
  a.scales = s_at.data();
  a.copies = copies.has_value() ? c_at.data() : nullptr;
  a.sizes = sizes.data();
  a.dtypes = dtypes.data();
  a.grad_dtypes = g_dtypes.data();
  a.copy_dtypes = c_dtypes.data();
}

std::optional<at::Tensor> Step::run() {
  if (a.count == 0) return norm;
  if (lists.empty()) runtime_error("a step runs once");
  const at::cuda::OptionalCUDAGuard guard(device);
  // the kernel writes past autograd's sight: a graph that saved a tensor has to notice
  for (const Refs* refs : {&l.params, &l.firsts, &l.seconds, &l.scales, &l.copies})
    for (const at::Tensor* o : *refs) o->unsafeGetTensorImpl()->bump_version();
  check_status(fssim_adamw_step(&a, current_stream()));
  lists.clear();
  held.clear();
  return norm;
}

std::optional<at::Tensor> adamw_step_(const py::list& params, const py::list& grads, const py::list& exp_avgs,
                                      const py::list& exp_avg_sqs, const OptList& scales, const Number& step,
                                      const Number& lr, double beta1, double beta2, double eps, double weight_decay,
                                      bool maximize, std::optional<double> max_norm, const OptTensor& norm_in,
                                      const OptList& copies, int64_t seed) {
  return Step(params, grads, exp_avgs, exp_avg_sqs, scales, step, lr, beta1, beta2, eps, weight_decay, maximize,
              max_norm, norm_in, copies, seed)
      .run();
}

}  // namespace

void bind_adamw(py::module& m) {
  m.def("adamw_step_", &adamw_step_, py::arg("params"), py::arg("grads"), py::arg("exp_avgs"),
        py::arg("exp_avg_sqs"), py::arg("scales"), py::arg("step"), py::arg("lr"), py::arg("beta1"),
        py::arg("beta2"), py::arg("eps"), py::arg("weight_decay"), py::arg("maximize"), py::arg("max_norm"),
        py::arg("norm"), py::arg("copies"), py::arg("seed"));
  py::class_<Step>(m, "AdamWStep", "A checked step of adamw_step_'s arguments, which run() takes once")
      .def(py::init<const py::list&, const py::list&, const py::list&, const py::list&, const OptList&, const Number&,
                    const Number&, double, double, double, double, bool, std::optional<double>, const OptTensor&,
                    const OptList&, int64_t>())
      .def("run", &Step::run);
}
