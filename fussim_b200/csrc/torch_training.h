// What the bindings of the training-step operators share: checks of arguments, their texts, and
// tensors as the C ABI takes them.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "fussim_b200.h"

void bind_training(py::module& m);
void bind_adamw(py::module& m);
void bind_block_norm(py::module& m);

namespace fssim_torch {

inline void check_status(int st) {
  if (st == FSSIM_OK) return;
  throw std::runtime_error(std::string("fussim_b200: ") + fssim_status_string(st) + ": " +
                           fssim_last_error());
}

inline fssim_stream_t current_stream() {
  return reinterpret_cast<fssim_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FSSIM_F32;
    case at::kHalf: return FSSIM_F16;
    case at::kBFloat16: return FSSIM_BF16;
    default: throw std::invalid_argument("unsupported dtype for fussim_b200");
  }
}

inline at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

using OptTensor = std::optional<at::Tensor>;

// A lazily negated view (the imaginary part of a conjugate) holds its numbers with the other sign.
inline at::Tensor resolved(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
inline OptTensor resolved(const OptTensor& t) { return t.has_value() ? OptTensor(resolved(*t)) : t; }

[[noreturn]] inline void value_error(const std::string& msg) { throw std::invalid_argument(msg); }
[[noreturn]] inline void runtime_error(const std::string& msg) { throw std::runtime_error(msg); }

inline std::string shape_text(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}
inline std::string type_text(at::ScalarType t) { return std::string(c10::toString(t)); }
inline bool known_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

inline void require_cuda(const char* what) {
  if (!at::hasCUDA() || at::cuda::device_count() == 0)
    runtime_error(std::string("CUDA is not available. ") + what + " requires a CUDA-capable GPU.");
}

// A tracer records the operators that torch dispatches: of a call here it would keep the allocation
// of the result and not the launches.
inline void refuse_tracing(const char* what) {
  using Key = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(Key::PROXY).has_value())
    runtime_error(std::string(what) + " cannot be traced (torch.jit.trace, make_fx, torch.export): its kernels "
                  "are launched outside torch's dispatcher");
}

// Nor is there a forward-mode derivative: a result without a tangent would stand for a zero one.
inline void refuse_tangent(const at::Tensor& t, const char* name, const char* what) {
  if (t._fw_grad(/*level=*/0).defined())
    runtime_error(std::string(what) + " has no forward-mode derivative, but " + name + " carries a tangent");
}

// Models have hundreds of gradients and a call's device time is tens of microseconds, so the
// tensors are read where the caller's list holds them (no copies of their handles) and in one pass.
using Refs = std::vector<const at::Tensor*>;

inline const at::Tensor& tensor_of(py::handle h, const char* what, size_t index) {
  if (!THPVariable_Check(h.ptr()))
    throw py::type_error(std::string(what) + " must be tensors, but that at index " + std::to_string(index) +
                         " is not");
  return THPVariable_Unpack(h.ptr());
}

inline Refs refs_of(const py::list& list, const char* what) {
  Refs refs;
  refs.reserve(list.size());
  for (size_t i = 0; i < list.size(); ++i) refs.push_back(&tensor_of(PyList_GET_ITEM(list.ptr(), i), what, i));
  return refs;
}

// Tensors whose numbers fill their memory are taken as they lie; others, and lazily negated views, go
// through a dense copy.
inline bool as_it_lies(const at::Tensor& t) { return t.is_non_overlapping_and_dense() && !t.is_neg(); }
inline at::Tensor dense_copy(const at::Tensor& t) { return resolved(t).contiguous(); }

// The memory of a tensor, and where the tensor stands in the call.
struct Span {
  uintptr_t begin, end;
  int64_t index;
  bool out;
};

// Refuses dense tensors that are written (out) and overlap another.
void check_spans(std::vector<Span>& spans);
// The tensors fit the gradients' operators (`what`), and are on the GPU.
void check_grads(const Refs& grads, const char* what);
// Their norm, a 0-d FP32 tensor; of none: zero.
at::Tensor norm_of(const Refs& grads);
at::Tensor zero_norm();

}  // namespace fssim_torch
