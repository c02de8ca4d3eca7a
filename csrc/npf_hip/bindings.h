// Helpers of the binding files, and what each of them adds to npf._hip_C.
#pragma once

#include <ATen/TracerMode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <hip/hip_runtime.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "type_codes.h"

void npf_bind_norms(pybind11::module_& m);      // ext_norms.cpp
void npf_bind_diff_attn(pybind11::module_& m);  // ext_diff_attn.cpp

// a kernel's code for the type, or an error that names the argument
inline int npf_type_code(const torch::Tensor& t, const char* name,
                         bool f64 = false) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return NPF_F32;
    case torch::kBFloat16: return NPF_BF16;
    case torch::kFloat16: return NPF_F16;
    case torch::kFloat64:
      if (f64) return NPF_F64;
      [[fallthrough]];
    default:
      TORCH_CHECK_TYPE(false, name, " has type ", t.scalar_type(),
                       ", which the kernel does not take");
  }
}

// The operators read and write memory themselves, past torch's dispatcher.  What
// it would do for a call is refused rather than left out: recording it in a
// trace (which would hold the first call's result as a constant) ...
inline void npf_check_call(const char* op) {
  using c10::impl::TorchDispatchModeKey;
  TORCH_CHECK_NOT_IMPLEMENTED(
      !at::tracer::impl::is_dispatch_enabled() &&
          !c10::impl::TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY)
               .has_value(),
      op, " cannot be traced; NPF_DISABLE_OPS=", op,
      " chooses the composed form");
}

// ... and what a tensor holds outside of its memory: a forward-mode tangent, or
// all of a wrapper (of vmap, of a fake tensor) that has no memory of its own.
inline void npf_check_plain(const torch::Tensor& t, const char* op) {
  if (!t.defined()) return;
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrappers(
      {DispatchKey::Python, DispatchKey::FuncTorchBatched,
       DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize,
       DispatchKey::Batched});
  TORCH_CHECK_NOT_IMPLEMENTED(!t.key_set().has_any(wrappers), op,
                              " takes no tensor that wraps another");
  TORCH_CHECK_NOT_IMPLEMENTED(
      !t._fw_grad(/*level=*/0).defined(), op,
      " has no forward-mode derivative; NPF_DISABLE_OPS=", op,
      " chooses the composed form");
}

// Memory holds the values of a negated view (the imaginary part of a conjugate)
// with the other sign, and there is none of a gradient that torch knows to be
// zero.
inline torch::Tensor npf_signed(const torch::Tensor& t) {
  if (!t.defined()) return t;
  if (t._is_zerotensor()) return torch::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

// Contiguous memory beside `on`, from the allocator itself: torch::empty's way
// there through the dispatcher takes longer than a launch (a layer norm with
// its gradients makes 6 such calls: 67 us of host time, with torch::empty 70).
inline torch::Tensor npf_empty(at::IntArrayRef sizes, at::ScalarType type,
                               const torch::Tensor& on) {
  return torch::Tensor(
      at::detail::empty_cuda(sizes, type, on.device(), std::nullopt));
}

// What a forward pass saved may come back through the program's own hooks
// (offloading, compression): it has to be what the kernels read.
inline void npf_check_saved(const torch::Tensor& t, const torch::Tensor& like,
                            at::ScalarType type, at::IntArrayRef sizes,
                            const char* op) {
  TORCH_CHECK_VALUE(t.defined() && t.device() == like.device() &&
                        t.layout() == torch::kStrided &&
                        t.scalar_type() == type && t.sizes() == sizes &&
                        !t.is_neg() && !t._is_zerotensor(),
                    op, ": a saved tensor came back changed");
  npf_check_plain(t, op);
}

inline void npf_check(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

// Gradients of an operator that is differentiable once: where a graph is built
// over its backward pass, a second derivative is an error rather than zero.
inline torch::autograd::variable_list npf_once(
    torch::autograd::variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list some;
  for (const auto& g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_());
  if (some.empty()) return grads;
  const int64_t n = (int64_t)some.size();
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is differentiable once", n);
  some = (*error)(std::move(some));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = some[i++];
  return grads;
}
