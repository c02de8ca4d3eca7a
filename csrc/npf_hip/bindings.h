// Helpers of the binding files, and what each of them adds to npf._hip_C.
#pragma once

#include <hip/hip_runtime.h>
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

inline void npf_check(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}
