// Bindings of layer norm and of gradient norm and clipping.

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <limits>

#include "bindings.h"
#include "grad_norm.h"
#include "layernorm.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

void* ptr_of(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

void check_rows(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.sizes() == like.sizes(), name,
                    " must have the shape ", like.sizes(), ", has ",
                    t.sizes());
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " must be on ",
                    like.device());
  TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type(), name,
                   " must have type ", like.scalar_type());
  TORCH_CHECK_VALUE(t.size(1) < 2 || t.stride(1) == 1, name,
                    " must have contiguous rows");
}

void check_columns(const OptTensor& t, const Tensor& x, const char* name) {
  if (!t) return;
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(1) &&
                        t->is_contiguous() && t->device() == x.device(),
                    name, " must be a contiguous [", x.size(1), "] on ",
                    x.device());
}

NpfLayerNormArgs norm_args(const Tensor& x, const OptTensor& residual,
                           const OptTensor& weight, const OptTensor& bias) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && x.size(1) > 0,
                    "layer_norm takes rows of at least one value on a GPU");
  TORCH_CHECK_VALUE(x.size(1) <= std::numeric_limits<int>::max(),
                    "layer_norm: rows are too wide");
  check_rows(x, x, "x");
  if (residual) check_rows(*residual, x, "residual");
  check_columns(weight, x, "weight");
  check_columns(bias, x, "bias");
  TORCH_CHECK_TYPE(!weight || !bias ||
                       weight->scalar_type() == bias->scalar_type(),
                   "weight and bias must have the same type");
  NpfLayerNormArgs a{};
  a.x = x.data_ptr();
  a.residual = ptr_of(residual);
  a.weight = ptr_of(weight);
  a.bias = ptr_of(bias);
  a.x_stride = x.stride(0);
  a.residual_stride = residual ? residual->stride(0) : 0;
  a.rows = x.size(0);
  a.width = (int)x.size(1);
  const OptTensor& w = weight ? weight : bias;
  a.weight_type = w ? npf_type_code(*w, "weight", true) : (int)NPF_F32;
  return a;
}

// (y, mean, rstd); the last two are empty unless `save`
std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(
    const Tensor& x, const OptTensor& residual, const OptTensor& weight,
    const OptTensor& bias, double eps, bool save) {
  NpfLayerNormArgs a = norm_args(x, residual, weight, bias);
  const int type = npf_type_code(x, "x");
  c10::DeviceGuard guard(x.device());
  Tensor y = torch::empty({x.size(0), x.size(1)}, x.options());
  auto f32 = x.options().dtype(torch::kFloat32);
  Tensor mean = torch::empty({save ? x.size(0) : 0}, f32);
  Tensor rstd = torch::empty({save ? x.size(0) : 0}, f32);
  if (a.rows == 0) return {y, mean, rstd};
  a.y = y.data_ptr();
  a.mean = save ? mean.data_ptr<float>() : nullptr;
  a.rstd = save ? rstd.data_ptr<float>() : nullptr;
  a.eps = (float)eps;
  npf_check(npf_layernorm_fwd(a, type, at::hip::getCurrentHIPStream()),
            "layer_norm");
  return {y, mean, rstd};
}

// (dx, dweight, dbias); those that are not asked for are None
std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_bwd(
    const Tensor& dy, const Tensor& x, const OptTensor& residual,
    const OptTensor& weight, const OptTensor& bias, const Tensor& mean,
    const Tensor& rstd, bool need_dx, bool need_dweight, bool need_dbias) {
  NpfLayerNormArgs a = norm_args(x, residual, weight, bias);
  const int type = npf_type_code(x, "x");
  check_rows(dy, x, "dy");
  TORCH_CHECK_VALUE(dy.is_contiguous(), "dy must be contiguous");
  TORCH_CHECK_VALUE(mean.numel() == x.size(0) && rstd.numel() == x.size(0),
                    "mean and rstd must hold one value a row");
  need_dweight = need_dweight && weight;
  need_dbias = need_dbias && bias;
  c10::DeviceGuard guard(x.device());
  OptTensor dx, dweight, dbias, partial;
  if (need_dx) dx = torch::empty({x.size(0), x.size(1)}, x.options());
  if (a.rows == 0) {
    if (need_dweight) dweight = torch::zeros_like(*weight);
    if (need_dbias) dbias = torch::zeros_like(*bias);
    return {dx, dweight, dbias};
  }
  if (need_dweight) dweight = torch::empty_like(*weight);
  if (need_dbias) dbias = torch::empty_like(*bias);
  if (need_dweight || need_dbias) {
    a.parts = npf_layernorm_parts(a, type);
    partial = torch::empty({a.parts, 2, x.size(1)},
                           x.options().dtype(torch::kFloat32));
    a.partial = partial->data_ptr<float>();
  }
  a.dy = dy.data_ptr();
  a.y = ptr_of(dx);
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.dweight = ptr_of(dweight);
  a.dbias = ptr_of(dbias);
  npf_check(npf_layernorm_bwd(a, type, at::hip::getCurrentHIPStream()),
            "layer_norm backward");
  return {dx, dweight, dbias};
}

int norm_code(double p) {
  if (p == 1.) return NPF_NORM_1;
  if (p == 2.) return NPF_NORM_2;
  TORCH_CHECK_VALUE(p == std::numeric_limits<double>::infinity(),
                    "norm_type must be 1, 2 or inf, is ", p);
  return NPF_NORM_INF;
}

// The gradients as spans of memory.  Neighbours in memory become one span
// (gradients that are views of one buffer, in order, are read as that buffer).
std::vector<NpfGradSpans> spans_of(const std::vector<Tensor>& grads) {
  std::vector<NpfGradSpans> all;
  auto size_of = [](int type) {
    return type == NPF_F64 ? 8 : type == NPF_F32 ? 4 : 2;
  };
  for (const Tensor& g : grads) {
    TORCH_CHECK_VALUE(g.is_cuda() && g.device() == grads[0].device(),
                      "all gradients must be on one GPU");
    TORCH_CHECK_VALUE(g.is_non_overlapping_and_dense(),
                      "gradients must be dense in memory");
    const int type = npf_type_code(g, "a gradient", true);
    if (g.numel() == 0) continue;
    char* p = static_cast<char*>(g.data_ptr());
    if (!all.empty() && all.back().n > 0) {
      NpfGradSpans& s = all.back();
      const int k = s.n - 1;
      if (s.type[k] == type &&
          static_cast<char*>(s.ptr[k]) + s.count[k] * size_of(type) == p) {
        s.count[k] += g.numel();
        continue;
      }
    }
    if (all.empty() || all.back().n == kGradSpans) all.emplace_back();
    NpfGradSpans& s = all.back();
    s.ptr[s.n] = p;
    s.count[s.n] = g.numel();
    s.type[s.n++] = (unsigned char)type;
  }
  for (NpfGradSpans& s : all) {
    long chunks = 0;
    for (int i = 0; i < s.n; ++i) {
      s.first_chunk[i] = (int)chunks;
      const long per = kGradChunkBytes / size_of(s.type[i]);
      chunks += (s.count[i] + per - 1) / per;
      TORCH_CHECK(chunks < std::numeric_limits<int>::max(),
                  "gradients are too large");
    }
    s.first_chunk[s.n] = (int)chunks;
  }
  return all;
}

// two gradients over the same memory would be scaled twice at once
void check_apart(const std::vector<NpfGradSpans>& all) {
  std::vector<std::pair<char*, char*>> at;
  for (const NpfGradSpans& s : all)
    for (int i = 0; i < s.n; ++i) {
      char* p = static_cast<char*>(s.ptr[i]);
      const int size =
          s.type[i] == NPF_F64 ? 8 : s.type[i] == NPF_F32 ? 4 : 2;
      at.emplace_back(p, p + s.count[i] * size);
    }
  std::sort(at.begin(), at.end());
  for (size_t i = 1; i < at.size(); ++i)
    TORCH_CHECK_VALUE(at[i].first >= at[i - 1].second,
                      "clipped gradients must not share memory");
}

// norm of all gradients; max_norm >= 0 also scales them in place
Tensor grad_norm(const std::vector<Tensor>& grads, double norm_type,
                 double max_norm) {
  const int norm = norm_code(norm_type);
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  std::vector<NpfGradSpans> all = spans_of(grads);
  const bool clip = max_norm >= 0.;
  if (clip) check_apart(all);
  c10::DeviceGuard guard(grads[0].device());
  auto options = torch::dtype(torch::kFloat32).device(grads[0].device());
  int type = NPF_F32;  // of the norm: as wide as the widest gradient
  for (const Tensor& g : grads)
    if (g.scalar_type() == torch::kFloat64) type = NPF_F64;
  Tensor total = torch::empty(
      {}, options.dtype(type == NPF_F64 ? torch::kFloat64 : torch::kFloat32));
  if (all.empty()) return total.zero_();
  int n = 0;
  for (const NpfGradSpans& s : all) n += npf_grad_blocks(s.first_chunk[s.n]);
  Tensor partial = torch::empty({n}, options.dtype(torch::kFloat64));
  auto stream = at::hip::getCurrentHIPStream();
  double* p = partial.data_ptr<double>();
  for (const NpfGradSpans& s : all) {
    npf_check(npf_grad_partial(s, norm, p, stream), "grad_norm");
    p += npf_grad_blocks(s.first_chunk[s.n]);
  }
  p = partial.data_ptr<double>();
  void* t = total.data_ptr();
  if (!clip) {
    npf_check(npf_grad_total(p, n, norm, t, type, stream), "grad_norm");
    return total;
  }
  for (const NpfGradSpans& s : all) {
    npf_check(npf_grad_scale(s, p, n, norm, max_norm, t, type, stream),
              "clip_grad_norm_");
    t = nullptr;
  }
  for (const Tensor& g : grads) g.unsafeGetTensorImpl()->bump_version();
  return total;
}

}  // namespace

void npf_bind_norms(pybind11::module_& m) {
  m.def("layer_norm_fwd", &layer_norm_fwd, "layer norm forward");
  m.def("layer_norm_bwd", &layer_norm_bwd,
        "layer norm backward -> (dx, dweight, dbias)");
  m.def("grad_norm", &grad_norm,
        "norm of many gradients; max_norm >= 0 clips them in place");
}
