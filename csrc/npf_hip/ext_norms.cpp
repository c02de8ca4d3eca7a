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

void* ptr_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

OptTensor some(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}

// [..., D] as [rows, D] with contiguous rows; copied only where no stride
// describes the rows
Tensor rows_of(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

void check_like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == x.sizes(), name, " must have the shape ",
                    x.sizes(), ", has ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ",
                    x.device());
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name,
                   " must have type ", x.scalar_type());
}

void check_columns(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1) &&
                        t.device() == x.device(),
                    name, " must have ", x.size(-1), " values on ",
                    x.device());
}

// The rows (x, residual as rows_of leaves them), weight and bias contiguous;
// residual, weight and bias may be undefined.
NpfLayerNormArgs norm_args(const Tensor& x, const Tensor& residual,
                           const Tensor& weight, const Tensor& bias) {
  NpfLayerNormArgs a{};
  a.x = x.data_ptr();
  a.residual = ptr_of(residual);
  a.weight = ptr_of(weight);
  a.bias = ptr_of(bias);
  a.x_stride = x.stride(0);
  a.residual_stride = residual.defined() ? residual.stride(0) : 0;
  a.rows = x.size(0);
  a.width = (int)x.size(1);
  const Tensor& w = weight.defined() ? weight : bias;
  a.weight_type = w.defined() ? npf_type_code(w, "weight", true) : (int)NPF_F32;
  return a;
}

// [2, rows]: means, and inverse deviations
void set_stats(NpfLayerNormArgs& a, const Tensor& stats) {
  a.mean = stats.data_ptr<float>();
  a.rstd = a.mean + a.rows;
}

// `stats` are filled where they are defined
void layer_norm_forward(const Tensor& x, const Tensor& residual,
                        const Tensor& weight, const Tensor& bias, double eps,
                        Tensor& y, const Tensor& stats) {
  NpfLayerNormArgs a = norm_args(x, residual, weight, bias);
  if (a.rows == 0) return;
  a.y = y.data_ptr();
  if (stats.defined()) set_stats(a, stats);
  a.eps = (float)eps;
  npf_check(npf_layernorm_fwd(a, npf_type_code(x, "x"),
                              at::hip::getCurrentHIPStream()),
            "layer_norm");
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x,
                        const OptTensor& residual_, const OptTensor& weight_,
                        const OptTensor& bias_, double eps) {
    const Tensor residual = residual_.value_or(Tensor());
    const Tensor weight = weight_.value_or(Tensor());
    const Tensor bias = bias_.value_or(Tensor());
    const Tensor xr = rows_of(x), rr = rows_of(residual);
    Tensor y = npf_empty(x.sizes(), x.scalar_type(), x);
    const Tensor stats = npf_empty({2, xr.size(0)}, torch::kFloat32, x);
    layer_norm_forward(xr, rr, weight, bias, eps, y, stats);
    auto needs = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    ctx->saved_data["needs"] =
        (int64_t)(needs(x) + 2 * needs(residual) + 4 * needs(weight) +
                  8 * needs(bias));
    ctx->save_for_backward({xr, rr, weight, bias, stats});
    return y;
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const Tensor &x = saved[0], &residual = saved[1], &weight = saved[2],
                 &bias = saved[3], &stats = saved[4];
    npf_check_plain(grads[0], "layer_norm");
    const Tensor& like = grads[0];
    const int64_t D = like.size(-1), rows = like.numel() / D;
    for (const Tensor* t : {&x, &residual})
      if (t == &x || t->defined()) {
        npf_check_saved(*t, like, like.scalar_type(), {rows, D}, "layer_norm");
        TORCH_CHECK_VALUE(D == 1 || t->stride(1) == 1,
                          "layer_norm: a saved tensor came back changed");
      }
    for (const Tensor* t : {&weight, &bias, &stats})
      if (t == &stats || t->defined()) {
        npf_check_saved(*t, like,
                        t == &stats ? torch::kFloat32 : t->scalar_type(),
                        t == &stats ? at::IntArrayRef{2, rows}
                                    : at::IntArrayRef{D},
                        "layer_norm");
        TORCH_CHECK_VALUE(t->is_contiguous(),
                          "layer_norm: a saved tensor came back changed");
      }
    c10::DeviceGuard guard(x.device());
    NpfLayerNormArgs a = norm_args(x, residual, weight, bias);
    const Tensor dy = npf_signed(grads[0]).contiguous();
    Tensor dx, dweight, dbias, partial;
    if (needs & 3) dx = npf_empty(dy.sizes(), dy.scalar_type(), dy);
    if (needs & 4)
      dweight = npf_empty(weight.sizes(), weight.scalar_type(), weight);
    if (needs & 8) dbias = npf_empty(bias.sizes(), bias.scalar_type(), bias);
    if (a.rows == 0) {
      if (dweight.defined()) dweight.zero_();
      if (dbias.defined()) dbias.zero_();
    } else {
      const int type = npf_type_code(x, "x");
      if (needs & 12) {
        a.parts = npf_layernorm_parts(a, type);
        partial = npf_empty({a.parts, 2, x.size(1)}, torch::kFloat32, x);
        a.partial = partial.data_ptr<float>();
      }
      a.dy = dy.data_ptr();
      a.y = ptr_of(dx);
      set_stats(a, stats);
      a.dweight = ptr_of(dweight);
      a.dbias = ptr_of(dbias);
      npf_check(npf_layernorm_bwd(a, type, at::hip::getCurrentHIPStream()),
                "layer_norm backward");
    }
    return npf_once(
        {needs & 1 ? dx : Tensor(), needs & 2 ? dx : Tensor(), dweight, dbias,
         Tensor()},
        "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x_, const OptTensor& residual_,
                  const OptTensor& weight_, const OptTensor& bias_,
                  double eps) {
  npf_check_call("layer_norm");
  npf_check_plain(x_, "layer_norm");
  for (const OptTensor* t : {&residual_, &weight_, &bias_})
    if (*t) npf_check_plain(**t, "layer_norm");
  const Tensor x = npf_signed(x_);
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1 && x.size(-1) > 0,
                    "layer_norm takes rows of at least one value on a GPU");
  TORCH_CHECK_VALUE(x.size(-1) <= std::numeric_limits<int>::max() / 2,
                    "layer_norm: rows are too wide");
  npf_type_code(x, "x");
  const Tensor residual = npf_signed(residual_.value_or(Tensor()));
  Tensor weight = npf_signed(weight_.value_or(Tensor()));
  Tensor bias = npf_signed(bias_.value_or(Tensor()));
  if (residual.defined()) check_like(residual, x, "residual");
  if (weight.defined()) {
    check_columns(weight, x, "weight");
    weight = weight.contiguous();
  }
  if (bias.defined()) {
    check_columns(bias, x, "bias");
    bias = bias.contiguous();
  }
  TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() ||
                       weight.scalar_type() == bias.scalar_type(),
                   "weight and bias must have the same type");
  c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled())
    for (const Tensor* t : {&x, &residual, (const Tensor*)&weight,
                            (const Tensor*)&bias})
      if (t->defined() && t->requires_grad())
        return LayerNorm::apply(x, some(residual), some(weight), some(bias),
                                eps);
  Tensor y = npf_empty(x.sizes(), x.scalar_type(), x);
  layer_norm_forward(rows_of(x), rows_of(residual), weight, bias, eps, y,
                     Tensor());
  return y;
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
    TORCH_CHECK_VALUE(g.is_non_overlapping_and_dense() && !g.is_neg() &&
                          !g._is_zerotensor(),
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

// norm of the gradients of all parameters that have one; max_norm >= 0 also
// scales them in place
Tensor grad_norm(const std::vector<Tensor>& params, double norm_type,
                 double max_norm) {
  npf_check_call("grad_norm");
  const int norm = norm_code(norm_type);
  std::vector<Tensor> grads;
  grads.reserve(params.size());
  for (const Tensor& p : params) {
    const Tensor& g = p.grad();
    if (!g.defined()) continue;
    TORCH_CHECK_TYPE(g.layout() == torch::kStrided,
                     "gradients must be dense floating tensors");
    npf_check_plain(g, "grad_norm");
    grads.push_back(g);
  }
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  std::vector<NpfGradSpans> all = spans_of(grads);
  const bool clip = max_norm >= 0.;
  if (clip) check_apart(all);
  c10::DeviceGuard guard(grads[0].device());
  int type = NPF_F32;  // of the norm: as wide as the widest gradient
  for (const Tensor& g : grads)
    if (g.scalar_type() == torch::kFloat64) type = NPF_F64;
  Tensor total = npf_empty(
      {}, type == NPF_F64 ? torch::kFloat64 : torch::kFloat32, grads[0]);
  if (all.empty()) return total.zero_();
  int n = 0;
  for (const NpfGradSpans& s : all) n += npf_grad_blocks(s.first_chunk[s.n]);
  Tensor partial = npf_empty({n}, torch::kFloat64, grads[0]);
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
  // (an inference tensor raises here, before any gradient changes)
  for (const Tensor& g : grads) g.unsafeGetTensorImpl()->bump_version();
  for (const NpfGradSpans& s : all) {
    npf_check(npf_grad_scale(s, p, n, norm, max_norm, t, type, stream),
              "clip_grad_norm_");
    t = nullptr;
  }
  return total;
}

}  // namespace

void npf_bind_norms(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm, "layer norm over the last axis");
  m.def("grad_norm", &grad_norm,
        "norm of the parameters' gradients; max_norm >= 0 clips them in place");
}
