// Bindings of differential attention.

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <limits>

#include "bindings.h"
#include "diff_attn.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

NpfHeads heads_of(const Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

void check_heads(const Tensor& t, const Tensor& q, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be [batch, heads, length, size]");
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == q.device(), name,
                    " must be on the GPU of the queries");
  TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), name,
                   " must have the type of the queries");
  TORCH_CHECK_VALUE(t.size(3) == 1 || t.stride(3) == 1, name,
                    " must be contiguous along its last axis");
}

// memory [B, length, heads, size], as the projection that follows wants it
Tensor heads_like(const Tensor& q, int64_t B, int64_t H, int64_t L,
                  int64_t size) {
  return torch::empty({B, L, H, size}, q.options()).transpose(1, 2);
}

NpfDiffAttnArgs common_args(const Tensor& q, const Tensor& k, const Tensor& v,
                            const Tensor& lam, double scale,
                            const OptTensor& lengths) {
  check_heads(q, q, "queries");
  check_heads(k, q, "keys");
  check_heads(v, q, "values");
  NpfDiffAttnArgs a{};
  const int64_t most = std::numeric_limits<int>::max() / 2;
  TORCH_CHECK_VALUE(q.size(0) <= 65535 && q.size(1) <= 65535 &&
                        q.size(1) * q.size(2) <= most && k.size(2) <= most,
                    "differential_attention: too many rows");
  a.B = (int)q.size(0);
  a.H = (int)q.size(1);
  a.Q = (int)q.size(2);
  a.D = (int)(q.size(3) / 2);
  a.Hk = (int)k.size(1);
  a.K = (int)k.size(2);
  a.Dv = (int)v.size(3);
  TORCH_CHECK_VALUE(q.size(3) == 2 * a.D && k.size(3) == 2 * a.D && a.D >= 1 &&
                        a.D <= 128,
                    "queries and keys must hold two maps of 1 to 128 values");
  TORCH_CHECK_VALUE(a.Dv >= 1 && a.Dv <= 256,
                    "values must have 1 to 256 values a head");
  TORCH_CHECK_VALUE(k.size(0) == a.B && v.size(0) == a.B &&
                        v.size(1) == a.Hk && v.size(2) == a.K,
                    "keys and values must match each other and the batch");
  TORCH_CHECK_VALUE(a.Hk >= 1 && a.H % a.Hk == 0,
                    "query heads must be a multiple of key heads");
  TORCH_CHECK_VALUE(lam.device() == q.device() &&
                        (lam.dim() == 0 ||
                         (lam.dim() == 1 && lam.size(0) == a.H)),
                    "lam must be a number or one a query head, on the GPU");
  a.lam = lam.data_ptr();
  a.lam_type = npf_type_code(lam, "lam", true);
  a.lam_heads = lam.dim() == 0 ? 1 : a.H;
  a.lam_stride = lam.dim() == 0 ? 0 : (int)lam.stride(0);
  if (lengths) {
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == a.B &&
                          lengths->device() == q.device() &&
                          lengths->is_contiguous(),
                      "key_lengths must be a contiguous [", a.B,
                      "] on the GPU of the queries");
    TORCH_CHECK_TYPE(lengths->scalar_type() == torch::kInt32 ||
                         lengths->scalar_type() == torch::kInt64,
                     "key_lengths must be int32 or int64");
    a.lengths = lengths->data_ptr();
    a.lengths64 = lengths->scalar_type() == torch::kInt64;
  }
  a.type = npf_type_code(q, "queries");
  a.scale = (float)scale;
  TORCH_CHECK_VALUE(npf_diff_attn_plan(a),
                    "differential_attention: sizes ", a.D, " and ", a.Dv,
                    " of a head are too large");
  a.q = heads_of(q);
  a.k = heads_of(k);
  a.v = heads_of(v);
  return a;
}

// (out, o2, lse); the last two are empty unless `save`
std::tuple<Tensor, Tensor, Tensor> diff_attn_fwd(
    const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam,
    double scale, const OptTensor& lengths, bool save) {
  NpfDiffAttnArgs a = common_args(q, k, v, lam, scale, lengths);
  c10::DeviceGuard guard(q.device());
  Tensor out = heads_like(q, a.B, a.H, a.Q, a.Dv);
  Tensor o2 = save ? heads_like(q, a.B, a.H, a.Q, a.Dv)
                   : torch::empty({0}, q.options());
  Tensor lse = torch::empty({save ? (long)a.B * a.H * a.Q * 2 : 0},
                            q.options().dtype(torch::kFloat32));
  if (out.numel() == 0) return {out, o2, lse};
  a.out = heads_of(out);
  if (save) {
    a.o2 = heads_of(o2);
    a.lse = lse.data_ptr<float>();
  }
  Tensor split;
  if (const size_t bytes = npf_diff_attn_workspace(a)) {
    split = torch::empty({(long)bytes}, q.options().dtype(torch::kUInt8));
    a.split = split.data_ptr();
  }
  npf_check(npf_diff_attn_fwd(a, at::hip::getCurrentHIPStream()),
            "differential_attention");
  return {out, o2, lse};
}

// (dq, dk, dv, dlam); those that are not asked for are None
std::tuple<OptTensor, OptTensor, OptTensor, OptTensor> diff_attn_bwd(
    const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
    const Tensor& lam, const Tensor& out, const Tensor& o2, const Tensor& lse,
    double scale, const OptTensor& lengths, bool need_dq, bool need_dk,
    bool need_dv, bool need_dlam) {
  NpfDiffAttnArgs a = common_args(q, k, v, lam, scale, lengths);
  check_heads(dout, q, "dout");
  TORCH_CHECK_VALUE(dout.sizes() == out.sizes() && o2.sizes() == out.sizes(),
                    "dout must have the shape of the output");
  c10::DeviceGuard guard(q.device());
  OptTensor dq, dk, dv, dlam;
  if (need_dq) dq = heads_like(q, a.B, a.H, a.Q, 2 * a.D);
  if (need_dk) dk = heads_like(k, a.B, a.Hk, a.K, 2 * a.D);
  if (need_dv) dv = heads_like(v, a.B, a.Hk, a.K, a.Dv);
  if (need_dlam) dlam = torch::empty(lam.sizes(), lam.options());
  if (out.numel() == 0 || a.K == 0) {
    for (OptTensor* t : {&dq, &dk, &dv, &dlam})
      if (*t) (*t)->zero_();
    return {dq, dk, dv, dlam};
  }
  auto f32 = q.options().dtype(torch::kFloat32);
  const long rows = (long)a.B * a.H * a.Q;
  Tensor stats = torch::empty({rows, 4}, f32);
  Tensor dlam_rows = torch::empty({rows}, f32);
  a.out = heads_of(out);
  a.o2 = heads_of(o2);
  a.dout = heads_of(dout);
  a.lse = lse.data_ptr<float>();
  a.stats = stats.data_ptr<float>();
  a.dlam_rows = dlam_rows.data_ptr<float>();
  if (dq) a.dq = heads_of(*dq);
  if (dk) a.dk = heads_of(*dk);
  if (dv) a.dv = heads_of(*dv);
  if (dlam) a.dlam = dlam->data_ptr();
  npf_check(npf_diff_attn_bwd(a, at::hip::getCurrentHIPStream()),
            "differential_attention backward");
  return {dq, dk, dv, dlam};
}

}  // namespace

void npf_bind_diff_attn(pybind11::module_& m) {
  m.def("diff_attn_fwd", &diff_attn_fwd,
        "differential attention forward -> (out, o2, lse)");
  m.def("diff_attn_bwd", &diff_attn_bwd,
        "differential attention backward -> (dq, dk, dv, dlam)");
}
