// Bindings of differential attention.

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <limits>

#include "bindings.h"
#include "diff_attn.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr const char* kName = "differential_attention";

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
  return torch::Tensor(at::detail::empty_strided_cuda(
      {B, H, L, size}, {L * H * size, size, H * size, 1}, q.scalar_type(),
      q.device()));
}

NpfDiffAttnArgs common_args(const Tensor& q, const Tensor& k, const Tensor& v,
                            const Tensor& lam, double scale,
                            const Tensor& lengths) {
  check_heads(q, q, "queries");
  check_heads(k, q, "keys");
  check_heads(v, q, "values");
  NpfDiffAttnArgs a{};
  // rows are counted in 31 bits, up to a block's behind the last one; offsets
  // in memory are not
  const int64_t most = std::numeric_limits<int>::max() - 1024;
  TORCH_CHECK_VALUE(q.size(0) * q.size(1) * q.size(2) <= most &&
                        q.size(0) * k.size(1) * k.size(2) <= most &&
                        k.size(2) <= most / 2 && q.size(2) <= most / 2,
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
  TORCH_CHECK_VALUE(v.size(3) >= 1 && v.size(3) <= 256,
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
  a.lam_stride = lam.dim() == 0 ? 0 : lam.stride(0);
  if (lengths.defined()) {
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == a.B &&
                          lengths.device() == q.device() &&
                          lengths.is_contiguous(),
                      "key_lengths must have ", a.B,
                      " values on the GPU of the queries");
    TORCH_CHECK_TYPE(lengths.scalar_type() == torch::kInt32 ||
                         lengths.scalar_type() == torch::kInt64,
                     "key_lengths must be int32 or int64");
    a.lengths = lengths.data_ptr();
    a.lengths64 = lengths.scalar_type() == torch::kInt64;
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

// out, and where `save` the second map's part and the statistics
Tensor attn_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                    const Tensor& lam, double scale, const Tensor& lengths,
                    bool save, Tensor* o2, Tensor* lse) {
  NpfDiffAttnArgs a = common_args(q, k, v, lam, scale, lengths);
  // (what the backward pass would refuse is refused here)
  TORCH_CHECK_VALUE(npf_diff_attn_fits(a, false) &&
                        (!save || npf_diff_attn_fits(a, true)),
                    "differential_attention: too many heads and rows for a "
                    "launch");
  Tensor out = heads_like(q, a.B, a.H, a.Q, a.Dv);
  a.out = heads_of(out);
  if (save) {
    *o2 = heads_like(q, a.B, a.H, a.Q, a.Dv);
    *lse = npf_empty({(long)a.B * a.H * a.Q * 2}, torch::kFloat32, q);
    a.o2 = heads_of(*o2);
    a.lse = lse->data_ptr<float>();
  }
  if (out.numel() == 0) return out;
  Tensor split;
  if (const long floats = npf_diff_attn_workspace(a)) {
    split = npf_empty({floats}, torch::kFloat32, q);
    a.split = split.data_ptr();
  }
  npf_check(npf_diff_attn_fwd(a, at::hip::getCurrentHIPStream()),
            "differential_attention");
  return out;
}

// along the last axis the kernels take contiguous values alone
Tensor as_heads(const Tensor& t_) {
  const Tensor t = npf_signed(t_);
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

struct DiffAttn : torch::autograd::Function<DiffAttn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& k,
                        const Tensor& q, const Tensor& v, const Tensor& lam,
                        const OptTensor& lengths_, double scale) {
    const Tensor lengths = lengths_.value_or(Tensor());
    Tensor o2, lse;
    Tensor out =
        attn_forward(q, k, v, lam, scale, lengths, true, &o2, &lse);
    ctx->saved_data["needs"] =
        (int64_t)(k.requires_grad() + 2 * q.requires_grad() +
                  4 * v.requires_grad() + 8 * lam.requires_grad());
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({k, q, v, lam, lengths, out, o2, lse});
    return out;
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const Tensor &k = saved[0], &q = saved[1], &v = saved[2], &lam = saved[3],
                 &lengths = saved[4], &out = saved[5], &o2 = saved[6],
                 &lse = saved[7];
    npf_check_plain(grads[0], kName);
    // (common_args looks at their sizes, types and strides)
    for (const Tensor* t : {&k, &q, &v, &lam})
      npf_check_saved(*t, grads[0], t->scalar_type(), t->sizes(), kName);
    if (lengths.defined())
      npf_check_saved(lengths, q, lengths.scalar_type(), lengths.sizes(), kName);
    c10::DeviceGuard guard(q.device());
    NpfDiffAttnArgs a = common_args(q, k, v, lam,
                                    ctx->saved_data["scale"].toDouble(),
                                    lengths);
    const std::vector<int64_t> sizes = {a.B, a.H, a.Q, a.Dv};
    for (const Tensor* t : {&out, &o2}) {
      npf_check_saved(*t, q, q.scalar_type(), sizes, kName);
      check_heads(*t, q, "the saved result");
    }
    npf_check_saved(lse, q, torch::kFloat32, {(long)a.B * a.H * a.Q * 2}, kName);
    TORCH_CHECK_VALUE(grads[0].sizes() == sizes && lse.is_contiguous(), kName,
                      ": a saved tensor came back changed");
    const Tensor dout = as_heads(grads[0]);
    check_heads(dout, q, "dout");
    Tensor dk, dq, dv, dlam;
    if (needs & 1) dk = heads_like(k, a.B, a.Hk, a.K, 2 * a.D);
    if (needs & 2) dq = heads_like(q, a.B, a.H, a.Q, 2 * a.D);
    if (needs & 4) dv = heads_like(v, a.B, a.Hk, a.K, a.Dv);
    if (needs & 8) dlam = npf_empty(lam.sizes(), lam.scalar_type(), q);
    if (out.numel() == 0 || a.K == 0) {
      for (Tensor* t : {&dk, &dq, &dv, &dlam})
        if (t->defined()) t->zero_();
    } else {
      const long rows = (long)a.B * a.H * a.Q;
      Tensor stats = npf_empty({(4 + a.dq_splits) * rows}, torch::kFloat32, q);
      // parts of split sums
      Tensor dq_part, dk_part, dv_part;
      auto parts = [&](Tensor& part, const Tensor& grad, int splits) {
        if (!grad.defined() || splits == 1) return (float*)nullptr;
        part = npf_empty({splits * grad.numel()}, torch::kFloat32, q);
        return part.data_ptr<float>();
      };
      a.dq_part = parts(dq_part, dq, a.dq_splits);
      a.dk_part = parts(dk_part, dk, a.dkv_splits);
      a.dv_part = parts(dv_part, dv, a.dkv_splits);
      Tensor reach;
      if (a.v_chunks) {
        reach = npf_empty({(long)a.B * a.Hk * (a.v_chunks + a.o_chunks)},
                          torch::kFloat32, q);
        a.reach = reach.data_ptr<float>();
      }
      a.out = heads_of(out);
      a.o2 = heads_of(o2);
      a.dout = heads_of(dout);
      a.lse = lse.data_ptr<float>();
      a.stats = stats.data_ptr<float>();
      a.dlam_rows = a.stats + 4 * rows;
      if (dq.defined()) a.dq = heads_of(dq);
      if (dk.defined()) a.dk = heads_of(dk);
      if (dv.defined()) a.dv = heads_of(dv);
      if (dlam.defined()) a.dlam = dlam.data_ptr();
      npf_check(npf_diff_attn_bwd(a, at::hip::getCurrentHIPStream()),
                "differential_attention backward");
    }
    return npf_once({dk, dq, dv, dlam, Tensor(), Tensor()},
                    "differential_attention");
  }
};

Tensor differential_attention(const Tensor& k_, const Tensor& q_,
                              const Tensor& v_, const Tensor& lam_,
                              double scale, const OptTensor& lengths_) {
  npf_check_call(kName);
  for (const Tensor* t : {&k_, &q_, &v_, &lam_}) npf_check_plain(*t, kName);
  if (lengths_) npf_check_plain(*lengths_, kName);
  const Tensor k = as_heads(k_), q = as_heads(q_), v = as_heads(v_);
  const Tensor lam = npf_signed(lam_);
  OptTensor lengths;
  if (lengths_) lengths = npf_signed(*lengths_).contiguous();
  c10::DeviceGuard guard(q.device());
  if (at::GradMode::is_enabled() &&
      (k.requires_grad() || q.requires_grad() || v.requires_grad() ||
       lam.requires_grad()))
    return DiffAttn::apply(k, q, v, lam, lengths, scale);
  return attn_forward(q, k, v, lam, scale, lengths.value_or(Tensor()), false,
                      nullptr, nullptr);
}

}  // namespace

void npf_bind_diff_attn(pybind11::module_& m) {
  m.def("differential_attention", &differential_attention,
        "difference of two softmax maps times the values");
}
