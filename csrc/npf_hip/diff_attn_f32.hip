// Differential attention for one type (a file each, to build side by side).

#include "diff_attn_impl.h"

hipError_t npf_diff_attn_fwd_f32(const NpfDiffAttnArgs& a, hipStream_t stream) {
  return npf_attn::typed<float>(a, false, stream);
}

hipError_t npf_diff_attn_bwd_f32(const NpfDiffAttnArgs& a, hipStream_t stream) {
  return npf_attn::typed<float>(a, true, stream);
}
