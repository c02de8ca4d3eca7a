// Arguments of the differential attention kernels (diff_attn*.hip).
#pragma once

#include <hip/hip_runtime.h>

struct NpfHeads {
  void* p;        // [B, heads, length, size], `size` values contiguous
  long b, h, l;   // strides in values
};

struct NpfDiffAttnArgs {
  NpfHeads q, k, v;       // [B, H, Q, 2D], [B, Hk, K, 2D], [B, Hk, K, Dv]
  NpfHeads out, o2;       // [B, H, Q, Dv]; o2 (the second map's part) or null
  NpfHeads dout;          // backward
  NpfHeads dq, dk, dv;    // backward; null where not asked for
  float* lse;             // [B, H, Q, 2]: log2 of each map's sum of exponents
  float* stats;           // backward: [B, H, Q, 4]: lse_1, lse_2, delta_1, _2
  float* dlam_rows;       // backward: [dq_splits, B, H, Q]
  void* dlam;             // backward: [lam_heads], or null
  const void* lam;
  const void* lengths;    // [B] int32 or int64, or null
  void* split;            // forward: the parts of a result that is joined
  float* dq_part;         // backward: parts of a split sum, [dq_splits, B, H,
  float* dk_part;         // Q, 2D] and [dkv_splits, B, Hk, K, 2D or Dv], where
  float* dv_part;         // there are several
  float* reach;           // backward, fp16: [B * Hk, v_chunks + o_chunks], the
                          // largest norms of rows of values and of dout
  float scale;
  int B, H, Hk, Q, K, D, Dv;
  int type, lam_type;
  long lam_stride;
  int lam_heads;          // values of lam: H or 1
  int lengths64;
  // the plan
  int pad;     // D and Dv / 2 are padded to this
  int waves;   // of a forward block, for each map
  int splits;  // parts of the key axis, forward
  int dq_splits;   // parts of the key axis, and of the query axis, backward
  int dkv_splits;
  int v_chunks;    // of a key head's rows of values, and of its queries' rows
  int o_chunks;    // of dout; 0 where `reach` is not wanted
  int v_rows;      // of a chunk, whole steps of kReachRows
  int o_rows;
};

constexpr int kReachRows = 64;

// fills the plan; false where no kernel covers the sizes
bool npf_diff_attn_plan(NpfDiffAttnArgs&);
// whether each launch of a pass has fewer than 2^32 threads, as HIP asks
bool npf_diff_attn_fits(const NpfDiffAttnArgs&, bool backward);
// floats of `split`
long npf_diff_attn_workspace(const NpfDiffAttnArgs&);
hipError_t npf_diff_attn_fwd(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_bwd(const NpfDiffAttnArgs&, hipStream_t);
