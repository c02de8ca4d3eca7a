// Arguments of the differential attention kernels (diff_attn.hip).
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
  float* delta;           // backward: [B, H, Q, 2]: dout . (each map's part)
  double* dlam_partial;   // backward: [B, H, parts]
  void* dlam;             // backward: [lam_heads], or null
  const void* lam;
  const void* lengths;    // [B] int32 or int64, or null
  void* split;            // forward over a split key axis: its workspace
  float scale;
  int B, H, Hk, Q, K, D, Dv;
  int type, lam_type, lam_stride;
  int lam_heads;          // values of lam: H or 1
  int lengths64;
  int parts;
  int splits;
};

// rows of dlam_partial for each head of a batch entry
int npf_diff_attn_parts(int Q);
hipError_t npf_diff_attn_fwd(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_bwd(const NpfDiffAttnArgs&, hipStream_t);
