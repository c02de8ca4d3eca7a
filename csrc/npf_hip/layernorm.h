// Arguments of the layer norm kernels (layernorm.hip).
#pragma once

#include <hip/hip_runtime.h>

struct NpfLayerNormArgs {
  const void* x;         // [rows, width], rows x_stride values apart
  const void* residual;  // the same, or null
  const void* weight;    // [width] or null
  const void* bias;      // [width] or null
  const void* dy;        // backward: [rows, width] contiguous
  void* y;               // forward: y; backward: dx, or null;
                         // [rows, width] contiguous
  float* mean;           // [rows]; forward: written where not null
  float* rstd;           // [rows]
  float* partial;        // backward: [parts, 2, width], or null
  void* dweight;         // backward: [width] or null
  void* dbias;           // backward: [width] or null
  long x_stride, residual_stride;
  long rows;
  int width;
  int parts;
  int weight_type;  // of weight, bias and their gradients
  float eps;
};

// rows of `partial` that the backward pass fills for this problem
int npf_layernorm_parts(const NpfLayerNormArgs&, int type);
hipError_t npf_layernorm_fwd(const NpfLayerNormArgs&, int type, hipStream_t);
hipError_t npf_layernorm_bwd(const NpfLayerNormArgs&, int type, hipStream_t);
