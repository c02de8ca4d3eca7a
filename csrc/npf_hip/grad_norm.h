// Arguments of the gradient norm and clipping kernels (grad_norm.hip).
#pragma once

#include <hip/hip_runtime.h>

constexpr int kGradSpans = 160;         // spans of memory a launch takes
constexpr long kGradChunkBytes = 32768;  // of a span a block takes at a time

// Spans of gradient memory; passed by value, so that a captured launch holds
// the addresses and no table has to be copied to the GPU.
struct NpfGradSpans {
  void* ptr[kGradSpans];
  long count[kGradSpans];          // values
  int first_chunk[kGradSpans + 1];  // chunks before each span, and in all
  unsigned char type[kGradSpans];
  int n;
};

enum NpfNormType { NPF_NORM_1 = 0, NPF_NORM_2 = 1, NPF_NORM_INF = 2 };

// blocks (and so partial sums) of a launch over this many chunks
int npf_grad_blocks(int chunks);
// partial[0 .. blocks) of one launch's spans
hipError_t npf_grad_partial(const NpfGradSpans&, int norm, double* partial,
                            hipStream_t);
// total = norm of all partials
hipError_t npf_grad_total(const double* partial, int n, int norm, void* total,
                          int total_type, hipStream_t);
// spans *= min(1, max_norm / (norm + 1e-6)); also writes total where not null
hipError_t npf_grad_scale(const NpfGradSpans&, const double* partial, int n,
                          int norm, double max_norm, void* total,
                          int total_type, hipStream_t);
