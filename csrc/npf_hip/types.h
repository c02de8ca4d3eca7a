// Element types of the kernels that take fp32, bf16 and fp16 alike.
#pragma once

#include <hip/hip_runtime.h>

#include "type_codes.h"

using npf_bf16 = __bf16;
using npf_f16 = _Float16;

// Accesses of up to 16 bytes at any alignment: global memory takes wide loads
// and stores at every byte address on gfx950, so odd widths and unaligned
// views need no narrow path of their own.
template <typename T, int N>
__device__ __forceinline__ void load_pack(T (&dst)[N], const T* src) {
  __builtin_memcpy(&dst, src, sizeof(T) * N);
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* dst, const T (&src)[N]) {
  __builtin_memcpy(dst, &src, sizeof(T) * N);
}

// one value of a tensor whose type is known by its code alone
__device__ __forceinline__ float load_coded(const void* p, int type, long i) {
  switch (type) {
    case NPF_F32: return static_cast<const float*>(p)[i];
    case NPF_BF16: return (float)static_cast<const npf_bf16*>(p)[i];
    case NPF_F16: return (float)static_cast<const npf_f16*>(p)[i];
    default: return (float)static_cast<const double*>(p)[i];
  }
}

__device__ __forceinline__ void store_coded(void* p, int type, long i,
                                            double v) {
  switch (type) {
    case NPF_F32: static_cast<float*>(p)[i] = (float)v; break;
    case NPF_BF16: static_cast<npf_bf16*>(p)[i] = (npf_bf16)(float)v; break;
    case NPF_F16: static_cast<npf_f16*>(p)[i] = (npf_f16)(float)v; break;
    default: static_cast<double*>(p)[i] = v;
  }
}
