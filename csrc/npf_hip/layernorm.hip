// Layer norm over the last axis, forward and backward.
//
//   z = x (+ residual);  mu = mean(z);  rstd = (mean((z - mu)^2) + eps)^-1/2
//   h = (z - mu) rstd;   y = h w + b
//   g = dy w;  dz = rstd (g - mean(g) - h mean(g h))
//   dw = sum over rows of dy h;  db = sum over rows of dy
//
// Statistics and sums are held in 32 bits; a value is rounded once, at its
// store.  The sum of x and residual is never rounded: the backward pass takes
// it from the two inputs again, which costs the read that a stored sum would
// cost and saves its write.

#include "common.h"
#include "layernorm.h"
#include "types.h"

namespace {

constexpr int kThreads = 256;

// sum over the block, in every thread; `smem` holds one float a wave
__device__ __forceinline__ float block_sum(float x, float* smem) {
  x = wave_allreduce_sum(x);
  const int waves = blockDim.x / NPF_WAVE;
  __syncthreads();
  if ((threadIdx.x & (NPF_WAVE - 1)) == 0) smem[threadIdx.x / NPF_WAVE] = x;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < waves; ++w) s += smem[w];
  return s;
}

template <typename T>
__device__ __forceinline__ float load_z(const NpfLayerNormArgs& a, long row,
                                        int c) {
  float z = (float)static_cast<const T*>(a.x)[row * a.x_stride + c];
  if (a.residual)
    z += (float)static_cast<const T*>(
        a.residual)[row * a.residual_stride + c];
  return z;
}

__device__ __forceinline__ float load_weight(const NpfLayerNormArgs& a,
                                             int c) {
  return a.weight ? load_coded(a.weight, a.weight_type, c) : 1.f;
}

// one block a row, three passes over it
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ln_fwd_loop(NpfLayerNormArgs a) {
  __shared__ float smem[kThreads / NPF_WAVE];
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float s = 0.f;
    for (int c = threadIdx.x; c < a.width; c += kThreads)
      s += load_z<T>(a, row, c);
    const float mean = block_sum(s, smem) / a.width;
    s = 0.f;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float d = load_z<T>(a, row, c) - mean;
      s += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(s, smem) / a.width + a.eps);
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      float y = (load_z<T>(a, row, c) - mean) * rstd * load_weight(a, c);
      if (a.bias) y += load_coded(a.bias, a.weight_type, c);
      static_cast<T*>(a.y)[row * a.width + c] = (T)y;
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    ln_dx_loop(NpfLayerNormArgs a) {
  __shared__ float smem[kThreads / NPF_WAVE];
  const T* dy = static_cast<const T*>(a.dy);
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, sgh = 0.f;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float g = (float)dy[row * a.width + c] * load_weight(a, c);
      sg += g;
      sgh += g * (load_z<T>(a, row, c) - mean) * rstd;
    }
    sg = block_sum(sg, smem) / a.width;
    sgh = block_sum(sgh, smem) / a.width;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float g = (float)dy[row * a.width + c] * load_weight(a, c);
      const float h = (load_z<T>(a, row, c) - mean) * rstd;
      static_cast<T*>(a.y)[row * a.width + c] = (T)(rstd * (g - sg - h * sgh));
    }
  }
}

// sums of dy h and dy over one part of the rows: a thread a column
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ln_dw_part(NpfLayerNormArgs a) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.width) return;
  float dw = 0.f, db = 0.f;
  for (long row = blockIdx.y; row < a.rows; row += a.parts) {
    const float dy = (float)static_cast<const T*>(a.dy)[row * a.width + c];
    dw += dy * (load_z<T>(a, row, c) - a.mean[row]) * a.rstd[row];
    db += dy;
  }
  a.partial[(2L * blockIdx.y) * a.width + c] = dw;
  a.partial[(2L * blockIdx.y + 1) * a.width + c] = db;
}

// the parts' sums, in their order: 16 columns and 16 slices of the parts a block
__global__ void __launch_bounds__(kThreads) ln_dw_join(NpfLayerNormArgs a) {
  __shared__ float smem[2][16][17];
  const int cl = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cl;
  float dw = 0.f, db = 0.f;
  if (c < a.width)
    for (int p = slice; p < a.parts; p += 16) {
      dw += a.partial[2L * p * a.width + c];
      db += a.partial[(2L * p + 1) * a.width + c];
    }
  smem[0][slice][cl] = dw;
  smem[1][slice][cl] = db;
  __syncthreads();
  if (slice > 1 || c >= a.width) return;
  float s = 0.f;
  for (int i = 0; i < 16; ++i) s += smem[slice][i][cl];
  void* out = slice == 0 ? a.dweight : a.dbias;
  if (out) store_coded(out, a.weight_type, c, s);
}

unsigned blocks_for(long rows) {
  return (unsigned)(rows < 4096 ? rows : 4096);
}

template <typename T>
hipError_t launch_bwd(const NpfLayerNormArgs& a, bool need_dx,
                      hipStream_t stream) {
  if (need_dx)
    ln_dx_loop<T><<<blocks_for(a.rows), kThreads, 0, stream>>>(a);
  if (a.partial) {
    ln_dw_part<T><<<dim3((a.width + kThreads - 1) / kThreads, a.parts),
                    kThreads, 0, stream>>>(a);
    ln_dw_join<<<(a.width + 15) / 16, kThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

int npf_layernorm_parts(long rows, int, int) {
  return (int)(rows < 128 ? rows : 128);
}

hipError_t npf_layernorm_fwd(const NpfLayerNormArgs& a, int type,
                             hipStream_t stream) {
  const unsigned n = blocks_for(a.rows);
  switch (type) {
    case NPF_F32: ln_fwd_loop<float><<<n, kThreads, 0, stream>>>(a); break;
    case NPF_BF16: ln_fwd_loop<npf_bf16><<<n, kThreads, 0, stream>>>(a); break;
    case NPF_F16: ln_fwd_loop<npf_f16><<<n, kThreads, 0, stream>>>(a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t npf_layernorm_bwd(const NpfLayerNormArgs& a, int type, bool need_dx,
                             hipStream_t stream) {
  switch (type) {
    case NPF_F32: return launch_bwd<float>(a, need_dx, stream);
    case NPF_BF16: return launch_bwd<npf_bf16>(a, need_dx, stream);
    case NPF_F16: return launch_bwd<npf_f16>(a, need_dx, stream);
    default: return hipErrorInvalidValue;
  }
}
