// Norm of many gradient tensors taken as one vector, and clipping by it.
//
//   n = (sum |g|^p)^(1/p), p = 1, 2 or inf;  c = min(1, max_norm / (n + 1e-6))
//   g *= c
//
// One launch leaves a partial sum a block, the next adds all partials in their
// order (every block for itself: a few thousand values) and scales.  No
// atomics, so the result does not change between runs.  Sums are held in 64
// bits: squares of 32-bit values neither overflow nor lose small terms.
//
// Measured (one MI355X), 492 MB of bf16 in 48 tensors: norm 114 us (4.3 TB/s;
// reading alone, a sum of 1 GiB reaches 4.0), scaling 154 us (6.4 TB/s, part
// of it from the cache that the norm has filled): memory bounds both.  32
// tensors of one small model (1 MB): 6 and 5 us, launches.

#include "common.h"
#include "grad_norm.h"
#include "types.h"

namespace {

constexpr int kThreads = 256;
// 492 MB of bf16, both passes with 512, 1024, 2048, 4096 blocks: 280, 268, 278,
// 286 us.
constexpr int kMostBlocks = 1024;

__device__ __forceinline__ double join(double a, double b, int norm) {
  if (norm != NPF_NORM_INF) return a + b;
  return (a > b || a != a) ? a : b;  // NaN stays
}

__device__ __forceinline__ double value_of(double v, int norm) {
  return norm == NPF_NORM_2 ? v * v : fabs(v);
}

__device__ __forceinline__ double block_join(double x, int norm,
                                             double* smem) {
  for (int off = NPF_WAVE / 2; off > 0; off >>= 1)
    x = join(x, __shfl_xor(x, off, NPF_WAVE), norm);
  if ((threadIdx.x & (NPF_WAVE - 1)) == 0) smem[threadIdx.x / NPF_WAVE] = x;
  __syncthreads();
  x = smem[0];
  for (int w = 1; w < kThreads / NPF_WAVE; ++w) x = join(x, smem[w], norm);
  return x;
}

__device__ __forceinline__ double norm_of(const double* partial, int n,
                                          int norm, double* smem) {
  double s = 0.;
  for (int i = threadIdx.x; i < n; i += kThreads)
    s = join(s, partial[i], norm);
  s = block_join(s, norm, smem);
  return norm == NPF_NORM_2 ? sqrt(s) : s;
}

__device__ __forceinline__ int size_of(int type) {
  return type == NPF_F64 ? 8 : type == NPF_F32 ? 4 : 2;
}

// the span that holds a chunk
__device__ __forceinline__ int span_of(const NpfGradSpans& s, int chunk) {
  int lo = 0, hi = s.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (s.first_chunk[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// A chunk is 32 KiB: 8 accesses of 16 bytes a thread, all in flight at once.
template <typename T>
__device__ __forceinline__ double sum_chunk(const T* p, long n, int norm) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr long kFull = kGradChunkBytes / (long)sizeof(T);
  double s = 0.;
  if (n == kFull) {
    T v[8][V];
    double part[4] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      load_pack(v[k], p + (k * kThreads + threadIdx.x) * V);
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
        part[k & 3] = join(part[k & 3], value_of((double)v[k][i], norm), norm);
    return join(join(part[0], part[1], norm), join(part[2], part[3], norm),
                norm);
  }
  long i = (long)threadIdx.x * V;
  for (; i + V <= n; i += kThreads * V) {
    T v[V];
    load_pack(v, p + i);
#pragma unroll
    for (int k = 0; k < V; ++k) s = join(s, value_of((double)v[k], norm), norm);
  }
  for (; i < n; ++i) s = join(s, value_of((double)p[i], norm), norm);
  return s;
}

template <typename T, typename C>
__device__ __forceinline__ void scale_chunk(T* p, long n, C c) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr long kFull = kGradChunkBytes / (long)sizeof(T);
  if (n == kFull) {
    T v[8][V];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      load_pack(v[k], p + (k * kThreads + threadIdx.x) * V);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = (T)((C)v[k][i] * c);
      store_pack(p + (k * kThreads + threadIdx.x) * V, v[k]);
    }
    return;
  }
  long i = (long)threadIdx.x * V;
  for (; i + V <= n; i += kThreads * V) {
    T v[V];
    load_pack(v, p + i);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (T)((C)v[k] * c);
    store_pack(p + i, v);
  }
  for (; i < n; ++i) p[i] = (T)((C)p[i] * c);
}

__global__ void __launch_bounds__(kThreads)
    grad_partial(NpfGradSpans s, int norm, double* partial) {
  __shared__ double smem[kThreads / NPF_WAVE];
  double sum = 0.;
  for (int c = blockIdx.x; c < s.first_chunk[s.n]; c += gridDim.x) {
    const int i = span_of(s, c);
    const long per = kGradChunkBytes / size_of(s.type[i]);
    const long at = (long)(c - s.first_chunk[i]) * per;
    const long n = s.count[i] - at < per ? s.count[i] - at : per;
    double part;
    switch (s.type[i]) {
      case NPF_F32: part = sum_chunk((const float*)s.ptr[i] + at, n, norm); break;
      case NPF_BF16: part = sum_chunk((const npf_bf16*)s.ptr[i] + at, n, norm); break;
      case NPF_F16: part = sum_chunk((const npf_f16*)s.ptr[i] + at, n, norm); break;
      default: part = sum_chunk((const double*)s.ptr[i] + at, n, norm);
    }
    sum = join(sum, part, norm);
  }
  sum = block_join(sum, norm, smem);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads)
    grad_total(const double* partial, int n, int norm, void* total,
               int total_type) {
  __shared__ double smem[kThreads / NPF_WAVE];
  const double t = norm_of(partial, n, norm, smem);
  if (threadIdx.x == 0) store_coded(total, total_type, 0, t);
}

__global__ void __launch_bounds__(kThreads)
    grad_scale(NpfGradSpans s, const double* partial, int n, int norm,
               double max_norm, void* total,
               int total_type) {
  __shared__ double smem[kThreads / NPF_WAVE];
  const double t = norm_of(partial, n, norm, smem);
  if (total && blockIdx.x == 0 && threadIdx.x == 0) store_coded(total, total_type, 0, t);
  const double ratio = max_norm / (t + 1e-6);
  if (ratio >= 1.) return;  // nothing to change
  // (a norm that is no number makes every gradient none)
  const float scale = (float)ratio;
  // from the last chunk back: what the first pass read last is still cached
  for (int c = s.first_chunk[s.n] - 1 - (int)blockIdx.x; c >= 0;
       c -= gridDim.x) {
    const int i = span_of(s, c);
    // a factor next to 1 is not 1 in 64 bits alone
    if (scale == 1.f && s.type[i] != NPF_F64) continue;
    const long per = kGradChunkBytes / size_of(s.type[i]);
    const long at = (long)(c - s.first_chunk[i]) * per;
    const long m = s.count[i] - at < per ? s.count[i] - at : per;
    switch (s.type[i]) {
      case NPF_F32: scale_chunk((float*)s.ptr[i] + at, m, scale); break;
      case NPF_BF16: scale_chunk((npf_bf16*)s.ptr[i] + at, m, scale); break;
      case NPF_F16: scale_chunk((npf_f16*)s.ptr[i] + at, m, scale); break;
      default: scale_chunk((double*)s.ptr[i] + at, m, ratio);
    }
  }
}

}  // namespace

int npf_grad_blocks(int chunks) {
  return chunks < kMostBlocks ? chunks : kMostBlocks;
}

hipError_t npf_grad_partial(const NpfGradSpans& s, int norm, double* partial,
                            hipStream_t stream) {
  grad_partial<<<npf_grad_blocks(s.first_chunk[s.n]), kThreads, 0, stream>>>(
      s, norm, partial);
  return hipGetLastError();
}

hipError_t npf_grad_total(const double* partial, int n, int norm, void* total,
                          int total_type, hipStream_t stream) {
  grad_total<<<1, kThreads, 0, stream>>>(partial, n, norm, total,
                                          total_type);
  return hipGetLastError();
}

hipError_t npf_grad_scale(const NpfGradSpans& s, const double* partial, int n,
                          int norm, double max_norm, void* total,
                          int total_type, hipStream_t stream) {
  grad_scale<<<npf_grad_blocks(s.first_chunk[s.n]), kThreads, 0, stream>>>(
      s, partial, n, norm, max_norm, total, total_type);
  return hipGetLastError();
}
