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

#include <type_traits>

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

// Measured (one MI355X): 16384 x 4096 bf16 with residual, forward 83 us (402
// MB, 4.9 TB/s), backward 125 us (537 MB and 34 MB of parts, 4.6 TB/s) and 12
// us to join the parts; a copy of 1 GiB moves 5.2 TB/s, so memory bounds both.
// 16384 x 32 fp32: 3.6, 5.0 and 3.0 us, launches; 5001 x 1001 fp16: 10, 13 and
// 5 us.

// ------------------------- rows held in registers ------------------------- //
//
// kLanes threads hold a row, each kPacks vectors of 16 bytes, and the block
// passes over rows with the weights (and in the backward pass its columns'
// sums) in registers: every value is read once.  Below a wave's width a wave
// holds several rows.

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <int kLanes>
constexpr int kBlock = kLanes > kThreads ? kLanes : kThreads;

// both sums over the threads of a row.  `smem` alternates between rows, so
// that one barrier a row is enough.
template <int kLanes>
__device__ __forceinline__ void row_sums(float& x, float& y, float2* smem) {
#pragma unroll
  for (int off = (kLanes < 64 ? kLanes : 64) / 2; off > 0; off >>= 1) {
    x += __shfl_xor(x, off, 64);
    y += __shfl_xor(y, off, 64);
  }
  if constexpr (kLanes > 64) {
    if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = float2{x, y};
    __syncthreads();
    x = y = 0.f;
#pragma unroll
    for (int w = 0; w < kLanes / 64; ++w) {
      x += smem[w].x;
      y += smem[w].y;
    }
  }
}

// kPacks vectors of one row; columns from `width` on become zeros
template <typename T, typename U, int kLanes, int kPacks>
__device__ __forceinline__ void load_row(float (&dst)[kPacks][kVec<T>],
                                         const U* row, int lane, int width) {
#pragma unroll
  for (int p = 0; p < kPacks; ++p) {
    const int c = (p * kLanes + lane) * kVec<T>;
    U v[kVec<T>];
    if (c + kVec<T> <= width) {
      load_pack(v, row + c);
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i)
        v[i] = c + i < width ? row[c + i] : (U)0.f;
    }
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) dst[p][i] = (float)v[i];
  }
}

template <typename T, int kLanes, int kPacks>
__device__ __forceinline__ void store_row(
    T* row, const float (&src)[kPacks][kVec<T>], int lane, int width) {
#pragma unroll
  for (int p = 0; p < kPacks; ++p) {
    const int c = (p * kLanes + lane) * kVec<T>;
    T v[kVec<T>];
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) v[i] = (T)src[p][i];
    if (c + kVec<T> <= width) {
      store_pack(row + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i)
        if (c + i < width) row[c + i] = v[i];
    }
  }
}

template <typename T, int kLanes, int kPacks>
__device__ __forceinline__ void load_z_row(float (&z)[kPacks][kVec<T>],
                                           const NpfLayerNormArgs& a, long row,
                                           int lane) {
  load_row<T, T, kLanes>(z, static_cast<const T*>(a.x) + row * a.x_stride,
                         lane, a.width);
  if (a.residual) {
    float r[kPacks][kVec<T>];
    load_row<T, T, kLanes>(
        r, static_cast<const T*>(a.residual) + row * a.residual_stride, lane,
        a.width);
#pragma unroll
    for (int p = 0; p < kPacks; ++p)
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) z[p][i] += r[p][i];
  }
}

template <typename T, typename W, int kLanes, int kPacks>
__global__ void __launch_bounds__(kBlock<kLanes>)
    ln_fwd_rows(NpfLayerNormArgs a) {
  constexpr int V = kVec<T>, kRows = kBlock<kLanes> / kLanes;
  __shared__ float2 smem[2][kLanes / 64 + 1];
  const int lane = threadIdx.x % kLanes;
  float w[kPacks][V], b[kPacks][V];
  if (a.weight)
    load_row<T, W, kLanes>(w, static_cast<const W*>(a.weight), lane, a.width);
  if (a.bias)
    load_row<T, W, kLanes>(b, static_cast<const W*>(a.bias), lane, a.width);
  for (long row0 = (long)blockIdx.x * kRows; row0 < a.rows;
       row0 += (long)gridDim.x * kRows) {
    const long row = row0 + threadIdx.x / kLanes;
    const bool live = kRows == 1 || row < a.rows;
    float z[kPacks][V] = {};
    if (live) load_z_row<T, kLanes>(z, a, row, lane);
    float s = 0.f, unused = 0.f;
#pragma unroll
    for (int p = 0; p < kPacks; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) s += z[p][i];
    row_sums<kLanes>(s, unused, smem[0]);
    const float mean = s / a.width;
    s = 0.f;
#pragma unroll
    for (int p = 0; p < kPacks; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        z[p][i] -= mean;
        if ((p * kLanes + lane) * V + i < a.width) s += z[p][i] * z[p][i];
      }
    row_sums<kLanes>(s, unused, smem[1]);
    const float rstd = 1.f / sqrtf(s / a.width + a.eps);
    if (!live) continue;
#pragma unroll
    for (int p = 0; p < kPacks; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        z[p][i] *= rstd;
        if (a.weight) z[p][i] *= w[p][i];
        if (a.bias) z[p][i] += b[p][i];
      }
    store_row<T, kLanes>(static_cast<T*>(a.y) + row * a.width, z, lane,
                         a.width);
    if (lane == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, typename W, int kLanes, int kPacks>
__global__ void __launch_bounds__(kBlock<kLanes>)
    ln_bwd_rows(NpfLayerNormArgs a) {
  constexpr int V = kVec<T>, kRows = kBlock<kLanes> / kLanes;
  __shared__ float2 smem[2][kLanes / 64 + 1];
  const int lane = threadIdx.x % kLanes;
  float w[kPacks][V], dw[kPacks][V] = {}, db[kPacks][V] = {};
  if (a.weight)
    load_row<T, W, kLanes>(w, static_cast<const W*>(a.weight), lane, a.width);
  const float inv = 1.f / a.width;
  int turn = 0;
  for (long row0 = (long)blockIdx.x * kRows; row0 < a.rows;
       row0 += (long)gridDim.x * kRows, turn ^= 1) {
    const long row = row0 + threadIdx.x / kLanes;
    const bool live = kRows == 1 || row < a.rows;
    float h[kPacks][V] = {}, g[kPacks][V] = {};
    float mean = 0.f, rstd = 0.f;
    if (live) {
      load_z_row<T, kLanes>(h, a, row, lane);
      load_row<T, T, kLanes>(g, static_cast<const T*>(a.dy) + row * a.width,
                             lane, a.width);
      mean = a.mean[row];
      rstd = a.rstd[row];
    }
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int p = 0; p < kPacks; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[p][i] = (h[p][i] - mean) * rstd;
        // (behind the row's end g is zero, so h is of no account)
        dw[p][i] += g[p][i] * h[p][i];
        db[p][i] += g[p][i];
        if (a.weight) g[p][i] *= w[p][i];
        sg += g[p][i];
        sgh += g[p][i] * h[p][i];
      }
    if (!a.y) continue;
    row_sums<kLanes>(sg, sgh, smem[turn]);
    sg *= inv;
    sgh *= inv;
    if (!live) continue;
#pragma unroll
    for (int p = 0; p < kPacks; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i)
        g[p][i] = rstd * (g[p][i] - sg - h[p][i] * sgh);
    store_row<T, kLanes>(static_cast<T*>(a.y) + row * a.width, g, lane,
                         a.width);
  }
  if (!a.partial) return;
  // the block's sums over its rows: lanes of a wave that hold the same
  // columns, then the waves
  constexpr int kShared = kLanes < 256 ? kBlock<kLanes> / 64 : 1;
  constexpr int kCols = (kLanes < 64 ? kLanes : 64) * kPacks * V;
  __shared__ float cols[kShared > 1 ? kShared : 1][kShared > 1 ? kCols : 1];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* out = a.partial + (2L * blockIdx.x + k) * a.width;
    if constexpr (kShared == 1) {
#pragma unroll
      for (int p = 0; p < kPacks; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (p * kLanes + lane) * V + i;
          if (c < a.width) out[c] = k ? db[p][i] : dw[p][i];
        }
    } else {
      __syncthreads();
#pragma unroll
      for (int p = 0; p < kPacks; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float x = k ? db[p][i] : dw[p][i];
#pragma unroll
          for (int off = 32; off >= kLanes; off >>= 1)
            x += __shfl_xor(x, off, 64);
          if ((threadIdx.x & 63) < kLanes)
            cols[threadIdx.x >> 6][(p * kLanes + lane) * V + i] = x;
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += kBlock<kLanes>) {
        float x = cols[0][c];
#pragma unroll
        for (int s = 1; s < kShared; ++s) x += cols[s][c];
        out[c] = x;
      }
    }
  }
}

// ----------------------------- rows of any width -------------------------- //

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

// the parts' sums, in their order: 16 columns and 64 slices of the parts a
// block at a time, weight and bias in blocks of their own
__global__ void __launch_bounds__(1024) ln_dw_join(NpfLayerNormArgs a) {
  __shared__ float smem[64][17];
  const int cl = threadIdx.x & 15, slice = threadIdx.x >> 4;
  void* out = blockIdx.y == 0 ? a.dweight : a.dbias;
  if (!out) return;
  for (int c0 = blockIdx.x * 16; c0 < a.width; c0 += gridDim.x * 16) {
    const int c = c0 + cl;
    float s = 0.f;
    if (c < a.width)
#pragma unroll 4
      for (int p = slice; p < a.parts; p += 64)
        s += a.partial[(2L * p + blockIdx.y) * a.width + c];
    smem[slice][cl] = s;
    __syncthreads();
    if (slice == 0 && c < a.width) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < 64; ++i) s += smem[i][cl];
      store_coded(out, a.weight_type, c, s);
    }
    __syncthreads();
  }
}

// -------------------------------- dispatch -------------------------------- //

// Vectors of 16 bytes in a row decide: up to 64 of them, one a lane in the
// smallest group of lanes that holds the row; up to 256, a wave with up to
// kMost a lane; then 256 and 1024 threads.  Wider rows, and weights of a type
// that is neither the rows' nor fp32, take the loop.
template <typename T>
constexpr int kMost = sizeof(T) == 4 ? 4 : 2;  // 16 values a lane

constexpr int kLoop = 0;

struct Layout {
  int lanes, packs;
};

template <typename T>
Layout layout_of(int width) {
  const int vecs = (width + kVec<T> - 1) / kVec<T>;
  for (int lanes = 4; lanes <= 64; lanes *= 2)
    if (vecs <= lanes) return {lanes, 1};
  for (int lanes : {64, 256, 1024})
    for (int packs = 1; packs <= kMost<T>; packs *= 2)
      if (vecs <= lanes * packs) return {lanes, packs};
  return {kLoop, 0};
}

template <typename T>
unsigned blocks_of(Layout l, long rows, long most) {
  const long per = l.lanes > kThreads ? 1 : kThreads / l.lanes;
  const long n = (rows + per - 1) / per;
  return (unsigned)(n < most ? n : most);
}

// calls f with the layout as compile-time numbers
template <typename T, typename F>
void with_layout(Layout l, F f) {
#define NPF_CASE(L, P)                                             \
  if (l.lanes == L && l.packs == P) {                              \
    f(std::integral_constant<int, L>{}, std::integral_constant<int, P>{}); \
    return;                                                        \
  }
  NPF_CASE(4, 1) NPF_CASE(8, 1) NPF_CASE(16, 1) NPF_CASE(32, 1)
  NPF_CASE(64, 1) NPF_CASE(64, 2) NPF_CASE(256, 1) NPF_CASE(256, 2)
  NPF_CASE(1024, 1) NPF_CASE(1024, 2)
  if constexpr (kMost<T> == 4) {
    NPF_CASE(64, 4) NPF_CASE(256, 4) NPF_CASE(1024, 4)
  }
#undef NPF_CASE
}

// Blocks of a pass, and so parts of the weight's sums.  16384 x 4096 bf16 with
// 512, 1024, 2048 blocks: forward 136, 83, 87 us, backward with its join 180,
// 137, 170 us.
constexpr long kBlocks = 1024;
constexpr int kLoopParts = 128;
constexpr int kJoinColumns = 1 << 24;  // of a launch of ln_dw_join

template <typename T, typename W>
void fwd_rows(const NpfLayerNormArgs& a, Layout l, hipStream_t stream) {
  const unsigned n = blocks_of<T>(l, a.rows, kBlocks);
  with_layout<T>(l, [&](auto lanes, auto packs) {
    ln_fwd_rows<T, W, lanes(), packs()>
        <<<n, kBlock<lanes()>, 0, stream>>>(a);
  });
}

template <typename T, typename W>
void bwd_rows(const NpfLayerNormArgs& a, Layout l, hipStream_t stream) {
  const unsigned n = blocks_of<T>(l, a.rows, kBlocks);
  with_layout<T>(l, [&](auto lanes, auto packs) {
    ln_bwd_rows<T, W, lanes(), packs()>
        <<<n, kBlock<lanes()>, 0, stream>>>(a);
  });
}

template <typename T>
Layout layout_for(const NpfLayerNormArgs& a, int type) {
  if (a.weight_type != type && a.weight_type != NPF_F32) return {kLoop, 0};
  return layout_of<T>(a.width);
}

template <typename T>
hipError_t launch_fwd(const NpfLayerNormArgs& a, int type,
                      hipStream_t stream) {
  const Layout l = layout_for<T>(a, type);
  if (l.lanes == kLoop)
    ln_fwd_loop<T><<<blocks_of<T>({256, 1}, a.rows, 4096), kThreads, 0,
                     stream>>>(a);
  else if (a.weight_type == type)
    fwd_rows<T, T>(a, l, stream);
  else
    fwd_rows<T, float>(a, l, stream);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_bwd(const NpfLayerNormArgs& a, int type,
                      hipStream_t stream) {
  const Layout l = layout_for<T>(a, type);
  if (l.lanes != kLoop) {
    if (a.weight_type == type)
      bwd_rows<T, T>(a, l, stream);
    else
      bwd_rows<T, float>(a, l, stream);
  } else {
    if (a.y)
      ln_dx_loop<T><<<blocks_of<T>({256, 1}, a.rows, 4096), kThreads, 0,
                      stream>>>(a);
    if (a.partial)
      ln_dw_part<T><<<dim3((a.width + kThreads - 1) / kThreads, a.parts),
                      kThreads, 0, stream>>>(a);
  }
  if (a.partial) {
    // (a launch has fewer than 2^32 threads: the widest rows take turns)
    const unsigned n = a.width >= kJoinColumns ? kJoinColumns : a.width;
    ln_dw_join<<<dim3((n + 15) / 16, 2), 1024, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T>
int parts_of(const NpfLayerNormArgs& a, int type) {
  const Layout l = layout_for<T>(a, type);
  if (l.lanes == kLoop) return (int)(a.rows < kLoopParts ? a.rows : kLoopParts);
  return (int)blocks_of<T>(l, a.rows, kBlocks);
}

}  // namespace

int npf_layernorm_parts(const NpfLayerNormArgs& a, int type) {
  switch (type) {
    case NPF_F32: return parts_of<float>(a, type);
    case NPF_BF16: return parts_of<npf_bf16>(a, type);
    default: return parts_of<npf_f16>(a, type);
  }
}

hipError_t npf_layernorm_fwd(const NpfLayerNormArgs& a, int type,
                             hipStream_t stream) {
  switch (type) {
    case NPF_F32: return launch_fwd<float>(a, type, stream);
    case NPF_BF16: return launch_fwd<npf_bf16>(a, type, stream);
    case NPF_F16: return launch_fwd<npf_f16>(a, type, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t npf_layernorm_bwd(const NpfLayerNormArgs& a, int type,
                             hipStream_t stream) {
  switch (type) {
    case NPF_F32: return launch_bwd<float>(a, type, stream);
    case NPF_BF16: return launch_bwd<npf_bf16>(a, type, stream);
    case NPF_F16: return launch_bwd<npf_f16>(a, type, stream);
    default: return hipErrorInvalidValue;
  }
}
