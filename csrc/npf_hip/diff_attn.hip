// Differential attention: the difference of two softmax maps.
//
//   S_i = scale q_i k_i^T;  P_i = softmax(S_i);  O = (P_1 - lam P_2) V
//   G = dO V^T;  delta_i = rowsum(dO * (P_i V))
//   dS_1 = P_1 (G - delta_1);  dS_2 = -lam P_2 (G - delta_2)
//   dq_i = scale dS_i k_i;  dk_i = scale dS_i^T q_i
//   dV = (P_1 - lam P_2)^T dO;  dlam = -sum delta_2
//
// Statistics are kept in units of log2: P_i = exp2(S_i log2(e) - lse_i).

#include "common.h"
#include "diff_attn.h"
#include "types.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.0e38f;

template <typename T>
__device__ __forceinline__ T* row_of(const NpfHeads& t, int b, int h, long l) {
  return static_cast<T*>(t.p) + b * t.b + h * t.h + l * t.l;
}

__device__ __forceinline__ int keys_of(const NpfDiffAttnArgs& a, int b) {
  if (!a.lengths) return a.K;
  const long n = a.lengths64 ? static_cast<const long*>(a.lengths)[b]
                             : static_cast<const int*>(a.lengths)[b];
  return n < 0 ? 0 : n > a.K ? a.K : (int)n;
}

__device__ __forceinline__ float lam_of(const NpfDiffAttnArgs& a, int h) {
  return load_coded(a.lam, a.lam_type, (long)h * a.lam_stride);
}

// one wave a query row
template <typename T>
__global__ void __launch_bounds__(64) fwd_row(NpfDiffAttnArgs a) {
  __shared__ float sq[256];
  __shared__ float sp[2][64];
  const int lane = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / (a.H / a.Hk);
  const int n = keys_of(a, b);
  const float s2 = a.scale * kLog2e;
  for (long r = blockIdx.x; r < a.Q; r += gridDim.x) {
    __syncthreads();
    for (int d = lane; d < 2 * a.D; d += 64)
      sq[d] = (float)row_of<T>(a.q, b, h, r)[d];
    float m[2] = {kLowest, kLowest}, l[2] = {0.f, 0.f};
    float o[2][4] = {};
    for (int k0 = 0; k0 < n; k0 += 64) {
      __syncthreads();
      const int kn = n - k0 < 64 ? n - k0 : 64;
      for (int i = 0; i < 2; ++i) {
        float s = kLowest;
        if (lane < kn) {
          const T* kp = row_of<T>(a.k, b, hk, k0 + lane) + i * a.D;
          s = 0.f;
          for (int d = 0; d < a.D; ++d) s += sq[i * a.D + d] * (float)kp[d];
          s *= s2;
        }
        const float mn = fmaxf(m[i], wave_allreduce_max(s));
        const float p = lane < kn ? exp2f(s - mn) : 0.f;
        const float c = exp2f(m[i] - mn);
        l[i] = l[i] * c + wave_allreduce_sum(p);
        m[i] = mn;
        sp[i][lane] = p;
        for (int j = 0; j < 4; ++j) o[i][j] *= c;
      }
      __syncthreads();
      for (int k = 0; k < kn; ++k) {
        const T* vp = row_of<T>(a.v, b, hk, k0 + k);
        for (int j = 0; j < 4; ++j)
          if (lane + 64 * j < a.Dv) {
            const float v = (float)vp[lane + 64 * j];
            o[0][j] += sp[0][k] * v;
            o[1][j] += sp[1][k] * v;
          }
      }
    }
    const float lam = lam_of(a, h);
    for (int j = 0; j < 4; ++j)
      if (lane + 64 * j < a.Dv) {
        const float o1 = n ? o[0][j] / l[0] : 0.f;
        const float o2 = n ? o[1][j] / l[1] : 0.f;
        row_of<T>(a.out, b, h, r)[lane + 64 * j] = (T)(o1 - lam * o2);
        if (a.o2.p) row_of<T>(a.o2, b, h, r)[lane + 64 * j] = (T)o2;
      }
    if (a.lse && lane < 2)
      a.lse[(((long)b * a.H + h) * a.Q + r) * 2 + lane] =
          n ? m[lane] + log2f(l[lane]) : 0.f;
  }
}

// delta_i of a row a wave, and this block's part of dlam
template <typename T>
__global__ void __launch_bounds__(256) bwd_delta(NpfDiffAttnArgs a) {
  __shared__ double part[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int h = blockIdx.y, b = blockIdx.z;
  const float lam = lam_of(a, h);
  double sum = 0.;
  for (int i = 0; i < 16; ++i) {
    const long r = (long)blockIdx.x * 64 + w * 16 + i;
    if (r >= a.Q) break;
    float d1 = 0.f, d2 = 0.f;
    for (int c = lane; c < a.Dv; c += 64) {
      const float g = (float)row_of<T>(a.dout, b, h, r)[c];
      const float o2 = (float)row_of<T>(a.o2, b, h, r)[c];
      d1 += g * ((float)row_of<T>(a.out, b, h, r)[c] + lam * o2);
      d2 += g * o2;
    }
    d1 = wave_allreduce_sum(d1);
    d2 = wave_allreduce_sum(d2);
    if (lane == 0) {
      float* p = a.delta + (((long)b * a.H + h) * a.Q + r) * 2;
      p[0] = d1;
      p[1] = d2;
    }
    sum += d2;
  }
  if (lane == 0) part[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    a.dlam_partial[((long)b * a.H + h) * a.parts + blockIdx.x] =
        part[0] + part[1] + part[2] + part[3];
}

// dlam of one head (of all heads where lam is one number)
__global__ void __launch_bounds__(256) bwd_dlam(NpfDiffAttnArgs a,
                                                int heads) {
  __shared__ double smem[256];
  double s = 0.;
  const long per = (long)heads * a.parts;
  for (long i = threadIdx.x; i < a.B * per; i += 256) {
    const long b = i / per, j = i % per;
    s += a.dlam_partial[(b * a.H + blockIdx.x * heads) * a.parts + j];
  }
  smem[threadIdx.x] = s;
  __syncthreads();
  for (int n = 128; n > 0; n >>= 1) {
    if (threadIdx.x < n) smem[threadIdx.x] += smem[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) store_coded(a.dlam, a.lam_type, blockIdx.x, -smem[0]);
}

// one wave a query row
template <typename T>
__global__ void __launch_bounds__(64) bwd_dq_row(NpfDiffAttnArgs a) {
  __shared__ float sq[256], sg[256];
  __shared__ float sd[2][64];
  const int lane = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / (a.H / a.Hk);
  const int n = keys_of(a, b);
  const float lam = lam_of(a, h);
  for (long r = blockIdx.x; r < a.Q; r += gridDim.x) {
    __syncthreads();
    for (int d = lane; d < 2 * a.D; d += 64)
      sq[d] = (float)row_of<T>(a.q, b, h, r)[d];
    for (int d = lane; d < a.Dv; d += 64)
      sg[d] = (float)row_of<T>(a.dout, b, h, r)[d];
    const long st = (((long)b * a.H + h) * a.Q + r) * 2;
    float dq[4] = {};
    for (int k0 = 0; k0 < n; k0 += 64) {
      __syncthreads();
      const int kn = n - k0 < 64 ? n - k0 : 64;
      float ds[2] = {0.f, 0.f};
      if (lane < kn) {
        const T* kp = row_of<T>(a.k, b, hk, k0 + lane);
        const T* vp = row_of<T>(a.v, b, hk, k0 + lane);
        float g = 0.f, s[2] = {0.f, 0.f};
        for (int d = 0; d < a.Dv; ++d) g += sg[d] * (float)vp[d];
        for (int i = 0; i < 2; ++i) {
          for (int d = 0; d < a.D; ++d)
            s[i] += sq[i * a.D + d] * (float)kp[i * a.D + d];
          const float p = exp2f(s[i] * a.scale * kLog2e - a.lse[st + i]);
          ds[i] = p * (g - a.delta[st + i]) * (i ? -lam : 1.f) * a.scale;
        }
      }
      sd[0][lane] = ds[0];
      sd[1][lane] = ds[1];
      __syncthreads();
      for (int k = 0; k < kn; ++k) {
        const T* kp = row_of<T>(a.k, b, hk, k0 + k);
        for (int j = 0; j < 4; ++j) {
          const int d = lane + 64 * j;
          if (d < 2 * a.D) dq[j] += sd[d >= a.D][k] * (float)kp[d];
        }
      }
    }
    for (int j = 0; j < 4; ++j)
      if (lane + 64 * j < 2 * a.D)
        row_of<T>(a.dq, b, h, r)[lane + 64 * j] = (T)dq[j];
  }
}

// one wave a key row
template <typename T>
__global__ void __launch_bounds__(64) bwd_dkv_row(NpfDiffAttnArgs a) {
  __shared__ float sk[256], sv[256];
  __shared__ float sd[3][64];
  const int lane = threadIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int group = a.H / a.Hk;
  const int n = keys_of(a, b);
  for (long r = blockIdx.x; r < a.K; r += gridDim.x) {
    __syncthreads();
    for (int d = lane; d < 2 * a.D; d += 64)
      sk[d] = (float)row_of<T>(a.k, b, hk, r)[d];
    for (int d = lane; d < a.Dv; d += 64)
      sv[d] = (float)row_of<T>(a.v, b, hk, r)[d];
    float dk[4] = {}, dv[4] = {};
    for (int h = hk * group; r < n && h < (hk + 1) * group; ++h) {
      const float lam = lam_of(a, h);
      for (int q0 = 0; q0 < a.Q; q0 += 64) {
        __syncthreads();
        const int qn = a.Q - q0 < 64 ? a.Q - q0 : 64;
        float ds[2] = {0.f, 0.f}, p[2] = {0.f, 0.f};
        if (lane < qn) {
          const long st = (((long)b * a.H + h) * a.Q + q0 + lane) * 2;
          const T* qp = row_of<T>(a.q, b, h, q0 + lane);
          const T* gp = row_of<T>(a.dout, b, h, q0 + lane);
          float g = 0.f, s[2] = {0.f, 0.f};
          for (int d = 0; d < a.Dv; ++d) g += sv[d] * (float)gp[d];
          for (int i = 0; i < 2; ++i) {
            for (int d = 0; d < a.D; ++d)
              s[i] += sk[i * a.D + d] * (float)qp[i * a.D + d];
            p[i] = exp2f(s[i] * a.scale * kLog2e - a.lse[st + i]);
            ds[i] = p[i] * (g - a.delta[st + i]) * (i ? -lam : 1.f) * a.scale;
          }
        }
        sd[0][lane] = ds[0];
        sd[1][lane] = ds[1];
        sd[2][lane] = p[0] - lam * p[1];
        __syncthreads();
        for (int q = 0; q < qn; ++q) {
          const T* qp = row_of<T>(a.q, b, h, q0 + q);
          const T* gp = row_of<T>(a.dout, b, h, q0 + q);
          for (int j = 0; j < 4; ++j) {
            const int d = lane + 64 * j;
            if (d < 2 * a.D) dk[j] += sd[d >= a.D][q] * (float)qp[d];
            if (d < a.Dv) dv[j] += sd[2][q] * (float)gp[d];
          }
        }
      }
    }
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 64 * j;
      if (a.dk.p && d < 2 * a.D) row_of<T>(a.dk, b, hk, r)[d] = (T)dk[j];
      if (a.dv.p && d < a.Dv) row_of<T>(a.dv, b, hk, r)[d] = (T)dv[j];
    }
  }
}

unsigned rows_grid(int rows) { return rows < 65536 ? rows : 65536; }

template <typename T>
hipError_t launch_bwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  bwd_delta<T><<<dim3(a.parts, a.H, a.B), 256, 0, stream>>>(a);
  if (a.dlam) {
    bwd_dlam<<<a.lam_heads, 256, 0, stream>>>(a, a.H / a.lam_heads);
  }
  if (a.dq.p)
    bwd_dq_row<T><<<dim3(rows_grid(a.Q), a.H, a.B), 64, 0, stream>>>(a);
  if (a.dk.p || a.dv.p)
    bwd_dkv_row<T><<<dim3(rows_grid(a.K), a.Hk, a.B), 64, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

int npf_diff_attn_parts(int Q) { return (Q + 63) / 64; }

hipError_t npf_diff_attn_fwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  const dim3 grid(rows_grid(a.Q), a.H, a.B);
  switch (a.type) {
    case NPF_F32: fwd_row<float><<<grid, 64, 0, stream>>>(a); break;
    case NPF_BF16: fwd_row<npf_bf16><<<grid, 64, 0, stream>>>(a); break;
    case NPF_F16: fwd_row<npf_f16><<<grid, 64, 0, stream>>>(a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t npf_diff_attn_bwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  switch (a.type) {
    case NPF_F32: return launch_bwd<float>(a, stream);
    case NPF_BF16: return launch_bwd<npf_bf16>(a, stream);
    case NPF_F16: return launch_bwd<npf_f16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}
