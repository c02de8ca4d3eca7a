// Differential attention: the plan, the join of a split key axis, and the
// backward pass's row sums.  The products are in diff_attn_impl.h.

#include "diff_attn_impl.h"

hipError_t npf_diff_attn_fwd_f32(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_fwd_bf16(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_fwd_f16(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_bwd_f32(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_bwd_bf16(const NpfDiffAttnArgs&, hipStream_t);
hipError_t npf_diff_attn_bwd_f16(const NpfDiffAttnArgs&, hipStream_t);

namespace {

using namespace npf_attn;

// one block a row: 4 slices of the splits, each over both maps' values
constexpr int kJoinThreads = 1024;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join(NpfDiffAttnArgs a) {
  __shared__ float part[4][2][256];
  __shared__ float weight_sum[2];
  const int group = a.H / a.Hk, rows = group * a.Q;
  const int row = blockIdx.x % rows, bh = blockIdx.x / rows;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int h = hk * group + row / a.Q, q = row % a.Q;
  const long step = split_row_floats(a.Dv);
  const float* w = static_cast<const float*>(a.split) +
                   (long)blockIdx.x * a.splits * step;
  const int slice = threadIdx.x >> 8, t = threadIdx.x & 255;
  float top[2] = {kLowest, kLowest};
  for (int s = threadIdx.x & 63; s < a.splits; s += 64)
    for (int m = 0; m < 2; ++m) top[m] = fmaxf(top[m], w[s * step + 2 * m]);
  for (int m = 0; m < 2; ++m) top[m] = wave_allreduce_max(top[m]);
  if (threadIdx.x < 64) {
    for (int m = 0; m < 2; ++m) {
      float l = 0.f;
      for (int s = threadIdx.x; s < a.splits; s += 64)
        l += exp2f(w[s * step + 2 * m] - top[m]) * w[s * step + 2 * m + 1];
      l = wave_allreduce_sum(l);
      if (threadIdx.x == 0) weight_sum[m] = l;
    }
  }
  float o[2] = {0.f, 0.f};
  if (t < a.Dv) {
#pragma unroll 4
    for (int s = slice; s < a.splits; s += 4)
#pragma unroll
      for (int m = 0; m < 2; ++m)
        o[m] += exp2f(w[s * step + 2 * m] - top[m]) *
                w[s * step + 4 + m * a.Dv + t];
  }
  part[slice][0][t] = o[0];
  part[slice][1][t] = o[1];
  __syncthreads();
  if (slice > 0) return;
  const bool any = keys_of(a, b) > 0;
  if (t < a.Dv) {
    for (int m = 0; m < 2; ++m) {
      o[m] = part[0][m][t] + part[1][m][t] + part[2][m][t] + part[3][m][t];
      o[m] = any ? o[m] / weight_sum[m] : 0.f;
    }
    row_of<T>(a.out, b, h, q)[t] = (T)(o[0] - lam_of(a, h) * o[1]);
    if (a.o2.p) row_of<T>(a.o2, b, h, q)[t] = (T)o[1];
  }
  if (a.lse && t < 2)
    a.lse[(((long)b * a.H + h) * a.Q + q) * 2 + t] =
        any ? top[t] + __log2f(weight_sum[t]) : 0.f;
}

// delta_i of each row, beside its lse: kLanes lanes of 4 values a row
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) row_stats(NpfDiffAttnArgs a) {
  // (rows are checked to fit 31 bits; divisions of 64 bits would cost more
  // than the sums)
  const unsigned rows = (unsigned)a.B * a.H * a.Q;
  const unsigned r = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= rows) return;  // whole groups of lanes
  const int q = (int)(r % (unsigned)a.Q), bh = (int)(r / (unsigned)a.Q);
  const int h = bh % a.H, b = bh / a.H;
  const int c = (threadIdx.x % kLanes) * 4;
  const float lam = lam_of(a, h);
  float d1 = 0.f, d2 = 0.f;
  if (c < a.Dv) {
    const T* gp = row_of<T>(a.dout, b, h, q) + c;
    const T* op = row_of<T>(a.out, b, h, q) + c;
    const T* sp = row_of<T>(a.o2, b, h, q) + c;
    T g[4] = {}, o[4] = {}, s[4] = {};
    if (c + 4 <= a.Dv) {
      load_pack(g, gp);
      load_pack(o, op);
      load_pack(s, sp);
    } else {
      for (int i = 0; c + i < a.Dv; ++i) {
        g[i] = gp[i];
        o[i] = op[i];
        s[i] = sp[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d1 += (float)g[i] * ((float)o[i] + lam * (float)s[i]);
      d2 += (float)g[i] * (float)s[i];
    }
  }
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) {
    d1 += __shfl_xor(d1, off, 64);
    d2 += __shfl_xor(d2, off, 64);
  }
  if (threadIdx.x % kLanes == 0)
    reinterpret_cast<float4*>(a.stats)[r] =
        float4{a.lse[2L * r], a.lse[2L * r + 1], d1, d2};
}

// dlam of one head (of all heads where lam is one number)
__global__ void __launch_bounds__(1024) sum_dlam(NpfDiffAttnArgs a,
                                                 int heads) {
  __shared__ double smem[1024];
  double s = 0.;
  const long per = (long)heads * a.Q;
#pragma unroll 4
  for (long i = threadIdx.x; i < a.B * per; i += 1024)
    s += a.dlam_rows[(i / per * a.H + blockIdx.x * heads) * a.Q + i % per];
  smem[threadIdx.x] = s;
  __syncthreads();
  for (int n = 512; n > 0; n >>= 1) {
    if (threadIdx.x < n) smem[threadIdx.x] += smem[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) store_coded(a.dlam, a.lam_type, blockIdx.x, -smem[0]);
}

template <typename T>
void launch_row_stats(const NpfDiffAttnArgs& a, hipStream_t stream) {
  const long rows = (long)a.B * a.H * a.Q;
  auto blocks = [&](int lanes) {
    return (unsigned)((rows * lanes + 255) / 256);
  };
  if (a.Dv <= 32)
    row_stats<T, 8><<<blocks(8), 256, 0, stream>>>(a);
  else if (a.Dv <= 64)
    row_stats<T, 16><<<blocks(16), 256, 0, stream>>>(a);
  else if (a.Dv <= 128)
    row_stats<T, 32><<<blocks(32), 256, 0, stream>>>(a);
  else
    row_stats<T, 64><<<blocks(64), 256, 0, stream>>>(a);
}

}  // namespace

bool npf_diff_attn_plan(NpfDiffAttnArgs& a) {
  for (a.pad = 16; a.pad < a.D || 2 * a.pad < a.Dv; a.pad *= 2)
    if (a.pad == 128) return false;
  const long rows = (long)(a.H / a.Hk) * a.Q;
  const long heads = (long)a.B * a.Hk;
  a.waves = heads * ((rows + 127) / 128) >= kManyBlocks ? 4 : 1;
  // Few rows: the key axis is split until every SIMD has a wave, no part
  // below 256 keys.
  const long waves = heads * ((rows + 31) / 32);
  const long most = (a.K + 255) / 256;
  long splits = a.waves == 1 && waves > 0 && waves < 512 ? 1280 / waves : 1;
  splits = splits > most ? most : splits;
  a.splits = (int)(splits < 1 ? 1 : splits);
  return true;
}

size_t npf_diff_attn_workspace(const NpfDiffAttnArgs& a) {
  if (a.splits <= 1) return 0;
  return sizeof(float) * a.splits * split_row_floats(a.Dv) * a.B * a.H * a.Q;
}

hipError_t npf_diff_attn_fwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  hipError_t e = hipErrorInvalidValue;
  switch (a.type) {
    case NPF_F32: e = npf_diff_attn_fwd_f32(a, stream); break;
    case NPF_BF16: e = npf_diff_attn_fwd_bf16(a, stream); break;
    case NPF_F16: e = npf_diff_attn_fwd_f16(a, stream); break;
  }
  if (e != hipSuccess || a.splits <= 1) return e;
  const long rows = (long)a.B * a.H * a.Q;
  if (rows > 0x7fffffffL) return hipErrorInvalidConfiguration;
  switch (a.type) {
    case NPF_F32: join<float><<<(unsigned)rows, kJoinThreads, 0, stream>>>(a); break;
    case NPF_BF16: join<npf_bf16><<<(unsigned)rows, kJoinThreads, 0, stream>>>(a); break;
    default: join<npf_f16><<<(unsigned)rows, kJoinThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

hipError_t npf_diff_attn_bwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  if ((long)a.B * a.H * a.Q > 0x7fffffffL) return hipErrorInvalidConfiguration;
  hipError_t e = hipErrorInvalidValue;
  switch (a.type) {
    case NPF_F32:
      launch_row_stats<float>(a, stream);
      e = npf_diff_attn_bwd_f32(a, stream);
      break;
    case NPF_BF16:
      launch_row_stats<npf_bf16>(a, stream);
      e = npf_diff_attn_bwd_bf16(a, stream);
      break;
    case NPF_F16:
      launch_row_stats<npf_f16>(a, stream);
      e = npf_diff_attn_bwd_f16(a, stream);
      break;
  }
  if (e != hipSuccess || !a.dlam) return e;
  sum_dlam<<<a.lam_heads, 1024, 0, stream>>>(a, a.H / a.lam_heads);
  return hipGetLastError();
}
