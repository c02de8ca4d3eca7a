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

// Join of a split forward pass.  Many splits (few rows): one block a row, 4
// slices of the splits, each over both maps' values.
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
    row_of<T>(a.out, b, h, q)[t] =
        (T)(any ? o[0] - lam_of(a, h) * o[1] : 0.f);
    if (a.o2.p) row_of<T>(a.o2, b, h, q)[t] = (T)o[1];
  }
  if (a.lse && t < 2)
    a.lse[(((long)b * a.H + h) * a.Q + q) * 2 + t] =
        any ? top[t] + __log2f(weight_sum[t]) : 0.f;
}

// Few splits (many rows): kLanes lanes of 4 values a row.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) join_rows(NpfDiffAttnArgs a) {
  const unsigned rows = (unsigned)a.B * a.H * a.Q;
  const unsigned r = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= rows) return;
  const unsigned each = (unsigned)(a.H / a.Hk) * a.Q;
  const int row = (int)(r % each), bh = (int)(r / each);
  const int b = bh / a.Hk;
  const int h = bh % a.Hk * (a.H / a.Hk) + row / a.Q, q = row % a.Q;
  const int c = (threadIdx.x % kLanes) * 4;
  const int count = a.Dv - c < 4 ? a.Dv - c : 4;
  const long step = split_row_floats(a.Dv);
  const float* w = static_cast<const float*>(a.split) + (long)r * a.splits * step;
  float mx[2] = {kLowest, kLowest}, l[2] = {0.f, 0.f}, o[2][4] = {};
  for (int s = 0; s < a.splits; ++s)
    for (int m = 0; m < 2; ++m) mx[m] = fmaxf(mx[m], w[s * step + 2 * m]);
  for (int s = 0; s < a.splits; ++s)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float* p = w + s * step;
      const float f = exp2f(p[2 * m] - mx[m]);
      l[m] += f * p[2 * m + 1];
      float v[4] = {};
      if (count == 4)
        load_pack(v, p + 4 + m * a.Dv + c);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < count) v[i] = p[4 + m * a.Dv + c + i];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[m][i] += f * v[i];
    }
  const bool any = keys_of(a, b) > 0;
  const float lam = lam_of(a, h);
  float x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = any ? o[1][i] / l[1] : 0.f;
    x[i] = any ? o[0][i] / l[0] - lam * y[i] : 0.f;
  }
  if (count > 0) {
    store4(row_of<T>(a.out, b, h, q) + c, count, x[0], x[1], x[2], x[3]);
    if (a.o2.p)
      store4(row_of<T>(a.o2, b, h, q) + c, count, y[0], y[1], y[2], y[3]);
  }
  if (a.lse && c == 0) {
    float* p = a.lse + (((long)b * a.H + h) * a.Q + q) * 2;
    for (int m = 0; m < 2; ++m) p[m] = any ? mx[m] + __log2f(l[m]) : 0.f;
  }
}

// Sum of the parts of a split gradient, in their order: rows of `size` values.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256)
    join_grads(NpfHeads out, const float* part, int B, int H, int L, int size,
               int splits) {
  const unsigned rows = (unsigned)B * H * L;
  const unsigned r = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= rows) return;
  const int l = (int)(r % (unsigned)L), bh = (int)(r / (unsigned)L);
  const int c = (threadIdx.x % kLanes) * 4;
  const int count = size - c < 4 ? size - c : 4;
  if (count <= 0) return;
  float x[4] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float* p = part + ((long)s * rows + r) * size + c;
    float v[4] = {};
    if (count == 4)
      load_pack(v, p);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < count) v[i] = p[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += v[i];
  }
  store4(row_of<T>(out, bh / H, bh % H, l) + c, count, x[0], x[1], x[2], x[3]);
}

// For gradients of keys and values alone, without the dq kernel that would
// leave them: delta_i of each row, beside its lse: kLanes lanes of 4 values a row
template <typename T, int kLanes>
__global__ void __launch_bounds__(256)
    row_stats(NpfDiffAttnArgs a, unsigned first) {
  // (rows are checked to fit 31 bits; divisions of 64 bits would cost more
  // than the sums)
  const unsigned rows = (unsigned)a.B * a.H * a.Q;
  const unsigned r = first + blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
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
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < a.Dv) {
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

// The largest norm of a chunk of rows of values, or of dout times the larger of
// 1 and |lam|; keys that are not there, and rows without keys, do not count.
// (A NaN is left out: it makes every gradient that its row meets NaN.)
// Measured: 16 x 4 heads, 1024 x 1024, maps of 16: 6 us of a step of 141; 2 x 16
// heads on 4, 4096 x 4096, maps of 64: 22 us (48 MB) of 1835.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) row_reach(NpfDiffAttnArgs a) {
  __shared__ float smem[4];
  const int heads = a.B * a.Hk, bh = blockIdx.x % heads;
  const int chunk = blockIdx.x / heads, b = bh / a.Hk, hk = bh % a.Hk;
  const int group = a.H / a.Hk, n = keys_of(a, b);
  const bool of_values = chunk < a.v_chunks;
  const int step = of_values ? a.v_rows : a.o_rows;
  const int row0 = (of_values ? chunk : chunk - a.v_chunks) * step;
  int rows = of_values ? n : n > 0 ? group * a.Q : 0;
  rows = rows - row0 < step ? rows : row0 + step;
  const int c = (threadIdx.x % kLanes) * 4;
  const int count = a.Dv - c < 4 ? a.Dv - c : 4;
  constexpr int kEach = kReachRows * kLanes / 256;
  float most = 0.f;
  for (int at = row0; at < rows; at += kReachRows) {
    // every row's loads before the first sum: one wait for memory, not one a row
    T v[kEach][4] = {};
    float weight[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int row = at + i * (256 / kLanes) + threadIdx.x / kLanes;
      weight[i] = 1.f;
      if (row >= rows) continue;
      const int h = of_values ? hk : hk * group + row / a.Q;
      const T* p = (of_values ? row_of<T>(a.v, b, h, row)
                              : row_of<T>(a.dout, b, h, row % a.Q)) + c;
      if (!of_values) weight[i] = fmaxf(1.f, fabsf(lam_of(a, h)));
      if (count == 4) {
        load_pack(v[i], p);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < count) v[i][e] = p[e];
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (float)v[i][e] * (float)v[i][e];
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1)
        s += __shfl_xor(s, off, 64);
      most = fmaxf(most, sqrtf(s) * weight[i]);
    }
  }
  most = wave_allreduce_max(most);
  if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0)
    a.reach[(long)bh * (a.v_chunks + a.o_chunks) + chunk] =
        fmaxf(fmaxf(smem[0], smem[1]), fmaxf(smem[2], smem[3]));
}

// dlam of one head after the other (of all heads where lam is one number)
constexpr int kDlamBlocks = 1 << 20;

__global__ void __launch_bounds__(1024) sum_dlam(NpfDiffAttnArgs a,
                                                 int heads) {
  __shared__ double smem[1024];
  // (sizes are checked to fit 31 bits)
  const unsigned per = (unsigned)heads * a.Q;
  const unsigned all = (unsigned)a.dq_splits * a.B * per;
  for (int h = blockIdx.x; h < a.lam_heads; h += gridDim.x) {
    double s = 0.;
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < all; i += 1024)
      s += a.dlam_rows[(long)(i / per * a.H + h * heads) * a.Q + i % per];
    smem[threadIdx.x] = s;
    __syncthreads();
    for (int n = 512; n > 0; n >>= 1) {
      if (threadIdx.x < n) smem[threadIdx.x] += smem[threadIdx.x + n];
      __syncthreads();
    }
    if (threadIdx.x == 0) store_coded(a.dlam, a.lam_type, h, -smem[0]);
    __syncthreads();
  }
}

// lanes of 4 values for a row of `size`, as a compile-time number
template <typename F>
void with_lanes(int size, F f) {
  if (size <= 32)
    f(std::integral_constant<int, 8>{});
  else if (size <= 64)
    f(std::integral_constant<int, 16>{});
  else if (size <= 128)
    f(std::integral_constant<int, 32>{});
  else
    f(std::integral_constant<int, 64>{});
}

unsigned row_blocks(long rows, int lanes) {
  return (unsigned)((rows * lanes + 255) / 256);
}

// whether a split pass has so many parts that a block joins one row
bool many(int splits) { return splits > 8; }

template <typename T>
hipError_t join_forward(const NpfDiffAttnArgs& a, hipStream_t stream) {
  const long rows = (long)a.B * a.H * a.Q;
  if (many(a.splits))
    join<T><<<(unsigned)rows, kJoinThreads, 0, stream>>>(a);
  else
    with_lanes(a.Dv, [&](auto lanes) {
      join_rows<T, lanes()>
          <<<row_blocks(rows, lanes()), 256, 0, stream>>>(a);
    });
  return hipGetLastError();
}

template <typename T>
void stats(const NpfDiffAttnArgs& a, hipStream_t stream) {
  if (a.dq.p || a.dlam) return;
  // (a launch has fewer than 2^32 threads: of 2^25 rows 64 lanes at most)
  const long rows = (long)a.B * a.H * a.Q;
  for (long first = 0; first < rows; first += 1L << 25) {
    const long some = rows - first < 1L << 25 ? rows - first : 1L << 25;
    with_lanes(a.Dv, [&](auto lanes) {
      row_stats<T, lanes()><<<row_blocks(some, lanes()), 256, 0, stream>>>(
          a, (unsigned)first);
    });
  }
}

template <typename T>
void reach(const NpfDiffAttnArgs& a, hipStream_t stream) {
  if constexpr (kScaledGrads<T>)
    with_lanes(a.Dv, [&](auto lanes) {
      row_reach<T, lanes()>
          <<<(unsigned)a.B * a.Hk * (a.v_chunks + a.o_chunks), 256, 0, stream>>>(
              a);
    });
}

template <typename T>
void join_one(const NpfHeads& out, const float* part, int B, int H, int L,
              int size, int splits, hipStream_t stream) {
  if (!out.p || splits == 1) return;
  with_lanes(size, [&](auto lanes) {
    join_grads<T, lanes()><<<row_blocks((long)B * H * L, lanes()), 256, 0,
                             stream>>>(out, part, B, H, L, size, splits);
  });
}

template <typename T>
hipError_t join_backward(const NpfDiffAttnArgs& a, hipStream_t stream) {
  join_one<T>(a.dq, a.dq_part, a.B, a.H, a.Q, 2 * a.D, a.dq_splits, stream);
  join_one<T>(a.dk, a.dk_part, a.B, a.Hk, a.K, 2 * a.D, a.dkv_splits, stream);
  join_one<T>(a.dv, a.dv_part, a.B, a.Hk, a.K, a.Dv, a.dkv_splits, stream);
  return hipGetLastError();
}

// Parts of an axis of `length` so that `blocks` become as many as the chip holds;
// none shorter than `least`, whose work would not pay for the join.
int parts_for(long blocks, long wanted, int length, int least) {
  if (blocks <= 0 || 2 * blocks > wanted) return 1;
  const long most = length / least;
  const long n = wanted / blocks;
  return (int)(n < most ? (n < 1 ? 1 : n) : (most < 1 ? 1 : most));
}

}  // namespace

bool npf_diff_attn_plan(NpfDiffAttnArgs& a) {
  for (a.pad = 16; a.pad < a.D || 2 * a.pad < a.Dv; a.pad *= 2)
    if (a.pad == 128) return false;
  const long rows = (long)(a.H / a.Hk) * a.Q;
  const long heads = (long)a.B * a.Hk;
  // Rows that fit one wave get a block of one wave, the others share tiles
  // between four.
  a.waves = rows <= 32 ? 1 : 4;
  // Blocks that the chip holds at once: of one wave by their LDS (4 tiles of
  // 32 or 64 rows), of more by their registers (see kResident, kFwdResident).
  const int row_bytes = 2 * a.pad * (a.type == NPF_F32 ? 4 : 2);
  const long wanted1 = row_bytes <= 256 ? 1280 : row_bytes == 512 ? 512 : 256;
  const long wanted = row_bytes <= 256 ? 512 : 256;
  const long row_blocks4 = heads * ((rows + 127) / 128);
  // (fp32 products are worth a join from 128 keys on: 8 x 8 heads of 96, 256 x
  // 256, 92 us to 81)
  a.splits = a.waves == 1 ? parts_for(heads, wanted1, a.K, 64)
                          : parts_for(row_blocks4, wanted, a.K,
                                      a.type == NPF_F32 ? 128 : 256);
  a.dq_splits = parts_for(row_blocks4, wanted, a.K, 256);
  a.dkv_splits =
      parts_for(heads * ((a.K + 127) / 128), wanted, (int)rows, 256);
  if (a.type == NPF_F16) {
    // no more than 1024 chunks, as every block reads them all (2 heads of 64, 4 x
    // 1000000, a step: with up to 256 chunks 1731 us, 1024 1508, 15625 1966; the
    // same in bf16, which needs none, 1308)
    auto chunks = [](int n, int* each) {
      const int steps = (n + kReachRows - 1) / kReachRows;
      *each = (steps + 1023) / 1024 * kReachRows;
      return *each ? (n + *each - 1) / *each : 0;
    };
    a.v_chunks = chunks(a.K, &a.v_rows);
    a.o_chunks = chunks((int)rows, &a.o_rows);
  }
  return true;
}

bool npf_diff_attn_fits(const NpfDiffAttnArgs& a, bool backward) {
  const long rows = (long)(a.H / a.Hk) * a.Q, heads = (long)a.B * a.Hk;
  const long tiles = heads * ((rows + 127) / 128);
  auto fits = [](long blocks, long threads) {
    return blocks <= 0xffffffffL / threads;
  };
  // (joins are of few rows: parts are planned where blocks are few)
  if (!backward)
    return a.waves == 1 ? fits(heads * a.splits * ((rows + 31) / 32), 128)
                        : fits(tiles * a.splits, 512);
  return fits(tiles * a.dq_splits, 256) &&
         fits(heads * ((a.K + 127) / 128) * a.dkv_splits, 256) &&
         fits(heads * ((long)a.v_chunks + a.o_chunks), 256);
}

long npf_diff_attn_workspace(const NpfDiffAttnArgs& a) {
  if (a.splits <= 1) return 0;
  return split_row_floats(a.Dv) * a.splits * a.B * a.H * a.Q;
}

hipError_t npf_diff_attn_fwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  if ((long)a.B * a.H * a.Q > 0x7fffffffL) return hipErrorInvalidConfiguration;
  hipError_t e = hipErrorInvalidValue;
  switch (a.type) {
    case NPF_F32: e = npf_diff_attn_fwd_f32(a, stream); break;
    case NPF_BF16: e = npf_diff_attn_fwd_bf16(a, stream); break;
    case NPF_F16: e = npf_diff_attn_fwd_f16(a, stream); break;
  }
  if (e != hipSuccess || a.splits <= 1) return e;
  switch (a.type) {
    case NPF_F32: return join_forward<float>(a, stream);
    case NPF_BF16: return join_forward<npf_bf16>(a, stream);
    default: return join_forward<npf_f16>(a, stream);
  }
}

hipError_t npf_diff_attn_bwd(const NpfDiffAttnArgs& a, hipStream_t stream) {
  if ((long)a.dq_splits * a.B * a.H * a.Q > 0x7fffffffL ||
      (long)a.B * a.Hk * a.K > 0x7fffffffL ||
      (long)a.B * a.Hk * (a.v_chunks + a.o_chunks) > 0x7fffffffL)
    return hipErrorInvalidConfiguration;
  hipError_t e = hipErrorInvalidValue;
  switch (a.type) {
    case NPF_F32:
      stats<float>(a, stream);
      e = npf_diff_attn_bwd_f32(a, stream);
      if (e == hipSuccess) e = join_backward<float>(a, stream);
      break;
    case NPF_BF16:
      stats<npf_bf16>(a, stream);
      e = npf_diff_attn_bwd_bf16(a, stream);
      if (e == hipSuccess) e = join_backward<npf_bf16>(a, stream);
      break;
    case NPF_F16:
      reach<npf_f16>(a, stream);
      stats<npf_f16>(a, stream);
      e = npf_diff_attn_bwd_f16(a, stream);
      if (e == hipSuccess) e = join_backward<npf_f16>(a, stream);
      break;
  }
  if (e != hipSuccess || !a.dlam) return e;
  // (a launch has fewer than 2^32 threads)
  const int blocks = a.lam_heads <= kDlamBlocks ? a.lam_heads : kDlamBlocks;
  sum_dlam<<<blocks, 1024, 0, stream>>>(a, a.H / a.lam_heads);
  return hipGetLastError();
}
