// The differential attention kernels, for one type and padded size.
//
//   S_i = scale q_i k_i^T;  P_i = softmax(S_i);  O = (P_1 - lam P_2) V
//   G = dO V^T;  delta_i = rowsum(dO * (P_i V))
//   dS_1 = P_1 (G - delta_1);  dS_2 = -lam P_2 (G - delta_2)
//   dq_i = scale dS_i k_i;  dk_i = scale dS_i^T q_i
//   dV = (P_1 - lam P_2)^T dO;  dlam = -sum P_2 * G
//
// Scores are held in units of log2: P_i = exp2(S_i log2(e) - lse_i).  The rows
// of one key head are its group's query heads one after the other, so heads
// that share keys share their tiles, also where each has one query.
#pragma once

#include "diff_attn_tile.h"

namespace npf_attn {

// kPad: a map's values, padded; a row of any operand is 2 kPad wide
template <typename T, int kPad>
struct Shape {
  static constexpr int kWidth = 2 * kPad;
  static constexpr int kRowBytes = kWidth * (int)sizeof(T);
  // keys (or queries) a tile: two buffers of two tiles in 64 KiB
  static constexpr int kTile = kRowBytes <= 256 ? 64 : 32;
  static constexpr int kSteps = kPad / (2 * kChunk<T>);  // chunk pairs a map
  static constexpr int kBlocks = kWidth / 32;  // 32 columns of a whole row
  static constexpr int kMapBlocks = kPad / 32 > 0 ? kPad / 32 : 1;
};

// Columns that block n of map m starts at.  Maps of 16 share one block: each
// accumulates it whole and keeps its half.
template <int kPad>
__host__ __device__ constexpr int map_col(int m, int n) {
  return kPad == 16 ? 0 : m * kPad + 32 * n;
}

__host__ __device__ inline int split_keys(int n, int splits, int tile) {
  const int tiles = (n + tile - 1) / tile;
  return (tiles + splits - 1) / splits * tile;
}

// A partial result of a split key axis: for each row both maps' running
// maximum and sum, and both sums of values, all in fp32.
__host__ __device__ inline long split_row_floats(int Dv) { return 2L * Dv + 4; }

// exp2 of score * c - m over one tile, into s; returns the lane's sum
__device__ __forceinline__ float exp_tile(f32x16& s, float c, float m) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -m));
    sum += s[i];
  }
  return sum;
}

template <typename T, int kPad, int kWaves>
__global__ void __launch_bounds__(64 * kWaves)
    diff_fwd(NpfDiffAttnArgs a) {
  using S = Shape<T, kPad>;
  using Lds = Tile<T, S::kWidth>;
  constexpr int kTile = kWaves == 1 ? 32 : S::kTile;
  constexpr int kTileBytes = kTile * S::kRowBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int group = a.H / a.Hk, rows = group * a.Q;
  const int row_tiles = (rows + 32 * kWaves - 1) / (32 * kWaves);
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int row_tile = id % row_tiles, bh = id / row_tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int row = (row_tile * kWaves + (threadIdx.x >> 6)) * 32 + col;
  const bool live = row < rows;
  const int h = hk * group + (live ? row / a.Q : 0);
  const int q = live ? row % a.Q : 0;

  const int n = keys_of(a, b);
  int begin = 0, end = n;
  if (a.splits > 1) {
    const int per = split_keys(n, a.splits, kTile);
    begin = split * per < n ? split * per : n;
    end = n - begin < per ? n : begin + per;
  }

  u32x4 qf[2][S::kSteps];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int u = 0; u < S::kSteps; ++u) {
      const ChunkOf c =
          chunk_of_maps<T, kPad>((m * S::kSteps + u) * 2 + half, a.D);
      qf[m][u] = u32x4{0, 0, 0, 0};
      if (live) qf[m][u] = load_chunk(row_of<T>(a.q, b, h, q), c);
    }

  f32x16 o[2][S::kBlocks];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j) o[m][j] = f32x16{};
  float mx[2] = {kLowest, kLowest}, l[2] = {0.f, 0.f};
  const float c = a.scale * kLog2e;

  Stage<T, S::kWidth, kTile, 64 * kWaves> stage;
  const int chunk = (int)threadIdx.x % Lds::kChunks;
  const ChunkOf kc = chunk_of_maps<T, kPad>(chunk, a.D);
  const ChunkOf vc = chunk_of_row<T>(chunk, a.Dv);
  const T* kp = row_of<T>(a.k, b, hk, 0);
  const T* vp = row_of<T>(a.v, b, hk, 0);
  if (begin < end) {
    stage.load(kp, a.k.l, kc, vp, a.v.l, vc, begin, end);
    stage.store(lds, lds + kTileBytes);
  }
  __syncthreads();
  int buffer = 0;
  for (int k0 = begin; k0 < end; k0 += kTile, buffer ^= 1) {
    const bool more = k0 + kTile < end;
    if (more) stage.load(kp, a.k.l, kc, vp, a.v.l, vc, k0 + kTile, end);
    const char* kt = lds + buffer * 2 * kTileBytes;
    const char* vt = kt + kTileBytes;
#pragma unroll
    for (int sub = 0; sub < kTile; sub += 32) {
      if (k0 + sub >= end) break;
      f32x16 s[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        s[m] = f32x16{};
#pragma unroll
        for (int u = 0; u < S::kSteps; ++u)
          s[m] = mma_chunk<T>(
              Lds::rows(kt, sub + col, (m * S::kSteps + u) * 2 + half),
              qf[m][u], s[m]);
      }
      if (k0 + sub + 32 > end) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + sub + reg_row(i) + 4 * half >= end)
            s[0][i] = s[1][i] = -INFINITY;
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float top = s[m][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[m][i]);
        top = both_max(top) * c;
        // The maximum is raised only where it is exceeded by 2^8: exponents
        // stay below that, far from any type's end, and most tiles leave the
        // sums as they are.
        if (__any(top > mx[m] + 8.f)) {
          const float up = fmaxf(mx[m], top);
          const float f = __builtin_amdgcn_exp2f(mx[m] - up);
          mx[m] = up;
          l[m] *= f;
#pragma unroll
          for (int j = 0; j < S::kBlocks; ++j) o[m][j] *= f;
        }
        l[m] += exp_tile(s[m], c, mx[m]);
      }
      const Operand<T> p[2] = {Operand<T>(s[0]), Operand<T>(s[1])};
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j) {
        f32x16* const acc[2] = {&o[0][j], &o[1][j]};
        Lds::template transposed<2>(vt, sub, 32 * j, lane, p, acc);
      }
    }
    if (more)
      stage.store(lds + (buffer ^ 1) * 2 * kTileBytes,
                  lds + (buffer ^ 1) * 2 * kTileBytes + kTileBytes);
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < 2; ++m) l[m] = both_sum(l[m]);
  if (!live) return;
  if (a.splits > 1) {
    float* w = static_cast<float*>(a.split) +
               ((long)bh * rows + row) * a.splits * split_row_floats(a.Dv) +
               split * split_row_floats(a.Dv);
    if (half == 0) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        w[2 * m] = mx[m];
        w[2 * m + 1] = l[m];
      }
    }
    w += 4;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * j + 8 * g + 4 * half;
          const f32x16& x = o[m][j];
          store4(w + m * a.Dv + d, a.Dv - d, x[4 * g], x[4 * g + 1],
                 x[4 * g + 2], x[4 * g + 3]);
        }
    return;
  }
  const float lam = lam_of(a, h);
  // rows without keys: zeros; all else divides, so that sums that are no
  // number show
  const float i1 = n ? 1.f / l[0] : 0.f, i2 = n ? 1.f / l[1] : 0.f;
  T* out = row_of<T>(a.out, b, h, q);
  T* o2 = a.o2.p ? row_of<T>(a.o2, b, h, q) : nullptr;
#pragma unroll
  for (int j = 0; j < S::kBlocks; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * j + 8 * g + 4 * half;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = o[1][j][4 * g + e] * i2;
        x[e] = o[0][j][4 * g + e] * i1 - lam * y[e];
      }
      store4(out + d, a.Dv - d, x[0], x[1], x[2], x[3]);
      if (o2) store4(o2 + d, a.Dv - d, y[0], y[1], y[2], y[3]);
    }
  if (a.lse && half == 0) {
    float* p = a.lse + (((long)b * a.H + h) * a.Q + q) * 2;
#pragma unroll
    for (int m = 0; m < 2; ++m) p[m] = n ? mx[m] + __log2f(l[m]) : 0.f;
  }
}

// dq, and each row's part of dlam: a wave holds 32 query rows and passes over
// the keys
template <typename T, int kPad, int kWaves>
__global__ void __launch_bounds__(64 * kWaves)
    diff_bwd_dq(NpfDiffAttnArgs a) {
  using S = Shape<T, kPad>;
  using Lds = Tile<T, S::kWidth>;
  constexpr int kTile = S::kTile;
  constexpr int kTileBytes = kTile * S::kRowBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int group = a.H / a.Hk, rows = group * a.Q;
  const int row_tiles = (rows + 32 * kWaves - 1) / (32 * kWaves);
  const int row_tile = blockIdx.x % row_tiles, bh = blockIdx.x / row_tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int row = (row_tile * kWaves + (threadIdx.x >> 6)) * 32 + col;
  const bool live = row < rows;
  const int h = hk * group + (live ? row / a.Q : 0);
  const int q = live ? row % a.Q : 0;
  const int n = keys_of(a, b);
  const long stat = ((long)b * a.H + h) * a.Q + q;

  u32x4 qf[2][S::kSteps], gf[2 * S::kSteps];
#pragma unroll
  for (int u = 0; u < 2 * S::kSteps; ++u) {
    u32x4 x{0, 0, 0, 0};
    gf[u] = x;
    if (live) {
      x = load_chunk(row_of<T>(a.q, b, h, q),
                     chunk_of_maps<T, kPad>(u * 2 + half, a.D));
      gf[u] = load_chunk(row_of<T>(a.dout, b, h, q),
                         chunk_of_row<T>(u * 2 + half, a.Dv));
    }
    qf[u / S::kSteps][u % S::kSteps] = x;
  }
  float4 st = {0.f, 0.f, 0.f, 0.f};
  if (live) st = reinterpret_cast<const float4*>(a.stats)[stat];
  const float lam = lam_of(a, h), c = a.scale * kLog2e;

  f32x16 dq[2][S::kMapBlocks];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < S::kMapBlocks; ++j) dq[m][j] = f32x16{};
  float dlam = 0.f;

  Stage<T, S::kWidth, kTile, 64 * kWaves> stage;
  const int chunk = (int)threadIdx.x % Lds::kChunks;
  const ChunkOf kc = chunk_of_maps<T, kPad>(chunk, a.D);
  const ChunkOf vc = chunk_of_row<T>(chunk, a.Dv);
  const T* kp = row_of<T>(a.k, b, hk, 0);
  const T* vp = row_of<T>(a.v, b, hk, 0);
  if (n > 0) {
    stage.load(kp, a.k.l, kc, vp, a.v.l, vc, 0, n);
    stage.store(lds, lds + kTileBytes);
  }
  __syncthreads();
  int buffer = 0;
  for (int k0 = 0; k0 < n; k0 += kTile, buffer ^= 1) {
    const bool more = k0 + kTile < n;
    if (more) stage.load(kp, a.k.l, kc, vp, a.v.l, vc, k0 + kTile, n);
    const char* kt = lds + buffer * 2 * kTileBytes;
    const char* vt = kt + kTileBytes;
#pragma unroll
    for (int sub = 0; sub < kTile; sub += 32) {
      if (k0 + sub >= n) break;
      f32x16 s[2], g{};
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        s[m] = f32x16{};
#pragma unroll
        for (int u = 0; u < S::kSteps; ++u)
          s[m] = mma_chunk<T>(
              Lds::rows(kt, sub + col, (m * S::kSteps + u) * 2 + half),
              qf[m][u], s[m]);
      }
#pragma unroll
      for (int u = 0; u < 2 * S::kSteps; ++u)
        g = mma_chunk<T>(Lds::rows(vt, sub + col, u * 2 + half), gf[u], g);
      const bool edge = k0 + sub + 32 > n;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], c, -st.x));
        float p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][i], c, -st.y));
        if (edge && k0 + sub + reg_row(i) + 4 * half >= n) p1 = p2 = 0.f;
        dlam = __builtin_fmaf(p2, g[i], dlam);
        s[0][i] = p1 * (g[i] - st.z);
        s[1][i] = p2 * (g[i] - st.w) * -lam;
      }
      const Operand<T> ds[2] = {Operand<T>(s[0]), Operand<T>(s[1])};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < S::kMapBlocks; ++j) {
          const Operand<T> one[1] = {ds[m]};
          f32x16* const acc[1] = {&dq[m][j]};
          Lds::template transposed<1>(kt, sub, map_col<kPad>(m, j), lane, one,
                                      acc);
        }
    }
    if (more)
      stage.store(lds + (buffer ^ 1) * 2 * kTileBytes,
                  lds + (buffer ^ 1) * 2 * kTileBytes + kTileBytes);
    __syncthreads();
  }

  dlam = both_sum(dlam);
  if (!live) return;
  if (half == 0) a.dlam_rows[stat] = dlam;
  if (!a.dq.p) return;
  T* out = row_of<T>(a.dq, b, h, q);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < S::kMapBlocks; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (kPad == 16 && g / 2 != m) continue;
        const int d = (kPad == 16 ? 8 * (g % 2) : 32 * j + 8 * g) + 4 * half;
        const f32x16 x = dq[m][j] * a.scale;
        store4(out + m * a.D + d, a.D - d, x[4 * g], x[4 * g + 1],
               x[4 * g + 2], x[4 * g + 3]);
      }
}

// dk and dv: a wave holds 32 keys and passes over the queries of the heads
// that share them
template <typename T, int kPad, int kWaves, bool kDk, bool kDv>
__global__ void __launch_bounds__(64 * kWaves)
    diff_bwd_dkv(NpfDiffAttnArgs a) {
  using S = Shape<T, kPad>;
  using Lds = Tile<T, S::kWidth>;
  constexpr int kTile = S::kTile;
  constexpr int kTileBytes = kTile * S::kRowBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // both buffers' statistics, one array each of lse_1, lse_2, delta_1, delta_2
  float(*stats)[4][kTile] =
      reinterpret_cast<float(*)[4][kTile]>(lds + 4 * kTileBytes);

  const int group = a.H / a.Hk;
  const int key_tiles = (a.K + 32 * kWaves - 1) / (32 * kWaves);
  const int key_tile = blockIdx.x % key_tiles, bh = blockIdx.x / key_tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int key = (key_tile * kWaves + (threadIdx.x >> 6)) * 32 + col;
  const int n = keys_of(a, b);
  const bool live = key < n;
  const float c = a.scale * kLog2e;

  u32x4 kf[2][S::kSteps], vf[2 * S::kSteps];
#pragma unroll
  for (int u = 0; u < 2 * S::kSteps; ++u) {
    u32x4 x{0, 0, 0, 0};
    vf[u] = x;
    if (live) {
      x = load_chunk(row_of<T>(a.k, b, hk, key),
                     chunk_of_maps<T, kPad>(u * 2 + half, a.D));
      if (kDk)
        vf[u] = load_chunk(row_of<T>(a.v, b, hk, key),
                           chunk_of_row<T>(u * 2 + half, a.Dv));
    }
    kf[u / S::kSteps][u % S::kSteps] = x;
  }
  f32x16 dk[2][S::kMapBlocks], dv[S::kBlocks];
#pragma unroll
  for (int j = 0; j < S::kMapBlocks; ++j) dk[0][j] = dk[1][j] = f32x16{};
#pragma unroll
  for (int j = 0; j < S::kBlocks; ++j) dv[j] = f32x16{};

  // (head, tile) pairs in one sequence; none where the block has no keys
  const int q_tiles = (a.Q + kTile - 1) / kTile;
  const int steps =
      key_tile * 32 * kWaves < n ? group * q_tiles : 0;
  Stage<T, S::kWidth, kTile, 64 * kWaves> stage;
  const int chunk = (int)threadIdx.x % Lds::kChunks;
  const ChunkOf qc = chunk_of_maps<T, kPad>(chunk, a.D);
  const ChunkOf gc = chunk_of_row<T>(chunk, a.Dv);
  float4 st;
  auto load = [&](int step) {
    const int h = hk * group + step / q_tiles;
    const int q0 = step % q_tiles * kTile;
    stage.load(row_of<T>(a.q, b, h, 0), a.q.l, qc, row_of<T>(a.dout, b, h, 0),
               a.dout.l, gc, q0, a.Q);
    const int q = q0 + (int)threadIdx.x;
    // rows that are not there have no weight
    st = float4{-kLowest, -kLowest, 0.f, 0.f};
    if (threadIdx.x < kTile && q < a.Q)
      st = reinterpret_cast<const float4*>(
          a.stats)[((long)b * a.H + h) * a.Q + q];
  };
  auto store = [&](int buffer) {
    stage.store(lds + buffer * 2 * kTileBytes,
                lds + buffer * 2 * kTileBytes + kTileBytes);
    if (threadIdx.x < kTile) {
      stats[buffer][0][threadIdx.x] = st.x;
      stats[buffer][1][threadIdx.x] = st.y;
      stats[buffer][2][threadIdx.x] = st.z;
      stats[buffer][3][threadIdx.x] = st.w;
    }
  };
  if (steps > 0) {
    load(0);
    store(0);
  }
  __syncthreads();
  int buffer = 0;
  for (int step = 0; step < steps; ++step, buffer ^= 1) {
    const bool more = step + 1 < steps;
    if (more) load(step + 1);
    const float lam = lam_of(a, hk * group + step / q_tiles);
    const int q0 = step % q_tiles * kTile;
    const char* qt = lds + buffer * 2 * kTileBytes;
    const char* gt = qt + kTileBytes;
#pragma unroll
    for (int sub = 0; sub < kTile; sub += 32) {
      if (q0 + sub >= a.Q) break;
      f32x16 s[2], g{};
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        s[m] = f32x16{};
#pragma unroll
        for (int u = 0; u < S::kSteps; ++u)
          s[m] = mma_chunk<T>(
              Lds::rows(qt, sub + col, (m * S::kSteps + u) * 2 + half),
              kf[m][u], s[m]);
      }
      if (kDk) {
#pragma unroll
        for (int u = 0; u < 2 * S::kSteps; ++u)
          g = mma_chunk<T>(Lds::rows(gt, sub + col, u * 2 + half), vf[u], g);
      }
      f32x16 map;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = sub + 8 * r + 4 * half;
        const f32x4 lse1 = *(const f32x4*)&stats[buffer][0][at];
        const f32x4 lse2 = *(const f32x4*)&stats[buffer][1][at];
        const f32x4 d1 = *(const f32x4*)&stats[buffer][2][at];
        const f32x4 d2 = *(const f32x4*)&stats[buffer][3][at];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * r + e;
          const float p1 =
              __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], c, -lse1[e]));
          const float p2 =
              __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][i], c, -lse2[e])) *
              lam;
          map[i] = p1 - p2;
          s[0][i] = p1 * (g[i] - d1[e]);
          s[1][i] = p2 * (d2[e] - g[i]);
        }
      }
      if (kDv) {
        const Operand<T> p[1] = {Operand<T>(map)};
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) {
          f32x16* const acc[1] = {&dv[j]};
          Lds::template transposed<1>(gt, sub, 32 * j, lane, p, acc);
        }
      }
      if (kDk) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const Operand<T> ds[1] = {Operand<T>(s[m])};
#pragma unroll
          for (int j = 0; j < S::kMapBlocks; ++j) {
            f32x16* const acc[1] = {&dk[m][j]};
            Lds::template transposed<1>(qt, sub, map_col<kPad>(m, j), lane, ds,
                                        acc);
          }
        }
      }
    }
    if (more) store(buffer ^ 1);
    __syncthreads();
  }

  if (key >= a.K) return;
  // keys behind the last one take no part, whatever their lanes hold
  if (kDk && a.dk.p) {
    T* out = row_of<T>(a.dk, b, hk, key);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < S::kMapBlocks; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (kPad == 16 && g / 2 != m) continue;
          const int d = (kPad == 16 ? 8 * (g % 2) : 32 * j + 8 * g) + 4 * half;
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = live ? dk[m][j][4 * g + e] * a.scale : 0.f;
          store4(out + m * a.D + d, a.D - d, x[0], x[1], x[2], x[3]);
        }
  }
  if (kDv && a.dv.p) {
    T* out = row_of<T>(a.dv, b, hk, key);
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * j + 8 * g + 4 * half;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = live ? dv[j][4 * g + e] : 0.f;
        store4(out + d, a.Dv - d, x[0], x[1], x[2], x[3]);
      }
  }
}

// -------------------------------- launches -------------------------------- //

template <typename K>
hipError_t launch(K kernel, long blocks, int threads, int lds,
                  const NpfDiffAttnArgs& a, hipStream_t stream) {
  if (blocks > 0x7fffffffL) return hipErrorInvalidConfiguration;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  kernel<<<(unsigned)blocks, threads, lds, stream>>>(a);
  return hipGetLastError();
}

template <typename T, int kPad>
hipError_t fwd_sized(const NpfDiffAttnArgs& a, hipStream_t stream) {
  using S = Shape<T, kPad>;
  const long heads = (long)a.B * a.Hk, rows = (long)(a.H / a.Hk) * a.Q;
  if (a.waves == 1)
    return launch(diff_fwd<T, kPad, 1>, heads * ((rows + 31) / 32) * a.splits,
                  64, 4 * 32 * S::kRowBytes, a, stream);
  return launch(diff_fwd<T, kPad, 4>, heads * ((rows + 127) / 128) * a.splits,
                256, 4 * S::kTile * S::kRowBytes, a, stream);
}

template <typename T, int kPad>
hipError_t bwd_sized(const NpfDiffAttnArgs& a, hipStream_t stream) {
  using S = Shape<T, kPad>;
  const long heads = (long)a.B * a.Hk, rows = (long)(a.H / a.Hk) * a.Q;
  const int lds = 4 * S::kTile * S::kRowBytes;
  if (a.dq.p || a.dlam) {
    const hipError_t e = launch(diff_bwd_dq<T, kPad, 4>,
                                heads * ((rows + 127) / 128), 256, lds, a,
                                stream);
    if (e != hipSuccess) return e;
  }
  const long blocks = heads * ((a.K + 127) / 128);
  const int more = 2 * 4 * S::kTile * (int)sizeof(float);
  if constexpr (sizeof(T) == 4 && kPad == 128) {
    // both gradients at once would not fit a wave's registers
    if (a.dk.p) {
      const hipError_t e = launch(diff_bwd_dkv<T, kPad, 4, true, false>, blocks,
                                  256, lds + more, a, stream);
      if (e != hipSuccess) return e;
    }
    if (a.dv.p)
      return launch(diff_bwd_dkv<T, kPad, 4, false, true>, blocks, 256,
                    lds + more, a, stream);
    return hipSuccess;
  } else {
    if (!a.dk.p && !a.dv.p) return hipSuccess;
    return launch(diff_bwd_dkv<T, kPad, 4, true, true>, blocks, 256, lds + more,
                  a, stream);
  }
}

template <typename T>
hipError_t fwd_typed(const NpfDiffAttnArgs& a, hipStream_t stream) {
  switch (a.pad) {
    case 16: return fwd_sized<T, 16>(a, stream);
    case 32: return fwd_sized<T, 32>(a, stream);
    case 64: return fwd_sized<T, 64>(a, stream);
    default: return fwd_sized<T, 128>(a, stream);
  }
}

template <typename T>
hipError_t bwd_typed(const NpfDiffAttnArgs& a, hipStream_t stream) {
  switch (a.pad) {
    case 16: return bwd_sized<T, 16>(a, stream);
    case 32: return bwd_sized<T, 32>(a, stream);
    case 64: return bwd_sized<T, 64>(a, stream);
    default: return bwd_sized<T, 128>(a, stream);
  }
}

}  // namespace npf_attn
