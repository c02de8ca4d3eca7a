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
  // tiles of 32 that a backward wave takes through a pass at once
  static constexpr int kSubs = sizeof(T) == 2 ? (kPad <= 32 ? 2 : 1)
                                              : (kPad <= 16 ? 2 : 1);
  // What a wave's registers hold decides how the gradients share launches: of
  // the keys both at once, else dk and dv apart, else dk of each map apart; of
  // the queries both maps at once, else apart.  (Long: dk and dv apart 959 us,
  // together 1260; heads of 128, 2 x 8 x 1024 x 1024, a whole step with dk of
  // each map apart: bf16 308 us, together 517.)
  static constexpr bool kBothGrads = kPad * (int)sizeof(T) < 128;
  static constexpr bool kDkMapsApart = kPad == 128;
  static constexpr bool kDqMapsApart = kPad * (int)sizeof(T) > 256;
  // whether the dq kernel keeps its queries in LDS rather than in registers
  // (long: 529 us, 704 with one wave a SIMD, 814 with two that spill)
  static constexpr bool kQueriesInLds = sizeof(T) == 2 && kPad == 64;
  static constexpr int kSteps = kPad / (2 * kChunk<T>);  // chunk pairs a map

  // The widest fp32 products are taken in two parts, and leave out the second,
  // the last quarter, where it is padding alone (a step at heads of 96: 1178 us
  // to 907); the others are taken whole (such questions at heads of 64: 503 us
  // to 570).  Steps of a part, of n in all:
  static constexpr int kParts = sizeof(T) == 4 && kPad == 128 ? 2 : 1;
  __host__ __device__ static constexpr int from(int n, int part) {
    return part ? n - n / 4 : 0;
  }
  __host__ __device__ static constexpr int upto(int n, int part) {
    return part + 1 < kParts ? n - n / 4 : n;
  }
  // of `all` padded values `size` are there
  __device__ static __forceinline__ bool taken(int part, int all, int size) {
    return part == 0 || 4 * size > 3 * all;
  }

  static constexpr int kBlocks = kWidth / 32;  // 32 columns of a whole row
  static constexpr int kMapBlocks = kPad / 32 > 0 ? kPad / 32 : 1;
};

// Waves a SIMD is to hold: two, in half of the registers each and with every
// matrix result in ordinary registers, up to 128 bytes of a map; else one.
// Kernels of one map go to twice the size in 16 bits, where the next rows do
// not pass through registers (kDirect).  (Long training bf16, dk and dv in one
// launch that spills: 4349 us; apart, 958.  Steps of 2 x 8 heads, 1024 x 1024,
// rows through registers, two waves and one: bf16 heads of 60 230 and 300 us,
// though dk and dv then spill 27 to 32 registers, heads of 20 107 and 107, fp32
// heads of 18 277 and 332; kernels of one map at bf16 heads of 100 547 and 495.)
template <typename T, int kPad, bool kDirect, bool kOneMap = false>
constexpr int kResident =
    kPad * (int)sizeof(T) <= (kOneMap && kDirect && sizeof(T) == 2 ? 256 : 128)
        ? 2 : 1;

// The same of the forward kernel, whose waves hold one map; rows on their way
// through registers (not kDirect) need room too.  (Long: 430 us; waves with
// both maps 475 with two a SIMD, 794 with one.  128 registers hold all but 9 at
// 128 bytes a map, 2 at 64.)
template <typename T, int kPad, bool kDirect>
constexpr int kFwdResident =
    kPad * (int)sizeof(T) <= (kDirect ? 128 : 64) ? 4
    : kPad * (int)sizeof(T) <= (kDirect ? 512 : 256) ? 2 : 1;

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

// exp2 of score * c - m over one tile, into s; returns the lane's sum of them
// and `sum`
__device__ __forceinline__ float exp_tile(f32x16& s, float c, float m,
                                          float sum) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -m));
    sum += s[i];
  }
  return sum;
}

// Measured (one MI355X; "long": 2 x 16 heads on 4, 4096 x 4096, maps of 64,
// bf16; "image": 16 x 4 heads, 1024 x 1024, maps of 16):
//
//            long bf16               image bf16   bound by
//   forward  430 us, 0.64 PFLOP/s      34 us      vector and matrix unit (long:
//   dq       525 us                    53 us      478 + 393 of 746 thousand
//   dk, dv   569 + 390 us              51 us      clocks a SIMD, forward)
// 8 heads of 128, 4096 x 4096, bf16: forward 203 us, 0.68 PFLOP/s.
//
// A pair of scores costs two exponents (8 clocks a 64-lane wave each) and about
// 8 other vector operations a lane, and little of a wave's products and vector
// work overlaps, however many waves a SIMD has.  LDS is read at less than a
// third of its rate (long), and but for 0.4% of dq's reads without bank conflicts.

// Forward: a wave holds 32 query rows and one map, and passes over the keys; a
// block has kRowWaves waves for each map, which share the tiles (the first
// map's waves move the keys', the second's the values') and meet at the end.
// With up to 32 rows a head, blocks of one wave a map split the keys between
// them (single queries against 32768 keys, 200 MB of bf16: 59 us, 3.4 TB/s,
// with the join).
template <typename T, int kPad, int kRowWaves, bool kDirect>
__global__ void __launch_bounds__(128 * kRowWaves,
                                  (kFwdResident<T, kPad, kDirect>))
    diff_fwd(NpfDiffAttnArgs a) {
  using S = Shape<T, kPad>;
  using Lds = Tile<T, S::kWidth>;
  constexpr int kTile = kRowWaves == 1 ? 32 * S::kSubs : S::kTile;
  // tiles of 32 that a wave takes through a pass at once: what fits a quarter
  // of a SIMD's registers (8 heads of 32, 4096^2, bf16: 93 us, with two 110)
  constexpr int kSubs = kPad <= 16 ? 2 : 1;
  // With few rows memory bounds the kernel, and the maps keep what rounding to
  // 16 bits leaves of them (single queries against 32768 keys: 57 to 59 us, and
  // the result's error falls from 1.48 to 1.0 times that of its last rounding).
  // With many rows it would cost more than it gives: a step 128 -> 141 us
  // (image), 1740 -> 2020 (long), padded fp16, 7 x 8 heads of 48, 333 x 2049, 53
  // -> 81; errors there are 1.4 to 1.5 times the last rounding's.
  constexpr bool kTwice = sizeof(T) == 2 && kRowWaves == 1;
  constexpr int kTileBytes = kTile * S::kRowBytes;
  // two objects, so that it shows that the next tiles' loads do not touch
  // what is being read
  __shared__ __attribute__((aligned(16))) char even[2 * kTileBytes];
  __shared__ __attribute__((aligned(16))) char odd[2 * kTileBytes];

  const int group = a.H / a.Hk, rows = group * a.Q;
  const int row_tiles = (rows + 32 * kRowWaves - 1) / (32 * kRowWaves);
  // Neighbouring blocks take different batch entries and heads: long and short
  // contexts spread over the chip, and as blocks are dealt to the 8 XCDs in
  // turn, those of one head mostly share an L2.  With few rows nothing is
  // shared, and neighbours in memory are read at a time (single queries
  // against 32768 keys: 15% faster).
  const int heads = a.B * a.Hk;
  int bh, row_tile, split;
  if (kRowWaves == 1) {
    split = blockIdx.x % a.splits;
    row_tile = blockIdx.x / a.splits % row_tiles;
    bh = blockIdx.x / a.splits / row_tiles;
  } else {
    bh = blockIdx.x % heads;
    row_tile = blockIdx.x / heads % row_tiles;
    split = blockIdx.x / heads / row_tiles;
  }
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = wave / kRowWaves, row_wave = wave % kRowWaves;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int row = (row_tile * kRowWaves + row_wave) * 32 + col;
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

  u32x4 qf[S::kSteps];
#pragma unroll
  for (int u = 0; u < S::kSteps; ++u) {
    qf[u] = u32x4{0, 0, 0, 0};
    if (live)
      qf[u] = load_chunk(
          row_of<T>(a.q, b, h, q),
          chunk_of_maps<T, kPad>((m * S::kSteps + u) * 2 + half, a.D));
  }

  f32x16 o[S::kBlocks];
#pragma unroll
  for (int j = 0; j < S::kBlocks; ++j) o[j] = f32x16{};
  float mx = kLowest, l = 0.f;
  const float c = a.scale * kLog2e;

  // one tile from LDS; kEdge: it may reach behind the last key
  const int rows_base = Lds::rows_base(lane) ^ (m * S::kSteps << 5);
  const int cols_base = Lds::cols_base(lane);
  auto pass = [&](auto edge, int k0, const char* kt) {
    constexpr bool kEdge = decltype(edge)::value;
    const char* vt = kt + kTileBytes;
    const int rb = fresh(rows_base), cb = fresh(cols_base);
#pragma unroll
    for (int sub0 = 0; sub0 < kTile; sub0 += 32 * kSubs) {
      if (kEdge && k0 + sub0 >= end) break;
      f32x16 s[kSubs];
#pragma unroll
      for (int t = 0; t < kSubs; ++t) {
        s[t] = f32x16{};
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
          if (!S::taken(part, kPad, a.D)) continue;
#pragma unroll
          for (int u = S::from(S::kSteps, part);
               u < S::upto(S::kSteps, part); ++u) {
            s[t] =
                mma_chunk<T>(Lds::rows(kt, rb, sub0 + 32 * t, u), qf[u], s[t]);
          }
        }
      }
      if constexpr (kEdge) {
#pragma unroll
        for (int t = 0; t < kSubs; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (k0 + sub0 + 32 * t + reg_row(i) + 4 * half >= end)
              s[t][i] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int t = 0; t < kSubs; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = larger(top, s[t][i]);
      top = both_max(top) * c;
      // The maximum is raised only where it is exceeded by 2^8: exponents stay
      // below that, far from any type's end, and most tiles leave the sums as
      // they are.  In fp16 it is held 2^7 too low, so that exponents reach from
      // 2^15 down to steps of 2^-24: values below 2^-24 of the largest, of
      // which a long context may hold most, count on down to 2^-31.  (Not
      // where scores are so large that their products' rounding nears that.)
      float under = 0.f;
      if (std::is_same<T, npf_f16>::value && fabsf(top) < 1048576.f)
        under = 7.f;
      if (__any(top > mx + (8.f + under))) {
        const float up = fmaxf(mx, top - under);
        const float f = __builtin_amdgcn_exp2f(mx - up);
        mx = up;
        l *= f;
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) o[j] *= f;
      }
#pragma unroll
      for (int t = 0; t < kSubs; ++t) {
        l = exp_tile(s[t], c, mx, l);
        const Product<T, S::kWidth, kTwice> p(s[t]);
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
          if (!S::taken(part, 2 * kPad, a.Dv)) continue;
#pragma unroll
          for (int j = S::from(S::kBlocks, part);
               j < S::upto(S::kBlocks, part); ++j)
            p.add(vt, cb, sub0 + 32 * t, 32 * j, o[j]);
        }
      }
    }
  };

  // what this wave's threads move
  Stage<T, S::kWidth, kTile, 64 * kRowWaves, kDirect> stage;
  const T* from = row_of<T>(m ? a.v : a.k, b, hk, 0);
  const long from_l = m ? a.v.l : a.k.l;
  const int per = m ? Lds::kChunks : Lds::kChunks / 2;
  const int size = m ? a.Dv : a.D;
  const int tid = row_wave * 64 + lane, to = m * kTileBytes;
  auto step = [&](int k0, const char* now, char* then) {
    const int next = k0 + kTile;
    if (next < end)
      stage.load(from, from_l, per, size, next, end, tid, then + to);
    pass(std::false_type{}, k0, now);
    if (next < end) stage.store(end - next, tid, then + to);
    __syncthreads();
  };
  stage.clear(per, size, tid, even + to);
  stage.clear(per, size, tid, odd + to);
  __syncthreads();
  if (begin < end) {
    stage.load(from, from_l, per, size, begin, end, tid, even + to);
    stage.store(end - begin, tid, even + to);
  }
  __syncthreads();
  const int full = (end - begin) / kTile;
  int k0 = begin;
  for (int t = 0; t < full;) {
    step(k0, even, odd);
    k0 += kTile;
    if (++t == full) break;
    step(k0, odd, even);
    k0 += kTile;
    ++t;
  }
  if (k0 < end) pass(std::true_type{}, k0, full & 1 ? odd : even);

  l = both_sum(l);
  if (a.splits > 1) {
    if (!live) return;
    float* w = static_cast<float*>(a.split) +
               (((long)bh * rows + row) * a.splits + split) *
                   split_row_floats(a.Dv);
    if (half == 0) {
      w[2 * m] = mx;
      w[2 * m + 1] = l;
    }
    w += 4 + m * a.Dv;
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * j + 8 * g + 4 * half;
        store4(w + d, a.Dv - d, o[j][4 * g], o[j][4 * g + 1], o[j][4 * g + 2],
               o[j][4 * g + 3]);
      }
    return;
  }
  // rows without keys: zeros; all else divides, so that sums that are no
  // number show
  const float inv = n ? 1.f / l : 0.f;
  if (a.lse && half == 0 && live)
    a.lse[(((long)b * a.H + h) * a.Q + q) * 2 + m] =
        n ? mx + __log2f(l) : 0.f;
  // The second map's results go to the first map's wave of the same rows, four
  // registers of all lanes (a piece) at a time, through what the tiles held.
  constexpr int kPieces = 2 * kTileBytes / (1024 * kRowWaves);  // of each array
  static_assert(kPieces * 1024 * kRowWaves == 2 * kTileBytes);
  auto piece = [&](int i) {
    char* at = i / kPieces % 2 ? odd : even;
    return reinterpret_cast<f32x4*>(
        at + ((i % kPieces * kRowWaves + row_wave) * 64 + lane) * 16);
  };
  const float lam = n ? lam_of(a, h) : 0.f;  // (it may be inf)
  T* out = row_of<T>(m ? a.o2 : a.out, b, h, q);
  const bool stores = live && (m == 0 || a.o2.p);
#pragma unroll
  for (int i0 = 0; i0 < 4 * S::kBlocks; i0 += 2 * kPieces) {
    __syncthreads();
    if (m) {
#pragma unroll
      for (int i = i0; i < i0 + 2 * kPieces && i < 4 * S::kBlocks; ++i) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = o[i / 4][i % 4 * 4 + e] * inv;
        *piece(i) = y;
        const int d = 8 * i + 4 * half;
        if (stores) store4(out + d, a.Dv - d, y[0], y[1], y[2], y[3]);
      }
    }
    __syncthreads();
    if (m == 0) {
#pragma unroll
      for (int i = i0; i < i0 + 2 * kPieces && i < 4 * S::kBlocks; ++i) {
        const f32x4 y = *piece(i);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = o[i / 4][i % 4 * 4 + e] * inv - lam * y[e];
        const int d = 8 * i + 4 * half;
        if (stores) store4(out + d, a.Dv - d, x[0], x[1], x[2], x[3]);
      }
    }
  }
}

constexpr int kBwdWaves = 4;  // of a backward block

// dq of the maps in kMaps (bits), and with the second map each row's part of
// dlam: a wave holds 32 query rows and passes over the keys
template <typename T, int kPad, bool kDirect, int kMaps>
__global__ void __launch_bounds__(64 * kBwdWaves, (kResident<T, kPad, kDirect>))
    diff_bwd_dq(NpfDiffAttnArgs a) {
  using S = Shape<T, kPad>;
  using Lds = Tile<T, S::kWidth>;
  constexpr int kWaves = kBwdWaves;
  constexpr bool kInLds = S::kQueriesInLds;
  constexpr int kTile = kInLds ? 32 * S::kSubs : S::kTile;
  constexpr int kSubs = S::kSubs;
  // For heads of up to 32 the maps' gradients keep what rounding to 16 bits
  // leaves of them.  Rows of them sum to zero, so what the keys of a row share
  // (scale q_i, more of it the fewer values a head has) cancels in dq but not in
  // the rounding: rounded once, dq's error is 1.53 times that of its own last
  // rounding at heads of 16 (now 1.07; a step 125 us rather than 117, image) and
  // 1.44 times at heads of 64 (1.02; 1855 us rather than 1740, long).
  constexpr bool kTwice = sizeof(T) == 2 && kPad <= 32;
  constexpr int kTileBytes = kTile * S::kRowBytes;
  // two objects, so that it shows that the next tiles' loads do not touch
  // what is being read
  __shared__ __attribute__((aligned(16))) char even[2 * kTileBytes];
  __shared__ __attribute__((aligned(16))) char odd[2 * kTileBytes];
  __shared__ __attribute__((
      aligned(16))) char held[kInLds ? 32 * kWaves * S::kRowBytes : 16];

  const int group = a.H / a.Hk, rows = group * a.Q;
  const int row_tiles = (rows + 32 * kWaves - 1) / (32 * kWaves);
  const int heads = a.B * a.Hk, bh = blockIdx.x % heads;
  const int row_tile = blockIdx.x / heads % row_tiles;
  const int split = blockIdx.x / heads / row_tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int row = (row_tile * kWaves + (threadIdx.x >> 6)) * 32 + col;
  const bool live = row < rows;
  const int h = hk * group + (live ? row / a.Q : 0);
  const int q = live ? row % a.Q : 0;
  const int keys = keys_of(a, b);
  int begin = 0, n = keys;  // this split's
  if (a.dq_splits > 1) {
    const int per = split_keys(n, a.dq_splits, kTile);
    begin = split * per < n ? split * per : n;
    n = n - begin < per ? n : begin + per;
  }
  const long stat = ((long)b * a.H + h) * a.Q + q;

  const int rows_base = Lds::rows_base(lane), cols_base = Lds::cols_base(lane);
  char* own = held + (kInLds ? (threadIdx.x >> 6) * 32 * S::kRowBytes : 0);
  u32x4 qf[kInLds ? 1 : 2 * S::kSteps], gf[2 * S::kSteps];
#pragma unroll
  for (int u = 0; u < 2 * S::kSteps; ++u) {
    u32x4 x{0, 0, 0, 0};
    gf[u] = x;
    if (live) {
      x = load_chunk(row_of<T>(a.q, b, h, q),
                     chunk_of_maps<T, kPad>(u * 2 + half, a.D));
      gf[u] = load_chunk(row_of<T>(a.dout, b, h, q),
                         chunk_of_row<T, kPad>(u * 2 + half, a.Dv));
    }
    if constexpr (kInLds)  // read by the lanes that write it alone
      *reinterpret_cast<u32x4*>(own + (rows_base ^ (u << 5))) = x;
    else
      qf[u] = x;
  }
  // rows without keys have no part in any gradient, whatever lam and dout hold
  const float lam = keys ? lam_of(a, h) : 0.f, c = a.scale * kLog2e;
  // the row's statistics; the dk/dv kernel finds them in a.stats
  float4 st = {0.f, 0.f, 0.f, 0.f};
  float square = 0.f;  // of the row of dout
#pragma unroll
  for (int u = 0; u < 2 * S::kSteps; ++u) {
    if (!live || keys == 0) break;
    const ChunkOf at = chunk_of_row<T, kPad>(u * 2 + half, a.Dv);
    T g[kChunk<T>], o[kChunk<T>], o2[kChunk<T>];
    const u32x4 x = load_chunk(row_of<T>(a.out, b, h, q), at);
    const u32x4 y = load_chunk(row_of<T>(a.o2, b, h, q), at);
    __builtin_memcpy(g, &gf[u], 16);
    __builtin_memcpy(o, &x, 16);
    __builtin_memcpy(o2, &y, 16);
#pragma unroll
    for (int i = 0; i < kChunk<T>; ++i) {
      st.z += (float)g[i] * ((float)o[i] + lam * (float)o2[i]);
      st.w += (float)g[i] * (float)o2[i];
      if (kScaledGrads<T>) square += (float)g[i] * (float)g[i];
    }
  }
  st.z = both_sum(st.z);
  st.w = both_sum(st.w);
  // maps are taken 2^e times as large, each row's by its own e
  float e = 0.f;
  if constexpr (kScaledGrads<T>)
    e = reach_exponent(
        reach_bound(sqrtf(both_sum(square)) * fmaxf(1.f, fabsf(lam)),
                    reach_of_values(a, bh)));
  const float back = kScaledGrads<T> ? __builtin_amdgcn_exp2f(-e) : 1.f;
  if (live) {
    st.x = a.lse[2 * stat];
    st.y = a.lse[2 * stat + 1];
    if ((kMaps & 1) && half == 0 && split == 0)
      reinterpret_cast<float4*>(a.stats)[stat] = st;
  }

  f32x16 dq[2][S::kMapBlocks];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < S::kMapBlocks; ++j) dq[m][j] = f32x16{};
  // sum of P_2 (G - delta_2), which is zero but for the rounding that delta_2
  // has seen: with delta_2 it makes the exact sum of P_2 G
  float dlam = 0.f;
  const float apart = st.z - st.w;

  StagePair<T, S::kWidth, kTile, 64 * kWaves, kDirect> stage;
  const T* kp = row_of<T>(a.k, b, hk, 0);
  const T* vp = row_of<T>(a.v, b, hk, 0);
  auto pass = [&](auto edge, int k0, const char* kt) {
    constexpr bool kEdge = decltype(edge)::value;
    const char* vt = kt + kTileBytes;
    const int rb = fresh(rows_base), cb = fresh(cols_base);
#pragma unroll
    for (int sub0 = 0; sub0 < kTile; sub0 += 32 * kSubs) {
      if (kEdge && k0 + sub0 >= n) break;
      f32x16 g[kSubs];
#pragma unroll
      for (int t = 0; t < kSubs; ++t) {
        // the products start from -delta_1, which costs what zeros would
#pragma unroll
        for (int i = 0; i < 16; ++i) g[t][i] = -st.z;
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
          if (!S::taken(part, 2 * kPad, a.Dv)) continue;
#pragma unroll
          for (int u = S::from(2 * S::kSteps, part);
               u < S::upto(2 * S::kSteps, part); ++u) {
            g[t] =
                mma_chunk<T>(Lds::rows(vt, rb, sub0 + 32 * t, u), gf[u], g[t]);
          }
        }
      }
      if (kSubs == 1) __builtin_amdgcn_sched_barrier(0);
      // one map after the other: a second tile of scores would not fit
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (!(kMaps >> m & 1)) continue;
        f32x16 s[kSubs];
#pragma unroll
        for (int t = 0; t < kSubs; ++t) {
          s[t] = f32x16{};
#pragma unroll
          for (int part = 0; part < S::kParts; ++part) {
            if (!S::taken(part, kPad, a.D)) continue;
#pragma unroll
            for (int i = S::from(S::kSteps, part);
                 i < S::upto(S::kSteps, part); ++i) {
              const int u = m * S::kSteps + i;
              u32x4 x;
              if constexpr (kInLds)
                x = Lds::rows(own, rb, 0, u);
              else
                x = qf[u];
              s[t] = mma_chunk<T>(Lds::rows(kt, rb, sub0 + 32 * t, u), x, s[t]);
            }
          }
        }
        const float lse = (m ? st.y : st.x) - e;
#pragma unroll
        for (int t = 0; t < kSubs; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, -lse));
            if (kEdge && k0 + sub0 + 32 * t + reg_row(i) + 4 * half >= n)
              p = 0.f;
            s[t][i] = p * (m ? g[t][i] + apart : g[t][i]);
            if (m) dlam += s[t][i];
          }
          const Product<T, S::kWidth, kTwice> ds(s[t]);
#pragma unroll
          for (int part = 0; part < S::kParts; ++part) {
            if (!S::taken(part, kPad, a.D)) continue;
#pragma unroll
            for (int j = S::from(S::kMapBlocks, part);
                 j < S::upto(S::kMapBlocks, part); ++j)
              ds.add(kt, cb, sub0 + 32 * t, map_col<kPad>(m, j), dq[m][j]);
          }
        }
        if (kSubs == 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto step = [&](int k0, const char* now, char* then) {
    const int next = k0 + kTile;
    if (next < n)
      stage.load(kp, a.k.l, vp, a.v.l, a.D, a.Dv, next, n, then);
    pass(std::false_type{}, k0, now);
    if (next < n) stage.store(n - next, then);
    __syncthreads();
  };
  stage.clear(a.D, a.Dv, even);
  stage.clear(a.D, a.Dv, odd);
  __syncthreads();
  if (begin < n) {
    stage.load(kp, a.k.l, vp, a.v.l, a.D, a.Dv, begin, n, even);
    stage.store(n - begin, even);
  }
  __syncthreads();
  const int full = (n - begin) / kTile;
  int k0 = begin;
  for (int t = 0; t < full;) {
    step(k0, even, odd);
    k0 += kTile;
    if (++t == full) break;
    step(k0, odd, even);
    k0 += kTile;
    ++t;
  }
  if (k0 < n) pass(std::true_type{}, k0, full & 1 ? odd : even);

  dlam = both_sum(dlam) * back + (split == 0 ? st.w : 0.f);
  if (!live) return;
  const long part = (long)split * a.B * a.H * a.Q + stat;
  if ((kMaps & 2) && half == 0) a.dlam_rows[part] = dlam;
  if (!a.dq.p) return;
  T* out = row_of<T>(a.dq, b, h, q);
  float* sum = a.dq_part + part * 2 * a.D;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < (kMaps >> m & 1 ? S::kMapBlocks : 0); ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (kPad == 16 && g / 2 != m) continue;
        const int d = (kPad == 16 ? 8 * (g % 2) : 32 * j + 8 * g) + 4 * half;
        const f32x16 x = dq[m][j] * back * (m ? -lam * a.scale : a.scale);
        if (a.dq_splits > 1)
          store4(sum + m * a.D + d, a.D - d, x[4 * g], x[4 * g + 1],
                 x[4 * g + 2], x[4 * g + 3]);
        else
          store4(out + m * a.D + d, a.D - d, x[4 * g], x[4 * g + 1],
                 x[4 * g + 2], x[4 * g + 3]);
      }
}

// dk of the maps in kMaps (bits) and, with kDv, dv: a wave holds 32 keys and
// passes over the queries of the heads that share them
template <typename T, int kPad, bool kDirect, int kMaps, bool kDv>
__global__ void __launch_bounds__(
    64 * kBwdWaves, (kResident<T, kPad, kDirect, !kDv && kMaps != 3>))
    diff_bwd_dkv(NpfDiffAttnArgs a) {
  using S = Shape<T, kPad>;
  using Lds = Tile<T, S::kWidth>;
  constexpr int kWaves = kBwdWaves;
  constexpr bool kDk = kMaps != 0;
  constexpr int kTile = kDk && !S::kBothGrads ? 32 : S::kTile;
  constexpr int kTileBytes = kTile * S::kRowBytes;
  // two objects, so that it shows that the next tiles' loads do not touch
  // what is being read
  __shared__ __attribute__((aligned(16))) char even[2 * kTileBytes];
  __shared__ __attribute__((aligned(16))) char odd[2 * kTileBytes];
  // Of each tile's queries what the products start from, and what parts the
  // two maps: the scores' -lse_i / c in 16 bits, where the maps' rounding hides
  // that they are summed at that size (lse_i in 32 bits); -delta_1 and
  // delta_2 - delta_1 (for scaled maps lam times that).
  constexpr bool kFromLse = sizeof(T) == 2;
  __shared__ __attribute__((aligned(16))) float even_stats[4][kTile];
  __shared__ __attribute__((aligned(16))) float odd_stats[4][kTile];

  const int group = a.H / a.Hk;
  const int key_tiles = (a.K + 32 * kWaves - 1) / (32 * kWaves);
  const int heads = a.B * a.Hk, bh = blockIdx.x % heads;
  const int key_tile = blockIdx.x / heads % key_tiles;
  const int split = blockIdx.x / heads / key_tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int key = (key_tile * kWaves + (threadIdx.x >> 6)) * 32 + col;
  const int n = keys_of(a, b);
  const bool live = key < n;
  const float c = a.scale * kLog2e;
  const int rows_base = Lds::rows_base(lane), cols_base = Lds::cols_base(lane);

  u32x4 kf[2][S::kSteps], vf[2 * S::kSteps];
#pragma unroll
  for (int u = 0; u < 2 * S::kSteps; ++u) {
    u32x4 x{0, 0, 0, 0}, y{0, 0, 0, 0};
    if (live) {
      x = load_chunk(row_of<T>(a.k, b, hk, key),
                     chunk_of_maps<T, kPad>(u * 2 + half, a.D));
      if (kDk)
        y = load_chunk(row_of<T>(a.v, b, hk, key),
                       chunk_of_row<T, kPad>(u * 2 + half, a.Dv));
    }
    kf[u / S::kSteps][u % S::kSteps] = x;
    vf[u] = y;
  }
  f32x16 dk[2][S::kMapBlocks], dv[S::kBlocks];
#pragma unroll
  for (int j = 0; j < S::kMapBlocks; ++j) dk[0][j] = dk[1][j] = f32x16{};
#pragma unroll
  for (int j = 0; j < S::kBlocks; ++j) dv[j] = f32x16{};

  // Maps are taken 2^e times as large, all rows' by one e: they meet in sums.
  // For dv, P_1 - lam P_2 is rounded as 2^ea times itself, below 2^15 as well.
  float e = 0.f, ea = 0.f;
  if constexpr (kScaledGrads<T>) {
    if (kDv) {
      float most = 0.f;
      for (int i = lane; i < group; i += 64)
        most = fmaxf(most, fabsf(lam_of(a, hk * group + i)));
      ea = reach_exponent(1.f + wave_allreduce_max(most));
    }
    e = kDk ? reach_exponent(
                  reach_bound(reach_of_dout(a, bh), reach_of_values(a, bh)))
            : ea;
  }
  auto power = [](float x) {
    return kScaledGrads<T> ? __builtin_amdgcn_exp2f(x) : 1.f;
  };
  const float back = power(-e), dv_back = power(-ea), to_dv = power(ea - e);

  // (head, tile) pairs in one sequence, this split's part of it; none where
  // the block has no keys
  const int q_tiles = (a.Q + kTile - 1) / kTile;
  const int per = (group * q_tiles + a.dkv_splits - 1) / a.dkv_splits;
  const int step0 = split * per;
  int steps = group * q_tiles;
  steps = steps - step0 < per ? steps : step0 + per;
  if (key_tile * 32 * kWaves >= n) steps = 0;
  StagePair<T, S::kWidth, kTile, 64 * kWaves, kDirect> stage;
  float4 st;
  float lam = 0.f, next_lam = 0.f;
  // the tile that is being loaded
  int next_h = hk * group + step0 / q_tiles, next_q = step0 % q_tiles * kTile;
  auto load = [&](char* to) {
    next_lam = lam_of(a, next_h);
    stage.load(row_of<T>(a.q, b, next_h, 0), a.q.l,
               row_of<T>(a.dout, b, next_h, 0), a.dout.l, a.D, a.Dv, next_q,
               a.Q, to);
    const int q = next_q + (int)threadIdx.x;
    // rows that are not there have no weight
    st = float4{INFINITY, INFINITY, 0.f, 0.f};
    if (threadIdx.x < kTile && q < a.Q)
      st = reinterpret_cast<const float4*>(
          a.stats)[((long)b * a.H + next_h) * a.Q + q];
  };
  auto store = [&](char* to, float (*to_stats)[kTile]) {
    stage.store(a.Q - next_q, to);
    if (threadIdx.x < kTile) {
      if (kScaledGrads<T>) {
        st.x -= e;
        st.y -= e;
      }
      to_stats[0][threadIdx.x] = kFromLse ? -st.x / c : st.x;
      to_stats[1][threadIdx.x] = kFromLse ? -st.y / c : st.y;
      to_stats[2][threadIdx.x] = -st.z;
      to_stats[3][threadIdx.x] =
          kScaledGrads<T> ? next_lam * (st.w - st.z) : st.w - st.z;
    }
    next_q += kTile;
    if (next_q >= a.Q) {
      next_q = 0;
      ++next_h;
    }
  };
  auto pass = [&](const char* qt, const float (*stats)[kTile]) {
    const char* gt = qt + kTileBytes;
    const int rb = fresh(rows_base), cb = fresh(cols_base);
#pragma unroll
    for (int sub = 0; sub < kTile; sub += 32) {
      f32x16 p[2], x;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (!kDv && !(kMaps >> m & 1)) continue;
        p[m] = kFromLse ? rows16(stats[m], sub, half) : f32x16{};
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
          if (!S::taken(part, kPad, a.D)) continue;
#pragma unroll
          for (int u = S::from(S::kSteps, part);
               u < S::upto(S::kSteps, part); ++u) {
            p[m] = mma_chunk<T>(Lds::rows(qt, rb, sub, m * S::kSteps + u),
                                kf[m][u], p[m]);
          }
        }
        if constexpr (kFromLse) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            p[m][i] = __builtin_amdgcn_exp2f(p[m][i] * c);
        } else {
          const f32x16 lse = rows16(stats[m], sub, half);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            p[m][i] =
                __builtin_amdgcn_exp2f(__builtin_fmaf(p[m][i], c, -lse[i]));
        }
        // (scaled maps take lam in the two sums below instead)
        if (m && !kScaledGrads<T>) p[m] *= lam;
      }
      if (kDv) {
        const float lam_dv = lam * to_dv;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (kScaledGrads<T>)
            x[i] = __builtin_fmaf(-lam_dv, p[1][i], p[0][i] * to_dv);
          else
            x[i] = p[0][i] - p[1][i];
        }
        const Operand<T> map[1] = {Operand<T>(x)};
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
          if (!S::taken(part, 2 * kPad, a.Dv)) continue;
#pragma unroll
          for (int j = S::from(S::kBlocks, part);
               j < S::upto(S::kBlocks, part); ++j) {
            f32x16* const acc[1] = {&dv[j]};
            Lds::template transposed<1>(gt, cb, sub, 32 * j, map, acc);
            // (reads of later columns would be taken ahead into registers that
            // are not there)
            if (kPad * (int)sizeof(T) > 256) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      if (kDk) {
        x = rows16(stats[2], sub, half);
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
          if (!S::taken(part, 2 * kPad, a.Dv)) continue;
#pragma unroll
          for (int u = S::from(2 * S::kSteps, part);
               u < S::upto(2 * S::kSteps, part); ++u) {
            x = mma_chunk<T>(Lds::rows(gt, rb, sub, u), vf[u], x);
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (!(kMaps >> m & 1)) continue;
          if (m == 0) {
            p[m] *= x;
          } else if constexpr (kScaledGrads<T>) {
            const f32x16 apart = rows16(stats[3], sub, half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              p[m][i] *= __builtin_fmaf(-lam, x[i], apart[i]);
          } else {
            p[m] *= rows16(stats[3], sub, half) - x;
          }
          const Operand<T> ds[1] = {Operand<T>(p[m])};
#pragma unroll
          for (int part = 0; part < S::kParts; ++part) {
            if (!S::taken(part, kPad, a.D)) continue;
#pragma unroll
            for (int j = S::from(S::kMapBlocks, part);
                 j < S::upto(S::kMapBlocks, part); ++j) {
              f32x16* const acc[1] = {&dk[m][j]};
              Lds::template transposed<1>(qt, cb, sub, map_col<kPad>(m, j), ds,
                                          acc);
            }
          }
        }
      }
      // (the next tile's reads, taken ahead, would not fit the registers)
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto turn = [&](int step, const char* now, const float (*now_stats)[kTile],
                  char* then, float (*then_stats)[kTile]) {
    const bool more = step + 1 < steps;
    lam = next_lam;
    if (more) load(then);
    pass(now, now_stats);
    if (more) store(then, then_stats);
    __syncthreads();
  };
  stage.clear(a.D, a.Dv, even);
  stage.clear(a.D, a.Dv, odd);
  __syncthreads();
  if (step0 < steps) {
    load(even);
    store(even, even_stats);
  }
  __syncthreads();
  for (int step = step0; step < steps;) {
    turn(step, even, even_stats, odd, odd_stats);
    if (++step == steps) break;
    turn(step, odd, odd_stats, even, even_stats);
    ++step;
  }

  if (key >= a.K) return;
  // keys behind the last one take no part, whatever their lanes hold
  const long part = ((long)split * a.B * a.Hk + bh) * a.K + key;
  if (kDk && a.dk.p) {
    T* out = row_of<T>(a.dk, b, hk, key);
    float* sum = a.dk_part + part * 2 * a.D;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < (kMaps >> m & 1 ? S::kMapBlocks : 0); ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (kPad == 16 && g / 2 != m) continue;
          const int d = (kPad == 16 ? 8 * (g % 2) : 32 * j + 8 * g) + 4 * half;
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i] = live ? dk[m][j][4 * g + i] * back * a.scale : 0.f;
          if (a.dkv_splits > 1)
            store4(sum + m * a.D + d, a.D - d, x[0], x[1], x[2], x[3]);
          else
            store4(out + m * a.D + d, a.D - d, x[0], x[1], x[2], x[3]);
        }
  }
  if (kDv && a.dv.p) {
    T* out = row_of<T>(a.dv, b, hk, key);
    float* sum = a.dv_part + part * a.Dv;
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * j + 8 * g + 4 * half;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = live ? dv[j][4 * g + i] * dv_back : 0.f;
        if (a.dkv_splits > 1)
          store4(sum + d, a.Dv - d, x[0], x[1], x[2], x[3]);
        else
          store4(out + d, a.Dv - d, x[0], x[1], x[2], x[3]);
      }
  }
}

// -------------------------------- launches -------------------------------- //

template <typename K>
hipError_t launch(K kernel, long blocks, int threads, const NpfDiffAttnArgs& a,
                  hipStream_t stream) {
  if (blocks > 0x7fffffffL) return hipErrorInvalidConfiguration;
  kernel<<<(unsigned)blocks, threads, 0, stream>>>(a);
  return hipGetLastError();
}

template <typename T, int kPad, bool kDirect>
hipError_t fwd_sized(const NpfDiffAttnArgs& a, hipStream_t stream) {
  const long heads = (long)a.B * a.Hk, rows = (long)(a.H / a.Hk) * a.Q;
  const long each = heads * a.splits;
  if (a.waves == 1)
    return launch(diff_fwd<T, kPad, 1, kDirect>, each * ((rows + 31) / 32),
                  128, a, stream);
  return launch(diff_fwd<T, kPad, 4, kDirect>, each * ((rows + 127) / 128),
                512, a, stream);
}

template <typename T, int kPad, bool kDirect>
hipError_t bwd_sized(const NpfDiffAttnArgs& a, hipStream_t stream) {
  const long heads = (long)a.B * a.Hk, rows = (long)(a.H / a.Hk) * a.Q;
  using S = Shape<T, kPad>;
  hipError_t e = hipSuccess;
  auto dq = [&](auto maps) {
    if (e == hipSuccess)
      e = launch(diff_bwd_dq<T, kPad, kDirect, decltype(maps)::value>,
                 heads * a.dq_splits * ((rows + 127) / 128), 256, a, stream);
  };
  auto dkv = [&](auto maps, auto with_dv) {
    if (e == hipSuccess)
      e = launch(diff_bwd_dkv<T, kPad, kDirect, decltype(maps)::value,
                              decltype(with_dv)::value>,
                 heads * a.dkv_splits * ((a.K + 127) / 128), 256, a, stream);
  };
  using None = std::integral_constant<int, 0>;
  using First = std::integral_constant<int, 1>;
  using Second = std::integral_constant<int, 2>;
  using Both = std::integral_constant<int, 3>;
  if (a.dq.p || a.dlam) {
    if constexpr (S::kDqMapsApart) {
      dq(First{});
      dq(Second{});
    } else {
      dq(Both{});
    }
  }
  if constexpr (S::kBothGrads) {
    if (a.dk.p || a.dv.p) dkv(Both{}, std::true_type{});
  } else {
    if (a.dk.p) {
      if constexpr (S::kDkMapsApart) {
        dkv(First{}, std::false_type{});
        dkv(Second{}, std::false_type{});
      } else {
        dkv(Both{}, std::false_type{});
      }
    }
    if (a.dv.p) dkv(None{}, std::true_type{});
  }
  return e;
}

// whether rows can move to LDS by themselves: 16-byte aligned
template <typename T>
bool direct(const NpfHeads& t) {
  const long n = kChunk<T>;
  return reinterpret_cast<size_t>(t.p) % 16 == 0 && t.b % n == 0 &&
         t.h % n == 0 && t.l % n == 0 && t.l < (1 << 24);
}

template <typename T, int kPad>
hipError_t sized(const NpfDiffAttnArgs& a, bool bwd, hipStream_t stream) {
  if (a.D % kChunk<T> == 0 && a.Dv % kChunk<T> == 0 && direct<T>(a.k) &&
      direct<T>(a.v) && (!bwd || (direct<T>(a.q) && direct<T>(a.dout))))
    return bwd ? bwd_sized<T, kPad, true>(a, stream)
               : fwd_sized<T, kPad, true>(a, stream);
  return bwd ? bwd_sized<T, kPad, false>(a, stream)
             : fwd_sized<T, kPad, false>(a, stream);
}

template <typename T>
hipError_t typed(const NpfDiffAttnArgs& a, bool bwd, hipStream_t stream) {
  switch (a.pad) {
    case 16: return sized<T, 16>(a, bwd, stream);
    case 32: return sized<T, 32>(a, bwd, stream);
    case 64: return sized<T, 64>(a, bwd, stream);
    default: return sized<T, 128>(a, bwd, stream);
  }
}

}  // namespace npf_attn
