// Tiles and matrix products of the differential attention kernels.
//
// All products use 32x32 matrix instructions.  A wave's result tile has its
// column in the lane (lane & 31) and 16 rows in registers: register i of lane
// half h = lane >> 5 holds row  8 (i / 4) + 4 h + i % 4.  Two facts carry the
// kernels:
//
// - with the score tile taken as (row = key, column = query), a query's
//   statistics need no more than a register reduction and one exchange between
//   the lane halves;
// - a tile in that layout is an operand of the next product as it stands: its
//   registers hold 16 rows of one column, and the order of the summed axis is
//   free as long as the other operand follows it.  The other operand, read
//   against its rows (a transposed read of LDS), follows it.
//
// Operands in LDS are row-major tiles of 16-byte chunks.  A row's chunks are
// permuted by an XOR with a function of the row, chosen so that both reads
// spread over all 64 banks: 16 rows at one chunk (an operand read along its
// rows), and 4 + 4 rows at 64 contiguous bytes (the transposed read).
#pragma once

#include "common.h"
#include "diff_attn.h"
#include "types.h"

#include <type_traits>

namespace npf_attn {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using s16x4 = __attribute__((ext_vector_type(4))) short;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.0e38f;  // below every finite score

// the row that register i holds in lane half 0
__host__ __device__ constexpr int reg_row(int i) {
  return 8 * (i / 4) + i % 4;
}

template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);  // values of a chunk

// ------------------------------ products -------------------------------- //

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(float a, float b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

template <typename T> struct Vec8;
template <> struct Vec8<npf_bf16> { using type = bf16x8; };
template <> struct Vec8<npf_f16> { using type = f16x8; };

// c += a b^T over one chunk a lane half: 16 values of the summed axis in 16
// bits, 8 (as four products) in 32
template <typename T>
__device__ __forceinline__ f32x16 mma_chunk(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    using V = typename Vec8<T>::type;
    return mma(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a);
    const f32x4 y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = mma(x[i], y[i], c);
    return c;
  }
}

// A 32x32 tile of map values or of their gradients as an operand.  In 16 bits
// its values are rounded here; statistics have seen them in 32.
template <typename T>
struct Operand {
  using V = typename Vec8<T>::type;
  V v[2];
  __device__ __forceinline__ explicit Operand(const f32x16& x) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[t][e] = (T)x[8 * t + e];
  }
  // what the rounding of x has left (exact in 32 bits), to be rounded in turn
  __device__ __forceinline__ f32x16 rest(f32x16 x) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const u32x4 pairs = __builtin_bit_cast(u32x4, v[t]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float y;
        if constexpr (std::is_same<T, npf_bf16>::value) {
          // (from the pair as it stands: else each value is rounded anew)
          const unsigned u = pairs[e / 2];
          y = __builtin_bit_cast(float, e & 1 ? u & 0xffff0000u : u << 16);
        } else {
          y = (float)v[t][e];
        }
        x[8 * t + e] -= y;
      }
    }
    return x;
  }
};
template <>
struct Operand<float> {
  f32x16 v;
  __device__ __forceinline__ explicit Operand(const f32x16& x) : v(x) {}
};

// -------------------------------- tiles ---------------------------------- //

// A value the compiler is to compute with anew: the many addresses that follow
// from it would otherwise be kept over a loop, each in a register.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <typename T, int kWidth>
struct Tile {
  static constexpr int kRowBytes = kWidth * (int)sizeof(T);
  static constexpr int kChunks = kRowBytes / 16;

  __device__ static __forceinline__ int permute(int row) {
    const int low = (row >> 2) & 3;
    if constexpr (kRowBytes == 64) return low;
    if constexpr (kRowBytes == 128) return low | (((row >> 1) & 1) << 2);
    return low | ((row & 3) << 2);
  }
  __device__ static __forceinline__ int at(int row, int chunk) {
    return row * kRowBytes + ((chunk ^ permute(row)) << 4);
  }

  // Where a lane reads along rows: its row of 32, its half's chunk 0.  The
  // chunks of a row, and the 32-row blocks of a tile, are then constants away
  // (XOR for the former).
  __device__ static __forceinline__ int rows_base(int lane) {
    return at(lane & 31, lane >> 5);
  }
  // chunk 2 pair + half of row row0 + lane % 32
  __device__ static __forceinline__ u32x4 rows(const char* tile, int base,
                                               int row0, int pair) {
    return *reinterpret_cast<const u32x4*>(tile + row0 * kRowBytes +
                                           (base ^ (pair << 5)));
  }

  // where a lane reads against rows
  __device__ static __forceinline__ int cols_base(int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      // lane j of 16 names 4 values of row j / 4, and gets 4 rows of column j
      const int j = lane & 15;
      return at(4 * half + (j >> 2), 2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) +
             (j & 1) * 8;
    } else {
      const int col = lane & 31;
      return at(4 * half, col >> 2) + (col & 3) * 4;
    }
  }

  // acc[lane % 32 of columns col0 ..][column of p] += tile^T p over the 32
  // rows from row0 on, for both maps' p at once
  template <int kMaps>
  __device__ static __forceinline__ void transposed(
      const char* tile, int base, int row0, int col0, const Operand<T> (&p)[kMaps],
      f32x16* const (&acc)[kMaps]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s16x4 part[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          // rows 16 t + 8 a + ...: 8 rows on, bit 1 of the permutation flips
          const char* src = tile + (row0 + 16 * t + 8 * a) * kRowBytes +
                            (base ^ (permute(8 * a) << 4) ^ (col0 << 1));
          part[a] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(src));
        }
        const auto both = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3,
                                                  4, 5, 6, 7);
        const auto v = __builtin_bit_cast(typename Vec8<T>::type, both);
#pragma unroll
        for (int m = 0; m < kMaps; ++m) *acc[m] = mma(v, p[m].v[t], *acc[m]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = *reinterpret_cast<const float*>(
            tile + (row0 + reg_row(i)) * kRowBytes +
            (base ^ (permute(reg_row(i)) << 4) ^ (col0 << 2)));
#pragma unroll
        for (int m = 0; m < kMaps; ++m) *acc[m] = mma(v, p[m].v[i], *acc[m]);
      }
    }
  }
};

// acc += tile^T x as Tile::transposed; kTwice: x is taken as the sum of its
// rounded values and of what rounding left, for 16 bits and more of each
template <typename T, int kWidth, bool kTwice>
struct Product {
  static constexpr int kParts = kTwice ? 2 : 1;
  Operand<T> p[kParts];
  __device__ __forceinline__ explicit Product(const f32x16& x)
      : Product(Operand<T>(x), x) {}
  __device__ __forceinline__ void add(const char* tile, int base, int row0,
                                      int col0, f32x16& acc) const {
    f32x16* at[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) at[i] = &acc;
    Tile<T, kWidth>::template transposed<kParts>(tile, base, row0, col0, p, at);
  }

 private:
  __device__ __forceinline__ Product(const Operand<T>& high, const f32x16& x)
      : p{high, Operand<T>(high.rest(x))} {}
};
template <typename T, int kWidth>
struct Product<T, kWidth, false> {
  Operand<T> p[1];
  __device__ __forceinline__ explicit Product(const f32x16& x)
      : p{Operand<T>(x)} {}
  __device__ __forceinline__ void add(const char* tile, int base, int row0,
                                      int col0, f32x16& acc) const {
    f32x16* const at[1] = {&acc};
    Tile<T, kWidth>::template transposed<1>(tile, base, row0, col0, p, at);
  }
};

// The chunk of a padded row that a thread moves: where its values stand in
// memory, and how many there are (the rest is padding).
struct ChunkOf {
  int offset, count;
};

// of a row in parts of `per` chunks (a power of two: a map's, or the row's), of
// which `size` values are there
template <typename T>
__device__ __forceinline__ ChunkOf chunk_of(int chunk, int per, int size) {
  const int in_part = (chunk & (per - 1)) * kChunk<T>;
  const int left = size - in_part;
  return {(chunk >= per ? size : 0) + in_part,
          left < 0 ? 0 : left > kChunk<T> ? kChunk<T> : left};
}

// of a row with two maps of `size` values, each padded to kPad
template <typename T, int kPad>
__device__ __forceinline__ ChunkOf chunk_of_maps(int chunk, int size) {
  return chunk_of<T>(chunk, kPad / kChunk<T>, size);
}

// of a row of up to 2 kPad values
template <typename T, int kPad>
__device__ __forceinline__ ChunkOf chunk_of_row(int chunk, int size) {
  return chunk_of<T>(chunk, 2 * kPad / kChunk<T>, size);
}

template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, ChunkOf c) {
  T v[kChunk<T>];
  if (c.count == kChunk<T>) {
    load_pack(v, row + c.offset);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk<T>; ++i)
      v[i] = i < c.count ? row[c.offset + i] : (T)0.f;
  }
  u32x4 r;
  __builtin_memcpy(&r, v, 16);
  return r;
}

// A tile of kRows rows on its way from memory to LDS, the next one under the
// products of this one.  kThreads threads move it, `tid` of them this one; a
// row is in parts of `per` chunks, of which `size` values are there.
//
// kDirect: 16-byte aligned rows of whole chunks.  The loads write LDS
// themselves and hold no registers; a wave's 64 chunks land side by side, so
// the permutation is in what each lane reads.  Chunks of padding are never
// written (`clear` makes them zeros once).  Rows behind the end read the last
// one again: no weight meets them, and what they hold has met a weight where it
// counts.
//
// Otherwise the chunks come through registers, each lane testing its own, and
// rows behind the end become zeros.
template <typename T, int kWidth, int kRows, int kThreads, bool kDirect>
struct Stage;

template <typename T, int kWidth, int kRows, int kThreads>
struct Stage<T, kWidth, kRows, kThreads, true> {
  using Lds = Tile<T, kWidth>;
  static constexpr int kCount = kRows * Lds::kChunks / kThreads;
  static_assert(kRows * Lds::kChunks % kThreads == 0 && Lds::kChunks <= 64);

  // Row pairs of the permutation repeat after 16 rows: where a step of all
  // threads is a multiple of that, one offset a lane serves every step.
  static constexpr int kStep = kThreads / Lds::kChunks;

  // All but the last tile are whole, and take their loads from a uniform
  // address and an offset of the lane that stays the same: no vector work a
  // load.
  __device__ __forceinline__ void load(const T* p, long l_, int per, int size,
                                       int row0, int end, int tid,
                                       char* tile) {
    p += row0 * l_;
    const int l = (int)l_, rows = end - row0;
    if (rows >= kRows)
      load_rows<true>(p, l, per, size, rows, tid, tile);
    else
      load_rows<false>(p, l, per, size, rows, tid, tile);
  }

  template <bool kWhole>
  __device__ __forceinline__ static void load_rows(const T* p, int l, int per,
                                                   int size, int rows, int tid,
                                                   char* tile) {
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      // chunk of lane 0 within the step, and its row
      const int first = wave * 64;
      int row = first / Lds::kChunks + lane / Lds::kChunks;
      const int chunk =
          lane % Lds::kChunks ^ Lds::permute(row + (kStep % 16 ? j * kStep : 0));
      if (!kWhole) {
        row += j * kStep;
        row = row < rows ? row : rows - 1;
      }
      const char* src = reinterpret_cast<const char*>(
          p + (kWhole ? (long)j * kStep * l : 0));  // the same for all lanes
      const ChunkOf c = chunk_of<T>(chunk, per, size);
      const unsigned at = (unsigned)(row * l + c.offset) * (int)sizeof(T);
      if (c.count > 0)
        __builtin_amdgcn_global_load_lds(
            (__attribute__((address_space(1))) void*)(src + at),
            (__attribute__((address_space(3))) void*)(tile +
                                                      (j * kThreads + first) *
                                                          16),
            16, 0, 0);
    }
  }

  // the tile becomes zeros, where some chunks will not be loaded
  __device__ __forceinline__ static void clear(int per, int size, int tid,
                                               char* tile) {
    if (size == per * kChunk<T>) return;
    for (int i = tid; i < kRows * Lds::kChunks; i += kThreads)
      reinterpret_cast<u32x4*>(tile)[i] = u32x4{0, 0, 0, 0};
  }

  // before the barrier that shows the tile to every wave
  __device__ __forceinline__ void store(int, int, char*) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), the other counters free
  }
};

template <typename T, int kWidth, int kRows, int kThreads>
struct Stage<T, kWidth, kRows, kThreads, false> {
  using Lds = Tile<T, kWidth>;
  static constexpr int kStep = kThreads / Lds::kChunks;  // rows at a time
  static constexpr int kCount = kRows / kStep;
  static_assert(kThreads % Lds::kChunks == 0 && kRows % kStep == 0);

  u32x4 x[kCount];

  __device__ __forceinline__ static void clear(int, int, int, char*) {}

  __device__ __forceinline__ void load(const T* p, long l, int per, int size,
                                       int row0, int end, int tid, char*) {
    const ChunkOf c = chunk_of<T>(tid % Lds::kChunks, per, size);
    const int first = row0 + tid / Lds::kChunks;
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      const int row = first + j * kStep;
      const int at = row < end ? row : end - 1;
      x[j] = load_chunk(p + at * l, c);
    }
  }

  // `count` rows of the tile are there
  __device__ __forceinline__ void store(int count, int tid, char* tile) {
    const int first = tid / Lds::kChunks, chunk = tid % Lds::kChunks;
    if (count < kRows) {
#pragma unroll
      for (int j = 0; j < kCount; ++j)
        if (first + j * kStep >= count) x[j] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < kCount; ++j)
      *reinterpret_cast<u32x4*>(tile + Lds::at(first + j * kStep, chunk)) =
          x[j];
  }
};

// Two tiles side by side, moved by all of a block's threads: rows of two maps
// of map_size values, and rows of row_size values.
template <typename T, int kWidth, int kRows, int kThreads, bool kDirect>
struct StagePair {
  using One = Stage<T, kWidth, kRows, kThreads, kDirect>;
  static constexpr int kChunks = kWidth / kChunk<T>;
  static constexpr int kTileBytes = kRows * kWidth * (int)sizeof(T);
  One x, y;

  __device__ __forceinline__ void load(const T* xp, long xl, const T* yp,
                                       long yl, int map_size, int row_size,
                                       int row0, int end, char* tiles) {
    const int tid = threadIdx.x;
    x.load(xp, xl, kChunks / 2, map_size, row0, end, tid, tiles);
    y.load(yp, yl, kChunks, row_size, row0, end, tid, tiles + kTileBytes);
  }
  __device__ __forceinline__ static void clear(int map_size, int row_size,
                                               char* tiles) {
    One::clear(kChunks / 2, map_size, threadIdx.x, tiles);
    One::clear(kChunks, row_size, threadIdx.x, tiles + kTileBytes);
  }
  __device__ __forceinline__ void store(int count, char* tiles) {
    x.store(count, threadIdx.x, tiles);
    y.store(count, threadIdx.x, tiles + kTileBytes);
  }
};

// ------------------------------- helpers --------------------------------- //

template <typename T>
__device__ __forceinline__ T* row_of(const NpfHeads& t, int b, int h, long l) {
  return static_cast<T*>(t.p) + b * t.b + h * t.h + l * t.l;
}

__device__ __forceinline__ int keys_of(const NpfDiffAttnArgs& a, int b) {
  if (!a.lengths) return a.K;
  const long n = a.lengths64 ? static_cast<const long*>(a.lengths)[b]
                             : (long)static_cast<const int*>(a.lengths)[b];
  return n < 0 ? 0 : n > a.K ? a.K : (int)n;
}

__device__ __forceinline__ float lam_of(const NpfDiffAttnArgs& a, int h) {
  return load_coded(a.lam, a.lam_type, h * a.lam_stride);
}

// In fp16 gradients of the maps are rounded as 2^e dS: unscaled, those above
// 65504 would become inf where the gradients that follow from them are finite.
// |dS| <= |G - delta|, and G and delta (a mean of G) are products of a row of
// dout and rows of values, so 2 |dO_i| max_j |V_j| bounds it; twice that, and
// the weight of the second map where it is above 1, leave room for the rounding
// that delta has seen.  e brings the bound just below 2^15, which keeps 40
// binary places under it from vanishing.
template <typename T>
constexpr bool kScaledGrads = std::is_same<T, npf_f16>::value;

__device__ __forceinline__ float reach_bound(float dout, float values) {
  return 4.f * dout * values;
}
// the largest e, within reason, with bound 2^e < 2^15; 0 where there is none
__device__ __forceinline__ float reach_exponent(float bound) {
  if (!(bound > 0.f && bound < INFINITY)) return 0.f;
  const int e = 15 - __builtin_amdgcn_frexp_expf(bound);
  return (float)(e < -60 ? -60 : e > 60 ? 60 : e);
}
// the largest of `chunks` of a head's chunks, in every lane of a wave
__device__ __forceinline__ float reach_of(const float* reach, int chunks) {
  float x = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < chunks; i += 64) x = fmaxf(x, reach[i]);
  return wave_allreduce_max(x);
}
__device__ __forceinline__ float reach_of_values(const NpfDiffAttnArgs& a,
                                                 int bh) {
  return reach_of(a.reach + (long)bh * (a.v_chunks + a.o_chunks), a.v_chunks);
}
__device__ __forceinline__ float reach_of_dout(const NpfDiffAttnArgs& a,
                                               int bh) {
  return reach_of(
      a.reach + (long)bh * (a.v_chunks + a.o_chunks) + a.v_chunks, a.o_chunks);
}

// x of the other lane half, for a reduction over both
struct Halves {
  float low, high;
};
__device__ __forceinline__ Halves halves(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned low = r[0], high = r[1];
  return {__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)};
}
// (NaN where one is: without the steps that keep it out)
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}
__device__ __forceinline__ float both_max(float x) {
  const Halves h = halves(x);
  return larger(h.low, h.high);
}
__device__ __forceinline__ float both_sum(float x) {
  const Halves h = halves(x);
  return h.low + h.high;
}

// one value a row of a 32-row block, in the order of a tile's registers
__device__ __forceinline__ f32x16 rows16(const float* of_row, int row0,
                                         int half) {
  f32x16 x;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const f32x4 y =
        *reinterpret_cast<const f32x4*>(of_row + row0 + 8 * r + 4 * half);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * r + i] = y[i];
  }
  return x;
}

// 4 consecutive values of a row, of which `count` exist
template <typename T>
__device__ __forceinline__ void store4(T* p, int count, float a, float b,
                                       float c, float d) {
  const T v[4] = {(T)a, (T)b, (T)c, (T)d};
  if (count >= 4) {
    store_pack(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) p[i] = v[i];
  }
}

}  // namespace npf_attn
