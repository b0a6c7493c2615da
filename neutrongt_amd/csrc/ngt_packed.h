// Tiles of the packed-window attention: 64 (or 32) rows of one head in LDS,
// read both as rows and as columns by the 32 x 32 matrix instructions.
//
// Lane layouts of the instructions (half = lane / 32, l = lane % 32):
//   D (32 x 32): lane holds D[8*(i/4) + 4*half + i%4][l], i < 16
//   bf16, K = 16: lane holds A[l][8*half + e] and B[8*half + e][l], e < 8
//   fp32, K = 2:  lane holds A[l][half] and B[half][l]
// A contraction may take its indices in any order as long as A and B agree,
// and the rows of A may be any 32 rows of the tile.  Both freedoms are used:
//  * row m of A is tile row 32t + 16*((m/4)%2) + 4*(m/8) + m%4, so that a lane
//    holds the scores of 16 CONSECUTIVE tile rows 32t + 16*half + i: its 16
//    bucket ids are one 16-byte load, and
//  * registers 8c .. 8c+7 of such a score tile are the B operand of K step c of
//    the next product as they are; its A operand is columns of the same tile
//    rows 32t + 16*half + 8c + e, which ds_read_b64_tr_b16 reads out of the
//    row-major tile (bf16 and pieces) or plain 4-byte reads do (fp32 heads wider
//    than 64: K = 2, one register a step).
// So one copy of a tile in LDS serves Q K^T, P V and every product of the
// backward, and no score leaves the registers.
//
// fp32 up to 64 wide is kept as three bf16 pieces (Pieces2 below): fp32 training of
// 9 windows of 33 to 1,777, heads of 16, 541 us on the fp32 instructions, 198 on pieces.
// Tiles are 16, 32, 64 or 128 wide; 16-wide ones halve a product's K against
// 32 for heads of 8 and 16 (8 heads of 8, 24 windows of 100 to 1,500: 119 -> 104 us).
//
// The 16-byte pieces of a row are permuted by swz(row), without padding.  LDS
// serves a 16-byte read in groups of lanes that are not 8 neighbours, so the
// bits were chosen by the conflict counter: with bits 1, 2 and 4 of the row
// (and 0 where a row fills all 64 banks) row reads and ds_read_b64_tr_b16 reads
// of every row size have none; with bits 0, 1 and 4 a row read took 12 clocks
// instead of 8.
#pragma once

#include "ngt_common.h"

#include <type_traits>

namespace ngt {
namespace packed {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Work-item and work-group ids as register reads: with the IEEE mode bit off
// (see build.py) the functions behind threadIdx and blockIdx are not inlined.
__device__ __forceinline__ int tid_x() { return static_cast<int>(__builtin_amdgcn_workitem_id_x()); }
__device__ __forceinline__ int wg_x() { return static_cast<int>(__builtin_amdgcn_workgroup_id_x()); }

// The wave's number in its block, known to be the same in all its lanes: what
// depends on it alone is decided once, on the scalar unit.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(tid_x() >> 6); }

__device__ __forceinline__ f32x16 fill16(float v) {
  f32x16 r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = v;
  return r;
}

// The bits of a value that may be a NaN.  These files are compiled as if there were none
// (see build.py), so a comparison of one may come out either way, and what is derived
// from its bits is not to be concluded from the arithmetic that made it.
__device__ __forceinline__ uint32_t bits_of(float x) {
  uint32_t b = __float_as_uint(x);
  asm("" : "+v"(b));
  return b;
}
__device__ __forceinline__ bool is_nan(float x) { return (bits_of(x) & 0x7fffffffu) > 0x7f800000u; }

// The two wave halves' values of a row, joined: v_permlane32_swap leaves the
// lower half's value in r[0] and the upper half's in r[1] of both.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// fp32 operands as three bf16 pieces: x = hi + mid + lo, each the rounding of
// what the ones before it leave.  Six of the nine products of two such operands
// reach fp32 precision (the three left out are below 2^-24 of the first), and
// the bf16 matrix instructions are 16 times as fast as the fp32 ones.  What lies
// below 2^-110 keeps fewer bits (its lower pieces fall below the type), a value above
// bf16's largest, 3.39e38, is an infinity, and a sum that an infinity enters may be NaN
// (infinity times a zero piece).
struct Pieces2 {
  uint32_t hi, mid, lo;
};
template <bool FINITE>
__device__ __forceinline__ Pieces2 split2(float a, float b) {
  auto low = [](uint32_t w) { return __uint_as_float(w << 16); };
  auto high = [](uint32_t w) { return __uint_as_float(w & 0xffff0000u); };
  Pieces2 r;
  r.hi = pack2_bf16(a, b);
  a -= low(r.hi), b -= high(r.hi);
  if constexpr (!FINITE) {  // an infinity is its first piece
    if ((r.hi & 0x7f80u) == 0x7f80u) a = 0.f;
    if ((r.hi & 0x7f800000u) == 0x7f800000u) b = 0.f;
  }
  r.mid = pack2_bf16(a, b);
  r.lo = pack2_bf16(a - low(r.mid), b - high(r.mid));
  return r;
}

// DP: the head size rounded up to 16, 32, 64 or 128; T: float or bf16_t.  fp32
// tiles up to 64 wide hold three planes of bf16 pieces, 32 rows of a plane side
// by side; wider ones (whose operands would fill the registers three times over)
// are fp32 and run on the fp32 instructions.
template <typename T, int DP>
struct Tile {
  static constexpr int kEs = static_cast<int>(sizeof(T));
  static constexpr bool kSplit = kEs == 4 && DP <= 64;
  static constexpr int kPlanes = kSplit ? 3 : 1;
  static constexpr int kPitch = DP * (kSplit ? 2 : kEs);  // bytes of a row of a plane
  static constexpr int kRow = kPitch * kPlanes;           // bytes of a row in LDS
  static constexpr int kPieces = kPitch / 16;  // 16-byte pieces of a plane's row
  static constexpr int kChunks = kPitch / 32;  // mma steps of a row
  static constexpr int kCols = DP < 32 ? 1 : DP / 32;  // 32-column blocks of a row
  static constexpr int kMemPieces = DP * kEs / 16;  // 16-byte pieces of a row in memory
  static constexpr int kRaw = kSplit ? 2 : 1;  // of them in one lane's share of a chunk

  // One lane's share of a chunk of an operand's row: 16 bytes at 32c + 16*half
  // of each plane.
  struct Op {
    u32x4 p[kPlanes];
  };

  __device__ static __forceinline__ int swz(int row) {
    int f = row >> 4 & 1;
    if constexpr (kPieces >= 4) f |= row >> 1 & 2;
    if constexpr (kPieces >= 8) f |= row << 1 & 4;
    if constexpr (kPieces >= 16) f |= row << 3 & 8;
    return f;
  }
  // of a row's piece in the first plane
  __device__ static __forceinline__ int offset(int row, int piece) {
    return (kPlanes > 1 ? (row >> 5) * 32 * kRow + (row & 31) * kPitch : row * kPitch) +
           ((piece ^ swz(row)) << 4);
  }
  // Row operand A of rows 32t ..: lane l's row (without 32t).
  __device__ static __forceinline__ int a_row(int l) {
    return 16 * ((l >> 2) & 1) + 4 * (l >> 3) + (l & 3);
  }
  __device__ static __forceinline__ Op load_a(const char* tile, int t, int c, int l, int half) {
    Op r;
#pragma unroll
    for (int n = 0; n < kPlanes; ++n)
      r.p[n] = *reinterpret_cast<const u32x4*>(tile + 32 * t * kRow + 32 * n * kPitch +
                                               offset(a_row(l), 2 * c + half));
    return r;
  }
  // An operand from a row's bytes in memory: kRaw times 16.
  __device__ static __forceinline__ Op op_of(const u32x4 (&raw)[kRaw]) {
    Op r;
    if constexpr (kSplit) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pieces2 x = split2<false>(__uint_as_float(raw[i / 2][2 * (i & 1)]),
                                        __uint_as_float(raw[i / 2][2 * (i & 1) + 1]));
        r.p[0][i] = x.hi, r.p[1][i] = x.mid, r.p[2][i] = x.lo;
      }
    } else {
      r.p[0] = raw[0];
    }
    return r;
  }
  // Writes one 16-byte piece of a row in memory to the tile.
  __device__ static __forceinline__ void put(char* tile, int row, int piece, const u32x4& w) {
    if constexpr (kSplit) {
      const Pieces2 a = split2<false>(__uint_as_float(w[0]), __uint_as_float(w[1]));
      const Pieces2 b = split2<false>(__uint_as_float(w[2]), __uint_as_float(w[3]));
      char* at = tile + offset(row, piece >> 1) + 8 * (piece & 1);
      *reinterpret_cast<uint2*>(at) = make_uint2(a.hi, b.hi);
      *reinterpret_cast<uint2*>(at + 32 * kPitch) = make_uint2(a.mid, b.mid);
      *reinterpret_cast<uint2*>(at + 64 * kPitch) = make_uint2(a.lo, b.lo);
    } else {
      *reinterpret_cast<u32x4*>(tile + offset(row, piece)) = w;
    }
  }

  // c += A B over one chunk of both rows (16 elements; 8 of whole fp32).
  __device__ static __forceinline__ f32x16 mma(const Op& a, const Op& b, f32x16 c) {
    if constexpr (kEs == 4 && !kSplit) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.p[0][i]),
                                                 __uint_as_float(b.p[0][i]), c, 0, 0, 0);
      return c;
    } else {
      auto step = [&](int i, int j) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.p[i]),
                                                    __builtin_bit_cast(bf16x8, b.p[j]), c, 0, 0, 0);
      };
      if constexpr (kSplit) step(2, 0), step(0, 2), step(1, 1), step(1, 0), step(0, 1);
      step(0, 0);
      return c;
    }
  }

  // acc[dt] (rows = columns 32dt .. of the tile) += tile^T p over tile rows
  // 32t .. 32t+31, p the lane's 16 values of those rows; for bf16 rounded to it,
  // or, with FINE, as two bf16 pieces (16 bits).
  template <bool FINE = false>
  __device__ static __forceinline__ void mma_cols(const char* tile, int t, const f32x16& p,
                                                  f32x16 (&acc)[kCols], int lane) {
    const int half = lane >> 5;
    if constexpr (kEs == 2 || kSplit) {
      const int j = lane & 15;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        Op b, rest;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (FINE && !kSplit) {
            const float x = p[8 * c + 2 * e], y = p[8 * c + 2 * e + 1];
            const uint32_t hi = pack2_bf16(x, y);
            b.p[0][e] = hi;
            rest.p[0][e] = pack2_bf16(x - __uint_as_float(hi << 16),
                                      y - __uint_as_float(hi & 0xffff0000u));
          } else if constexpr (kSplit) {
            const Pieces2 x = split2<true>(p[8 * c + 2 * e], p[8 * c + 2 * e + 1]);
            b.p[0][e] = x.hi, b.p[1][e] = x.mid, b.p[2][e] = x.lo;
          } else {
            b.p[0][e] = pack2_bf16(p[8 * c + 2 * e], p[8 * c + 2 * e + 1]);
          }
        }
        // rows j / 4 and then 4 further: of swz() only bit 1 depends on more than the lane
        const int row = 16 * half + (j >> 2);
        // (of a 16-wide tile columns 16 .. 31 are 0 .. 15 again: nobody reads those sums)
        const int piece = (DP < 32 ? 0 : 2 * ((lane >> 4) & 1)) + ((j & 3) >> 1);
        constexpr int kFlip = kPieces >= 4 ? 32 : 0;
        const int at = (piece ^ swz(row)) * 16 + 8 * (j & 1) + row * kPitch;
#pragma unroll
        for (int dt = 0; dt < kCols; ++dt) {
          Op a;
#pragma unroll
          for (int n = 0; n < kPlanes; ++n) {
            // the column block is bits 2 and 3 of the piece
            const char* base = tile + 32 * t * kRow + (32 * n + 8 * c) * kPitch;
            typedef __attribute__((address_space(3))) s16x4* lds4_t;
            const s16x4 lo =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(base + (at ^ (dt << 6))));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds4_t)(base + 4 * kPitch + (at ^ (dt << 6) ^ kFlip)));
            const uint2 lw = __builtin_bit_cast(uint2, lo), hw = __builtin_bit_cast(uint2, hi);
            a.p[n] = u32x4{lw.x, lw.y, hw.x, hw.y};
          }
          if constexpr (FINE && !kSplit) acc[dt] = mma(a, rest, acc[dt]);
          acc[dt] = mma(a, b, acc[dt]);
        }
      }
    } else {
      const int l = lane & 31;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = 16 * half + i;
#pragma unroll
        for (int dt = 0; dt < kCols; ++dt) {
          const float a = *reinterpret_cast<const float*>(
              tile + 32 * t * kPitch + offset(row, 8 * dt + (l >> 2)) + 4 * (l & 3));
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[i], acc[dt], 0, 0, 0);
        }
      }
    }
  }
};

// A lane's row of one head as the operands it supplies to mma, zero behind the
// row's d elements or where the row is not there.
template <typename T, int DP>
struct RowFrag {
  using L = Tile<T, DP>;
  typename L::Op w[L::kChunks];
  __device__ __forceinline__ void load(const T* __restrict__ row, bool ok, int d, int half) {
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c) {
      const int at = (2 * c + half) * 16 * L::kRaw;  // bytes
      u32x4 raw[L::kRaw];
#pragma unroll
      for (int i = 0; i < L::kRaw; ++i) {
        raw[i] = u32x4{0u, 0u, 0u, 0u};
        if (ok && at < d * L::kEs)
          raw[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(row) + at + 16 * i);
      }
      w[c] = L::op_of(raw);
    }
  }
  // -x for every element where `odd`
  __device__ __forceinline__ void negate(bool odd) {
    const uint32_t m = !odd ? 0u : L::kEs == 2 || L::kSplit ? 0x80008000u : 0x80000000u;
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
      for (int n = 0; n < L::kPlanes; ++n) w[c].p[n] ^= u32x4{m, m, m, m};
  }
};

// Reads through a buffer descriptor: 16 or 4 bytes at a byte offset of a base that
// is the same in all lanes; what lies at or behind `bytes` reads as zero, so a
// tile's missing rows cost neither a branch nor a select.
using Buffer = __amdgpu_buffer_rsrc_t;
constexpr int kMostBytes = 0x7fffff00;
constexpr int kNowhere = 0x7ffffff0;  // an offset behind every buffer's end
__device__ __forceinline__ Buffer make_buffer(const void* base, int64_t bytes) {
  const int n = bytes > kMostBytes ? kMostBytes : bytes < 0 ? 0 : static_cast<int>(bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, n, 0x00027000);
}
__device__ __forceinline__ u32x4 read16(Buffer b, int offset) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0));
}
__device__ __forceinline__ float read4(Buffer b, int offset) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, offset, 0, 0));
}

// The 16-byte pieces of ROWS rows of one head that one of N threads moves from
// memory to an LDS tile; rows behind the window's end and columns behind d are
// zero.  ROWS rows span less than 2^31 bytes (kMostRowBytes).
constexpr int64_t kMostRowBytes = (1 << 23) - 1;  // of 256 rows, and room for a last row
template <typename T, int DP, int ROWS, int N>
struct Stage {
  using L = Tile<T, DP>;
  static constexpr int kTotal = ROWS * L::kMemPieces;
  static constexpr int NV = (kTotal + N - 1) / N;
  u32x4 w[NV];
  int at[NV];
  __device__ __forceinline__ Stage(int64_t stride, int d, int tid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int r = (tid + i * N) / L::kMemPieces, p = (tid + i * N) % L::kMemPieces;
      at[i] = 16 * p < d * L::kEs ? r * static_cast<int>(stride) + 16 * p : kNowhere;
    }
  }
  // rows row0 .. of the n_rows at base, `stride` bytes apart
  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int n_rows, int d) {
    const Buffer b =
        make_buffer(reinterpret_cast<const char*>(base) + int64_t(row0) * stride,
                    row0 < n_rows ? int64_t(n_rows - row0 - 1) * stride + d * L::kEs : 0);
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = read16(b, at[i]);
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = tid + i * N;
      if (kTotal % N == 0 || e < kTotal) L::put(tile, e / L::kMemPieces, e % L::kMemPieces, w[i]);
    }
  }
};

// A block is RW x KS waves: RW waves of 32 rows each, KS of them on the same
// rows, each on its own 64 of the 64 * KS rows of the other side that a stage
// holds.  More row waves share a stage's tile among more rows; more sets
// shorten the longest block and fill the chip where rows are few.  At the end
// the sets' sums of a row wave are added in set order.
template <int RW, int KS>
struct Block {
  static constexpr int kThreads = 64 * RW * KS;
  static constexpr int kStage = 64 * KS;                        // rows of a stage
  static constexpr int kJoinBytes = (KS - 1) * RW * 64 * 16 * 4;  // of one accumulator
};

// Adds the sets' accumulators into set 0's; buf holds kJoinBytes.  Every wave
// calls it; the block's earlier reads of buf are done (a barrier is passed here).
template <int RW, int KS>
__device__ __forceinline__ void join_sets(f32x16& acc, char* buf, int rw, int set, int lane) {
  if constexpr (KS > 1) {
    float4* b = reinterpret_cast<float4*>(buf);
    __syncthreads();
    if (set > 0) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        b[(((set - 1) * RW + rw) * 4 + g) * 64 + lane] =
            make_float4(acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]);
    }
    __syncthreads();
    if (set == 0) {
#pragma unroll
      for (int s = 0; s < KS - 1; ++s)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 y = b[((s * RW + rw) * 4 + g) * 64 + lane];
          acc[4 * g] += y.x, acc[4 * g + 1] += y.y, acc[4 * g + 2] += y.z, acc[4 * g + 3] += y.w;
        }
    }
  }
}

// 4 consecutive values of a row.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 2) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
                       __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  } else {
    return *reinterpret_cast<const float4*>(p);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2_bf16(a, b), pack2_bf16(c, d));
  else
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}

// Bucket ids of a lane's 16 tile rows, and the bias table of one head in LDS:
// entries in log2 units, -inf (not attended) behind the n_buckets there are.
// Finite entries act as if within +-2^60: a row of the type's lowest values
// still gives every pair the same weight instead of none.
//
// A bias beyond kFar in a row's greatest score leaves no bits in fp32 for the base
// and the sum in one number, nor for starting a product from it: such rows subtract
// the base and then log2 of the sum, each by itself, and keep both (lse and, H * n_q
// further, the logarithm).  They are as rare as masks of large finite values: a wave
// that has one takes a few instructions a score more.
constexpr int kTable = 256;
constexpr float kFar = 256.f;
__device__ __forceinline__ bool is_far(float base) {  // an infinity or a NaN is not
  const uint32_t from = __float_as_uint(kFar);
  return (bits_of(base) & 0x7fffffffu) - from < 0x7f800000u - from;
}
template <typename T>
__device__ __forceinline__ void load_table(float* tab, const void* __restrict__ table, int table_f32,
                                           int n_buckets, int n_heads, int h, int tid,
                                           int n_threads) {
  for (int b = tid; b < kTable; b += n_threads) {
    float x = -INFINITY;
    if (b < n_buckets) {
      const int64_t at = int64_t(b) * n_heads + h;
      x = table_f32 ? static_cast<const float*>(table)[at]
                    : elem<T>::load(static_cast<const T*>(table) + at);
      const uint32_t mag = __float_as_uint(x) & 0x7fffffffu;
      if (mag < 0x7f800000u) x = fminf(fmaxf(x * kLog2e, -0x1p60f), 0x1p60f);
    }
    tab[b] = x;
  }
}
__device__ __forceinline__ int bucket_of(const u32x4& ids, int i) {
  return static_cast<int>((ids[i >> 2] >> (8 * (i & 3))) & 255u);
}

// The table's values for a lane's 16 ids.  All reads are under way before what
// follows (left to itself the compiler waits for each: 16 latencies a tile).
__device__ __forceinline__ f32x16 look_up(const float* tab, const u32x4& ids) {
  f32x16 v;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = tab[bucket_of(ids, i)];
  __builtin_amdgcn_sched_barrier(0);
  return v;
}

}  // namespace packed
}  // namespace ngt

namespace ngt {
namespace packed {

// The blocks there are: row waves and sets (Block).
struct Shape {
  int rw, ks;
};
// The most sets of a kernel: by the LDS of its tiles, and for the dK/dV pass,
// whose two accumulators and two operands fill a wave's registers, by those.
constexpr int most_sets(int row, bool dkv) {
  return row <= 192 ? 4 : row <= 384 && !dkv ? 2 : 1;
}
template <int MOST, typename F>
int with_shape(Shape s, F&& f) {
  using std::integral_constant;
  if (s.rw == 1) return f(integral_constant<int, 1>(), integral_constant<int, 1>());
  if constexpr (MOST >= 2) {
    if (s.ks == 2 && s.rw == 4) return f(integral_constant<int, 4>(), integral_constant<int, 2>());
    if (s.ks == 2) return f(integral_constant<int, 2>(), integral_constant<int, 2>());
  }
  if constexpr (MOST >= 4)
    if (s.ks == 4) return f(integral_constant<int, 2>(), integral_constant<int, 4>());
  if (s.rw == 4) return f(integral_constant<int, 4>(), integral_constant<int, 1>());
  return f(integral_constant<int, 2>(), integral_constant<int, 1>());
}

// ------------------------------------------------------- the backward's launch
struct BwdArgs {
  const int64_t* q_start;
  const int64_t* k_start;
  const int64_t* b_start;
  const int64_t* bt_start;
  const int2* items;
  int n_items;
  int H, Hkv, d, causal, n_buckets, table_f32;
  float scale;
  int64_t sq, sk, sv;  // bytes between rows
  int64_t n_q;
  const void* q;
  const void* k;
  const void* v;
  const void* go;
  const float* out32;
  const float* lse;
  float* dsum;  // [H, n_q]: -D, written by the dQ pass, read by the dK/dV pass
  const void* table;
  const uint8_t* ids;
  const uint8_t* ids_t;
  float* part_table;  // [H, items, n_buckets]
  void* gq;
  void* gk;
  void* gv;
  void* grad_table;
  int32_t hist_shift;
};
// log2 of the columns of a wave's sums per bucket in the dQ pass (doubles).  Fewer let
// more waves run, but more lanes of an instruction meet: 16, 8 in fp32, whose pairs take
// longer elsewhere, and for large tables (forward and backward, us, 32 | 16 | 8 columns:
// 3 windows of 1,000 to 3,333, 32 heads of 24, 64 buckets 1,185 | 1,135 | 1,227; 40 windows of
// 150 to 300, as many heads, 200 buckets 361 | 238 | 193; 4 windows of 750 to 1,500, 40
// buckets, fp32 739 | 716 | 656; 3,001 rows, 8 heads of 8, 10 buckets, fp32 279 | 275 | 289).
// The line at 100 buckets lies between the tables measured, 64 and 200.
inline int hist_shift(bool f32, int n_buckets) { return f32 || n_buckets > 100 ? 3 : 4; }

struct BwdPlan {
  const int2* items_q;
  const int2* items_k;
  int n_items_q;
  Shape dq, dkv;
  int64_t dq_blocks, dkv_blocks;
};
int packed_bwd(int dtype, const BwdPlan& p, const BwdArgs& a, hipStream_t st);

}  // namespace packed
}  // namespace ngt
