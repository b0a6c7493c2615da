// What the gated linear layer's tiled products share (ngt_gated.hip, ngt_gated_bwd.hip):
// the blocks' tiles, and stages of their operands from memory to LDS and from there to
// the matrix instructions.
#pragma once

#include "ngt_linear.h"

#include <initializer_list>

namespace ngt {

// What the forward keeps for the backward: zu act'(zg) and act(zg), the factors of dy, with 12
// bits of mantissa: the upper 16 bits of the fp32 as rows [M, 2 N], and the 4 bits behind
// them as one word for each 8 columns, in blocks of 32 rows by 32 columns (what a wave of the
// forward writes at a time).  Rounded to bf16
// there the gradients were off by 2.9e-3, of which rounding dz and the results makes 2.4e-3,
// which these leave; the bits cost an eighth of the bytes.
struct Keep {
  int64_t high_bytes, low_blocks;
  int32_t n, across;
  __host__ __device__ Keep(int64_t M, int32_t N)
      : high_bytes((4 * M * N + 255) / 256 * 256), low_blocks((M + 31) / 32), n(N), across((N + 63) / 64) {}
  __host__ __device__ int64_t bytes() const { return high_bytes + low_blocks * across * 2048; }
  __host__ __device__ uint16_t* high(void* keep, int64_t row, int part) const {
    return static_cast<uint16_t*>(keep) + (2 * row + part) * n;
  }
  // of column c, a multiple of 8
  __host__ __device__ uint32_t* low(void* keep, int64_t row, int part, int c) const {
    return reinterpret_cast<uint32_t*>(static_cast<char*>(keep) + high_bytes) +
           ((row / 32 * across + c / 64) * 4 + 2 * part + c % 64 / 32) * 128 + row % 32 * 4 + c % 32 / 8;
  }
  // bits 12 to 15 of the word's i-th column
  __device__ static uint32_t low_of(uint32_t w, int i) {
    const int at = 8 * (i & 3) + (i < 4 ? 4 : 0);
    return (at < 12 ? w << (12 - at) : w >> (at - 12)) & 0xf000u;
  }
};

// dz as the tiled products read it: blocks of 32 rows by 64 columns, 4 KB each, one after
// another along the columns of dzg and then of dzu, each layer's columns filled up with zeros
// to whole blocks and the rows to whole stages.  What a product brings to LDS at a time
// lies together in memory, whole and without masks, whether it takes dz by rows or by columns.
struct DzBlocks {
  int64_t row_blocks;
  int32_t per_layer;  // blocks along a layer's columns
  __host__ __device__ DzBlocks(int64_t M, int32_t N) : row_blocks((M + 63) / 64 * 2), per_layer((N + 63) / 64) {}
  __host__ __device__ int64_t across() const { return 2 * int64_t(per_layer); }
  __host__ __device__ int64_t bytes() const { return row_blocks * across() * 4096; }
};

// Backward products (ngt_gated_bwd.hip): dx = dzg Wg + dzu Wu, or, with the contraction split,
// parts of it, and dW = dz^T x, or parts of it over splits of the rows.  K is a multiple of 8.
struct GatedBwd {
  const uint16_t* dz;  // DzBlocks
  const uint16_t* x;   // [M, K]
  const uint16_t* wg;  // [N, K]
  const uint16_t* wu;
  uint16_t* dx;        // [M, K]
  void* dw[2];         // [N, K], where there is one split
  float* part;         // [splits][M][K] of dx, [splits][2 N][K] of dW
  int64_t M;
  int32_t N, K;
  int32_t dw_f32[2];
  int32_t parts;       // so also where there is one split
};
// A product's blocks: 64 fn columns each, and so many splits of `per_split` stages.
struct GatedShape {
  int32_t fn, splits, per_split;
};
GatedShape gated_dx_shape(int64_t M, int32_t N, int32_t K);
GatedShape gated_dw_shape(int64_t M, int32_t N, int32_t K);
int launch_gated_dx(const GatedBwd& g, const GatedShape& s, hipStream_t st);
int launch_gated_dw(const GatedBwd& g, const GatedShape& s, hipStream_t st);

namespace {

using packed::f32x16;
using packed::fill16;
using packed::tid_x;
using packed::wg_x;

constexpr int kStage = 64;  // contraction per LDS stage: rows of 128 bytes
using L = packed::Tile<bf16_t, kStage>;

// Rows that the tiled products take are below kFar: 32-bit offsets within 256 of them.
constexpr int64_t kFar = 1 << 21;
inline bool all_aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned16(p)) return false;
  return true;
}

// The block's tile: each XCD (block number mod 8) takes a contiguous run, in which the
// blocks under way at a time form a square, 8 rows of tiles side by side, so that its L2
// holds what they share.
struct TileAt {
  int m, n, split;
  bool there;
};
__device__ __forceinline__ TileAt tile_at(int tiles_m, int tiles_n, int splits) {
  constexpr int kRows = 8;
  const int tiles = tiles_m * tiles_n, total = tiles * splits, per = (total + 7) / 8;
  int id = (wg_x() % 8) * per + wg_x() / 8;
  if (wg_x() / 8 >= per || id >= total) return {0, 0, 0, false};
  const int split = id / tiles;
  id -= split * tiles;
  const int band = id / (kRows * tiles_n), in = id - band * kRows * tiles_n;
  const int rows = min(kRows, tiles_m - band * kRows);
  return {band * kRows + in % rows, in / rows, split, true};
}

// A buffer's descriptor in scalar registers: `bytes` from `base` (none where negative); what
// lies behind reads as zero.
__device__ __forceinline__ u32x4 descriptor(const void* base, int64_t bytes) {
  const auto at = reinterpret_cast<uint64_t>(base);
  const int64_t n = bytes > packed::kMostBytes ? packed::kMostBytes : bytes < 0 ? 0 : bytes;
  auto scalar = [](uint64_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
  };
  return {scalar(at), scalar(at >> 32 & 0xffffu), scalar(n), 0x00027000u};
}
__device__ __forceinline__ uint32_t lds_at(const char* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}
// 64 pieces of 16 bytes of a wave from memory to LDS, one after another from `to`.  The
// compiler does not know what this writes: with its builtin it waits for every such piece
// before any transposing read.  So the caller waits (all_there) and meets the other waves
// before it reads.  s_nop: m0, and scalar registers that a vector instruction wrote, need
// up to 5 instructions until a buffer instruction reads them.
__device__ __forceinline__ void bring(u32x4 from, int offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(to), "v"(offset), "s"(from)
               : "m0");
}
// Until all that this wave brings is there.
__device__ __forceinline__ void all_there() { wait_for_all_but<0>(); }
// Until all that this wave reads from LDS is there.
__device__ __forceinline__ void all_read() { __builtin_amdgcn_s_waitcnt(0xc07f); }
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// An operand with the contraction along its rows: a stage is 32-row pieces of 128 bytes a
// row, 4 KB, whose 16-byte pieces are permuted by swz(row).
struct RowsOperand {
  int v;      // the thread's offset in the first 32 rows
  int piece;  // its first element of the row
  int step;   // 32 rows
  __device__ __forceinline__ void init(int64_t stride) {
    const int r = tid_x() / 8;
    piece = 8 * (tid_x() % 8 ^ L::swz(r));
    v = 2 * (r * static_cast<int>(stride) + piece);
    step = 64 * static_cast<int>(stride);
  }
  // of rows `rows` (at most `most`) from `base`, at column k of `width`
  __device__ static __forceinline__ u32x4 source(const uint16_t* base, int rows, int most,
                                                 int64_t stride, int k, int width) {
    return descriptor(base + k, 2 * ((min(most, rows) - 1) * stride + width - k));
  }
  // rows 32 i ..
  __device__ __forceinline__ void load(u32x4 from, int i, int k, int width, uint32_t to) const {
    bring(from, k + piece < width ? v + i * step : packed::kNowhere, to);
  }
  // a lane's share of chunk c (16 of the contraction) of 32 rows, its row a_row(lane): 8
  // from 32 (c / 2) + 16 half + 8 (c % 2)
  __device__ static __forceinline__ L::Op frag(const char* tile, int t, int c, int lane) {
    L::Op r;
    r.p[0] = *reinterpret_cast<const u32x4*>(
        tile + 4096 * t + L::offset(L::a_row(lane & 31), 4 * (c >> 1) + 2 * (lane >> 5) + (c & 1)));
    return r;
  }
};

// A block of dz, which is 32 rows of a RowsOperand and half a tile of a ColsOperand alike.
struct BlockOperand {
  int v;  // the thread's offset in it
  __device__ __forceinline__ void init() {
    const int r = tid_x() / 8;
    v = 128 * r + 16 * (tid_x() % 8 ^ L::swz(r));
  }
  __device__ __forceinline__ void load(u32x4 from, int offset, uint32_t to) const {
    bring(from, v + offset, to);
  }
};

// An operand with the contraction across its rows: a stage is 64 rows of 64-column tiles,
// 128 bytes a row, 8 KB, permuted the same way.
struct ColsOperand {
  int v;     // the thread's offset in the first 32 rows of the first tile
  int col;   // its first column
  int step;  // 32 rows
  __device__ __forceinline__ void init(int64_t stride) {
    const int r = tid_x() / 8;
    col = 8 * (tid_x() % 8 ^ L::swz(r));
    v = 2 * (r * static_cast<int>(stride) + col);
    step = 64 * static_cast<int>(stride);
  }
  // of `rows` rows (a stage's at most) from `base`, with `cols` columns from it on
  __device__ static __forceinline__ u32x4 source(const uint16_t* base, int64_t rows, int64_t stride,
                                                 int cols) {
    return descriptor(base, 2 * ((rows < kStage ? rows - 1 : kStage - 1) * stride + cols));
  }
  // rows 32 (q % 2) .. of tile q / 2
  __device__ __forceinline__ void load(u32x4 from, int q, int cols, uint32_t to) const {
    bring(from, 64 * (q / 2) + col < cols ? v + q % 2 * step + 128 * (q / 2) : packed::kNowhere, to);
  }
  // the same share of chunk c of 32 columns; a lane's column is a_row(lane), because a
  // ds_read_b64_tr_b16 takes its four 8-byte pieces of a row from wherever its lanes point
  __device__ static __forceinline__ L::Op frag(const char* tile, int t, int c, int lane) {
    const int j = lane & 15, q = j & 3;
    const int row = 32 * (c >> 1) + 16 * (lane >> 5) + 8 * (c & 1) + (j >> 2);
    const int piece = 4 * (t & 1) + ((lane >> 4) & 1) + 2 * (q & 1);
    const char* base = tile + 8192 * (t >> 1);
    typedef __attribute__((address_space(3))) packed::s16x4* lds4_t;
    auto read = [&](int r) {
      return __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (lds4_t)(base + r * 128 + ((piece ^ L::swz(r)) << 4) + 8 * (q >> 1))));
    };
    const uint2 lo = read(row), hi = read(row + 4);
    L::Op r;
    r.p[0] = u32x4{lo.x, lo.y, hi.x, hi.y};
    return r;
  }
};

}  // namespace
}  // namespace ngt
