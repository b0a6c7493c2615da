// Linear layer with its epilogue: y = act(x W^T + b) + r in bf16, fp32 inside,
// and its backward up to the weight's gradient (ngt_wgrad.hip).  The encoder's
// FFN and output projections (NeutronGT/models/graphormer_dist_node_level.py:
// 18-30, 176-206) read and write their activations once instead of three times.
//
// x [M, K] and W [N, K] both have the contraction along their rows, so an MFMA
// takes W's rows as A and x's as B as they lie in LDS (16 bytes a lane), and D
// has outputs n in its registers: with the row order of ngt_packed.h a lane
// ends up with 16 consecutive outputs of one row, so bias, residual and result
// are 16-byte accesses.
//
// Rounded to bf16 besides the results: z, kept for the backward, and dz, the operand of dx,
// dW and db.  Trained with GELU (4,096 x 768 -> 768) the gradients are off by 2.41e-3 where
// rounding them alone makes 1.66e-3; nearly all of the rest is dz, which is an operand's type
// (z in fp32: 2.35e-3 for twice its bytes; act'(z) kept in bf16 instead of z: 3.03e-3).
#include "ngt_linear.h"

namespace ngt {
namespace {

using packed::f32x16;
using packed::fill16;
using packed::tid_x;
using packed::wg_x;

constexpr int kActNone = NGT_ACT_NONE, kActRelu = NGT_ACT_RELU, kActGelu = NGT_ACT_GELU;
constexpr int kStage = 64;  // contraction per LDS stage: rows of 128 bytes
using L = packed::Tile<bf16_t, kStage>;

struct GemmArgs {
  const uint16_t* x;  // [M, K], rows x_stride apart
  const uint16_t* w;  // [N, K]
  const uint16_t* bias;
  const uint16_t* r;  // [M, N]
  uint16_t* y;        // [M, N]
  uint16_t* z;        // [M, N] or null: before the activation
  int64_t x_stride;
  int32_t M, N, K, act;
  int32_t tiles_m, tiles_n;
};

template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (ACT == kActGelu) return z * normal(z).cdf;
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == kActGelu) {
    const Normal n = normal(z);
    return fmaf(z * 0.39894228040143268f, n.pdf, n.cdf);
  }
  return 1.f;
}

// 8 results from their sums and their pieces of bias and residual (zeros where
// there are none).
__device__ __forceinline__ void results8(int act, const float (&s)[8], const u32x4& bias,
                                         const u32x4& res, u32x4& y, u32x4& z) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s[i] + half_of(bias, i);
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
  if (act == kActGelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_of<kActGelu>(v[i]);
  } else if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_of<kActRelu>(v[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = pack2_bf16(v[2 * i] + half_of(res, 2 * i), v[2 * i + 1] + half_of(res, 2 * i + 1));
}

// 8 outputs n .. n+7 of row m.
template <bool ALIGNED>
__device__ __forceinline__ void finish8(const GemmArgs& a, int m, int n, const float (&s)[8]) {
  if (m >= a.M || n >= a.N) return;
  const int64_t at = int64_t(m) * a.N + n;
  u32x4 b = {0u, 0u, 0u, 0u}, r = {0u, 0u, 0u, 0u}, y, z;
  if (a.bias) b = load8<ALIGNED>(a.bias, n, a.N);
  if (a.r) r = load8<ALIGNED>(a.r + int64_t(m) * a.N, n, a.N);
  results8(a.act, s, b, r, y, z);
  if (ALIGNED || n + 8 <= a.N) {
    if constexpr (ALIGNED) {
      *reinterpret_cast<u32x4*>(a.y + at) = y;
      if (a.z) *reinterpret_cast<u32x4*>(a.z + at) = z;
    } else {
      reinterpret_cast<Loose16*>(a.y + at)->w = y;
      if (a.z) reinterpret_cast<Loose16*>(a.z + at)->w = z;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < a.N) {
        a.y[at + i] = static_cast<uint16_t>(y[i / 2] >> (16 * (i & 1)));
        if (a.z) a.z[at + i] = static_cast<uint16_t>(z[i / 2] >> (16 * (i & 1)));
      }
  }
}

// One block: BM rows by BN outputs, 2 x 2 waves of (BM / 2) x (BN / 2), stages of 64
// of the contraction in LDS.  A 128 x 128 block's stage takes 512 clocks of the CU's
// MFMA, 512 of its reads from LDS, 256 of the writes there and 512 of its path from L2
// (32 KB at 64 bytes a clock); a 256 x 128 block has three quarters of that traffic per
// MFMA.
// BUFS = 1: read, wait, multiply; the 2 to 3 blocks of a CU fill each other's waits
// (10,007 x 4,096 -> 1,024 88 us, 113 us with the pieces read into registers and
// stored to LDS a stage later).
// BUFS = 4: three stages under way while one is multiplied, for a grid of at most one
// block a CU, where nothing else fills the waits (2,048 x 4,096 -> 1,024 41 us,
// BUFS = 1 64 us).
// What is left then is the wait for each stage's first fragments and, with GELU, the
// epilogue: some 110 clocks for a wave's 64 outputs, 7,200 a block, the MFMA time of
// 900 of the contraction (blocks on the same CU overlap it, a lone one does not).
template <int BM, int BN, int BUFS, bool ALIGNED>
__global__ __launch_bounds__(256) void k_gemm(GemmArgs a) {
  constexpr int FM = BM / 64, FN = BN / 64;  // 32 x 32 tiles of a wave
  constexpr int NX = BM * 8 / 256, NW = BN * 8 / 256;  // 16-byte pieces per thread
  constexpr int kTiles = (BM + BN) * 128, kMore = BUFS > 1 ? kTiles : 16;
  // arrays of their own, so that the compiler knows a read from one independent of
  // what is on its way to another
  __shared__ __align__(16) char s0[kTiles];
  __shared__ __align__(16) char s1[kMore];
  __shared__ __align__(16) char s2[kMore];
  __shared__ __align__(16) char s3[kMore];
  const int tid = tid_x(), lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  const int in_wave_order = 1024 * packed::wave_id();
  // each XCD (block number mod 8) takes a contiguous run of tiles, the tiles
  // of a row of x one after another: its L2 holds W and each row once
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8;
  const int id = (wg_x() % 8) * per + wg_x() / 8;
  if (wg_x() / 8 >= per || id >= total) return;  // block-uniform
  const int m0 = id / a.tiles_n * BM, n0 = id % a.tiles_n * BN;
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = fill16(0.f);

  // the next chunk's fragments are read before a chunk's products
  auto multiply = [&](const char* xs) {
    const char* ws = xs + BM * 128;
    L::Op fx[2][FM], fw[2][FN];
    auto read = [&](int c) {
#pragma unroll
      for (int i = 0; i < FM; ++i) fx[c & 1][i] = L::load_a(xs + wm * 128, i, c, l32, half);
#pragma unroll
      for (int j = 0; j < FN; ++j) fw[c & 1][j] = L::load_a(ws + wn * 128, j, c, l32, half);
    };
    read(0);
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c) {
      if (c + 1 < L::kChunks) read(c + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = L::mma(fw[c & 1][j], fx[c & 1][i], acc[i][j]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  if constexpr (ALIGNED) {
    // Rows that are not there read as zeros, a piece behind the row's end (the last
    // stage's) is sent behind the buffer's.  A wave's pieces lie one after another
    // in LDS, so the swizzle is in which piece of its row a thread reads.
    int ax[NX], aw[NW];
    auto piece = [&](int i) {
      const int r = (tid + i * 256) / 8;
      return 8 * (tid % 8 ^ L::swz(r));
    };
#pragma unroll
    for (int i = 0; i < NX; ++i)
      ax[i] = 2 * ((tid + i * 256) / 8 * static_cast<int>(a.x_stride) + piece(i));
#pragma unroll
    for (int i = 0; i < NW; ++i) aw[i] = 2 * ((tid + i * 256) / 8 * a.K + piece(i));
    auto fetch = [&](int k, char* to) {
      const packed::Buffer bx = packed::make_buffer(
          a.x + m0 * a.x_stride + k, 2 * ((min(BM, a.M - m0) - 1) * a.x_stride + a.K - k));
      const packed::Buffer bw = packed::make_buffer(
          a.w + int64_t(n0) * a.K + k, 2 * ((min(BN, a.N - n0) - 1) * int64_t(a.K) + a.K - k));
#pragma unroll
      for (int i = 0; i < NX; ++i)
        to_lds(bx, ax[i] | (k + piece(i) < a.K ? 0 : packed::kNowhere),
               to + 4096 * i + in_wave_order);
#pragma unroll
      for (int i = 0; i < NW; ++i)
        to_lds(bw, aw[i] | (k + piece(i) < a.K ? 0 : packed::kNowhere),
               to + BM * 128 + 4096 * i + in_wave_order);
    };
    if constexpr (BUFS == 1) {
      for (int k = 0; k < a.K; k += kStage) {
        __syncthreads();
        fetch(k, s0);
        wait_for_all_but<0>();
        __syncthreads();
        multiply(s0);
      }
    } else {
      auto step = [&](int k, char* to, const char* from) {
        // this wave's pieces of stage k are there; behind the barrier all waves' are,
        // and all have read what `to` held
        wait_for_all_but<2 * (NX + NW)>();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        fetch(k + 3 * kStage, to);  // (behind the last stage: zeros)
        multiply(from);
      };
      fetch(0, s0);
      fetch(kStage, s1);
      fetch(2 * kStage, s2);
      for (int k = 0;;) {
        step(k, s3, s0);
        if ((k += kStage) >= a.K) break;
        step(k, s0, s1);
        if ((k += kStage) >= a.K) break;
        step(k, s1, s2);
        if ((k += kStage) >= a.K) break;
        step(k, s2, s3);
        if ((k += kStage) >= a.K) break;
      }
      wait_for_all_but<0>();  // nothing is on its way to LDS when the block ends
    }
  } else {
    u32x4 px[NX], pw[NW];
    auto fetch = [&](int k) {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int e = tid + i * 256, row = m0 + e / 8;
        px[i] = u32x4{0u, 0u, 0u, 0u};
        if (row < a.M) px[i] = load8<false>(a.x + row * a.x_stride, k + 8 * (e % 8), a.K);
      }
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int e = tid + i * 256, row = n0 + e / 8;
        pw[i] = u32x4{0u, 0u, 0u, 0u};
        if (row < a.N) pw[i] = load8<false>(a.w + int64_t(row) * a.K, k + 8 * (e % 8), a.K);
      }
    };
    fetch(0);
    for (int k = 0; k < a.K; k += kStage) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int e = tid + i * 256;
        *reinterpret_cast<u32x4*>(s0 + L::offset(e / 8, e % 8)) = px[i];
      }
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int e = tid + i * 256;
        *reinterpret_cast<u32x4*>(s0 + BM * 128 + L::offset(e / 8, e % 8)) = pw[i];
      }
      __syncthreads();
      fetch(k + kStage);  // (behind the last stage: zeros)
      multiply(s0);
    }
  }
  if constexpr (ALIGNED) {
    // all pieces of bias and residual under way at once (waiting for each in its
    // turn took 7 us a block); what is not there reads as zero and is not written
    const int64_t base = int64_t(m0) * a.N + n0;
    const int64_t bytes = 2 * (int64_t(min(BM, a.M - m0) - 1) * a.N + min(BN, a.N - n0));
    const packed::Buffer br = packed::make_buffer(a.r + base, a.r ? bytes : 0);
    const packed::Buffer bb = packed::make_buffer(a.bias + n0, a.bias ? 2 * (a.N - n0) : 0);
    const packed::Buffer by = packed::make_buffer(a.y + base, bytes);
    const packed::Buffer bz = packed::make_buffer(a.z + base, a.z ? bytes : 0);
    auto at = [&](int i, int j, int e) {
      const int c = wn + 32 * j + 16 * half + 8 * e;
      return n0 + c < a.N ? 2 * ((wm + 32 * i + L::a_row(l32)) * a.N + c) : packed::kNowhere;
    };
    u32x4 bias[FN][2], res[FM][FN][2];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        bias[j][e] = packed::read16(bb, 2 * (wn + 32 * j + 16 * half + 8 * e));
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          res[i][j][e] = a.r ? packed::read16(br, at(i, j, e)) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float s[8];
          u32x4 y, z;
#pragma unroll
          for (int t = 0; t < 8; ++t) s[t] = acc[i][j][8 * e + t];
          results8(a.act, s, bias[j][e], res[i][j][e], y, z);
          __builtin_amdgcn_raw_buffer_store_b128(y, by, at(i, j, e), 0, 0);
          if (a.z) __builtin_amdgcn_raw_buffer_store_b128(z, bz, at(i, j, e), 0, 0);
        }
  } else {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float s[8];
#pragma unroll
          for (int t = 0; t < 8; ++t) s[t] = acc[i][j][8 * e + t];
          finish8<false>(a, m0 + wm + 32 * i + L::a_row(l32),
                         n0 + wn + 32 * j + 16 * half + 8 * e, s);
        }
  }
}

// Few outputs: one block 32 F rows by 32 F outputs straight from memory, its
// four waves every fourth 64 of the contraction each; their sums are added in
// wave order.
template <int F, bool ALIGNED>
__global__ __launch_bounds__(256) void k_gemm_few(GemmArgs a) {
  constexpr int kPitch = 36;  // floats
  __shared__ __align__(16) float red[4][32][kPitch];
  const int tid = tid_x(), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = packed::wave_id();
  const int m0 = wg_x() / a.tiles_n * (32 * F), n0 = wg_x() % a.tiles_n * (32 * F);
  const int row = L::a_row(l32);
  f32x16 acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = fill16(0.f);
  packed::Buffer bx, bw;
  if constexpr (ALIGNED) {
    bx = packed::make_buffer(a.x + m0 * a.x_stride,
                             2 * ((min(32 * F, a.M - m0) - 1) * a.x_stride + a.K));
    bw = packed::make_buffer(a.w + int64_t(n0) * a.K, 2 * (min(32 * F, a.N - n0) * int64_t(a.K)));
  }
  for (int k = 64 * wave; k < a.K; k += 256) {
    u32x4 fx[F][4], fw[F][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = k + 16 * c + 8 * half;
#pragma unroll
      for (int i = 0; i < F; ++i) {
        if constexpr (ALIGNED) {
          const int over = col < a.K ? 0 : packed::kNowhere;
          fx[i][c] =
              packed::read16(bx, 2 * ((32 * i + l32) * static_cast<int>(a.x_stride) + col) | over);
          fw[i][c] = packed::read16(bw, 2 * ((32 * i + row) * a.K + col) | over);
        } else {
          fx[i][c] = fw[i][c] = u32x4{0u, 0u, 0u, 0u};
          if (m0 + 32 * i + l32 < a.M)
            fx[i][c] = load8<false>(a.x + (m0 + 32 * i + l32) * a.x_stride, col, a.K);
          if (n0 + 32 * i + row < a.N)
            fw[i][c] = load8<false>(a.w + int64_t(n0 + 32 * i + row) * a.K, col, a.K);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
          acc[i][j] = L::mma({{fw[j][c]}}, {{fx[i][c]}}, acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) {
      if (i + j > 0) __syncthreads();
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(&red[wave][l32][16 * half + 4 * g]) =
            make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                        acc[i][j][4 * g + 3]);
      __syncthreads();
      if (tid < 128) {
        const int m = tid >> 2, n = (tid & 3) * 8;
        float s[8];
#pragma unroll
        for (int t = 0; t < 8; ++t)
          s[t] = ((red[0][m][n + t] + red[1][m][n + t]) + red[2][m][n + t]) + red[3][m][n + t];
        finish8<ALIGNED>(a, m0 + 32 * i + m, n0 + 32 * j + n, s);
      }
    }
}

// dz = dy act'(z), 8 elements a thread.
template <int ACT>
__global__ __launch_bounds__(256) void k_act_grad(const uint16_t* __restrict__ dy,
                                                  const uint16_t* __restrict__ z, int64_t n,
                                                  uint16_t* __restrict__ dz) {
  const int64_t step = int64_t(__builtin_amdgcn_grid_size_x()) * 8;
  for (int64_t i = (int64_t(wg_x()) * 256 + tid_x()) * 8; i < n; i += step) {
    if (i + 8 <= n) {
      const u32x4 g = *reinterpret_cast<const u32x4*>(dy + i);
      const u32x4 v = *reinterpret_cast<const u32x4*>(z + i);
      u32x4 o;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        o[t] = pack2_bf16(half_of(g, 2 * t) * act_grad<ACT>(half_of(v, 2 * t)),
                          half_of(g, 2 * t + 1) * act_grad<ACT>(half_of(v, 2 * t + 1)));
      *reinterpret_cast<u32x4*>(dz + i) = o;
    } else {
      for (int64_t t = i; t < n; ++t)
        dz[t] = f32_to_bf16(bf16_to_f32(dy[t]) * act_grad<ACT>(bf16_to_f32(z[t])));
    }
  }
}

// out[c][r] = in[r][c], 64 x 64 elements a block.
__global__ __launch_bounds__(256) void k_transpose(const uint16_t* __restrict__ in, int rows,
                                                   int cols, int tiles_c,
                                                   uint16_t* __restrict__ out) {
  __shared__ uint16_t t[64][66];
  const int r0 = wg_x() / tiles_c * 64, c0 = wg_x() % tiles_c * 64;
  // all reads under way at once: of what is there, not written where it is not
  uint16_t v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = tid_x() + 256 * i;
    v[i] = in[int64_t(min(r0 + e / 64, rows - 1)) * cols + min(c0 + e % 64, cols - 1)];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) t[(tid_x() + 256 * i) / 64][tid_x() % 64] = v[i];
  __syncthreads();
#pragma unroll
  for (int e = tid_x(); e < 4096; e += 256) {
    const int c = c0 + e / 64, r = r0 + e % 64;
    if (r < rows && c < cols) out[int64_t(c) * rows + r] = t[e % 64][e / 64];
  }
}

int launch_gemm(GemmArgs a, hipStream_t st) {
  KernelTimer timer_("linear_gemm", st);
  // 16-byte accesses, and 32-bit offsets within a tile's 256 rows
  constexpr int64_t kFar = 1 << 21;
  const bool al = a.K < kFar && a.N < kFar && a.x_stride < kFar && a.K % 8 == 0 &&
                  a.N % 8 == 0 && a.x_stride % 8 == 0 && aligned16(a.x) && aligned16(a.w) &&
                  aligned16(a.bias) && aligned16(a.r) && aligned16(a.y) && aligned16(a.z);
  auto tiles = [&](int bm, int bn) {
    a.tiles_m = (a.M + bm - 1) / bm;
    a.tiles_n = (a.N + bn - 1) / bn;
    return int64_t(a.tiles_m) * a.tiles_n;
  };
  auto run = [&](auto kernel, auto loose, int64_t n) {
    if (al) hipLaunchKernelGGL(kernel, dim3(unsigned(n)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(loose, dim3(unsigned(n)), dim3(256), 0, st, a);
  };
  auto eighths = [](int64_t n) { return (n + 7) / 8 * 8; };
  // By the count of 128 x 128 tiles, for the card's 256 CUs (us with bias, GELU and
  // residual: 32 | 64 rows a block | 128 in four buffers | 128 | 256).  Narrow blocks
  // while wider ones leave most CUs without work: 4,096 x 1,024 at 40 rows (32 tiles)
  // 6.6 | 11.3 | 15.1, 768 x 768 at 512 (24) 8.6 | 10.5 | 13.0; but at 1,024 (48)
  // 11.8 | 10.9 | 13.1, and 4,096 x 1,024 at 256 (64) 18.2 | 13.9 | 15.8.  Then whole
  // tiles through LDS: 768 x 768 at 2,048 (96) - | 19.9 | 13.3 | 15.0, and at 10,007 (474)
  // - | 62 | 27.9 | 24.7.  Tiles of 256 rows need several blocks on every CU and a long
  // contraction: 4,096 x 1,024 at 4,096 (512 of them) 52.2 | 47.3, at 32,768 404 | 387,
  // 1,024 x 4,096 at 32,768 317 | 285, but at 10,007 (320) 87.7 | 108, and 768 x 768 at
  // 32,768 57.0 | 63.1.
  const int64_t t128 = tiles(128, 128);
  if (t128 < 40) {
    run(k_gemm_few<1, true>, k_gemm_few<1, false>, tiles(32, 32));
  } else if (t128 < 80) {
    run(k_gemm_few<2, true>, k_gemm_few<2, false>, tiles(64, 64));
  } else if (t128 <= 256) {
    run(k_gemm<128, 128, 4, true>, k_gemm<128, 128, 1, false>, eighths(tiles(128, 128)));
  } else if (a.K < 1024 || tiles(256, 128) < 512) {
    run(k_gemm<128, 128, 1, true>, k_gemm<128, 128, 1, false>, eighths(tiles(128, 128)));
  } else {
    run(k_gemm<256, 128, 1, true>, k_gemm<256, 128, 1, false>, eighths(tiles(256, 128)));
  }
  NGT_HIP_CHECK(hipGetLastError());
  return NGT_OK;
}

int check_sizes(const char* fn, int64_t M, int32_t N, int32_t K, int act) {
  if (M < 0 || N < 1 || K < 1)
    return set_error(NGT_ERR_ARG, "%s: bad sizes rows=%lld n_out=%d n_in=%d", fn,
                     static_cast<long long>(M), N, K);
  if (act < kActNone || act > kActGelu) return set_error(NGT_ERR_ARG, "%s: activation %d", fn, act);
  // 32-bit rows, and fewer than 2^24 blocks of 256 threads for each of the tile
  // grids: y, dx and W's transpose
  auto blocks = [](int64_t r, int64_t c, int t) { return (r + t - 1) / t * ((c + t - 1) / t); };
  constexpr int64_t kMost = (1 << 24) - 8;
  if (M > (1 << 30) || blocks(M, N, 128) > kMost || blocks(M, K, 128) > kMost ||
      blocks(N, K, 64) > kMost)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: rows=%lld n_out=%d n_in=%d exceed the grid", fn,
                     static_cast<long long>(M), N, K);
  return NGT_OK;
}

}  // namespace
}  // namespace ngt

using namespace ngt;

extern "C" int ngt_linear_fwd(const void* x, int64_t x_stride, const void* w, const void* bias,
                              const void* residual, int64_t n_rows, int32_t n_out, int32_t n_in,
                              int32_t activation, void* y, void* z, void* stream) {
  const char* fn = "ngt_linear_fwd";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in, activation));
  if (n_rows == 0) return NGT_OK;
  if (!x || !w || !y) return set_error(NGT_ERR_ARG, "%s: null x, w or y", fn);
  if (x_stride < n_in) return set_error(NGT_ERR_ARG, "%s: x rows overlap", fn);
  GemmArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(w),
             static_cast<const uint16_t*>(bias), static_cast<const uint16_t*>(residual),
             static_cast<uint16_t*>(y), static_cast<uint16_t*>(z), x_stride,
             static_cast<int32_t>(n_rows), n_out, n_in, activation, 0, 0};
  return launch_gemm(a, static_cast<hipStream_t>(stream));
}

extern "C" int ngt_linear_bwd_workspace_bytes(int64_t n_rows, int32_t n_out, int32_t n_in,
                                              size_t* bytes) {
  NGT_CHECK_OK(check_sizes("ngt_linear_bwd_workspace_bytes", n_rows, n_out, n_in, kActNone));
  if (!bytes) return set_error(NGT_ERR_ARG, "ngt_linear_bwd_workspace_bytes: null bytes");
  *bytes = size_t(n_out) * n_in * 2;
  return NGT_OK;
}

extern "C" int ngt_linear_bwd(const void* dy, const void* z, const void* w, int64_t n_rows,
                              int32_t n_out, int32_t n_in, int32_t activation, void* dz, void* dx,
                              void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "ngt_linear_bwd";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in, activation));
  if (n_rows == 0) return NGT_OK;
  if (!dy || (activation != kActNone && (!z || !dz)))
    return set_error(NGT_ERR_ARG, "%s: null dy, z or dz", fn);
  if (activation != kActNone && !(aligned16(dy) && aligned16(z) && aligned16(dz)))
    return set_error(NGT_ERR_ARG, "%s: dy, z and dz must be 16-byte aligned", fn);
  const size_t need = size_t(n_out) * n_in * 2;
  if (dx && !w) return set_error(NGT_ERR_ARG, "%s: null w", fn);
  if (dx && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu or not 16-byte aligned", fn,
                     workspace_bytes, need);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (activation != kActNone) {
    KernelTimer timer_("linear_act_grad", st);
    const int64_t n = n_rows * n_out, blocks = (n + 2047) / 2048;
    hipLaunchKernelGGL(activation == kActGelu ? k_act_grad<kActGelu> : k_act_grad<kActRelu>,
                       dim3(unsigned(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st,
                       static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(z), n,
                       static_cast<uint16_t*>(dz));
    NGT_HIP_CHECK(hipGetLastError());
    dy = dz;
  }
  if (!dx) return NGT_OK;
  {
    KernelTimer timer_("linear_transpose", st);
    const int tc = (n_in + 63) / 64;
    const int64_t blocks = int64_t((n_out + 63) / 64) * tc;
    hipLaunchKernelGGL(k_transpose, dim3(unsigned(blocks)), dim3(256), 0, st,
                       static_cast<const uint16_t*>(w), n_out, n_in, tc,
                       static_cast<uint16_t*>(workspace));
    NGT_HIP_CHECK(hipGetLastError());
  }
  // dx = dz W: rows of W^T are the other operand
  GemmArgs a{static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(workspace), nullptr,
             nullptr, static_cast<uint16_t*>(dx), nullptr, n_out, static_cast<int32_t>(n_rows),
             n_in, n_out, kActNone, 0, 0};
  return launch_gemm(a, st);
}
