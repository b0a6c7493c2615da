// Gated linear layer, bf16: y = act(x Wg^T + bg) * (x Wu^T + bu), fp32 inside, and its
// backward:
//   dzg = dy zu act'(zg), dzu = dy act(zg);  dx = dzg Wg + dzu Wu,  dW = dz^T x,  db = sums of dz.
// The forward keeps the two factors of dy instead of zg and zu (Keep, ngt_gated.h), so
// that the backward forms no activation.
#include "ngt_gated.h"

#include <algorithm>
#include <cmath>
#include <utility>

namespace ngt {
namespace {

struct GatedArgs {
  const uint16_t* x;   // [M, K], rows x_stride apart
  const uint16_t* wg;  // [N, K]
  const uint16_t* wu;
  const uint16_t* bg;  // [N] or null
  const uint16_t* bu;
  uint16_t* y;         // [M, N]
  void* keep;          // Keep, or null
  int64_t x_stride;
  int32_t M, N, K, act;
  int32_t tiles_m, tiles_n;
  // where the contraction is split: [splits][2][M][N filled up to 8s], and a split's elements of it
  float* part;
  int32_t splits, per_split;
};
__host__ __device__ constexpr int32_t up8(int32_t n) { return (n + 7) / 8 * 8; }

// act(z) and act'(z).
struct Gate {
  float value, slope;
};
template <int ACT>
__device__ __forceinline__ Gate gate_of(float z) {
  if constexpr (ACT == NGT_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
    return {z * s, s * fmaf(z, 1.f - s, 1.f)};
  }
  if constexpr (ACT == NGT_ACT_GELU) {
    const Normal n = normal(z);
    return {z * n.cdf, fmaf(z * 0.39894228040143268f, n.pdf, n.cdf)};
  }
  if constexpr (ACT == NGT_ACT_RELU)
    return {z > 0.f ? z : (z != z ? z : 0.f), z > 0.f ? 1.f : 0.f};
  return {z, 1.f};
}

// f with the activation, and whether the backward's factors are wanted, as constants.
template <typename F>
__device__ __forceinline__ void with_act(int act, bool keep, F f) {
  auto go = [&](auto a) {
    if (keep) f(a, std::true_type{});
    else f(a, std::false_type{});
  };
  if (act == NGT_ACT_SILU) go(std::integral_constant<int, NGT_ACT_SILU>{});
  else if (act == NGT_ACT_GELU) go(std::integral_constant<int, NGT_ACT_GELU>{});
  else if (act == NGT_ACT_RELU) go(std::integral_constant<int, NGT_ACT_RELU>{});
  else go(std::integral_constant<int, NGT_ACT_NONE>{});
}

// Pieces of 8 results and, for the backward, of what it keeps, from their sums.
struct Results {
  u32x4 y, kg, ku;
  uint32_t lg, lu;
};
// 8 fp32 to 20 bits each, rounded to the nearest: their upper halves, and the 4 bits behind
// them, of the first four in the upper halves of the word's bytes, of the others in the lower.
// (A NaN stays one: no sum of bf16 products has all its lower bits set.)
__device__ __forceinline__ void keep8(const float (&v)[8], u32x4& high, uint32_t& low) {
  uint32_t u[8], b[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(v[i]) + 0x800u;
#pragma unroll
  for (int i = 0; i < 4; ++i) high[i] = __builtin_amdgcn_perm(u[2 * i + 1], u[2 * i], 0x07060302u);
#pragma unroll
  for (int i = 0; i < 2; ++i)  // bits 8 to 15 of four
    b[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[4 * i + 3], u[4 * i + 2], 0x0c0c0501u),
                                 __builtin_amdgcn_perm(u[4 * i + 1], u[4 * i], 0x0c0c0501u), 0x05040100u);
  low = (b[0] & 0xf0f0f0f0u) | (b[1] >> 4 & 0x0f0f0f0fu);
}
template <int ACT, bool KEEP>
__device__ __forceinline__ Results results8(const float (&zg)[8], const float (&zu)[8]) {
  Results r;
  r.lg = r.lu = 0u;
  float g[8], u[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int c = 2 * i + t;
      const Gate q = gate_of<ACT>(zg[c]);
      v[t] = q.value * zu[c], g[c] = zu[c] * q.slope, u[c] = q.value;
    }
    r.y[i] = pack2_bf16(v[0], v[1]);
  }
  if constexpr (KEEP) keep8(g, r.kg, r.lg), keep8(u, r.ku, r.lu);
  return r;
}

__device__ __forceinline__ void store8(uint16_t* row, int c, int n, const u32x4& v) {
  if (c + 8 <= n) {
    reinterpret_cast<Loose16*>(row + c)->w = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) row[c + i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
  }
}

// 8 outputs n .. n+7 (n a multiple of 8) of row m from their sums.
__device__ __forceinline__ void finish8(const GatedArgs& a, int m, int n, const float (&sg)[8],
                                        const float (&su)[8]) {
  if (m >= a.M || n >= a.N) return;
  u32x4 bg = {0u, 0u, 0u, 0u}, bu = {0u, 0u, 0u, 0u};
  if (a.bg) bg = load8<false>(a.bg, n, a.N);
  if (a.bu) bu = load8<false>(a.bu, n, a.N);
  float zg[8], zu[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) zg[t] = sg[t] + half_of(bg, t), zu[t] = su[t] + half_of(bu, t);
  Results r;
  with_act(a.act, a.keep != nullptr, [&](auto act, auto keep) {
    r = results8<act.value, keep.value>(zg, zu);
  });
  store8(a.y + int64_t(m) * a.N, n, a.N, r.y);
  if (a.keep) {
    const Keep k(a.M, a.N);
    store8(k.high(a.keep, m, 0), n, a.N, r.kg);
    store8(k.high(a.keep, m, 1), n, a.N, r.ku);
    *k.low(a.keep, m, 0, n) = r.lg;
    *k.low(a.keep, m, 1, n) = r.lu;
  }
}

// The same outputs' sums over a split of the contraction.
__device__ __forceinline__ void part8(const GatedArgs& a, int split, int m, int n,
                                      const float (&sg)[8], const float (&su)[8]) {
  if (m >= a.M || n >= a.N) return;
  float* to = a.part + (int64_t(2 * split) * a.M + m) * up8(a.N) + n;
#pragma unroll
  for (int t = 0; t < 8; t += 4) {
    *reinterpret_cast<float4*>(to + t) = make_float4(sg[t], sg[t + 1], sg[t + 2], sg[t + 3]);
    *reinterpret_cast<float4*>(to + int64_t(a.M) * up8(a.N) + t) =
        make_float4(su[t], su[t + 1], su[t + 2], su[t + 3]);
  }
}
// The splits' sums added in their order, and what becomes of them; 8 outputs a thread.
__global__ __launch_bounds__(256) void k_gated_join_fwd(GatedArgs a) {
  const int across = up8(a.N) / 8, i = wg_x() * 256 + tid_x();
  if (i >= a.M * across) return;
  const int64_t layer = int64_t(a.M) * across * 8;
  float s[2][8] = {};
#pragma unroll 4
  for (int c = 0; c < a.splits; ++c)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float* from = a.part + (2 * c + p) * layer + int64_t(i) * 8;
#pragma unroll
      for (int t = 0; t < 8; t += 4) {
        const float4 v = *reinterpret_cast<const float4*>(from + t);
        s[p][t] += v.x, s[p][t + 1] += v.y, s[p][t + 2] += v.z, s[p][t + 3] += v.w;
      }
    }
  const int m = i / across;
  finish8(a, m, (i - m * across) * 8, s[0], s[1]);
}

// The most blocks of a launch that grows with the matrices' elements, which may be more than the
// 2^32 threads that a launch stays below: with more to do each block takes several pieces.
constexpr int64_t kMostBlocks = 1 << 20;

// x, Wg and Wu with their rows filled up to 8s with zeros, one after another (of widths that are
// no multiple of 8: 2 x 8,193 rows of 2,049 25 us, 5 TB/s).
struct PackArgs {
  const uint16_t* from[3];
  int64_t rows[3];  // of the three, 0 where not wanted
  int64_t x_stride;
  uint16_t* to;
  int32_t k;
  int32_t blocks;
};
__global__ __launch_bounds__(256) void k_gated_pack(PackArgs a) {
  const int across = up8(a.k) / 8, together = across < 256 ? 256 / across : 1;
  const int r = tid_x() / across;
  if (across < 256 && r >= together) return;
  const int64_t all = a.rows[0] + a.rows[1] + a.rows[2];
  for (int64_t at = int64_t(wg_x()) * together + (across < 256 ? r : 0); at < all;
       at += int64_t(a.blocks) * together) {
    uint16_t* to = a.to + at * across * 8;
    int64_t row = at;
    int which = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (which == i && row >= a.rows[i]) row -= a.rows[i], ++which;
    const uint16_t* from = (which == 0 ? a.from[0] : which == 1 ? a.from[1] : a.from[2]) + row * (which == 0 ? a.x_stride : a.k);
    for (int c = across < 256 ? tid_x() - r * across : tid_x(); c < across; c += 256)
      *reinterpret_cast<u32x4*>(to + 8 * c) = load8<false>(from, 8 * c, a.k);
  }
}
// What of it in its workspace is what.
struct Packed {
  const uint16_t *x, *wg, *wu;
};
int launch_pack(PackArgs a, hipStream_t st, Packed* to) {
  const int across = up8(a.k) / 8, together = across < 256 ? 256 / across : 1;
  const int64_t rows = a.rows[0] + a.rows[1] + a.rows[2];
  a.blocks = static_cast<int32_t>(std::min((rows + together - 1) / together, kMostBlocks));
  hipLaunchKernelGGL(k_gated_pack, dim3(unsigned(a.blocks)), dim3(256), 0, st, a);
  NGT_HIP_CHECK(hipGetLastError());
  to->x = a.to, to->wg = a.to + a.rows[0] * up8(a.k), to->wu = to->wg + a.rows[1] * up8(a.k);
  return NGT_OK;
}

// Any sizes and 2-byte alignment.  One block: 64 rows by 64 outputs of both products,
// 2 x 2 waves of 32 x 32, stages of 64 of the contraction read into registers while the
// stage before is multiplied.  For rows that are not whole 16-byte pieces where filling them up
// does not pay (plan_fwd), and for other alignments.  32,768 rows, 768 -> 2,048 in it: 350 us
// (k_gated 215).
__global__ __launch_bounds__(256) void k_gated_any(GatedArgs a) {
  constexpr int NP = 64 * 8 / 256;  // 16-byte pieces per thread and operand
  __shared__ __align__(16) char lds[3][64 * 128];
  const int tid = tid_x(), lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  const int tiles = a.tiles_m * a.tiles_n, split = wg_x() / tiles, tile = wg_x() - split * tiles;
  const int m0 = tile / a.tiles_n * 64, n0 = tile % a.tiles_n * 64;
  const int first = split * a.per_split, end = min(first + a.per_split, a.K);
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x16 g = fill16(0.f), u = fill16(0.f);
  u32x4 p[3][NP];
  auto fetch = [&](int k) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int e = tid + i * 256, c = k + 8 * (e % 8), m = m0 + e / 8, n = n0 + e / 8;
      p[0][i] = p[1][i] = p[2][i] = u32x4{0u, 0u, 0u, 0u};
      if (m < a.M) p[0][i] = load8<false>(a.x + m * a.x_stride, c, a.K);
      if (n < a.N) {
        p[1][i] = load8<false>(a.wg + int64_t(n) * a.K, c, a.K);
        p[2][i] = load8<false>(a.wu + int64_t(n) * a.K, c, a.K);
      }
    }
  };
  fetch(first);
  for (int k = first; k < end; k += kStage) {
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int e = tid + i * 256;
        *reinterpret_cast<u32x4*>(lds[o] + L::offset(e / 8, e % 8)) = p[o][i];
      }
    __syncthreads();
    fetch(k + kStage);  // (behind the contraction: zeros)
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c) {
      const L::Op x = L::load_a(lds[0] + wm * 128, 0, c, l32, half);
      g = L::mma(L::load_a(lds[1] + wn * 128, 0, c, l32, half), x, g);
      u = L::mma(L::load_a(lds[2] + wn * 128, 0, c, l32, half), x, u);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float sg[8], su[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) sg[t] = g[8 * e + t], su[t] = u[8 * e + t];
    const int m = m0 + wm + L::a_row(l32), n = n0 + wn + 16 * half + 8 * e;
    if (a.splits > 1) part8(a, split, m, n, sg, su);
    else finish8(a, m, n, sg, su);
  }
}

// Few rows, aligned: a block is 16 NT outputs of both layers for up to 16 MT rows, its waves
// every WAVES-th 64 of the contraction each, weights and rows straight from memory to
// registers; their sums meet in LDS and are added in wave order.  Bound by the weights'
// bytes (33 rows, 2,048 -> 8,192: 18 us, 3.7 TB/s; a library product of that size 19), or,
// where those are few, by one wait for memory and the join (5 rows, 768 -> 768: 5 us).
template <int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_gated_few(GatedArgs a) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  constexpr int kTiles = 2 * NT * MT;
  __shared__ __align__(16) float red[WAVES][kTiles][16][20];  // [x row][output], padded
  const int lane = tid_x() & 63, wave = packed::wave_id(), quad = lane >> 4, l16 = lane & 15;
  const int split = __builtin_amdgcn_workgroup_id_y(), n0 = wg_x() * 16 * NT;
  const int first = split * a.per_split, end = min(first + a.per_split, a.K);
  f32x4 acc[2][NT][MT];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[p][j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // a row that is not there is the last one again: nobody reads what comes of it
  const uint16_t *x[MT], *w[2][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = a.x + min(16 * i + l16, a.M - 1) * a.x_stride;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t at = int64_t(min(n0 + 16 * j + l16, a.N - 1)) * a.K;
    w[0][j] = a.wg + at, w[1][j] = a.wu + at;
  }
  struct Step {
    u32x4 x[2][MT], w[2][2][NT];
  };
  auto fetch = [&](int k) {
    Step s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = k + 32 * h + 8 * quad;
      const bool there = c < end;
      auto read = [&](const uint16_t* row) {
        return there ? *reinterpret_cast<const u32x4*>(row + c) : u32x4{0u, 0u, 0u, 0u};
      };
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int j = 0; j < NT; ++j) s.w[h][p][j] = read(w[p][j]);
#pragma unroll
      for (int i = 0; i < MT; ++i) s.x[h][i] = read(x[i]);
    }
    return s;
  };
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[p][j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(packed::bf16x8, s.w[h][p][j]),
                __builtin_bit_cast(packed::bf16x8, s.x[h][i]), acc[p][j][i], 0, 0, 0);
  };
  constexpr int kApart = 64 * WAVES;
  Step now = fetch(first + 64 * wave);
  for (int k = first + 64 * wave; k < end; k += kApart) {
    const Step next = fetch(k + kApart);
    multiply(now);
    now = next;
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        *reinterpret_cast<f32x4*>(&red[wave][(p * NT + j) * MT + i][l16][4 * quad]) = acc[p][j][i];
  __syncthreads();
  for (int e = tid_x(); e < 16 * MT * NT * 2; e += 64 * WAVES) {
    const int m = e / (2 * NT), j = e % (2 * NT) / 2, half = e % 2;
    if (m >= a.M) break;
    float s[2][8];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int t = 0; t < 8; ++t) s[p][t] = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v)
#pragma unroll
        for (int t = 0; t < 8; ++t)
          s[p][t] += red[v][(p * NT + j) * MT + m / 16][m % 16][8 * half + t];
    }
    if (a.splits > 1) part8(a, split, m, n0 + 16 * j + 8 * half, s[0], s[1]);
    else finish8(a, m, n0 + 16 * j + 8 * half, s[0], s[1]);
  }
}

// dz = [dzg | dzu], and the biases' gradients: part_b[chunk][2 N], sums of the
// unrounded products.  A block: 256 columns of chunk_rows rows, 8 columns a thread.  WHOLE: whole
// pieces, else any width and 2-byte alignment.  Bound by memory: 32,768 by 2,048 moves 738 MB in
// 142 to 147 us, 5.1 TB/s, as a copy does.
template <bool WHOLE>
__global__ __launch_bounds__(256) void k_gated_dz(const uint16_t* __restrict__ dy,
                                                  void* keep, int64_t rows,
                                                  int32_t n, int32_t tiles_n, int32_t chunk_rows,
                                                  uint16_t* __restrict__ dz,
                                                  float* __restrict__ part_b) {
  __shared__ float red[2][8][256];
  const int64_t chunk = wg_x() / tiles_n;
  const int cg = tid_x() & 31, lane = tid_x() >> 5;
  const int c = (wg_x() - static_cast<int>(chunk) * tiles_n) * 256 + 8 * cg;
  const DzBlocks blocks(rows, n);
  const Keep kept(rows, n);
  const int64_t end = blocks.row_blocks * 32;  // of what is written
  const int64_t r0 = chunk * chunk_rows, r1 = r0 + chunk_rows < end ? r0 + chunk_rows : end;
  float sum[2][8];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int t = 0; t < 8; ++t) sum[p][t] = 0.f;
  if (c < 64 * blocks.per_layer) {
#pragma unroll 2
    for (int64_t row = r0 + lane; row < r1; row += 8) {
      u32x4 g = {0u, 0u, 0u, 0u}, v[2] = {g, g};
      uint32_t low[2] = {0u, 0u};
      if (row < rows && c < n) {
        g = load8<WHOLE>(dy + row * n, c, n);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint16_t* from = kept.high(keep, row, p);
          // the last time that it is read
          if constexpr (WHOLE)
            v[p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + c));
          else
            v[p] = load8<false>(from, c, n);
          low[p] = *kept.low(keep, row, p, c);
        }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        u32x4 o;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float k0 = __uint_as_float(v[p][t] << 16 | Keep::low_of(low[p], 2 * t));
          const float k1 = __uint_as_float((v[p][t] & 0xffff0000u) | Keep::low_of(low[p], 2 * t + 1));
          const float lo = half_of(g, 2 * t) * k0, hi = half_of(g, 2 * t + 1) * k1;
          sum[p][2 * t] += lo, sum[p][2 * t + 1] += hi;
          o[t] = pack2_bf16(lo, hi);
        }
        *reinterpret_cast<u32x4*>(dz + (row / 32 * blocks.across() + p * blocks.per_layer + c / 64) * 2048 +
                                  row % 32 * 64 + c % 64) = o;
      }
    }
  }
  if (!part_b) return;
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int t = 0; t < 8; ++t) red[p][lane][8 * cg + t] = sum[p][t];
  __syncthreads();
  const int col = c - 8 * cg + tid_x();
  if (col >= n) return;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    float s = 0.f;
#pragma unroll
    for (int l = 0; l < 8; ++l) s += red[p][l][tid_x()];
    part_b[(2 * chunk + p) * n + col] = s;
  }
}

// The parameters' gradients in their types: of each weight the splits' sums added in their
// order, 4 elements a thread; of the biases the chunks', 8 lanes a column that take every
// 8th, added in their order.  Bound by the sums' bytes: 2 x 2,048 x 768 in two splits 12 us.
struct JoinArgs {
  const float* part;    // [splits][2 N][K filled up to 8s]
  const float* part_b;  // [chunks][2 N]
  void* dw[2];
  void* db[2];
  int64_t nk;           // N K
  int32_t n, k, splits, chunks, blocks_w;
  int32_t dw_f32[2], db_f32[2];
};
__device__ __forceinline__ void put(void* to, int64_t i, bool f32, float v) {
  if (f32) static_cast<float*>(to)[i] = v;
  else static_cast<uint16_t*>(to)[i] = f32_to_bf16(v);
}
__global__ __launch_bounds__(256) void k_gated_join(JoinArgs a) {
  __shared__ float red[8][32];
  if (wg_x() < a.blocks_w) {
    const int pitch = up8(a.k);
    const int64_t all = 2 * int64_t(a.n) * pitch;
    for (int64_t at = (int64_t(wg_x()) * 256 + tid_x()) * 4; at < all; at += int64_t(a.blocks_w) * 1024) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int c = 0; c < a.splits; ++c) {
        const float4 v = *reinterpret_cast<const float4*>(a.part + c * all + at);
        s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
      }
      // the element of the weights, and how many of the four there are
      int64_t i = at;
      int there = 4;
      if (pitch != a.k) {
        const int64_t row = at / pitch;
        const int c = static_cast<int>(at - row * pitch);
        i = row * a.k + c, there = min(a.k - c, 4);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (!a.dw[w]) continue;
        const int64_t o = i - w * a.nk;
        const bool f32 = a.dw_f32[w];
        if (pitch == a.k && o >= 0 && o + 4 <= a.nk) {
          if (f32) *reinterpret_cast<float4*>(static_cast<float*>(a.dw[w]) + o) = make_float4(s[0], s[1], s[2], s[3]);
          else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.dw[w]) + o) = make_uint2(pack2_bf16(s[0], s[1]), pack2_bf16(s[2], s[3]));
        } else {
          for (int t = 0; t < there; ++t)
            if (o + t >= 0 && o + t < a.nk) put(a.dw[w], o + t, f32, s[t]);
        }
      }
    }
    return;
  }
  const int col = (wg_x() - a.blocks_w) * 32 + tid_x() % 32, lane = tid_x() / 32;
  float s = 0.f;
  if (col < 2 * a.n)
#pragma unroll 8
    for (int c = lane; c < a.chunks; c += 8) s += a.part_b[int64_t(c) * 2 * a.n + col];
  red[lane][tid_x() % 32] = s;
  __syncthreads();
  if (lane != 0 || col >= 2 * a.n) return;
  s = 0.f;
#pragma unroll
  for (int l = 0; l < 8; ++l) s += red[l][tid_x()];
  const int w = col >= a.n;
  if (a.db[w]) put(a.db[w], col - w * a.n, a.db_f32[w], s);
}

// dx from the splits' sums, added in their order, 8 elements a thread.
__global__ __launch_bounds__(256) void k_gated_join_dx(const float* __restrict__ part, int32_t splits,
                                                       int64_t M, int32_t K,
                                                       uint16_t* __restrict__ dx) {
  const int across = up8(K) / 8;
  const int64_t i = int64_t(wg_x()) * 256 + tid_x();
  if (i >= M * across) return;
  float s[8] = {};
#pragma unroll 8
  for (int c = 0; c < splits; ++c) {
    const float* p = part + (c * M * across + i) * 8;
    const float4 v = *reinterpret_cast<const float4*>(p), w = *reinterpret_cast<const float4*>(p + 4);
    s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
    s[4] += w.x, s[5] += w.y, s[6] += w.z, s[7] += w.w;
  }
  u32x4 o;
#pragma unroll
  for (int t = 0; t < 4; ++t) o[t] = pack2_bf16(s[2 * t], s[2 * t + 1]);
  const int64_t m = i / across;
  store8(dx + m * K, static_cast<int>(i - m * across) * 8, K, o);
}

// Rows of x and W of whole 16-byte pieces, of y too where WHOLE.  One block: 64 FM rows by 64
// outputs of both layers, 2 x 2 waves, each FM tiles of 32 x 32 of the gate and the same of the
// other layer.  A wave takes a stage's operands into registers before it multiplies, so the
// one buffer is free for the next stage while it does, and two blocks on a CU fill each
// other's reads.
// 10,007 rows, 1,024 -> 4,096 without keep: 160 us, 1,050 TFLOP/s (a library product of the
// same size and nothing else 143); 32,768 rows, 768 -> 2,048 with keep: 258, of which the loop is
// 185 (its products and LDS reads alone 146, its loads alone 111), the rest arithmetic and 470 MB
// of stores, which the loops of other blocks do not hide.  Measured at the first size: 256 rows
// by 128 outputs in 8 waves with two buffers 175 us, 192 by 64 in two blocks with two buffers 168.
// At FM = 4 the loop takes all 256 registers that two blocks leave a lane: 4 or 5 that the results
// need wait in scratch memory, written before the loop and read once after it.
template <int FM, bool WHOLE>
__global__ __launch_bounds__(256, 2) void k_gated(GatedArgs a) {
  constexpr int BM = 64 * FM, kRowsBytes = BM * 128;
  __shared__ __align__(16) char lds[FM > 1 ? 49152 : kRowsBytes + 128 * 128];
  const int lane = tid_x() & 63, wave = packed::wave_id(), half = lane >> 5;
  constexpr bool kSplit = FM == 1;  // (taller tiles are for many blocks)
  const TileAt at = tile_at(a.tiles_m, a.tiles_n, kSplit ? a.splits : 1);
  if (!at.there) return;  // block-uniform
  const int m0 = at.m * BM, n0 = at.n * 64;
  const int first = kSplit ? at.split * a.per_split : 0;
  const int end = kSplit ? min(first + a.per_split, a.K) : a.K;
  const bool parts = kSplit && a.splits > 1;
  const int wm = (wave >> 1) * FM, wn = wave & 1;  // in 32s
  // A lane has outputs n .. n+15 of row a_row(lane) of each tile; its sums begin with their biases.
  const int n = n0 + 32 * wn + 16 * half;
  f32x16 g[FM], u[FM];
  g[0] = u[0] = fill16(0.f);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (a.bg && !parts) {
      const u32x4 b = load8<false>(a.bg, n + 8 * e, a.N);
#pragma unroll
      for (int t = 0; t < 8; ++t) g[0][8 * e + t] = half_of(b, t);
    }
    if (a.bu && !parts) {
      const u32x4 b = load8<false>(a.bu, n + 8 * e, a.N);
#pragma unroll
      for (int t = 0; t < 8; ++t) u[0][8 * e + t] = half_of(b, t);
    }
  }
#pragma unroll
  for (int i = 1; i < FM; ++i) g[i] = g[0], u[i] = u[0];
  RowsOperand x, w;
  x.init(a.x_stride), w.init(a.K);
  const uint32_t mine = lds_at(lds) + 1024 * wave;
  // 32 rows of Wg, the same of Wu, the next of Wg, of Wu: a wave of a block's two columns of
  // waves has its own beside one another
  auto fetch = [&](int k) {
    const u32x4 fx = RowsOperand::source(a.x + m0 * a.x_stride, a.M - m0, BM, a.x_stride, k, a.K);
#pragma unroll
    for (int i = 0; i < 2 * FM; ++i) x.load(fx, i, k, a.K, mine + 4096 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 32 * (i >> 1);
      const u32x4 fw = RowsOperand::source((i & 1 ? a.wu : a.wg) + int64_t(n) * a.K, a.N - n, 32, a.K,
                                           k, a.K);
      w.load(fw, 0, k, a.K, mine + kRowsBytes + 4096 * i);
    }
  };
  fetch(first);
  for (int k = first; k < end; k += kStage) {
    all_there();
    meet();
    L::Op fx[L::kChunks][FM], fw[L::kChunks][2];
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c) {
#pragma unroll
      for (int j = 0; j < 2; ++j) fw[c][j] = RowsOperand::frag(lds + kRowsBytes, 2 * wn + j, c, lane);
#pragma unroll
      for (int i = 0; i < FM; ++i) fx[c][i] = RowsOperand::frag(lds, wm + i, c, lane);
    }
    all_read();
    meet();
    fetch(k + kStage);  // (behind the contraction: zeros)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        g[i] = L::mma(fw[c][0], fx[c][i], g[i]);
        u[i] = L::mma(fw[c][1], fx[c][i], u[i]);
      }
    __builtin_amdgcn_sched_barrier(0);
  }
  all_there();  // nothing is on its way to LDS any more, of any wave
  if (parts) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sg[8], su[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) sg[t] = g[0][8 * e + t], su[t] = u[0][8 * e + t];
      part8(a, at.split, m0 + 32 * wm + L::a_row(lane & 31), n + 8 * e, sg, su);
    }
    return;
  }
  meet();
  // The results go through LDS, 64 rows at a time in two buffers, so that a store's lanes fill
  // the 128 bytes of each of 8 rows (64 bytes of 16: 265 us instead of 258 in the second size
  // above, and 12 % more bytes written).  f: 16 neighbouring lanes meet all 64 banks.
  const int back = 16 * wave + lane / 8, n_back = n0 + 8 * (lane % 8);
  auto slot = [&](int i, int kind, int row, int piece) {
    const int f = (row >> 1 & 3) | (row >> 2 & 4);
    return reinterpret_cast<u32x4*>(lds + 24576 * (i & 1) + 8192 * kind + 128 * row + 16 * (piece ^ f));
  };
  const Keep kept(a.M, a.N);
  with_act(a.act, a.keep != nullptr, [&](auto act, auto keep) {
    constexpr bool KEEP = decltype(keep)::value;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = L::a_row(lane & 31), m = m0 + 32 * (wm + i) + row, at = 32 * (wave >> 1) + row;
      uint2 lg, lu;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sg[8], su[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) sg[t] = g[i][8 * e + t], su[t] = u[i][8 * e + t];
        const Results r = results8<act.value, KEEP>(sg, su);
        *slot(i, 0, at, 4 * wn + 2 * half + e) = r.y;
        if constexpr (KEEP) {
          *slot(i, 1, at, 4 * wn + 2 * half + e) = r.kg, *slot(i, 2, at, 4 * wn + 2 * half + e) = r.ku;
          (e ? lg.y : lg.x) = r.lg, (e ? lu.y : lu.x) = r.lu;
        }
      }
      if constexpr (KEEP)
        if (m < a.M && n < a.N) {  // (both words are there, whatever N)
          *reinterpret_cast<uint2*>(kept.low(a.keep, m, 0, n)) = lg;
          *reinterpret_cast<uint2*>(kept.low(a.keep, m, 1, n)) = lu;
        }
      all_read();
      meet();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = back + 8 * q, m_back = m0 + 32 * ((r >> 5) * FM + i) + (r & 31);
        const u32x4 y = *slot(i, 0, r, lane % 8);
        u32x4 kg, ku;
        if constexpr (KEEP) kg = *slot(i, 1, r, lane % 8), ku = *slot(i, 2, r, lane % 8);
        if (m_back >= a.M || n_back >= a.N) continue;
        if constexpr (!WHOLE) {
          store8(a.y + int64_t(m_back) * a.N, n_back, a.N, y);
          if constexpr (KEEP) {
            store8(kept.high(a.keep, m_back, 0), n_back, a.N, kg);
            store8(kept.high(a.keep, m_back, 1), n_back, a.N, ku);
          }
          continue;
        }
        *reinterpret_cast<u32x4*>(a.y + int64_t(m_back) * a.N + n_back) = y;
        if constexpr (KEEP) {
          __builtin_nontemporal_store(kg, reinterpret_cast<u32x4*>(kept.high(a.keep, m_back, 0) + n_back));
          __builtin_nontemporal_store(ku, reinterpret_cast<u32x4*>(kept.high(a.keep, m_back, 1) + n_back));
        }
      }
    }
  });
}

// How a backward is cut, and where its workspace holds what.
struct BwdPlan {
  GatedShape dx, dw;
  bool packed;         // widths that are no multiple of 8: x and W filled up, results by way of sums
  int32_t chunk_rows;  // of a block of k_gated_dz
  int64_t chunks;
  size_t dz, part, part_b, pack, bytes;  // part: dx's sums, then the weights'
};
BwdPlan plan_bwd(int64_t M, int32_t N, int32_t K) {
  BwdPlan p;
  const int32_t pitch = up8(K);
  p.dx = gated_dx_shape(M, N, pitch), p.dw = gated_dw_shape(M, N, pitch);
  p.packed = pitch != K;
  // 1,024 blocks where there are rows enough, of 8 rows a pass (2,048 -> 8,192 us at 64 rows: 6, at
  // 128 rows a block 12; 768 -> 2,048 at 511: 8 and 20)
  p.chunk_rows = 128;
  while (p.chunk_rows > 8 && (M + p.chunk_rows - 1) / p.chunk_rows * ((N + 255) / 256) < 1024)
    p.chunk_rows /= 2;
  // (M filled up to whole blocks of dz)
  p.chunks = M == 0 ? 0 : ((M + 63) / 64 * 64 + p.chunk_rows - 1) / p.chunk_rows;
  auto align = [](size_t b) { return (b + 255) & ~size_t(255); };
  auto sums = [&](const GatedShape& s, int64_t rows) {
    return s.splits > 1 || p.packed ? size_t(s.splits) * rows * pitch * sizeof(float) : 0;
  };
  p.dz = 0;
  p.part = align(DzBlocks(M, N).bytes());
  p.part_b = p.part + align(std::max(sums(p.dx, M), sums(p.dw, 2 * int64_t(N))));
  p.pack = p.part_b + align(size_t(p.chunks) * 2 * N * sizeof(float));
  p.bytes = p.pack + (p.packed ? (size_t(M) + 2 * N) * pitch * 2 : 0);
  return p;
}

// How a forward's contraction is split, in elements, where there are few blocks: each split's sums
// are written and read again (about 4 TB/s), so the best number is a square root, as in the
// backward; none below 4 stages of 64 each, nor where it saves less than the second launch and a
// block's start and end again, 8 us.  us, one split / several: 1,024 outputs of 4,096 at 64 rows 27 /
// 17, at 65 43 / 19, at 1,200 48 / 43; 64 of 8,192 at 1 row 21 / 13, at 300 78 / 19; 255 of 8,191 at 65
// 118 / 26.
struct Split {
  int32_t splits, per_split;
};
Split split_of(int64_t M, int32_t N, int32_t K, double stage, int64_t stages, int32_t elements,
               int64_t most) {
  const double sums = 2e-6 / 4 * 8 * double(M) * N;
  const double want = std::sqrt(stage * double(stages) / sums);
  int64_t splits = want < double(most) ? std::llround(want) : most;
  if (splits < 2 || stage * double(stages) * (1.0 - 1.0 / double(splits)) < 8.0 + sums * double(splits))
    return {1, K};
  const int64_t per = (stages + splits - 1) / splits;
  return {static_cast<int32_t>((stages + per - 1) / per), static_cast<int32_t>(per * elements)};
}
constexpr int kFewRows = 64;
Split few_split(int64_t M, int32_t N, int32_t K) {
  // a step of the 8 waves takes 512 elements, and 1.2 us and the rows' share
  const int64_t stages = (int64_t(K) + 511) / 512;
  return split_of(M, N, K, 1.2 + 0.03 * double(M), stages, 512, std::min<int64_t>(512 / ((N + 15) / 16), stages));
}
Split tile_split(int64_t M, int32_t N, int32_t K) {
  const int64_t stages = (int64_t(K) + 63) / 64, tiles = (M + 63) / 64 * ((N + 63) / 64);
  return split_of(M, N, K, 0.65, stages, 64, std::min<int64_t>(768 / std::max<int64_t>(tiles, 1), stages / 4));
}
// Whether a forward fills up the rows of x and W first: its reading and writing (4 bytes an
// element at 5 TB/s) against what k_gated_any takes longer (us, it / filled up: 769 -> 2,049 at 1
// row 18 / 12, at 8,193 223 / 107; 2,049 -> 8,193 at 600 rows 162 / 97, at 129 57 and, were it filled up,
// 56).
bool fills_up(int64_t M, int32_t N, int32_t K) {
  return K % 8 != 0 && 3.0 + 0.8e-6 * double(M + 2 * int64_t(N)) * K < 6.0 + 3.6e-9 * double(M) * N * K;
}
struct FwdPlan {
  bool packed;
  size_t pack, bytes;
};
FwdPlan plan_fwd(int64_t M, int32_t N, int32_t K) {
  if (M == 0) return {false, 0, 0};
  FwdPlan p{fills_up(M, N, K), 0, 0};
  int32_t splits = tile_split(M, N, K).splits;
  if (M <= kFewRows) splits = std::max(splits, few_split(M, N, K).splits);
  p.pack = splits > 1 ? size_t(splits) * 2 * M * up8(N) * sizeof(float) : 0;
  p.bytes = p.pack + (p.packed ? (size_t(M) + 2 * N) * up8(K) * 2 : 0);
  return p;
}

int check_sizes(const char* fn, int64_t M, int32_t N, int32_t K) {
  if (M < 0 || N < 1 || K < 1)
    return set_error(NGT_ERR_ARG, "%s: bad sizes rows=%lld n_out=%d n_in=%d", fn,
                     static_cast<long long>(M), N, K);
  // 32-bit rows, and fewer than 2^24 blocks for each of the tile grids
  auto blocks = [](int64_t r, int64_t c, int t) { return (r + t - 1) / t * ((c + t - 1) / t); };
  constexpr int64_t kMost = (1 << 24) - 8;
  if (M > (1 << 30) || 2 * int64_t(N) >= kFar || K >= kFar || blocks(M, N, 64) > kMost || blocks(M, K, 64) > kMost ||
      blocks(N, K, 32) > kMost)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: rows=%lld n_out=%d n_in=%d exceed the grid", fn,
                     static_cast<long long>(M), N, K);
  return NGT_OK;
}

}  // namespace
}  // namespace ngt

using namespace ngt;

extern "C" int ngt_gated_keep_bytes(int64_t n_rows, int32_t n_out, size_t* bytes) {
  NGT_CHECK_OK(check_sizes("ngt_gated_keep_bytes", n_rows, n_out, 1));
  if (!bytes) return set_error(NGT_ERR_ARG, "ngt_gated_keep_bytes: null bytes");
  *bytes = static_cast<size_t>(Keep(n_rows, n_out).bytes());
  return NGT_OK;
}

extern "C" int ngt_gated_fwd_workspace_bytes(int64_t n_rows, int32_t n_out, int32_t n_in,
                                             size_t* bytes) {
  const char* fn = "ngt_gated_fwd_workspace_bytes";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (!bytes) return set_error(NGT_ERR_ARG, "%s: null bytes", fn);
  *bytes = plan_fwd(n_rows, n_out, n_in).bytes;
  return NGT_OK;
}

extern "C" int ngt_gated_fwd(const void* x, int64_t x_stride, const void* w_gate, const void* w_up,
                             const void* b_gate, const void* b_up, int64_t n_rows, int32_t n_out,
                             int32_t n_in, int32_t activation, void* y, void* keep, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* fn = "ngt_gated_fwd";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (activation < NGT_ACT_NONE || activation > NGT_ACT_SILU)
    return set_error(NGT_ERR_ARG, "%s: activation %d", fn, activation);
  if (n_rows == 0) return NGT_OK;
  if (!x || !w_gate || !w_up || !y) return set_error(NGT_ERR_ARG, "%s: null x, w or y", fn);
  if (x_stride < n_in) return set_error(NGT_ERR_ARG, "%s: x rows overlap", fn);
  if (!aligned16(keep)) return set_error(NGT_ERR_ARG, "%s: keep must be 16-byte aligned", fn);
  const FwdPlan p = plan_fwd(n_rows, n_out, n_in);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned16(workspace)))
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu or not 16-byte aligned", fn,
                     workspace_bytes, p.bytes);
  GatedArgs a{};
  a.x = static_cast<const uint16_t*>(x), a.x_stride = x_stride;
  a.wg = static_cast<const uint16_t*>(w_gate), a.wu = static_cast<const uint16_t*>(w_up);
  a.bg = static_cast<const uint16_t*>(b_gate), a.bu = static_cast<const uint16_t*>(b_up);
  a.y = static_cast<uint16_t*>(y), a.keep = keep, a.part = static_cast<float*>(workspace);
  a.M = static_cast<int32_t>(n_rows), a.N = n_out, a.K = n_in, a.act = activation;
  a.tiles_m = (a.M + 63) / 64, a.tiles_n = (a.N + 63) / 64;
  hipStream_t st = static_cast<hipStream_t>(stream);
  KernelTimer timer_("gated_fwd", st);
  if (p.packed) {
    Packed to;
    NGT_CHECK_OK(launch_pack({{a.x, a.wg, a.wu},
                              {n_rows, n_out, n_out},
                              x_stride,
                              reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + p.pack),
                              n_in, 0},
                             st, &to));
    a.x = to.x, a.wg = to.wg, a.wu = to.wu, a.K = up8(n_in), a.x_stride = a.K;
  }
  const bool aligned = a.K % 8 == 0 && a.x_stride % 8 == 0 && all_aligned16({a.x, a.wg, a.wu});
  // 1 and 64 rows, us, here and in the tiles of 64 rows: 768 -> 2,048 7, 9 and 14, 14; 2,048 -> 8,192
  // 17, 24 and 31, 31.
  if (aligned && n_rows <= kFewRows) {
    const Split s = few_split(n_rows, n_out, a.K);
    a.splits = s.splits, a.per_split = s.per_split;
    auto run = [&](auto mt) {
      constexpr int MT = decltype(mt)::value;
      // 32 outputs a block where that leaves 256 blocks (64 rows of 2,048 -> 8,192 25 us, 16 outputs
      // 32; of 768 -> 2,048 12 and 9)
      const int blocks = (n_out + 15) / 16;
      if (blocks >= 512)
        hipLaunchKernelGGL((k_gated_few<MT, 2, MT < 3 ? 8 : 4>),
                           dim3(unsigned((n_out + 31) / 32), a.splits), dim3(MT < 3 ? 512 : 256), 0,
                           st, a);
      else
        hipLaunchKernelGGL((k_gated_few<MT, 1, 8>), dim3(unsigned(blocks), a.splits), dim3(512), 0, st,
                           a);
    };
    if (n_rows <= 16) run(std::integral_constant<int, 1>{});
    else if (n_rows <= 32) run(std::integral_constant<int, 2>{});
    else if (n_rows <= 48) run(std::integral_constant<int, 3>{});
    else run(std::integral_constant<int, 4>{});
  } else {
    const Split s = tile_split(n_rows, n_out, a.K);
    a.splits = s.splits, a.per_split = s.per_split;
    if (aligned && a.x_stride < kFar) {
      auto run = [&](auto fm) {
        constexpr int FM = decltype(fm)::value;
        a.tiles_m = (a.M + 64 * FM - 1) / (64 * FM);
        const int64_t blocks = (int64_t(a.tiles_m) * a.tiles_n * (FM == 1 ? a.splits : 1) + 7) / 8 * 8;
        const bool whole = n_out % 8 == 0 && aligned16(y);
        hipLaunchKernelGGL((whole ? &k_gated<FM, true> : &k_gated<FM, false>), dim3(unsigned(blocks)),
                           dim3(256), 0, st, a);
      };
      // The tallest tile that leaves 384 blocks, three quarters of what the CUs hold (us with 256,
      // 128 and 64 rows: 2,048 -> 8,192 at 512 rows 46, 41, 49, at 1,024 66, 79, 93; 768 -> 2,048 at
      // 65 18, 14, 13, at 2,048 22, 19, 23, at 32,768 240, 261, 292).
      if (a.splits == 1 && (n_rows + 255) / 256 * a.tiles_n >= 384) run(std::integral_constant<int, 4>{});
      else if (a.splits == 1 && (n_rows + 127) / 128 * a.tiles_n >= 384) run(std::integral_constant<int, 2>{});
      else run(std::integral_constant<int, 1>{});
    } else {
      hipLaunchKernelGGL(k_gated_any, dim3(unsigned(int64_t(a.tiles_m) * a.tiles_n * a.splits)), dim3(256),
                         0, st, a);
    }
  }
  NGT_HIP_CHECK(hipGetLastError());
  if (a.splits > 1) {
    const int64_t pieces = n_rows * (up8(n_out) / 8);
    hipLaunchKernelGGL(k_gated_join_fwd, dim3(unsigned((pieces + 255) / 256)), dim3(256), 0, st, a);
    NGT_HIP_CHECK(hipGetLastError());
  }
  return NGT_OK;
}

extern "C" int ngt_gated_bwd_workspace_bytes(int64_t n_rows, int32_t n_out, int32_t n_in,
                                             size_t* bytes) {
  const char* fn = "ngt_gated_bwd_workspace_bytes";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (!bytes) return set_error(NGT_ERR_ARG, "%s: null bytes", fn);
  *bytes = plan_bwd(n_rows, n_out, n_in).bytes;
  return NGT_OK;
}

extern "C" int ngt_gated_bwd_tiles(int64_t n_rows, int32_t n_out, int32_t n_in, int32_t columns[2],
                                   int32_t splits[2]) {
  const char* fn = "ngt_gated_bwd_tiles";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (!columns || !splits) return set_error(NGT_ERR_ARG, "%s: null columns or splits", fn);
  const BwdPlan p = plan_bwd(n_rows, n_out, n_in);
  columns[0] = 64 * p.dx.fn, splits[0] = p.dx.splits;
  columns[1] = 64 * p.dw.fn, splits[1] = p.dw.splits;
  return NGT_OK;
}

extern "C" int ngt_gated_bwd(const void* dy, const void* keep, const void* x, const void* w_gate,
                             const void* w_up, int64_t n_rows, int32_t n_out, int32_t n_in,
                             const ngt_gated_grads* grads, void* workspace, size_t workspace_bytes,
                             void* stream) {
  const char* fn = "ngt_gated_bwd";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (!grads) return set_error(NGT_ERR_ARG, "%s: null grads", fn);
  const ngt_gated_grads& g = *grads;
  const bool want_w = g.dw_gate || g.dw_up, want_b = g.db_gate || g.db_up;
  if (n_rows > 0 && (!dy || !keep)) return set_error(NGT_ERR_ARG, "%s: null dy or keep", fn);
  if (n_rows > 0 && g.dx && (!w_gate || !w_up)) return set_error(NGT_ERR_ARG, "%s: null w", fn);
  if (n_rows > 0 && want_w && !x) return set_error(NGT_ERR_ARG, "%s: null x", fn);
  for (const auto& t : {std::pair<const void*, int32_t>(g.dw_gate, g.dw_gate_dtype),
                        {g.dw_up, g.dw_up_dtype}, {g.db_gate, g.db_gate_dtype},
                        {g.db_up, g.db_up_dtype}})
    if (t.first && t.second != NGT_F32 && t.second != NGT_BF16)
      return set_error(NGT_ERR_ARG, "%s: gradient dtype %d", fn, t.second);
  if (!all_aligned16({dy, keep, x, w_gate, w_up, g.dx, g.dw_gate, g.dw_up}))
    return set_error(NGT_ERR_ARG, "%s: matrices must be 16-byte aligned", fn);
  const BwdPlan p = plan_bwd(n_rows, n_out, n_in);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned16(workspace)))
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu or not 16-byte aligned", fn,
                     workspace_bytes, p.bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  auto* dz = reinterpret_cast<uint16_t*>(ws + p.dz);
  auto* part = reinterpret_cast<float*>(ws + p.part);
  auto* part_b = reinterpret_cast<float*>(ws + p.part_b);
  GatedBwd products{dz,
                    static_cast<const uint16_t*>(x),
                    static_cast<const uint16_t*>(w_gate),
                    static_cast<const uint16_t*>(w_up),
                    static_cast<uint16_t*>(g.dx),
                    {g.dw_gate, g.dw_up},
                    part,
                    n_rows,
                    n_out,
                    up8(n_in),
                    {g.dw_gate_dtype == NGT_F32, g.dw_up_dtype == NGT_F32},
                    p.packed};
  if (p.packed && n_rows > 0 && (g.dx || want_w)) {
    KernelTimer timer_("gated_pack", st);
    Packed to;
    NGT_CHECK_OK(launch_pack({{products.x, products.wg, products.wu},
                              {want_w ? n_rows : 0, g.dx ? n_out : 0, g.dx ? n_out : 0},
                              n_in,
                              reinterpret_cast<uint16_t*>(ws + p.pack),
                              n_in, 0},
                             st, &to));
    products.x = to.x, products.wg = to.wg, products.wu = to.wu;
  }
  if (n_rows > 0) {
    KernelTimer timer_("gated_dz", st);
    const int32_t tiles_n = (n_out + 255) / 256;
    hipLaunchKernelGGL(n_out % 8 == 0 ? &k_gated_dz<true> : &k_gated_dz<false>,
                       dim3(unsigned(p.chunks * tiles_n)), dim3(256), 0, st,
                       static_cast<const uint16_t*>(dy), const_cast<void*>(keep), n_rows, n_out,
                       tiles_n, p.chunk_rows, dz, want_b ? part_b : nullptr);
    NGT_HIP_CHECK(hipGetLastError());
  }
  if (n_rows > 0 && g.dx) {
    KernelTimer timer_("gated_dx", st);
    NGT_CHECK_OK(launch_gated_dx(products, p.dx, st));
    if (p.dx.splits > 1 || p.packed) {
      const int64_t blocks = (n_rows * (products.K / 8) + 255) / 256;
      hipLaunchKernelGGL(k_gated_join_dx, dim3(unsigned(blocks)), dim3(256), 0, st, part, p.dx.splits,
                         n_rows, n_in, products.dx);
      NGT_HIP_CHECK(hipGetLastError());
    }
  }
  if (want_w && n_rows > 0) {
    KernelTimer timer_("gated_dw", st);
    NGT_CHECK_OK(launch_gated_dw(products, p.dw, st));
  }
  const int32_t splits = n_rows > 0 ? p.dw.splits : 0;
  const bool join_w = want_w && (splits != 1 || p.packed);
  if (join_w || want_b) {
    KernelTimer timer_("gated_join", st);
    JoinArgs j{};
    j.part = part, j.part_b = part_b;
    j.dw[0] = g.dw_gate, j.dw[1] = g.dw_up, j.db[0] = g.db_gate, j.db[1] = g.db_up;
    j.dw_f32[0] = g.dw_gate_dtype == NGT_F32, j.dw_f32[1] = g.dw_up_dtype == NGT_F32;
    j.db_f32[0] = g.db_gate_dtype == NGT_F32, j.db_f32[1] = g.db_up_dtype == NGT_F32;
    j.nk = int64_t(n_out) * n_in, j.n = n_out, j.k = n_in, j.splits = splits;
    j.chunks = static_cast<int32_t>(p.chunks);
    j.blocks_w = join_w ? static_cast<int32_t>(std::min((2 * int64_t(n_out) * products.K + 1023) / 1024, kMostBlocks)) : 0;
    const int blocks_b = want_b ? (2 * n_out + 31) / 32 : 0;
    hipLaunchKernelGGL(k_gated_join, dim3(unsigned(j.blocks_w + blocks_b)), dim3(256), 0, st, j);
    NGT_HIP_CHECK(hipGetLastError());
  }
  return NGT_OK;
}
