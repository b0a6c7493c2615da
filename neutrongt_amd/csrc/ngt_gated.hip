// Gated linear layer, bf16: y = act(x Wg^T + bg) * (x Wu^T + bu), fp32 inside, and its
// backward up to the weights' gradients (ngt_wgrad.hip):
//   keep = [zu act'(zg) | act(zg)],  dz = [dzg | dzu] = dy * keep,  dx = dzg Wg + dzu Wu.
// The forward keeps the two factors of dy instead of zg and zu, so that the backward
// forms no activation; either way two roundings to bf16 stand between dy and dz.
#include "ngt_linear.h"

namespace ngt {
namespace {

using packed::f32x16;
using packed::fill16;
using packed::tid_x;
using packed::wg_x;

constexpr int kStage = 64;  // contraction per LDS stage: rows of 128 bytes
using L = packed::Tile<bf16_t, kStage>;

struct GatedArgs {
  const uint16_t* x;   // [M, K], rows x_stride apart
  const uint16_t* wg;  // [N, K]
  const uint16_t* wu;
  const uint16_t* bg;  // [N] or null
  const uint16_t* bu;
  uint16_t* y;         // [M, N]
  uint16_t* keep;      // [M, 2 N] or null
  int64_t x_stride;
  int32_t M, N, K, act;
  int32_t tiles_m, tiles_n;
};

// act(z) and act'(z).
struct Gate {
  float value, slope;
};
__device__ __forceinline__ Gate gate_of(int act, float z) {
  if (act == NGT_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
    return {z * s, s * fmaf(z, 1.f - s, 1.f)};
  }
  if (act == NGT_ACT_GELU) {
    const Normal n = normal(z);
    return {z * n.cdf, fmaf(z * 0.39894228040143268f, n.pdf, n.cdf)};
  }
  if (act == NGT_ACT_RELU) return {z > 0.f ? z : (z != z ? z : 0.f), z > 0.f ? 1.f : 0.f};
  return {z, 1.f};
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

// 8 outputs n .. n+7 of row m from their sums.
__device__ __forceinline__ void finish8(const GatedArgs& a, int m, int n, const float (&sg)[8],
                                        const float (&su)[8]) {
  if (m >= a.M || n >= a.N) return;
  u32x4 bg = {0u, 0u, 0u, 0u}, bu = {0u, 0u, 0u, 0u}, y, kg, ku;
  if (a.bg) bg = load8<false>(a.bg, n, a.N);
  if (a.bu) bu = load8<false>(a.bu, n, a.N);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[2], g[2], u[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float zu = su[2 * i + t] + half_of(bu, 2 * i + t);
      const Gate q = gate_of(a.act, sg[2 * i + t] + half_of(bg, 2 * i + t));
      v[t] = q.value * zu, g[t] = zu * q.slope, u[t] = q.value;
    }
    y[i] = pack2_bf16(v[0], v[1]);
    kg[i] = pack2_bf16(g[0], g[1]);
    ku[i] = pack2_bf16(u[0], u[1]);
  }
  store8(a.y + int64_t(m) * a.N, n, a.N, y);
  if (a.keep) {
    uint16_t* row = a.keep + int64_t(m) * 2 * a.N;
    store8(row, n, a.N, kg);
    store8(row + a.N, n, a.N, ku);
  }
}

// Any sizes and 2-byte alignment.  One block: 64 rows by 64 outputs of both products,
// 2 x 2 waves of 32 x 32, stages of 64 of the contraction read into registers while the
// stage before is multiplied.
__global__ __launch_bounds__(256) void k_gated_any(GatedArgs a) {
  constexpr int NP = 64 * 8 / 256;  // 16-byte pieces per thread and operand
  __shared__ __align__(16) char lds[3][64 * 128];
  const int tid = tid_x(), lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  const int m0 = wg_x() / a.tiles_n * 64, n0 = wg_x() % a.tiles_n * 64;
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
  fetch(0);
  for (int k = 0; k < a.K; k += kStage) {
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int e = tid + i * 256;
        *reinterpret_cast<u32x4*>(lds[o] + L::offset(e / 8, e % 8)) = p[o][i];
      }
    __syncthreads();
    fetch(k + kStage);  // (behind the last stage: zeros)
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
    finish8(a, m0 + wm + L::a_row(l32), n0 + wn + 16 * half + 8 * e, sg, su);
  }
}

// dz = [dy keep_g | dy keep_u], 8 columns a thread.
__global__ __launch_bounds__(256) void k_gated_dz(const uint16_t* __restrict__ dy,
                                                  const uint16_t* __restrict__ keep, int64_t rows,
                                                  int32_t n, uint16_t* __restrict__ dz) {
  const int64_t per_row = (n + 7) / 8, total = rows * per_row;
  const int64_t step = int64_t(__builtin_amdgcn_grid_size_x());
  for (int64_t i = int64_t(wg_x()) * 256 + tid_x(); i < total; i += step) {
    const int64_t row = i / per_row;
    const int c = static_cast<int>(i - row * per_row) * 8;
    const u32x4 g = load8<false>(dy + row * n, c, n);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const u32x4 v = load8<false>(keep + (2 * row + part) * n, c, n);
      u32x4 o;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        o[t] = pack2_bf16(half_of(g, 2 * t) * half_of(v, 2 * t),
                          half_of(g, 2 * t + 1) * half_of(v, 2 * t + 1));
      store8(dz + (2 * row + part) * n, c, n, o);
    }
  }
}

struct DxArgs {
  const uint16_t* dz;  // [M, 2 N]
  const uint16_t* wg;  // [N, K]
  const uint16_t* wu;
  uint16_t* dx;        // [M, K]
  int32_t M, N, K;
  int32_t tiles_k;
};

// dx = dzg Wg + dzu Wu at any sizes and alignment: the same blocks, 64 rows by 64 of K,
// contracted over the outputs of one layer and then of the other; W's stages are
// turned on their way to LDS.
__global__ __launch_bounds__(256) void k_gated_dx_any(DxArgs a) {
  constexpr int NP = 64 * 8 / 256;
  __shared__ __align__(16) char lz[64 * 128];
  __shared__ __align__(16) char lw[64 * 128];
  const int tid = tid_x(), lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  const int m0 = wg_x() / a.tiles_k * 64, k0 = wg_x() % a.tiles_k * 64;
  const int wm = (wave >> 1) * 32, wk = (wave & 1) * 32;
  f32x16 acc = fill16(0.f);
  for (int part = 0; part < 2; ++part) {
    const uint16_t* w = part ? a.wu : a.wg;
    for (int n0 = 0; n0 < a.N; n0 += kStage) {
      u32x4 z[NP], v[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int e = tid + i * 256, m = m0 + e / 8, n = n0 + e / 8;
        z[i] = v[i] = u32x4{0u, 0u, 0u, 0u};
        if (m < a.M) z[i] = load8<false>(a.dz + (int64_t(m) * 2 + part) * a.N, n0 + 8 * (e % 8), a.N);
        if (n < a.N) v[i] = load8<false>(w + int64_t(n) * a.K, k0 + 8 * (e % 8), a.K);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int e = tid + i * 256, r = e / 8, c = e % 8;
        *reinterpret_cast<u32x4*>(lz + L::offset(r, c)) = z[i];
#pragma unroll
        for (int t = 0; t < 8; ++t)
          *reinterpret_cast<uint16_t*>(lw + L::offset(8 * c + t, r / 8) + 2 * (r % 8)) =
              static_cast<uint16_t>(v[i][t / 2] >> (16 * (t & 1)));
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c)
        acc = L::mma(L::load_a(lw + wk * 128, 0, c, l32, half),
                     L::load_a(lz + wm * 128, 0, c, l32, half), acc);
    }
  }
  const int m = m0 + wm + L::a_row(l32);
  if (m >= a.M) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    u32x4 o;
#pragma unroll
    for (int t = 0; t < 4; ++t) o[t] = pack2_bf16(acc[8 * e + 2 * t], acc[8 * e + 2 * t + 1]);
    const int k = k0 + wk + 16 * half + 8 * e;
    if (k < a.K) store8(a.dx + int64_t(m) * a.K, k, a.K, o);
  }
}

int check_sizes(const char* fn, int64_t M, int32_t N, int32_t K) {
  if (M < 0 || N < 1 || K < 1)
    return set_error(NGT_ERR_ARG, "%s: bad sizes rows=%lld n_out=%d n_in=%d", fn,
                     static_cast<long long>(M), N, K);
  // 32-bit rows, and fewer than 2^24 blocks for each of the tile grids
  auto blocks = [](int64_t r, int64_t c, int t) { return (r + t - 1) / t * ((c + t - 1) / t); };
  constexpr int64_t kMost = (1 << 24) - 8;
  if (M > (1 << 30) || N > (1 << 29) || blocks(M, N, 64) > kMost || blocks(M, K, 64) > kMost)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: rows=%lld n_out=%d n_in=%d exceed the grid", fn,
                     static_cast<long long>(M), N, K);
  return NGT_OK;
}

}  // namespace
}  // namespace ngt

using namespace ngt;

extern "C" int ngt_gated_fwd(const void* x, int64_t x_stride, const void* w_gate, const void* w_up,
                             const void* b_gate, const void* b_up, int64_t n_rows, int32_t n_out,
                             int32_t n_in, int32_t activation, void* y, void* keep, void* stream) {
  const char* fn = "ngt_gated_fwd";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (activation < NGT_ACT_NONE || activation > NGT_ACT_SILU)
    return set_error(NGT_ERR_ARG, "%s: activation %d", fn, activation);
  if (n_rows == 0) return NGT_OK;
  if (!x || !w_gate || !w_up || !y) return set_error(NGT_ERR_ARG, "%s: null x, w or y", fn);
  if (x_stride < n_in) return set_error(NGT_ERR_ARG, "%s: x rows overlap", fn);
  GatedArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(w_gate),
              static_cast<const uint16_t*>(w_up), static_cast<const uint16_t*>(b_gate),
              static_cast<const uint16_t*>(b_up), static_cast<uint16_t*>(y),
              static_cast<uint16_t*>(keep), x_stride, static_cast<int32_t>(n_rows), n_out, n_in,
              activation, 0, 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  KernelTimer timer_("gated_fwd", st);
  a.tiles_m = (a.M + 63) / 64, a.tiles_n = (a.N + 63) / 64;
  hipLaunchKernelGGL(k_gated_any, dim3(unsigned(int64_t(a.tiles_m) * a.tiles_n)), dim3(256), 0, st,
                     a);
  NGT_HIP_CHECK(hipGetLastError());
  return NGT_OK;
}

extern "C" int ngt_gated_bwd_workspace_bytes(int64_t n_rows, int32_t n_out, int32_t n_in,
                                             size_t* bytes) {
  NGT_CHECK_OK(check_sizes("ngt_gated_bwd_workspace_bytes", n_rows, n_out, n_in));
  if (!bytes) return set_error(NGT_ERR_ARG, "ngt_gated_bwd_workspace_bytes: null bytes");
  *bytes = 0;
  return NGT_OK;
}

extern "C" int ngt_gated_bwd(const void* dy, const void* keep, const void* w_gate,
                             const void* w_up, int64_t n_rows, int32_t n_out, int32_t n_in,
                             void* dz, void* dx, void* workspace, size_t workspace_bytes,
                             void* stream) {
  const char* fn = "ngt_gated_bwd";
  NGT_CHECK_OK(check_sizes(fn, n_rows, n_out, n_in));
  if (n_rows == 0) return NGT_OK;
  if (!dy || !keep || !dz) return set_error(NGT_ERR_ARG, "%s: null dy, keep or dz", fn);
  if (dx && (!w_gate || !w_up)) return set_error(NGT_ERR_ARG, "%s: null w", fn);
  hipStream_t st = static_cast<hipStream_t>(stream);
  {
    KernelTimer timer_("gated_dz", st);
    const int64_t blocks = (n_rows * ((n_out + 7) / 8) + 255) / 256;
    hipLaunchKernelGGL(k_gated_dz, dim3(unsigned(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st,
                       static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(keep), n_rows,
                       n_out, static_cast<uint16_t*>(dz));
    NGT_HIP_CHECK(hipGetLastError());
  }
  if (!dx) return NGT_OK;
  KernelTimer timer_("gated_dx", st);
  DxArgs a{static_cast<const uint16_t*>(dz), static_cast<const uint16_t*>(w_gate),
           static_cast<const uint16_t*>(w_up), static_cast<uint16_t*>(dx),
           static_cast<int32_t>(n_rows), n_out, n_in, (n_in + 63) / 64};
  hipLaunchKernelGGL(k_gated_dx_any, dim3(unsigned((n_rows + 63) / 64 * a.tiles_k)), dim3(256), 0,
                     st, a);
  NGT_HIP_CHECK(hipGetLastError());
  return NGT_OK;
}
