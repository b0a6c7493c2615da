// RMS norm of query and key heads with a gain, and the rotation of their first
// components by the row's position, in one pass; forward and backward.  What stands
// between the projections of packed attention and the attention itself.
//
//   s = 1 / sqrt(mean(x^2) + eps),  h = x s,  u = h gain        (no gain: u = x)
//   y_a = m (u_a cos t - u_b sin t),  y_b = m (u_a sin t + u_b cos t),  t = position f
// and backward, with g = the transposed rotation of dy:
//   dgain = sum over rows and heads of g h,  w = g gain,  dx = s (w - h mean(w h)).
// s is formed again from x, which the backward reads anyway.
//
// Bound by memory: a head is read once and written once.  A lane holds 2 V of its
// components, V pairs (16 bytes twice where sizes and alignment allow), a group of
// lanes a head, so the mean is a few steps within the wave.  Cosines and sines are
// formed once for all heads of a row, in LDS: the angle in fp64 turns, of which only the
// part behind the quarter turn enters the fp32 functions, so that a far position
// costs no precision.
// bf16: 12,289 rows of 32 + 8 heads of 128 47 us, 5.4 TB/s; 32,768 rows of 32 + 32 heads of 24
// 40 forward, 5.0 TB/s, and 64 backward, 4.7 TB/s (its sums take the registers of two
// of the eight waves that the forward has on a SIMD).
#include "ngt_common.h"

#include <type_traits>

namespace ngt {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int kTableBytes = 16384;  // cosines and sines of a block's rows
// Blocks of a backward that a CU holds, by the registers of its sums, for pieces of `bytes`; a
// launch has about as many, each with a partial sum (bf16, 32,768 rows of 32 + 32 heads of 24:
// 1,024 blocks 76 us, 1,280 71, 1,536 67; 12,289 of 32 + 8 of 128: 768 86 us, 1,024 85, 1,280 90).
// The heads of 24 were measured with interleaved pairs.  In halves the kernel of 8-byte pieces of
// bf16 needs 4 registers more than six blocks leave it; it keeps them in scratch memory, two of
// them read once a head (32 + 32 heads of 24 68 us for 63, 16 + 16 of 40 67 for 65, both with the
// library's timer).  fp32 with a norm, five blocks: 16 + 16 heads of 24 62 us, 4.9 TB/s; of 64 167,
// 4.8 TB/s.
constexpr int bwd_blocks(int bytes, int es) { return bytes <= 8 ? 6 : es == 2 ? 4 : 5; }
constexpr int kBwdBlocks = 6 * 256;
inline size_t sums_bytes(int32_t d) { return size_t(kBwdBlocks + 2) * d * sizeof(float); }

// One of queries and keys, as the kernels see it.
struct Rows {
  const void* x;
  const void* gain;
  void* y;
  const void* dy;
  float* part;  // [blocks][d] of dgain, or null
  int64_t x_row, x_head, dy_row, dy_head;
  int32_t n_heads, gain_f32;
  int32_t tile_rows;  // rows of a tile
  int32_t splits;     // blocks that share a tile's heads
  int32_t tiles;
  int32_t blocks;
};

struct Args {
  Rows r[2];
  const void* positions;
  const double* turns;
  int64_t n_rows;
  float eps, by_cos, by_sin;  // the rotation's magnitude; by_sin negative: turned back
  int32_t d, dim, units, group_log;  // 2^group_log lanes a head
  int32_t pos64;
};

// cos and sin of 2 pi x, x in turns.
__device__ __forceinline__ float2 cos_sin(double x) {
  x -= rint(x);
  const double q = rint(4.0 * x);
  // less than an eighth of a turn is left, exact until it is rounded
  const float f = static_cast<float>(fma(q, -0.25, x));
  float s, c;
  sincospif(2.f * f, &s, &c);
  const int k = static_cast<int>(q) & 3;
  const float a = k & 1 ? -s : c, b = k & 1 ? c : s;
  return k & 2 ? make_float2(-a, -b) : make_float2(a, b);
}

template <typename T, int V>
struct Chunk {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];
  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  __device__ __forceinline__ static void store(T* __restrict__ p, const float* v) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      else if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
      else *p = v[0];
    } else {
      if constexpr (V == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]),
                                                  pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
      else if constexpr (V == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
      else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = pack2_bf16(v[0], v[1]);
      else p->x = static_cast<uint16_t>(pack2_bf16(v[0], 0.f));
    }
  }
};

// Sum over the 2^log adjacent lanes of a head, the same in all of them: within 16 lanes by
// lane permutations of the addition itself (neighbours, pairs, halves of 8 and of 16 mirrored).
template <int CTRL>
__device__ __forceinline__ float add_lanes(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float group_sum(float v, int log) {
  if (log > 0) v = add_lanes<0xb1>(v);   // quad_perm 1 0 3 2
  if (log > 1) v = add_lanes<0x4e>(v);   // quad_perm 2 3 0 1
  if (log > 2) v = add_lanes<0x141>(v);  // row_half_mirror
  if (log > 3) v = add_lanes<0x140>(v);  // row_mirror
  if (log > 4) v += shfl_xor(v, 16);
  if (log > 5) v += shfl_xor(v, 32);
  return v;
}

// 1 / sqrt(x): the instruction's result and a Newton step, within 1.5 half steps of fp32.
__device__ __forceinline__ float inverse_root(float x) {
  const float r = __builtin_amdgcn_rsqf(x);
  const float e = fmaf(-x * r, r, 1.f);
  // (0, infinities and NaN as they come: a step would make NaN of them)
  return x > 1e-30f && x < 1e30f ? fmaf(0.5f * r, e, r) : 1.f / sqrtf(x);
}

// V pairs of components of each of a lane's U units; INTER: pairs are adjacent.
template <typename T, int V, int U, bool INTER, bool BWD>
__global__ __launch_bounds__(kThreads, BWD ? bwd_blocks(V * sizeof(T), sizeof(T)) : 1) void k_norm_rotary(const Args a) {
  extern __shared__ float2 table[];  // [tile_rows][dim / 2]
  __shared__ float sums[BWD ? kThreads / kWave : 1][BWD ? kMaxDim : 1];
  const int tid = threadIdx.x;
  const bool second = int(blockIdx.x) >= a.r[0].blocks;  // block-uniform
  const Rows r = second ? a.r[1] : a.r[0];
  const int block = blockIdx.x - (second ? a.r[0].blocks : 0);
  const int pairs = a.dim / 2, lanes = 1 << a.group_log, groups = kThreads >> a.group_log;
  const int lane = tid & (lanes - 1), group = tid >> a.group_log;
  const bool norm = r.gain != nullptr;
  const float by_d = 1.f / static_cast<float>(a.d), by_heads = 1.f / static_cast<float>(r.n_heads);

  // where this lane's units lie in a head
  int at[U][2], turn[U];
  bool there[U], turned[U];
  float gain[U][2 * V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int unit = lane * U + u;
    there[u] = unit < a.units;
    turned[u] = 2 * V * unit < a.dim;
    turn[u] = turned[u] ? unit * V : 0;  // (its first pair)
    const bool apart = !INTER && turned[u];
    // (a lane without a unit reads the first one again)
    at[u][0] = !there[u] ? 0 : apart ? unit * V : 2 * V * unit;
    at[u][1] = !there[u] ? V : apart ? pairs + unit * V : 2 * V * unit + V;
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
      gain[u][i] = 1.f;
      if (norm && there[u]) {
        const int c = at[u][i / V] + i % V;
        gain[u][i] = r.gain_f32 ? static_cast<const float*>(r.gain)[c]
                                : bf16_to_f32(static_cast<const bf16_t*>(r.gain)[c].x);
      }
    }
  }
  float acc[U][2 * V];
  if constexpr (BWD)
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) acc[u][i] = 0.f;

  const int slot = block % r.splits, per_round = r.blocks / r.splits;
  for (int tile = block / r.splits; tile < r.tiles; tile += per_round) {
    const int64_t row0 = int64_t(tile) * r.tile_rows;
    const int rows = a.n_rows - row0 < r.tile_rows ? int(a.n_rows - row0) : r.tile_rows;
    const int items = rows * r.n_heads, step = groups * r.splits;
    // (below 2^17, so the quotient, half an item off the next whole number, is exact)
    auto row_of = [&](int item) { return static_cast<int>((item + 0.5f) * by_heads); };
    struct Head {
      Chunk<T, V> x[U][2], g[U][2];
    };
    auto fetch = [&](int item) {
      Head h;
      item = min(item, items - 1);  // behind the last: that one again
      const int row = row_of(item), head = item - row * r.n_heads;
      const T* x = static_cast<const T*>(r.x) + (row0 + row) * r.x_row + head * r.x_head;
      const T* g = static_cast<const T*>(r.dy) + (row0 + row) * r.dy_row + head * r.dy_head;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          h.x[u][c].load(x + at[u][c]);
          if constexpr (BWD) h.g[u][c].load(g + at[u][c]);
        }
      return h;
    };
    // the next head is on its way while one is computed, the first one while the cosines are
    int item = slot * groups + group;
    Head next = fetch(item);
    __syncthreads();
    for (int e = tid; e < rows * pairs; e += kThreads) {
      const int row = e / pairs;
      const double p = a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[row0 + row])
                               : static_cast<double>(static_cast<const int32_t*>(a.positions)[row0 + row]);
      const float2 cs = cos_sin(p * a.turns[e - row * pairs]);
      table[e] = make_float2(cs.x * a.by_cos, cs.y * a.by_sin);
    }
    __syncthreads();
    for (; item < items; item += step) {
      const Head now = next;
      next = fetch(item + step);
      const int row = row_of(item), head = item - row * r.n_heads;
      const int64_t to = ((row0 + row) * r.n_heads + head) * a.d;
      float v[U][2 * V];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) v[u][i] = now.x[u][i / V].get(i % V);
      float scale = 1.f;
      if (norm) {
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float q = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) q = fmaf(v[u][i], v[u][i], q);
          s += there[u] ? q : 0.f;
        }
        scale = inverse_root(fmaf(group_sum(s, a.group_log), by_d, a.eps));
      }
      float w[U][2 * V], dot = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float2* cs = table + row * pairs + turn[u];
        float in[2 * V];
#pragma unroll
        for (int i = 0; i < 2 * V; ++i)
          in[i] = BWD ? now.g[u][i / V].get(i % V) : norm ? v[u][i] * scale * gain[u][i] : v[u][i];
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) w[u][i] = in[i];
        if (turned[u]) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            constexpr int kA = INTER ? 2 : 1, kB = INTER ? 1 : V;
            const int ia = kA * j, ib = kA * j + kB;
            const float c = cs[j].x, s = cs[j].y;
            w[u][ia] = fmaf(in[ia], c, -(in[ib] * s));
            w[u][ib] = fmaf(in[ia], s, in[ib] * c);
          }
        }
        if constexpr (BWD)
          if (norm) {
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
              v[u][i] *= scale;
              acc[u][i] = fmaf(w[u][i], v[u][i], acc[u][i]);
              w[u][i] *= gain[u][i];
              q = fmaf(w[u][i], v[u][i], q);
            }
            dot += there[u] ? q : 0.f;
          }
      }
      if constexpr (BWD) {
        if (norm) {
          dot = group_sum(dot, a.group_log) * by_d;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) w[u][i] = scale * fmaf(-v[u][i], dot, w[u][i]);
        }
        if (!r.y) continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (there[u]) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            Chunk<T, V>::store(static_cast<T*>(r.y) + to + at[u][c], &w[u][c * V]);
        }
    }
  }
  if constexpr (BWD) {
    if (!r.part) return;  // block-uniform
    // the groups of a wave, then the waves in their order
    const int wave = tid / kWave;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) {
        for (int off = lanes; off < kWave; off <<= 1) acc[u][i] += shfl_xor(acc[u][i], off);
        if (tid % kWave < lanes && there[u]) sums[wave][at[u][i / V] + i % V] = acc[u][i];
      }
    __syncthreads();
    if (tid < a.d) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < kThreads / kWave; ++q) s += sums[q][tid];
      r.part[int64_t(block) * a.d + tid] = s;
    }
  }
}

// dgain: the blocks' sums added, 32 columns a block, 32 lanes a column that take
// every 32nd block; in fp64.
struct Join {
  const float* part[2];
  void* out[2];
  int32_t blocks[2], f32[2];
  int32_t d;
};
__global__ __launch_bounds__(1024) void k_join_gain(const Join j) {
  __shared__ double red[32][33];
  const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
  if (!j.out[which]) return;
  double s = 0.0;
  if (col < j.d) {
#pragma unroll 4
    for (int b = lane; b < j.blocks[which]; b += 32)
      s += static_cast<double>(j.part[which][int64_t(b) * j.d + col]);
  }
  red[lane][threadIdx.x % 32] = s;
  __syncthreads();
  if (lane != 0 || col >= j.d) return;
  for (int l = 1; l < 32; ++l) s += red[l][threadIdx.x];
  if (j.f32[which]) static_cast<float*>(j.out[which])[col] = static_cast<float>(s);
  else static_cast<bf16_t*>(j.out[which])[col].x = f32_to_bf16(static_cast<float>(s));
}

bool multiple(const void* p, int64_t a, int64_t b, int v, int es) {
  return reinterpret_cast<uintptr_t>(p) % (v * es) == 0 && a % v == 0 && b % v == 0;
}

int check(const char* fn, int dtype, const ngt_head_rows* q, const ngt_head_rows* k,
          int64_t n_rows, int32_t d, const ngt_rotation* rot, float eps, bool bwd) {
  if (dtype != NGT_F32 && dtype != NGT_BF16) return set_error(NGT_ERR_ARG, "%s: dtype %d", fn, dtype);
  if (n_rows < 0 || n_rows > kMaxRows)
    return set_error(NGT_ERR_ARG, "%s: n_rows=%lld", fn, static_cast<long long>(n_rows));
  if (d < 2 || d % 2 || d > kMaxDim)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: head_dim %d is not even or not within 2 .. %d", fn, d,
                     kMaxDim);
  if (!q) return set_error(NGT_ERR_ARG, "%s: null q", fn);
  if (!(eps >= 0.f)) return set_error(NGT_ERR_ARG, "%s: eps=%g", fn, double(eps));
  if (rot && (rot->dim < 0 || rot->dim % 2 || rot->dim > d))
    return set_error(NGT_ERR_ARG, "%s: %d rotated components of %d", fn, rot->dim, d);
  if (rot && rot->dim > 0 && rot->position_bytes != 4 && rot->position_bytes != 8)
    return set_error(NGT_ERR_ARG, "%s: positions of %d bytes", fn, rot->position_bytes);
  if (n_rows > 0 && rot && rot->dim > 0 && (!rot->positions || !rot->turns))
    return set_error(NGT_ERR_ARG, "%s: null positions or turns", fn);
  for (const ngt_head_rows* h : {q, k}) {
    if (!h) continue;
    if (h->n_heads < 1 || h->n_heads > (1 << 16))
      return set_error(NGT_ERR_ARG, "%s: %d heads", fn, h->n_heads);
    if (h->gain && h->gain_dtype != NGT_F32 && h->gain_dtype != NGT_BF16)
      return set_error(NGT_ERR_ARG, "%s: gain dtype %d", fn, h->gain_dtype);
    if (n_rows > 0 && ((!h->x && !(bwd && !h->gain)) || (bwd ? !h->dy : !h->y)))
      return set_error(NGT_ERR_ARG, "%s: null %s", fn, bwd ? "x or dy" : "x or y");
    if (h->dgain && !h->gain) return set_error(NGT_ERR_ARG, "%s: dgain without a gain", fn);
    if (h->x_row < 0 || h->x_head < 0 || h->dy_row < 0 || h->dy_head < 0)
      return set_error(NGT_ERR_ARG, "%s: negative stride", fn);
  }
  return NGT_OK;
}

template <typename T, int V, int U, bool BWD>
void launch(const Args& a, bool inter, int blocks, size_t lds, hipStream_t st) {
  auto kernel = inter ? &k_norm_rotary<T, V, U, true, BWD> : &k_norm_rotary<T, V, U, false, BWD>;
  hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kThreads), lds, st, a);
}

template <bool BWD>
int run(const char* fn, int dtype, const ngt_head_rows* q, const ngt_head_rows* k, int64_t n_rows,
        int32_t d, const ngt_rotation* rot, float eps, void* workspace, hipStream_t st) {
  const int es = dtype == NGT_F32 ? 4 : 2;
  Args a{};
  a.n_rows = n_rows, a.eps = eps, a.d = d;
  a.dim = rot ? rot->dim : 0;
  if (a.dim) {
    a.positions = rot->positions, a.turns = rot->turns;
    a.by_cos = rot->magnitude, a.by_sin = BWD ? -rot->magnitude : rot->magnitude;
    a.pos64 = rot->position_bytes == 8;
  }
  // A gradient without a norm is its dy turned back: x is not read, and where neither has a norm
  // the forward's kernel does it (fp32, 10,007 rows of 16 + 4 heads of 64: 20 us instead of 28).
  ngt_head_rows own[2];
  const ngt_head_rows* in[2] = {};
  bool sums = false;
  for (int i = 0; i < 2; ++i) {
    const ngt_head_rows* h = i ? k : q;
    if (!h) continue;
    own[i] = *h, in[i] = &own[i];
    if (!BWD) continue;
    if (h->gain) sums = true;
    else own[i].x = h->dy, own[i].x_row = h->dy_row, own[i].x_head = h->dy_head;
  }
  // the widest pieces that sizes and alignment allow
  int v = 16 / es;
  auto fits = [&](int n) {
    if (d % (2 * n) || a.dim % (2 * n)) return false;
    for (const ngt_head_rows* h : in) {
      if (!h) continue;
      if (!multiple(h->x, h->x_row, h->x_head, n, es) || !multiple(h->y, d, d, n, es)) return false;
      if (BWD && !multiple(h->dy, h->dy_row, h->dy_head, n, es)) return false;
    }
    return true;
  };
  while (v > 1 && !fits(v)) v /= 2;
  a.units = d / (2 * v);
  const int per_lane = v == 1 ? 2 : 1;
  while ((per_lane << a.group_log) < a.units) ++a.group_log;
  const int groups = kThreads >> a.group_log;
  int blocks = 0;
  Join join{};
  join.d = d;
  float* part = static_cast<float*>(workspace);
  for (int i = 0; i < 2; ++i) {
    Rows& r = a.r[i];
    const ngt_head_rows* h = in[i];
    if (!h || (BWD && !h->y && !h->dgain)) continue;
    r.x = h->x, r.gain = h->gain, r.y = h->y, r.dy = h->dy;
    r.x_row = h->x_row, r.x_head = h->x_head, r.dy_row = h->dy_row, r.dy_head = h->dy_head;
    r.n_heads = h->n_heads, r.gain_f32 = h->gain_dtype == NGT_F32;
    // 8 heads for each group, so that a row's cosines serve many (32,768 rows of 32 + 32 heads of 24,
    // forward and backward: 4 heads 126 us, 8 116, 16 118)
    int rows = 8 * groups / h->n_heads;
    const int most = a.dim ? kTableBytes / (a.dim * 4) : 1024;
    rows = rows < 1 ? 1 : rows > most ? most : rows;
    // .. unless that leaves CUs without a block (12,289 rows of 32 + 8 heads of 128: 512 blocks of
    // keys 48.6 us, 256 50.4, 1,024 48.4)
    while (rows > 1 && (n_rows + rows - 1) / rows < 512) rows /= 2;
    r.tile_rows = rows;
    const int64_t tiles = (n_rows + rows - 1) / rows;
    r.tiles = static_cast<int32_t>(tiles);
    // a backward's blocks by the tensors' work
    const int all = h->n_heads + (in[1 - i] ? in[1 - i]->n_heads : 0);
    int64_t most_blocks = sums ? int64_t(256 * bwd_blocks(v * es, es)) * h->n_heads / all : 1 << 20;
    if (most_blocks < 1) most_blocks = 1;
    const int rounds = (rows * h->n_heads + groups - 1) / groups;
    r.splits = 1;
    while (r.splits < rounds && r.splits < most_blocks && tiles * r.splits < 512) ++r.splits;
    int64_t n = tiles * r.splits;
    if (n > most_blocks) n = most_blocks / r.splits * r.splits;
    r.blocks = static_cast<int32_t>(n);
    blocks += r.blocks;
    if (BWD && h->dgain) {
      r.part = part;
      part += int64_t(r.blocks) * d;
      join.part[i] = r.part, join.out[i] = h->dgain, join.blocks[i] = r.blocks;
      join.f32[i] = r.gain_f32;
    }
  }
  if (blocks > 0) {
    KernelTimer timer_(BWD ? "norm_rotary_bwd" : "norm_rotary_fwd", st);
    const int tile = a.r[0].tile_rows > a.r[1].tile_rows ? a.r[0].tile_rows : a.r[1].tile_rows;
    const size_t lds = size_t(tile) * (a.dim / 2) * sizeof(float2);
    const bool inter = rot && rot->interleaved;
    auto go = [&](auto bwd) {
      constexpr bool B = decltype(bwd)::value;
      if (dtype == NGT_F32) {
        if (v == 4) launch<float, 4, 1, B>(a, inter, blocks, lds, st);
        else if (v == 2) launch<float, 2, 1, B>(a, inter, blocks, lds, st);
        else launch<float, 1, 2, B>(a, inter, blocks, lds, st);
      } else {
        if (v == 8) launch<bf16_t, 8, 1, B>(a, inter, blocks, lds, st);
        else if (v == 4) launch<bf16_t, 4, 1, B>(a, inter, blocks, lds, st);
        else if (v == 2) launch<bf16_t, 2, 1, B>(a, inter, blocks, lds, st);
        else launch<bf16_t, 1, 2, B>(a, inter, blocks, lds, st);
      }
    };
    if (sums) go(std::true_type{});
    else go(std::false_type{});
    NGT_HIP_CHECK(hipGetLastError());
  }
  if (BWD && (join.out[0] || join.out[1])) {
    KernelTimer timer_("norm_rotary_gain", st);
    hipLaunchKernelGGL(k_join_gain, dim3((d + 31) / 32, 2), dim3(1024), 0, st, join);
    NGT_HIP_CHECK(hipGetLastError());
  }
  return NGT_OK;
}

}  // namespace
}  // namespace ngt

using namespace ngt;

extern "C" int ngt_norm_rotary_fwd(int dtype, const ngt_head_rows* q, const ngt_head_rows* k,
                                   int64_t n_rows, int32_t d, const ngt_rotation* rotation,
                                   float eps, void* stream) {
  const char* fn = "ngt_norm_rotary_fwd";
  NGT_CHECK_OK(check(fn, dtype, q, k, n_rows, d, rotation, eps, false));
  if (n_rows == 0) return NGT_OK;
  return run<false>(fn, dtype, q, k, n_rows, d, rotation, eps, nullptr,
                    static_cast<hipStream_t>(stream));
}

extern "C" int ngt_norm_rotary_bwd_workspace_bytes(int64_t n_rows, int32_t d, size_t* bytes) {
  const char* fn = "ngt_norm_rotary_bwd_workspace_bytes";
  if (n_rows < 0 || n_rows > kMaxRows || d < 2 || d > kMaxDim || !bytes)
    return set_error(NGT_ERR_ARG, "%s: n_rows=%lld head_dim=%d", fn,
                     static_cast<long long>(n_rows), d);
  *bytes = sums_bytes(d);
  return NGT_OK;
}

extern "C" int ngt_norm_rotary_bwd(int dtype, const ngt_head_rows* q, const ngt_head_rows* k,
                                   int64_t n_rows, int32_t d, const ngt_rotation* rotation,
                                   float eps, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* fn = "ngt_norm_rotary_bwd";
  NGT_CHECK_OK(check(fn, dtype, q, k, n_rows, d, rotation, eps, true));
  const bool sums = q->dgain || (k && k->dgain);
  if (sums && n_rows > 0 &&
      (!workspace || workspace_bytes < sums_bytes(d) ||
       reinterpret_cast<uintptr_t>(workspace) % 16))
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu or not 16-byte aligned", fn,
                     workspace_bytes, sums_bytes(d));
  return run<true>(fn, dtype, q, k, n_rows, d, rotation, eps, workspace,
                   static_cast<hipStream_t>(stream));
}
