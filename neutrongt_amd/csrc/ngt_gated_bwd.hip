// The gated linear layer's two backward products over aligned sizes, both on one block
// shape: 256 by 64 FN outputs, 4 waves of 4 x FN tiles of 32 x 32 (accumulators in
// AGPRs), one block on a CU, contracted in stages of 64.
//   dx = dzg Wg + dzu Wu         rows of dz by columns of Wg, then of Wu
//   dW = dz^T x                  columns of dz by columns of x
// Two stages fit in LDS: one is multiplied while the next comes in.  Where there are fewer
// blocks than CUs the contraction is split over several, whose fp32 sums are added in order
// (512 rows of 2,048 -> 8,192: dx 69 us, 220 without).
// 32,768 rows of 768 -> 2,048: dx 205 us, dW 195 to 203, 1,010 to 1,050 TFLOP/s (library products of
// these sizes 189 and 308); the products alone take 132 to 144 there, the loads alone 144 to 165.
// Stages of 32 in five buffers took as long.
#include "ngt_gated.h"

#include <algorithm>
#include <cmath>

namespace ngt {
namespace {

enum Mode { kDx, kDw };

struct BwdArgs {
  GatedBwd g;
  GatedShape shape;
  int32_t tiles_m, tiles_n;
};

template <int FN, Mode MODE>
__global__ __launch_bounds__(256, 1) void k_gated_bwd(BwdArgs args) {
  constexpr int FM = 4, BM = 64 * FM, BN = 64 * FN;
  using A = std::conditional_t<MODE == kDx, RowsOperand, ColsOperand>;  // as it lies in LDS
  using B = ColsOperand;
  constexpr int kABytes = BM * 128, kStageBytes = (BM + BN) * 128;
  __shared__ __align__(16) char s0[kStageBytes];
  __shared__ __align__(16) char s1[kStageBytes];
  const GatedBwd& g = args.g;
  const int lane = tid_x() & 63, wave = packed::wave_id(), half = lane >> 5;
  const TileAt at = tile_at(args.tiles_m, args.tiles_n, args.shape.splits);
  if (!at.there) return;  // block-uniform
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int wm = (wave >> 1) * FM, wn = (wave & 1) * FN;  // in 32s
  const DzBlocks blocks(g.M, g.N);
  const int64_t across = blocks.across() * 4096;  // bytes of a row of blocks
  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = fill16(0.f);

  BlockOperand oa;
  B ob;
  oa.init(), ob.init(g.K);
  // the contraction: twice N (a stage holds one layer's), or the rows; this split's part of it
  const int layer_stages = blocks.per_layer;
  const int all = MODE == kDx ? 2 * layer_stages : static_cast<int>((g.M + kStage - 1) / kStage);
  const int first = at.split * args.shape.per_split;
  const int end = min(first + args.shape.per_split, all), stages = end - first;
  const int cols_b = g.K - n0;
  struct Source {
    u32x4 a, b;
  };
  // of the split's stage i; behind its last one all is zero
  auto source = [&](int i) {
    Source f;
    const int s = first + i;
    const bool there = s < end;
    const char* dz = reinterpret_cast<const char*>(g.dz);
    if constexpr (MODE == kDx) {
      const int up = s >= layer_stages, k = (s - (up ? layer_stages : 0)) * kStage;
      const int64_t from = m0 / 32 * across + int64_t(s) * 4096;
      f.a = descriptor(dz + from, there ? blocks.bytes() - from : 0);
      f.b = ColsOperand::source((up ? g.wu : g.wg) + int64_t(k) * g.K + n0, there ? g.N - k : 0, g.K,
                                cols_b);
    } else {
      const int64_t r = int64_t(s) * kStage, from = r / 32 * across + m0 / 64 * 4096;
      f.a = descriptor(dz + from, there ? blocks.bytes() - from : 0);
      f.b = ColsOperand::source(g.x + r * g.K + n0, there ? g.M - r : 0, g.K, cols_b);
    }
    return f;
  };
  constexpr int kLoadsA = 2 * FM, kLoads = kLoadsA + 2 * FN;
  const int down = static_cast<int>(across);
  auto load = [&](const Source& f, int q, uint32_t to) {
    if (q >= kLoads) return;
    to += 4096 * q;
    if (q >= kLoadsA) ob.load(f.b, q - kLoadsA, cols_b, to);
    else oa.load(f.a, MODE == kDx ? q * down : q % 2 * down + q / 2 * 4096, to);
  };
  L::Op fa[4][FM], fb[4][FN];
  constexpr int kFrags = FM + FN;
  auto read = [&](const char* from, int c, int r) {  // fragment r of chunk c
    if (r < FN) fb[c][r] = B::frag(from + kABytes, wn + r, c, lane);
    else fa[c][r - FN] = A::frag(from, wm + r - FN, c, lane);
  };
  // Chunk c's products, and between them reads of chunk c + 3 (of the next stage but for
  // c = 0) and what `also` does, in the order written: the compiler would gather them.
  constexpr int kGroups = 8;
  auto phase = [&](const char* from, int c, auto also) {
#pragma unroll
    for (int t = 0; t < kGroups; ++t) {
#pragma unroll
      for (int r = t * kFrags / kGroups; r < (t + 1) * kFrags / kGroups; ++r) read(from, (c + 3) % 4, r);
      also(t);
#pragma unroll
      for (int e = t * FM * FN / kGroups; e < (t + 1) * FM * FN / kGroups; ++e)
        acc[e / FN][e % FN] = L::mma(fb[c][e % FN], fa[c][e / FN], acc[e / FN][e % FN]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto nothing = [](int) {};
  const uint32_t mine0 = lds_at(s0) + 1024 * wave, mine1 = lds_at(s1) + 1024 * wave;
  // Stage s, of which three chunks are in registers.  Once the fourth is, of all waves, its
  // buffer takes stage s + 2, in two phases: all 16 loads in one phase took 190 us for the
  // 32,768 x 4,096 x 768 of dz^T x, in two 180, in three 184.
  auto step = [&](int s, const char* cur, const char* next, uint32_t mine) {
    phase(cur, 0, nothing);
    all_read();
    all_there();
    meet();
    const Source f = source(s + 2);
    phase(next, 1, [&](int t) { load(f, t, mine); });
    phase(next, 2, [&](int t) { load(f, kGroups + t, mine); });
    phase(next, 3, nothing);
  };
  const Source f0 = source(0), f1 = source(1);
#pragma unroll
  for (int q = 0; q < kLoads; ++q) load(f0, q, mine0);
#pragma unroll
  for (int q = 0; q < kLoads; ++q) load(f1, q, mine1);
  all_there();
  meet();
#pragma unroll
  for (int r = 0; r < 3 * kFrags; ++r) read(s0, r / kFrags, r % kFrags);
  for (int s = 0; s < stages; s += 2) {  // (an odd number's last one is of zeros)
    step(s, s0, s1, mine0);
    step(s + 1, s1, s0, mine1);
  }
  all_there();  // nothing is on its way to LDS when the block ends
  // a lane has 16 consecutive outputs of row a_row(lane) of each tile
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + 32 * (wm + i) + L::a_row(lane & 31);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + 32 * (wn + j) + 16 * half;
      // 16 columns of row `row` of a matrix: of fp32 sums or of results in bf16
      auto put = [&](void* to, int64_t row, bool f32) {
        if (f32) {
          float* p = static_cast<float*>(to) + row * g.K + n;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + 4 * e < g.K)
              *reinterpret_cast<float4*>(p + 4 * e) =
                  make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2],
                              acc[i][j][4 * e + 3]);
        } else {
          uint16_t* p = static_cast<uint16_t*>(to) + row * g.K + n;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u32x4 y;
#pragma unroll
            for (int t = 0; t < 4; ++t)
              y[t] = pack2_bf16(acc[i][j][8 * e + 2 * t], acc[i][j][8 * e + 2 * t + 1]);
            if (n + 8 * e < g.K) *reinterpret_cast<u32x4*>(p + 8 * e) = y;
          }
        }
      };
      const bool parts = args.shape.splits > 1 || g.parts;
      if constexpr (MODE == kDx) {
        if (m < g.M) put(parts ? static_cast<void*>(g.part) : g.dx, parts ? at.split * g.M + m : m, parts);
      } else {
        // m counts dz's columns with what fills up each layer's
        const int layer = m >= 64 * blocks.per_layer;
        const int64_t o = m - layer * 64 * blocks.per_layer;
        if (m < 64 * blocks.across() && o < g.N) {
          if (parts) put(g.part, (2 * int64_t(at.split) + layer) * g.N + o, true);
          else if (g.dw[layer]) put(g.dw[layer], o, g.dw_f32[layer]);
        }
      }
    }
  }
}

template <int FN, Mode MODE>
int launch_one(const GatedBwd& g, const GatedShape& shape, hipStream_t st) {
  BwdArgs a{g, shape, 0, 0};
  const int64_t m = MODE == kDx ? g.M : 64 * DzBlocks(g.M, g.N).across();
  a.tiles_m = static_cast<int32_t>((m + 255) / 256);
  a.tiles_n = (g.K + 64 * FN - 1) / (64 * FN);
  const int64_t blocks = (int64_t(a.tiles_m) * a.tiles_n * shape.splits + 7) / 8 * 8;
  hipLaunchKernelGGL((k_gated_bwd<FN, MODE>), dim3(unsigned(blocks)), dim3(256), 0, st, a);
  NGT_HIP_CHECK(hipGetLastError());
  return NGT_OK;
}
template <Mode MODE>
int launch(const GatedBwd& g, const GatedShape& shape, hipStream_t st) {
  return shape.fn == 4   ? launch_one<4, MODE>(g, shape, st)
         : shape.fn == 3 ? launch_one<3, MODE>(g, shape, st)
                         : launch_one<2, MODE>(g, shape, st);
}

// The cheapest blocks for m by K outputs over `stages` of contraction.  A stage of a block with
// 64 fn columns takes about fn + 2 units of time, some 0.3 us each (32,768 rows, 4,096 x 768:
// dx 1.31, 1.6, 1.76 us at fn = 2, 3, 4, dw 1.12, 1.55, 1.85), a block beside its stages about
// as much as 4 of them, and each round of 256 blocks comes after the one before.  Each of
// several splits costs its sums, `bytes` written and read again at some 4 TB/s: per + 4 stages
// and those sums are least where the splits are the square root of their quotient.
GatedShape shape_of(int64_t m, int32_t K, int64_t stages, int64_t bytes) {
  GatedShape best{4, 1, static_cast<int32_t>(stages)};
  if (m == 0 || stages == 0) return best;  // nothing is launched
  double cost = 1e300;
  for (int fn = 4; fn >= 2; --fn) {
    const int64_t tiles = (m + 255) / 256 * ((K + 64 * fn - 1) / (64 * fn));
    const double stage = 0.3 * (fn + 2), sums = 5e-7 * double(bytes);
    const double alone = double((tiles + 255) / 256) * stage * double(stages + 4);
    if (alone < cost) cost = alone, best = {fn, 1, static_cast<int32_t>(stages)};
    const double want = std::sqrt(stage * double(stages) / sums);
    const int64_t most = std::min<int64_t>(256 / tiles, stages / 4);
    const int64_t splits = want < double(most) ? std::llround(want) : most;
    if (splits < 2) continue;
    const int64_t per = (stages + splits - 1) / splits, used = (stages + per - 1) / per;
    const double c = stage * double(per + 4) + 3.0 + sums * double(used);
    if (c < cost) cost = c, best = {fn, static_cast<int32_t>(used), static_cast<int32_t>(per)};
  }
  return best;
}

}  // namespace

GatedShape gated_dx_shape(int64_t M, int32_t N, int32_t K) {
  return shape_of(M, K, DzBlocks(M, N).across(), 4 * M * K);
}
GatedShape gated_dw_shape(int64_t M, int32_t N, int32_t K) {
  return shape_of(64 * DzBlocks(M, N).across(), K, (M + kStage - 1) / kStage, int64_t(8) * N * K);
}
int launch_gated_dx(const GatedBwd& g, const GatedShape& s, hipStream_t st) {
  return launch<kDx>(g, s, st);
}
int launch_gated_dw(const GatedBwd& g, const GatedShape& s, hipStream_t st) {
  return launch<kDw>(g, s, st);
}

}  // namespace ngt
