// The gated linear layer's two backward products over aligned sizes, both on one block
// shape: 256 by 64 FN outputs, 4 waves of 4 x FN tiles of 32 x 32 (accumulators in
// AGPRs), one block on a CU, contracted in stages of 64.
//   dx = dzg Wg + dzu Wu         rows of dz by columns of Wg, then of Wu
//   part[split] = dz^T x         columns of dz by columns of x, over the split's rows
// Two stages fit in LDS: one is multiplied while the next comes in.
#include "ngt_gated.h"

namespace ngt {
namespace {

enum Mode { kDx, kDw };

struct BwdArgs {
  GatedBwd g;
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
  const TileAt at = tile_at(args.tiles_m, args.tiles_n, MODE == kDw ? g.splits : 1);
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
  // the contraction: twice N (a stage holds one layer's), or the split's rows
  const int half_stages = blocks.per_layer;
  const int64_t row0 = MODE == kDw ? at.split * g.split_rows : 0;
  const int64_t rows = g.M - row0 < g.split_rows ? g.M - row0 : g.split_rows;
  const int stages = MODE == kDx ? 2 * half_stages : static_cast<int>((rows + kStage - 1) / kStage);
  const int cols_b = g.K - n0;
  struct Source {
    u32x4 a, b;
  };
  // of stage s; behind the last one all is zero
  auto source = [&](int s) {
    Source f;
    const char* dz = reinterpret_cast<const char*>(g.dz);
    if constexpr (MODE == kDx) {
      const int up = s >= half_stages, k = (s - (up ? half_stages : 0)) * kStage;
      const int64_t from = m0 / 32 * across + int64_t(s) * 4096;
      f.a = descriptor(dz + from, s < stages ? blocks.bytes() - from : 0);
      f.b = ColsOperand::source((up ? g.wu : g.wg) + int64_t(k) * g.K + n0, g.N - k, g.K, cols_b);
    } else {
      const int64_t r = row0 + int64_t(s) * kStage, left = rows - int64_t(s) * kStage;
      const int64_t from = r / 32 * across + m0 / 64 * 4096;
      f.a = descriptor(dz + from, left > 0 ? blocks.bytes() - from : 0);
      f.b = ColsOperand::source(g.x + r * g.K + n0, left, g.K, cols_b);
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
      if constexpr (MODE == kDx) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          u32x4 y;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            y[t] = pack2_bf16(acc[i][j][8 * e + 2 * t], acc[i][j][8 * e + 2 * t + 1]);
          if (m < g.M && n + 8 * e < g.K) *reinterpret_cast<u32x4*>(g.dx + m * g.K + n + 8 * e) = y;
        }
      } else {
        // m counts dz's columns with what fills up each layer's
        const int layer = m >= 64 * blocks.per_layer;
        const int64_t o = m - layer * 64 * blocks.per_layer;
        float* to = g.part + ((2 * int64_t(at.split) + layer) * g.N + o) * g.K + n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (layer * 64 * blocks.per_layer + o < blocks.across() * 64 && o < g.N && n + 4 * e < g.K)
            *reinterpret_cast<float4*>(to + 4 * e) =
                make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2],
                            acc[i][j][4 * e + 3]);
      }
    }
  }
}

template <int FN, Mode MODE>
int launch(const GatedBwd& g, hipStream_t st) {
  BwdArgs a{g, 0, 0};
  const int64_t m = MODE == kDx ? g.M : 64 * DzBlocks(g.M, g.N).across();
  a.tiles_m = static_cast<int32_t>((m + 255) / 256);
  a.tiles_n = (g.K + 64 * FN - 1) / (64 * FN);
  const int64_t blocks = int64_t(a.tiles_m) * a.tiles_n * (MODE == kDw ? g.splits : 1);
  hipLaunchKernelGGL((k_gated_bwd<FN, MODE>), dim3(unsigned((blocks + 7) / 8 * 8)), dim3(256), 0, st,
                     a);
  NGT_HIP_CHECK(hipGetLastError());
  return NGT_OK;
}

// The rounds that 256 CUs need for so many blocks.  A stage of a block with 64 fn columns takes
// about fn + 2 units of time (32,768 rows, 4,096 x 768: dx 1.31, 1.6, 1.76 us at fn = 2, 3, 4,
// dw 1.12, 1.55, 1.85).
int64_t rounds(int64_t blocks) { return (blocks + 255) / 256; }

}  // namespace

int launch_gated_dx(const GatedBwd& g, hipStream_t st) {
  int best = 4;
  int64_t cost = INT64_MAX;
  for (int fn = 4; fn >= 2; --fn) {
    const int64_t c = (fn + 2) * rounds((g.M + 255) / 256 * ((g.K + 64 * fn - 1) / (64 * fn)));
    if (c < cost) cost = c, best = fn;
  }
  return best == 4 ? launch<4, kDx>(g, st) : best == 3 ? launch<3, kDx>(g, st) : launch<2, kDx>(g, st);
}

GatedDwShape gated_dw_shape(int64_t M, int32_t N, int32_t K) {
  const int64_t stages = (M + kStage - 1) / kStage;
  GatedDwShape best{4, 1};
  int64_t cost = INT64_MAX;
  for (int fn = 4; fn >= 2; --fn) {
    const int64_t tiles = (DzBlocks(M, N).across() + 3) / 4 * ((K + 64 * fn - 1) / (64 * fn));
    // a split has 4 stages at least
    int64_t splits = 256 / tiles;
    if (splits > stages / 4) splits = stages / 4;
    if (splits < 1) splits = 1;
    const int64_t c = (fn + 2) * rounds(tiles * splits) * ((stages + splits - 1) / splits);
    if (c < cost) cost = c, best = {fn, static_cast<int>(splits)};
  }
  return best;
}

int launch_gated_dw(const GatedBwd& g, int fn, hipStream_t st) {
  return fn == 4 ? launch<4, kDw>(g, st) : fn == 3 ? launch<3, kDw>(g, st) : launch<2, kDw>(g, st);
}

}  // namespace ngt
