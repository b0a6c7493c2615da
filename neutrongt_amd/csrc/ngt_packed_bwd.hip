// Attention over packed windows: the backward.
#include "ngt_packed.h"

namespace ngt {
namespace packed {
namespace {

constexpr int kRows = 64;  // rows of one stage

// dQ, D = G . out and the bias's gradient.  One block: NW * 32 query rows of
// one window and head, a wave 32 of them (lane = query); the window's keys pass
// through LDS 64 at a time.
//   S^T = K Q^T, dP^T = V G^T, P = exp2(S - lse), dS = P (dP - D), dQ^T += K^T dS^T
// HIST: the wave keeps 64 running sums per bucket, one a lane, so that every
// sum has a fixed order; the block adds them up at its end.
template <typename T, int DP, bool BIAS, bool HIST, int NW>
__global__ __launch_bounds__(64 * NW) void k_packed_dq(BwdArgs a) {
  using L = Tile<T, DP>;
  constexpr int N = 64 * NW;
  constexpr bool kAhead = (kRows * L::kPieces / N) * 8 <= 32;
  __shared__ __align__(16) char ks[kRows * L::kPitch];
  __shared__ __align__(16) char vs[kRows * L::kPitch];
  __shared__ float tab[BIAS ? kTable : 1];
  extern __shared__ float hist[];  // HIST: [NW][n_buckets + 1][64]
  const int tid = tid_x(), lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  const int bid = wg_x();
  const int kvh = bid % a.Hkv, grp = (bid / a.Hkv) % (a.H / a.Hkv);
  const int h = kvh * (a.H / a.Hkv) + grp;
  const int it = bid / a.H;
  const int2 item = a.items[it];
  const int64_t q0 = a.q_start[item.x], k0 = a.k_start[item.x];
  const int nq = static_cast<int>(a.q_start[item.x + 1] - q0);
  const int nk = static_cast<int>(a.k_start[item.x + 1] - k0);
  const int ahead = nk - nq;
  const int qi = item.y + wave * 32 + l32;
  const int qc = min(qi, nq - 1);
  const int lim = a.causal ? min(qc + ahead, nk - 1) : nk - 1;
  const int first_lim = a.causal ? min(item.y + wave * 32 + ahead, nk - 1) : nk - 1;
  const int last_q = min(item.y + wave * 32 + 31, nq - 1);
  const int wave_end = item.y + wave * 32 >= nq ? 0 : a.causal ? min(last_q + ahead + 1, nk) : nk;
  const int block_end = a.causal ? min(min(item.y + 32 * NW, nq) + ahead, nk) : nk;
  const T* kb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.k) + k0 * a.sk) +
                int64_t(kvh) * a.d;
  const T* vb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.v) + k0 * a.sv) +
                int64_t(kvh) * a.d;
  const int64_t row = ((q0 + qc) * a.H + h) * int64_t(a.d);
  RowFrag<T, DP> q, g;
  q.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.q) + (q0 + qc) * a.sq) +
             int64_t(h) * a.d,
         qi < nq, a.d, half);
  g.load(reinterpret_cast<const T*>(a.go) + row, qi < nq, a.d, half);
  // D: this half's chunks of the row, then both halves
  float D = 0.f;
#pragma unroll
  for (int c = 0; c < L::kChunks; ++c) {
    constexpr int kE = 16 / L::kEs;  // elements of a lane's 16 bytes
    const int at = (2 * c + half) * kE;
    if (at < a.d) {
#pragma unroll
      for (int e = 0; e < kE; e += 4) {
        const float4 o = *reinterpret_cast<const float4*>(a.out32 + row + at + e);
        float x[4];
        if constexpr (L::kEs == 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(g.w[c][i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = g.w[c][(e + i) / 2];
            x[i] = __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
          }
        }
        D = fmaf(x[0], o.x, fmaf(x[1], o.y, fmaf(x[2], o.z, fmaf(x[3], o.w, D))));
      }
    }
  }
  D = sum_halves(D);
  // a lane without a row has no weight anywhere
  const float lse = qi < nq ? a.lse[int64_t(h) * a.n_q + q0 + qi] : INFINITY;
  if (qi < nq && half == 0) a.dsum[int64_t(h) * a.n_q + q0 + qi] = D;

  const uint8_t* ids = nullptr;
  float* my_hist = nullptr;
  if constexpr (BIAS) {
    load_table(tab, reinterpret_cast<const T*>(a.table), a.n_buckets, a.H, h, tid, N);
    ids = a.ids + a.b_start[item.x] + int64_t(qc) * ((nk + 63) & ~63) + 16 * half;
  }
  if constexpr (HIST) {
    for (int i = tid; i < NW * (a.n_buckets + 1) * 64; i += N) hist[i] = 0.f;
    my_hist = hist + wave * (a.n_buckets + 1) * 64 + lane;
  }
  const float s2 = a.scale * kLog2e;
  f32x16 acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = fill16(0.f);

  Stage<T, DP, kRows, N> pk, pv;
  u32x4 idw[2];
  if constexpr (kAhead) {
    pk.load(kb, a.sk, 0, nk, a.d, tid);
    pv.load(vb, a.sv, 0, nk, a.d, tid);
  }
  for (int kt = 0; kt < block_end; kt += kRows) {
    if constexpr (BIAS) {
#pragma unroll
      for (int t = 0; t < 2; ++t) idw[t] = *reinterpret_cast<const u32x4*>(ids + kt + 32 * t);
    }
    __syncthreads();
    if constexpr (!kAhead) {
      pk.load(kb, a.sk, kt, nk, a.d, tid);
      pk.store(ks, tid);
      pv.load(vb, a.sv, kt, nk, a.d, tid);
      pv.store(vs, tid);
    } else {
      pk.store(ks, tid);
      pv.store(vs, tid);
    }
    __syncthreads();
    if constexpr (kAhead) {
      if (kt + kRows < block_end) {
        pk.load(kb, a.sk, kt + kRows, nk, a.d, tid);
        pv.load(vb, a.sv, kt + kRows, nk, a.d, tid);
      }
    }
    if (kt >= wave_end) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t == 1 && kt + 32 >= wave_end) break;
      f32x16 s = fill16(0.f), dp = fill16(-D);
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) {
        s = mma_rows<T>(L::load_a(ks, t, c, l32, half), q.w[c], s);
        dp = mma_rows<T>(L::load_a(vs, t, c, l32, half), g.w[c], dp);
      }
      const bool cut = kt + 32 * t + 31 > first_lim;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x;
        if constexpr (BIAS)
          x = fmaf(s[i], s2, tab[bucket_of(idw[t], i)]) - lse;
        else
          x = fmaf(s[i], s2, -lse);
        if (cut && kt + 32 * t + 16 * half + i > lim) x = -INFINITY;
        s[i] = __builtin_amdgcn_exp2f(x) * dp[i];
      }
      if constexpr (HIST) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int b = min(bucket_of(idw[t], i), a.n_buckets);
          atomicAdd(my_hist + b * 64, s[i]);  // the lane's own word: no other writes it
        }
      }
      L::mma_cols(ks, t, s, acc, lane);
    }
  }
  if (qi < nq) {
    T* o = reinterpret_cast<T*>(a.gq) + ((q0 + qi) * a.H + h) * int64_t(a.d);
#pragma unroll
    for (int c = 0; c < L::kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 32 * c + 8 * i + 4 * half;
        if (at < a.d)
          store4(o + at, acc[c][4 * i] * a.scale, acc[c][4 * i + 1] * a.scale,
                 acc[c][4 * i + 2] * a.scale, acc[c][4 * i + 3] * a.scale);
      }
  }
  if constexpr (HIST) {
    __syncthreads();
    for (int b = tid; b < a.n_buckets; b += N) {
      float sum = 0.f;
      for (int w = 0; w < NW; ++w) {
        const float* hw = hist + (w * (a.n_buckets + 1) + b) * 64;
        float s = 0.f;
        for (int i = 0; i < 64; ++i) s += hw[(i + b) & 63];  // from its own place: no bank twice
        sum += s;
      }
      a.part_table[(int64_t(h) * a.n_items + it) * a.n_buckets + b] = sum;
    }
  }
}

// dK and dV.  One block: NW * 32 keys of one window and key head, a wave 32 of
// them (lane = key); the rows of the group's heads that see them pass through
// LDS 64 at a time, head after head: dK and dV of shared heads are one sum.
//   S = Q K^T, dP = G V^T, P = exp2(S - lse), dS = P (dP - D)
//   dV^T += G^T P, dK^T += Q^T dS
template <typename T, int DP, bool BIAS, int NW>
__global__ __launch_bounds__(64 * NW) void k_packed_dkv(BwdArgs a) {
  using L = Tile<T, DP>;
  constexpr int N = 64 * NW;
  constexpr bool kAhead = (kRows * L::kPieces / N) * 8 <= 32;
  __shared__ __align__(16) char qs[kRows * L::kPitch];
  __shared__ __align__(16) char gs[kRows * L::kPitch];
  __shared__ __align__(16) float ls[kRows], ds[kRows];
  __shared__ float tab[BIAS ? kTable : 1];
  const int tid = tid_x(), lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  const int kvh = wg_x() % a.Hkv;
  const int2 item = a.items[wg_x() / a.Hkv];
  const int G = a.H / a.Hkv;
  const int64_t q0 = a.q_start[item.x], k0 = a.k_start[item.x];
  const int nq = static_cast<int>(a.q_start[item.x + 1] - q0);
  const int nk = static_cast<int>(a.k_start[item.x + 1] - k0);
  const int ahead = nk - nq;
  const int kj = item.y + wave * 32 + l32;
  const int kc = min(kj, nk - 1);
  // the first query that sees this key, the block's first key, the wave's last one
  const int lim = a.causal ? kc - ahead : 0;
  const int block_begin = a.causal ? max(0, item.y - ahead) & ~(kRows - 1) : 0;
  const int wave_begin = a.causal ? max(0, item.y + wave * 32 - ahead) : 0;
  const int last_lim = a.causal ? item.y + wave * 32 + 31 - ahead : 0;
  RowFrag<T, DP> k, v;
  k.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.k) + (k0 + kc) * a.sk) +
             int64_t(kvh) * a.d,
         kj < nk, a.d, half);
  v.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.v) + (k0 + kc) * a.sv) +
             int64_t(kvh) * a.d,
         kj < nk, a.d, half);
  const uint8_t* ids = nullptr;
  if constexpr (BIAS)
    ids = a.ids_t + a.bt_start[item.x] + int64_t(kc) * ((nq + 63) & ~63) + 16 * half;
  const float s2 = a.scale * kLog2e;
  f32x16 ak[L::kCols], av[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) ak[c] = fill16(0.f), av[c] = fill16(0.f);

  Stage<T, DP, kRows, N> pq, pg;
  float pl = 0.f, pd = 0.f;
  for (int grp = 0; grp < G; ++grp) {
    const int h = kvh * G + grp;
    const T* qb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.q) + q0 * a.sq) +
                  int64_t(h) * a.d;
    const T* gb = reinterpret_cast<const T*>(a.go) + (q0 * a.H + h) * int64_t(a.d);
    const int64_t sg = int64_t(a.H) * a.d * L::kEs;
    const float* lse = a.lse + int64_t(h) * a.n_q + q0;
    const float* dsum = a.dsum + int64_t(h) * a.n_q + q0;
    auto fetch = [&](int qt) {
      if (tid < kRows) {  // a row that is not there has no weight
        pl = qt + tid < nq ? lse[qt + tid] : INFINITY;
        pd = qt + tid < nq ? dsum[qt + tid] : 0.f;
      }
      if constexpr (kAhead) {
        pq.load(qb, a.sq, qt, nq, a.d, tid);
        pg.load(gb, sg, qt, nq, a.d, tid);
      }
    };
    if constexpr (BIAS) {
      __syncthreads();  // the last head's rows are done with its table
      load_table(tab, reinterpret_cast<const T*>(a.table), a.n_buckets, a.H, h, tid, N);
    }
    fetch(block_begin);
    for (int qt = block_begin; qt < nq; qt += kRows) {
      u32x4 idw[2];
      if constexpr (BIAS) {
#pragma unroll
        for (int t = 0; t < 2; ++t) idw[t] = *reinterpret_cast<const u32x4*>(ids + qt + 32 * t);
      }
      __syncthreads();
      if constexpr (!kAhead) {
        pq.load(qb, a.sq, qt, nq, a.d, tid);
        pq.store(qs, tid);
        pg.load(gb, sg, qt, nq, a.d, tid);
        pg.store(gs, tid);
      } else {
        pq.store(qs, tid);
        pg.store(gs, tid);
      }
      if (tid < kRows) ls[tid] = pl, ds[tid] = pd;
      __syncthreads();
      if (qt + kRows < nq) fetch(qt + kRows);
      if (qt + kRows <= wave_begin || item.y + wave * 32 >= nk) continue;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 s = fill16(0.f), dp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 y = *reinterpret_cast<const float4*>(ds + 32 * t + 16 * half + 4 * i);
          dp[4 * i] = -y.x, dp[4 * i + 1] = -y.y, dp[4 * i + 2] = -y.z, dp[4 * i + 3] = -y.w;
        }
#pragma unroll
        for (int c = 0; c < L::kChunks; ++c) {
          s = mma_rows<T>(L::load_a(qs, t, c, l32, half), k.w[c], s);
          dp = mma_rows<T>(L::load_a(gs, t, c, l32, half), v.w[c], dp);
        }
        const bool cut = qt + 32 * t < last_lim;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const float4 y = *reinterpret_cast<const float4*>(ls + 32 * t + 16 * half + 4 * i4);
          const float lv[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * i4 + j;
            float x;
            if constexpr (BIAS)
              x = fmaf(s[i], s2, tab[bucket_of(idw[t], i)]) - lv[j];
            else
              x = fmaf(s[i], s2, -lv[j]);
            if (cut && qt + 32 * t + 16 * half + i < lim) x = -INFINITY;
            s[i] = __builtin_amdgcn_exp2f(x);
            dp[i] *= s[i];
          }
        }
        L::mma_cols(gs, t, s, av, lane);
        L::mma_cols(qs, t, dp, ak, lane);
      }
    }
  }
  if (kj < nk) {
    const int64_t row = ((k0 + kj) * a.Hkv + kvh) * int64_t(a.d);
    T* ok = reinterpret_cast<T*>(a.gk) + row;
    T* ov = reinterpret_cast<T*>(a.gv) + row;
#pragma unroll
    for (int c = 0; c < L::kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 32 * c + 8 * i + 4 * half;
        if (at < a.d) {
          store4(ok + at, ak[c][4 * i] * a.scale, ak[c][4 * i + 1] * a.scale,
                 ak[c][4 * i + 2] * a.scale, ak[c][4 * i + 3] * a.scale);
          store4(ov + at, av[c][4 * i], av[c][4 * i + 1], av[c][4 * i + 2], av[c][4 * i + 3]);
        }
      }
  }
}

// dTable[b, h]: the work items' sums in a fixed order: 16 waves take every
// 16th item (lane = bucket), their sums are added in wave order.
template <typename T>
__global__ __launch_bounds__(1024) void k_packed_table_grad(const float* __restrict__ part,
                                                            int n_items, int n_buckets, int H,
                                                            T* __restrict__ grad) {
  __shared__ float red[16][64];
  const int tid = tid_x(), lane = tid & 63, w = tid >> 6;
  const int h = wg_x() % H, b = (wg_x() / H) * 64 + lane;
  float s = 0.f;
  if (b < n_buckets) {
#pragma unroll 4
    for (int i = w; i < n_items; i += 16) s += part[(int64_t(h) * n_items + i) * n_buckets + b];
  }
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && b < n_buckets) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    elem<T>::store(grad + int64_t(b) * H + h, s);
  }
}

template <typename T, int DP, bool BIAS, bool HIST>
int launch_dq(const BwdArgs& a, int nw, int64_t blocks, size_t lds, hipStream_t st) {
  KernelTimer timer_("packed_dq", st);
  auto run = [&](auto kernel) {
    if (lds)
      NGT_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(64 * nw), lds, st, a);
    NGT_HIP_CHECK(hipGetLastError());
    return int(NGT_OK);
  };
  if (nw == 4) return run(k_packed_dq<T, DP, BIAS, HIST, 4>);
  if (nw == 2) return run(k_packed_dq<T, DP, BIAS, HIST, 2>);
  return run(k_packed_dq<T, DP, BIAS, HIST, 1>);
}

template <typename T, int DP>
int bwd(const BwdPlan& p, const BwdArgs& base, hipStream_t st) {
  const bool bias = base.table != nullptr, hist = bias && base.grad_table;
  BwdArgs a = base;
  if (p.dq_blocks > 0) {
    a.items = p.items_q;
    a.n_items = p.n_items_q;
    const size_t lds = hist ? size_t(p.dq_waves) * (a.n_buckets + 1) * 256 : 0;
    NGT_CHECK_OK(hist   ? (launch_dq<T, DP, true, true>(a, p.dq_waves, p.dq_blocks, lds, st))
                 : bias ? (launch_dq<T, DP, true, false>(a, p.dq_waves, p.dq_blocks, 0, st))
                        : (launch_dq<T, DP, false, false>(a, p.dq_waves, p.dq_blocks, 0, st)));
  }
  if (p.dkv_blocks > 0) {
    KernelTimer timer_("packed_dkv", st);
    a.items = p.items_k;
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(unsigned(p.dkv_blocks)), dim3(64 * p.dkv_waves), 0, st, a);
    };
    if (bias) {
      if (p.dkv_waves == 4) run(k_packed_dkv<T, DP, true, 4>);
      else if (p.dkv_waves == 2) run(k_packed_dkv<T, DP, true, 2>);
      else run(k_packed_dkv<T, DP, true, 1>);
    } else {
      if (p.dkv_waves == 4) run(k_packed_dkv<T, DP, false, 4>);
      else if (p.dkv_waves == 2) run(k_packed_dkv<T, DP, false, 2>);
      else run(k_packed_dkv<T, DP, false, 1>);
    }
    NGT_HIP_CHECK(hipGetLastError());
  }
  if (hist) {
    KernelTimer timer_("packed_table_grad", st);
    hipLaunchKernelGGL(k_packed_table_grad<T>, dim3(unsigned(a.H * ((a.n_buckets + 63) / 64))),
                       dim3(1024), 0, st, a.part_table, p.dq_blocks > 0 ? p.n_items_q : 0,
                       a.n_buckets, a.H, static_cast<T*>(a.grad_table));
    NGT_HIP_CHECK(hipGetLastError());
  }
  return NGT_OK;
}

}  // namespace

int packed_bwd(int dtype, const BwdPlan& p, const BwdArgs& a, hipStream_t st) {
  const int dp = a.d <= 32 ? 32 : a.d <= 64 ? 64 : 128;
  if (dtype == NGT_F32)
    return dp == 32 ? bwd<float, 32>(p, a, st) : dp == 64 ? bwd<float, 64>(p, a, st)
                                                          : bwd<float, 128>(p, a, st);
  return dp == 32 ? bwd<bf16_t, 32>(p, a, st) : dp == 64 ? bwd<bf16_t, 64>(p, a, st)
                                                         : bwd<bf16_t, 128>(p, a, st);
}

}  // namespace packed
}  // namespace ngt
