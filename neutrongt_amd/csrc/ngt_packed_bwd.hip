// Attention over packed windows: the backward, from the rows' lse and the fp32 output.
//   P = e^(S - lse), D = g.out, dS = P (g V^T - D)
//   dQ = scale dS K, dK = scale dS^T Q, dV = P^T g, dTable[b, h] = sum of dS where id = b
// Two passes, one by queries (dQ, D, the table) and one by keys (dK, dV), so that every
// sum has one owner and one order; the scores are formed in both (14 d flops a pair
// instead of 10 d) and the exponential with them, which costs less than sums over blocks
// through memory would.  In bf16 P and dS are rounded to bf16 for their products, a half
// step of each term (dQ, dK and dV are then off by 1.38 to 1.44 times the rounding of the
// result; what two pieces cost stands in ngt_packed.hip); everything else is fp32.
// What bounds them: vector instructions a pair as in the forward (8 heads of 8, 24
// windows of 100 to 1,500: dQ 41, dK/dV 37 us).  At d = 64 causal no unit is busy for more
// than 34 % of the time in dQ (101 us) or 30 % in dK/dV (149 us): waits, of dK/dV's four sets
// before the diagonal for one another and of blocks of 66 KB for a place.  With the bias's
// gradient dQ is bound by LDS, a table entry and an addition of a double per pair, busy for
// 69 % of the time (3 windows of 1,000 to 3,333, 32 heads of 24: 408 us, dK/dV 345).
#include "ngt_packed.h"

namespace ngt {
namespace packed {
namespace {

// Adds a lane's 16 values to the wave's running sums of their buckets, in the
// lane's column: hist[bucket][l mod columns], doubles.  LDS adds a double in 9 clocks
// a wave instruction where a float takes 193 (3 a lane); reading, adding and
// writing back takes 10 and seven compares and selects a value.  The lanes of an
// instruction that meet in one sum are always the same ones, added in lane order.
__device__ __forceinline__ void add_to_buckets(double* hist, const u32x4& ids, const f32x16& x,
                                               int n_buckets, int shift) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    unsafeAtomicAdd(hist + (min(bucket_of(ids, i), n_buckets) << shift),
                    static_cast<double>(x[i]));
}

// dQ, D = G . out and the bias's gradient.  One block: RW * 32 query rows of
// one window and head (lane = query); the window's keys pass through LDS
// 64 * KS at a time.
//   S^T = K Q^T, dP^T = V G^T, P = exp2(S - lse), dS = P (dP - D), dQ^T += K^T dS^T
// HIST: the wave keeps 8 or 16 running sums per bucket (hist_shift), each of the same
// rows' pairs in the same order; the block adds them up at its end.
template <typename T, int DP, bool BIAS, bool HIST, int RW, int KS>
__global__ __launch_bounds__(64 * RW * KS) void k_packed_dq(BwdArgs a) {
  using L = Tile<T, DP>;
  using B = Block<RW, KS>;
  constexpr int N = B::kThreads, kRows = B::kStage;
  constexpr int kTileBytes = kRows * L::kRow;
  constexpr bool kAhead = (kRows * L::kMemPieces / N) * 8 <= 32;
  __shared__ __align__(16) char
      buf[2 * kTileBytes > B::kJoinBytes ? 2 * kTileBytes : B::kJoinBytes];
  __shared__ float tab[BIAS ? kTable : 1];
  extern __shared__ __align__(8) double hist[];  // HIST: [RW * KS][n_buckets + 1][columns]
  char *const ks = buf, *const vs = buf + kTileBytes;
  const int tid = tid_x(), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int wid = wave_id(), wave = wid % RW, set = wid / RW;
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
  const int block_end = a.causal ? min(min(item.y + 32 * RW, nq) + ahead, nk) : nk;
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
  // D: every other 4 elements of the row, then both halves
  float D = 0.f;
  if (qi < nq) {
    const T* gr = reinterpret_cast<const T*>(a.go) + row;
    for (int at = 4 * half; at < a.d; at += 8) {
      const float4 o = *reinterpret_cast<const float4*>(a.out32 + row + at);
      const float4 x = load4(gr + at);
      D = fmaf(x.x, o.x, fmaf(x.y, o.y, fmaf(x.z, o.z, fmaf(x.w, o.w, D))));
    }
  }
  D = sum_halves(D);
  // a lane without a row has no weight anywhere
  float lse = qi < nq ? a.lse[int64_t(h) * a.n_q + q0 + qi] : INFINITY;
  float far = 0.f, far_log = 0.f;  // of a row beyond kFar, whose lse is then 0 here
  if constexpr (BIAS) {
    if (is_far(lse)) {
      far = lse, lse = 0.f;
      far_log = a.lse[int64_t(a.H + h) * a.n_q + q0 + qi];
    }
  }
  const bool any_far = BIAS && __any(far != 0.f);
  if (qi < nq && half == 0 && set == 0) a.dsum[int64_t(h) * a.n_q + q0 + qi] = -D;

  const int ld = (nk + 63) & ~63;
  const uint8_t* ids = nullptr;  // of the block's first query
  double* my_hist = nullptr;
  const int cols = (1 << a.hist_shift) - 1;
  if constexpr (BIAS) {
    load_table<T>(tab, a.table, a.table_f32, a.n_buckets, a.H, h, tid, N);
    ids = a.ids + a.b_start[item.x] + int64_t(item.y) * ld;
  }
  if constexpr (HIST) {
    for (int i = tid; i < RW * KS * (a.n_buckets + 1) << a.hist_shift; i += N) hist[i] = 0.;
    my_hist = hist + (wid * (a.n_buckets + 1) << a.hist_shift) + (l32 & cols);
  }
  const float s2 = a.scale * kLog2e;
  // The bf16 matrix instructions round their sums down, a row's dP - D by some 2^-25 of
  // its terms; the bias's gradient adds up millions of them, so in fp32 odd rows take
  // everything with the other sign there, and what was rounded down cancels (fp32, 3,001
  // rows, 40 buckets: the gradient's error 2.8e-6 -> 4.3e-7 of its norm, no time).
  constexpr bool kTurn = HIST && sizeof(T) == 4;
  const float sign = kTurn && (l32 & 1) ? -1.f : 1.f;
  if constexpr (kTurn) g.negate(l32 & 1), D *= sign;
  // bf16 with a bias: the products start from -lse, in their units, and -D; in fp32
  // -lse would cost them bits there
  constexpr bool kFromLse = BIAS && sizeof(T) == 2;
  const f32x16 s_start = fill16(kFromLse ? -lse / s2 : 0.f), dp_start = fill16(-D);
  f32x16 acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = fill16(0.f);

  Stage<T, DP, kRows, N> pk(a.sk, a.d, tid), pv(a.sv, a.d, tid);
  u32x4 idw[2], id_next[2];
  const Buffer id_buf = make_buffer(ids, int64_t(min(32 * RW, nq - item.y)) * ld);
  const int id_at = (qc - item.y) * ld + 16 * half;
  auto fetch_ids = [&](int k1) {
    if constexpr (BIAS) {
#pragma unroll
      for (int t = 0; t < 2; ++t) id_next[t] = read16(id_buf, id_at + k1 + 32 * t);
    }
  };
  fetch_ids(64 * set);
  if constexpr (kAhead) {
    pk.load(kb, a.sk, 0, nk, a.d);
    pv.load(vb, a.sv, 0, nk, a.d);
  }
  const char* k_tile = ks + 64 * set * L::kRow;
  const char* v_tile = vs + 64 * set * L::kRow;
  for (int kt = 0; kt < block_end; kt += kRows) {
    __syncthreads();
    if constexpr (!kAhead) {
      pk.load(kb, a.sk, kt, nk, a.d);
      pk.store(ks, tid);
      pv.load(vb, a.sv, kt, nk, a.d);
      pv.store(vs, tid);
    } else {
      pk.store(ks, tid);
      pv.store(vs, tid);
    }
    __syncthreads();
    idw[0] = id_next[0], idw[1] = id_next[1];
    fetch_ids(kt + kRows + 64 * set);
    if constexpr (kAhead) {
      if (kt + kRows < block_end) {
        pk.load(kb, a.sk, kt + kRows, nk, a.d);
        pv.load(vb, a.sv, kt + kRows, nk, a.d);
      }
    }
    const int k1 = kt + 64 * set;  // this set's first key
    if (k1 >= wave_end) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t == 1 && k1 + 32 >= wave_end) break;
      f32x16 bias;
      if constexpr (BIAS) bias = look_up(tab, idw[t]);
      f32x16 s = s_start, dp = dp_start;
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) {
        s = L::mma(L::load_a(k_tile, t, c, l32, half), q.w[c], s);
        dp = L::mma(L::load_a(v_tile, t, c, l32, half), g.w[c], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = fmaf(s[i], s2, kFromLse ? bias[i] : BIAS ? bias[i] - lse : -lse);
      if (any_far) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (s[i] - far) - far_log;
      }
      if (k1 + 32 * t + 31 > first_lim) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k1 + 32 * t + 16 * half + i > lim) s[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]) * dp[i];
      if constexpr (HIST) add_to_buckets(my_hist, idw[t], s, a.n_buckets, a.hist_shift);
      // a row's dS add up to zero, so what its keys have in common cancels, and in heads
      // of up to 16 that is much of them: there dS goes in as two bf16 pieces (8 heads of
      // 8, 1,500 rows: dQ's error 1.6 -> 1.07 times that of rounding the result; 35 -> 45 us)
      L::template mma_cols<DP == 16>(k_tile, t, s, acc, lane);
    }
  }
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) join_sets<RW, KS>(acc[c], buf, wave, set, lane);
  if (qi < nq && set == 0) {
    const float by = sign * a.scale;
    T* o = reinterpret_cast<T*>(a.gq) + ((q0 + qi) * a.H + h) * int64_t(a.d);
#pragma unroll
    for (int c = 0; c < L::kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 32 * c + 8 * i + 4 * half;
        if (at < a.d)
          store4(o + at, acc[c][4 * i] * by, acc[c][4 * i + 1] * by, acc[c][4 * i + 2] * by,
                 acc[c][4 * i + 3] * by);
      }
  }
  if constexpr (HIST) {
    __syncthreads();
    for (int b = tid; b < a.n_buckets; b += N) {
      double sum = 0.;
      for (int w = 0; w < RW * KS; ++w) {
        const double* hw = hist + (w * (a.n_buckets + 1) + b << a.hist_shift);
        // from its own place: no bank twice; odd rows with their sign
        for (int i = 0; i <= cols; ++i)
          sum += kTurn && ((i + b) & 1) ? -hw[(i + b) & cols] : hw[(i + b) & cols];
      }
      a.part_table[(int64_t(h) * a.n_items + it) * a.n_buckets + b] = static_cast<float>(sum);
    }
  }
}

// dK and dV.  One block: RW * 32 keys of one window and key head (lane = key);
// the rows of the group's heads that see them pass through LDS 64 * KS at a
// time, head after head: dK and dV of shared heads are one sum.
//   S = Q K^T, dP = G V^T, P = exp2(S - lse), dS = P (dP - D)
//   dV^T += G^T P, dK^T += Q^T dS
// With a bias, whose table lookups it waits for, three waves a SIMD in the one shape whose
// registers allow it, four row waves in bf16 at 32: 32 heads of 24, 8,556 rows, 379 -> 343 us
// (without a bias 42 -> 45).  Held to three, the other shapes there spill 6 to 50 registers
// (300 windows of 8 to 32, 8 heads of 24: 20 us, 14 without the bound).
template <typename T, int DP, bool BIAS, int RW, int KS>
__global__ __launch_bounds__(64 * RW * KS,
                             BIAS && DP == 32 && sizeof(T) == 2 && RW == 4 && KS == 1 ? 3 : 1) void
k_packed_dkv(BwdArgs a) {
  using L = Tile<T, DP>;
  using B = Block<RW, KS>;
  constexpr int N = B::kThreads, kRows = B::kStage;
  constexpr int kTileBytes = kRows * L::kRow;
  constexpr bool kAhead = (kRows * L::kMemPieces / N) * 8 <= 32;
  __shared__ __align__(16) char
      buf[2 * kTileBytes > B::kJoinBytes ? 2 * kTileBytes : B::kJoinBytes];
  __shared__ __align__(16) float ls[kRows], ds[kRows];
  __shared__ float far[BIAS ? kRows : 1][2];  // of rows beyond kFar, whose ls is then 0
  __shared__ float tab[BIAS ? kTable : 1];
  char *const qs = buf, *const gs = buf + kTileBytes;
  const int tid = tid_x(), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int wid = wave_id(), wave = wid % RW, set = wid / RW;
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
  const int block_begin = a.causal ? max(0, item.y - ahead) & ~63 : 0;
  const int wave_begin = a.causal ? max(0, item.y + wave * 32 - ahead) : 0;
  const int last_lim = a.causal ? item.y + wave * 32 + 31 - ahead : 0;
  RowFrag<T, DP> k, v;
  k.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.k) + (k0 + kc) * a.sk) +
             int64_t(kvh) * a.d,
         kj < nk, a.d, half);
  v.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.v) + (k0 + kc) * a.sv) +
             int64_t(kvh) * a.d,
         kj < nk, a.d, half);
  const int ld = (nq + 63) & ~63;
  const uint8_t* ids = nullptr;  // of the block's first key
  if constexpr (BIAS) ids = a.ids_t + a.bt_start[item.x] + int64_t(item.y) * ld;
  const Buffer id_buf = make_buffer(ids, int64_t(min(32 * RW, nk - item.y)) * ld);
  const int id_at = (kc - item.y) * ld + 16 * half;
  const float s2 = a.scale * kLog2e;
  f32x16 ak[L::kCols], av[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) ak[c] = fill16(0.f), av[c] = fill16(0.f);

  const int64_t sg = int64_t(a.H) * a.d * L::kEs;
  Stage<T, DP, kRows, N> pq(a.sq, a.d, tid), pg(sg, a.d, tid);
  // bf16: the products start from -lse, in their units; in fp32 that would cost them
  // bits (9 windows of 33 to 1,777, heads of 16: dK's error 7.4e-7 -> 4.4e-7 of its norm)
  constexpr bool kFromLse = sizeof(T) == 2;
  const float lse_per = kFromLse ? -1.f / s2 : -1.f;
  float pl = 0.f, pl_log = 0.f, pd = 0.f;
  u32x4 idw[2], id_next[2];
  const char* q_tile = qs + 64 * set * L::kRow;
  const char* g_tile = gs + 64 * set * L::kRow;
  for (int grp = 0; grp < G; ++grp) {
    const int h = kvh * G + grp;
    const T* qb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.q) + q0 * a.sq) +
                  int64_t(h) * a.d;
    const T* gb = reinterpret_cast<const T*>(a.go) + (q0 * a.H + h) * int64_t(a.d);
    const Buffer lse = make_buffer(a.lse + int64_t(h) * a.n_q + q0, int64_t(nq) * 4);
    const Buffer lse_log = make_buffer(a.lse + int64_t(a.H + h) * a.n_q + q0,
                                       BIAS ? int64_t(nq) * 4 : 0);
    const Buffer dsum = make_buffer(a.dsum + int64_t(h) * a.n_q + q0, int64_t(nq) * 4);
    auto fetch = [&](int qt) {
      if constexpr (BIAS) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          id_next[t] = read16(id_buf, id_at + qt + 64 * set + 32 * t);
      }
      // (a row that is not there has no weight)
      pl = read4(lse, 4 * (qt + tid));
      pl = qt + tid < nq ? pl : INFINITY;
      if constexpr (BIAS) pl_log = read4(lse_log, 4 * (qt + tid));
      pd = read4(dsum, 4 * (qt + tid));
      if constexpr (kAhead) {
        pq.load(qb, a.sq, qt, nq, a.d);
        pg.load(gb, sg, qt, nq, a.d);
      }
    };
    if constexpr (BIAS) {
      __syncthreads();  // the last head's rows are done with its table
      load_table<T>(tab, a.table, a.table_f32, a.n_buckets, a.H, h, tid, N);
    }
    fetch(block_begin);
    for (int qt = block_begin; qt < nq; qt += kRows) {
      __syncthreads();
      if constexpr (!kAhead) {
        pq.load(qb, a.sq, qt, nq, a.d);
        pq.store(qs, tid);
        pg.load(gb, sg, qt, nq, a.d);
        pg.store(gs, tid);
      } else {
        pq.store(qs, tid);
        pg.store(gs, tid);
      }
      if (tid < kRows) {
        const bool two = BIAS && is_far(pl);
        ls[tid] = two ? 0.f : pl * lse_per, ds[tid] = pd;
        if constexpr (BIAS) far[tid][0] = two ? pl : 0.f, far[tid][1] = two ? pl_log : 0.f;
      }
      __syncthreads();
      idw[0] = id_next[0], idw[1] = id_next[1];
      if (qt + kRows < nq) fetch(qt + kRows);
      const int q1 = qt + 64 * set;  // this set's first query
      if (q1 + 64 <= wave_begin || q1 >= nq || item.y + wave * 32 >= nk) continue;
      bool any_far = false;
      if constexpr (BIAS) any_far = __any(far[64 * set + lane][0] != 0.f);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 bias;
        if constexpr (BIAS) bias = look_up(tab, idw[t]);
        f32x16 s, dp;  // start from -lse (bf16) and -D of the rows
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = 64 * set + 32 * t + 16 * half + 4 * i;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if constexpr (kFromLse) x = *reinterpret_cast<const float4*>(ls + at);
          const float4 y = *reinterpret_cast<const float4*>(ds + at);
          s[4 * i] = x.x, s[4 * i + 1] = x.y, s[4 * i + 2] = x.z, s[4 * i + 3] = x.w;
          dp[4 * i] = y.x, dp[4 * i + 1] = y.y, dp[4 * i + 2] = y.z, dp[4 * i + 3] = y.w;
        }
#pragma unroll
        for (int c = 0; c < L::kChunks; ++c) {
          s = L::mma(L::load_a(q_tile, t, c, l32, half), k.w[c], s);
          dp = L::mma(L::load_a(g_tile, t, c, l32, half), v.w[c], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (kFromLse) {
            s[i] = BIAS ? fmaf(s[i], s2, bias[i]) : s[i] * s2;
          } else {
            const float minus = ls[64 * set + 32 * t + 16 * half + i];
            s[i] = fmaf(s[i], s2, BIAS ? bias[i] + minus : minus);
          }
        }
        if constexpr (BIAS) {
          if (any_far) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float* by = far[64 * set + 32 * t + 16 * half + i];
              s[i] = (s[i] - by[0]) - by[1];
            }
          }
        }
        if (q1 + 32 * t < last_lim) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (q1 + 32 * t + 16 * half + i < lim) s[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = __builtin_amdgcn_exp2f(s[i]);
          dp[i] *= s[i];
        }
        L::mma_cols(g_tile, t, s, av, lane);
        L::mma_cols(q_tile, t, dp, ak, lane);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) {
    join_sets<RW, KS>(ak[c], buf, wave, set, lane);
    join_sets<RW, KS>(av[c], buf, wave, set, lane);
  }
  if (kj < nk && set == 0) {
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
int launch_dq(const BwdArgs& a, const BwdPlan& p, size_t lds, hipStream_t st) {
  KernelTimer timer_("packed_dq", st);
  return with_shape<most_sets(Tile<T, DP>::kRow, false)>(p.dq, [&](auto rw, auto ks) {
    auto kernel = k_packed_dq<T, DP, BIAS, HIST, rw.value, ks.value>;
    if (lds)
      NGT_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    hipLaunchKernelGGL(kernel, dim3(unsigned(p.dq_blocks)), dim3(64 * rw.value * ks.value), lds, st,
                       a);
    NGT_HIP_CHECK(hipGetLastError());
    return int(NGT_OK);
  });
}

template <typename T, int DP, bool BIAS>
int launch_dkv(const BwdArgs& a, const BwdPlan& p, hipStream_t st) {
  KernelTimer timer_("packed_dkv", st);
  return with_shape<most_sets(Tile<T, DP>::kRow, true)>(p.dkv, [&](auto rw, auto ks) {
    hipLaunchKernelGGL((k_packed_dkv<T, DP, BIAS, rw.value, ks.value>), dim3(unsigned(p.dkv_blocks)),
                       dim3(64 * rw.value * ks.value), 0, st, a);
    NGT_HIP_CHECK(hipGetLastError());
    return int(NGT_OK);
  });
}

template <typename T, int DP>
int bwd(const BwdPlan& p, const BwdArgs& base, hipStream_t st) {
  const bool bias = base.table != nullptr, hist = bias && base.grad_table;
  BwdArgs a = base;
  if (p.dq_blocks > 0) {
    a.items = p.items_q;
    a.n_items = p.n_items_q;
    const size_t lds = size_t(p.dq.rw) * p.dq.ks * (a.n_buckets + 1) * (size_t(8) << a.hist_shift);
    NGT_CHECK_OK(hist   ? (launch_dq<T, DP, true, true>(a, p, lds, st))
                 : bias ? (launch_dq<T, DP, true, false>(a, p, 0, st))
                        : (launch_dq<T, DP, false, false>(a, p, 0, st)));
  }
  if (p.dkv_blocks > 0) {
    a.items = p.items_k;
    NGT_CHECK_OK(bias ? (launch_dkv<T, DP, true>(a, p, st)) : (launch_dkv<T, DP, false>(a, p, st)));
  }
  if (hist) {
    KernelTimer timer_("packed_table_grad", st);
    auto run = [&](auto* grad) {
      hipLaunchKernelGGL(k_packed_table_grad<std::remove_pointer_t<decltype(grad)>>,
                         dim3(unsigned(a.H * ((a.n_buckets + 63) / 64))),
                         dim3(1024), 0, st, a.part_table, p.dq_blocks > 0 ? p.n_items_q : 0,
                         a.n_buckets, a.H, grad);
    };
    if (a.table_f32) run(static_cast<float*>(a.grad_table));
    else run(static_cast<T*>(a.grad_table));
    NGT_HIP_CHECK(hipGetLastError());
  }
  return NGT_OK;
}

}  // namespace

int packed_bwd(int dtype, const BwdPlan& p, const BwdArgs& a, hipStream_t st) {
  auto run = [&](auto t) {
    using T = decltype(t);
    return a.d <= 16   ? bwd<T, 16>(p, a, st)
           : a.d <= 32 ? bwd<T, 32>(p, a, st)
           : a.d <= 64 ? bwd<T, 64>(p, a, st)
                       : bwd<T, 128>(p, a, st);
  };
  return dtype == NGT_F32 ? run(float{}) : run(bf16_t{});
}

}  // namespace packed
}  // namespace ngt
