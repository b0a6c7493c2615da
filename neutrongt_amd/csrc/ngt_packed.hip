// Attention over packed windows: sequences of different lengths back to back,
// grouped heads, causal order, a learned bias per pair bucket.  Forward.
//   s_ij = scale q_i.k_j + table[id_ij, h],  o_i = sum_j e^(s_ij - lse_i) v_j over the
//   pairs that i sees,  lse_i = log sum_j e^s_ij (kept in log2 units for the backward)
// in one pass over a window's keys, with the running base and sum of each row in
// registers (RowSoftmax); no score goes to memory.  Scores, sums and statistics are
// fp32.  In bf16 a weight is rounded to bf16 for its product with v, a half step of each,
// as the result's own: the error is 1.24 to 1.4 times that of rounding the result, where two
// pieces of a weight bring it to 1.00 and cost a second product and six instructions a pair
// of weights (heads of 128 282 -> 364 us; with the backward's the same, heads of 64 343 ->
// 424, of 24 with a bias 1,019 -> 1,211, of 8 110 -> 133).  A caller who wants the weights in
// 32 bits passes fp32 rows: there they go in as three pieces.
//
// What bounds it.  1,024 pairs cost a SIMD 4 DP clocks of the matrix cores for both
// products and some 5.5 vector instructions a lane's score, the exponential four times as
// long as another: about 540 clocks, which set the pace for narrow heads and are as much as
// the products at 128.  There the two take turns instead of overlapping (matrix cores busy
// for 43 % of the time, vector units 40 %): 5 causal windows of 500 to 4,096, 32 heads of 128
// over 8, 268 us, 936 TFLOP/s of the pairs seen.  With a bias a pair adds a byte of ids from
// memory and a table entry from LDS, and the vector units are busy for 61 % of the time (3
// windows of 1,000 to 3,333, 32 heads of 24: 248 us).
#include "ngt_packed.h"

#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

namespace ngt {
namespace packed {
namespace {

constexpr float kRebase = 8.f;  // weights stay below 2^8 of a row's base

struct FwdArgs {
  const int64_t* q_start;
  const int64_t* k_start;
  const int64_t* b_start;
  const int2* items;
  int H, Hkv, d, causal, n_buckets, table_f32;
  float scale;
  int64_t sq, sk, sv;  // bytes between rows
  const void* q;
  const void* k;
  const void* v;
  const void* table;
  const uint8_t* ids;
  void* out;
  float* out32;
  float* lse;  // [H, n_q], log2 units; +inf for a row that attends to nothing (and kFar)
  int64_t n_q;
};

// The running softmax of a lane's row.  Scores x (log2 units times 1 / c2) come
// relative to the row's base m: the first product of a tile starts from -m
// (`start`, in product units) instead of 0, so that a weight costs a multiply
// and an exponential.  The base moves only when some row exceeds it by kRebase,
// so most tiles rescale nothing; weights and sums share the base, so this is
// exact.
template <bool BIAS>
struct RowSoftmax {
  float c2, per, step;  // per: product units per unit of x
  float m = 0.f;
  float thr = -INFINITY;  // -inf before the row's first key
  float l = 0.f;
  float far = 0.f;  // the base where it is beyond kFar: no product starts from it
  f32x16 start = fill16(0.f);
  __device__ __forceinline__ RowSoftmax(float c2_, float per_) : c2(c2_), per(per_), step(kRebase / c2_) {}

  template <int NT, int NC>
  __device__ __forceinline__ void weights(f32x16 (&x)[NT], f32x16 (&acc)[NC]) {
    if constexpr (BIAS) {
      if (__any(far != 0.f)) from_far(x, acc);
    }
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[t][i]);
    if (__any(mx > thr)) {
      mx = max_halves(mx);
      const bool first = thr == -INFINITY;
      const float up = !first ? fmaxf(mx, 0.f) : mx == -INFINITY ? 0.f : mx;
      const float f = first ? 0.f : __builtin_amdgcn_exp2f(-up * c2);
      if (mx > -INFINITY) thr = step;
      m += up;
      l *= f;
      restart();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[t][i] -= up;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][i] *= f;
    }
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[t][i] = __builtin_amdgcn_exp2f(x[t][i] * c2);
        s += x[t][i];
      }
    l += s;
  }
  __device__ __forceinline__ void restart() {
    if constexpr (BIAS) far = fabsf(m) < kFar ? 0.f : m;
    start = fill16(BIAS && far != 0.f ? 0.f : -m * per);
  }
  // Rows whose base is far have scores that are not relative to it yet.
  template <int NT, int NC>
  __device__ __forceinline__ void from_far(f32x16 (&x)[NT], f32x16 (&acc)[NC]) {
    const bool mine = far != 0.f;
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[t][i]);
    const float to = fmaxf(m, max_halves(mx));
    const float f = mine ? __builtin_amdgcn_exp2f(m - to) : 1.f, by = mine ? to : 0.f;
    l *= f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[t][i] -= by;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][i] *= f;
    if (mine) m = to;
    restart();
  }
  // The row's base in log2 units, -inf where it has seen no key, and its sum.  Where one
  // of its scores is NaN, so is the sum, and the base is 0: what joins such rows compares
  // only numbers.
  __device__ __forceinline__ void finish(float& base, float& sum) const {
    sum = sum_halves(l);
    base = is_nan(sum) ? 0.f : thr == -INFINITY ? thr : m * c2;
  }
};

// A row's sum is 0 (it saw no key), positive, or NaN where one of its scores is.
__device__ __forceinline__ bool saw_nothing(float sum) { return bits_of(sum) == 0u; }
__device__ __forceinline__ float inverse(float sum) { return saw_nothing(sum) ? 0.f : 1.f / sum; }

__device__ __forceinline__ void store_lse(const FwdArgs& a, int64_t at, float base, float sum) {
  const float log = __builtin_amdgcn_logf(sum);
  const bool none = saw_nothing(sum), nan = is_nan(sum);
  const bool far = a.table && is_far(base) && !none && !nan;
  a.lse[at] = none ? INFINITY : far ? base : base + log;
  if (a.table) a.lse[int64_t(a.H) * a.n_q + at] = far ? log : 0.f;
}

// One block: RW * 32 query rows of one window and head; the window's keys pass
// through LDS 64 * KS at a time (pick_shape says which and why).  The next stage's
// pieces are on their way while one is used.
template <typename T, int DP, bool BIAS, int RW, int KS>
__global__ __launch_bounds__(64 * RW * KS) void k_packed_fwd(FwdArgs a) {
  using L = Tile<T, DP>;
  using B = Block<RW, KS>;
  constexpr int N = B::kThreads, kKeys = B::kStage;
  constexpr int kTileBytes = kKeys * L::kRow;
  // registers for the next stage's pieces, where they are few enough
  constexpr bool kAhead = (kKeys * L::kMemPieces / N) * 8 <= 64;
  __shared__ __align__(16) char
      buf[2 * kTileBytes > B::kJoinBytes ? 2 * kTileBytes : B::kJoinBytes];
  __shared__ float tab[BIAS ? kTable : 1];
  __shared__ float ml[KS > 1 ? KS * RW : 1][2][64];
  char *const ks = buf, *const vs = buf + kTileBytes;
  const int tid = tid_x(), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int wid = tid >> 6, wave = wid % RW, set = wid / RW;
  // the heads that share K and V follow each other H_kv blocks apart: with 8
  // key heads all blocks of one of them run on one XCD, whose L2 holds them
  const int bid = wg_x();
  const int kvh = bid % a.Hkv, grp = (bid / a.Hkv) % (a.H / a.Hkv);
  const int h = kvh * (a.H / a.Hkv) + grp;
  const int2 item = a.items[bid / a.H];
  const int64_t q0 = a.q_start[item.x], k0 = a.k_start[item.x];
  const int nq = static_cast<int>(a.q_start[item.x + 1] - q0);
  const int nk = static_cast<int>(a.k_start[item.x + 1] - k0);
  const int ahead = nk - nq;
  const int qi = item.y + wave * 32 + l32;  // this lane's query
  const int qc = min(qi, nq - 1);
  const int lim = a.causal ? min(qc + ahead, nk - 1) : nk - 1;  // its last key
  const int first_lim = a.causal ? min(item.y + wave * 32 + ahead, nk - 1) : nk - 1;
  const int last_q = min(item.y + wave * 32 + 31, nq - 1);
  const int wave_end = item.y + wave * 32 >= nq ? 0 : a.causal ? min(last_q + ahead + 1, nk) : nk;
  const int block_end = a.causal ? min(min(item.y + 32 * RW, nq) + ahead, nk) : nk;
  const T* kb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.k) + k0 * a.sk) +
                int64_t(kvh) * a.d;
  const T* vb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.v) + k0 * a.sv) +
                int64_t(kvh) * a.d;
  RowFrag<T, DP> q;
  q.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.q) + (q0 + qc) * a.sq) +
             int64_t(h) * a.d,
         qi < nq, a.d, half);
  const int ld = (nk + 63) & ~63;
  const uint8_t* ids = nullptr;  // of the block's first query
  if constexpr (BIAS) {
    load_table<T>(tab, a.table, a.table_f32, a.n_buckets, a.H, h, tid, N);
    ids = a.ids + a.b_start[item.x] + int64_t(item.y) * ld;
  }
  const float s2 = a.scale * kLog2e;
  RowSoftmax<BIAS> sm(BIAS ? 1.f : s2, BIAS ? 1.f / s2 : 1.f);
  f32x16 acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = fill16(0.f);

  Stage<T, DP, kKeys, N> pk(a.sk, a.d, tid), pv(a.sv, a.d, tid);
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
  const char* kt_tile = ks + 64 * set * L::kRow;
  const char* vt_tile = vs + 64 * set * L::kRow;
  for (int kt = 0; kt < block_end; kt += kKeys) {
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
    fetch_ids(kt + kKeys + 64 * set);
    if constexpr (kAhead) {
      if (kt + kKeys < block_end) {
        pk.load(kb, a.sk, kt + kKeys, nk, a.d);
        pv.load(vb, a.sv, kt + kKeys, nk, a.d);
      }
    }
    const int k1 = kt + 64 * set;  // this set's first key
    if (k1 >= wave_end) continue;
    f32x16 bias[2];
    if constexpr (BIAS) bias[0] = look_up(tab, idw[0]), bias[1] = look_up(tab, idw[1]);
    f32x16 x[2] = {sm.start, sm.start};
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        x[t] = L::mma(L::load_a(kt_tile, t, c, l32, half), q.w[c], x[t]);
    if constexpr (BIAS) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[t][i] = fmaf(x[t][i], s2, bias[t][i]);
    }
    if (k1 + 63 > first_lim) {  // some key of the tile is behind some row's last one
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k1 + 32 * t + 16 * half + i > lim) x[t][i] = -INFINITY;
    }
    sm.weights(x, acc);
#pragma unroll
    for (int t = 0; t < 2; ++t) L::mma_cols(vt_tile, t, x[t], acc, lane);
  }

  float base, l;
  sm.finish(base, l);
  if constexpr (KS > 1) {
    ml[set * RW + wave][0][lane] = base;
    ml[set * RW + wave][1][lane] = l;
    __syncthreads();
    const float mine = base;
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) base = fmaxf(base, ml[s * RW + wave][0][lane]);
    auto factor = [&](float b) { return b == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(b - base); };
#pragma unroll
    for (int s = 0; s < KS; ++s)
      sum = fmaf(ml[s * RW + wave][1][lane], factor(ml[s * RW + wave][0][lane]), sum);
    const float f = factor(mine);
    l = sum;
#pragma unroll
    for (int c = 0; c < L::kCols; ++c) {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][i] *= f;
      join_sets<RW, KS>(acc[c], buf, wave, set, lane);
    }
    if (set > 0) return;
  }
  if (qi < nq) {
    const float r = inverse(l);
    T* o = reinterpret_cast<T*>(a.out) + ((q0 + qi) * a.H + h) * int64_t(a.d);
    float* o32 = a.out32 ? a.out32 + ((q0 + qi) * a.H + h) * int64_t(a.d) : nullptr;
#pragma unroll
    for (int c = 0; c < L::kCols; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * c + 8 * g + 4 * half;
        if (at < a.d) {
          store4(o + at, acc[c][4 * g] * r, acc[c][4 * g + 1] * r, acc[c][4 * g + 2] * r,
                 acc[c][4 * g + 3] * r);
          if (o32)
            store4(o32 + at, acc[c][4 * g] * r, acc[c][4 * g + 1] * r, acc[c][4 * g + 2] * r,
                   acc[c][4 * g + 3] * r);
        }
      }
    if (a.lse && half == 0) store_lse(a, int64_t(h) * a.n_q + q0 + qi, base, l);
  }
}

// ------------------------------------------------------- a few rows per window
struct FewArgs {
  FwdArgs f;
  int splits;
  float* part_ml;   // [windows * H_kv, splits, 32, 2]: base (log2 units) and sum
  float* part_acc;  // [windows * H_kv, splits, 32, DP rounded up to 32]
};

// The rows of one window and key head: row r is query r % nq of the group's
// head r / nq.  One block: the keys of one split, each wave its own tiles of
// 32 keys straight from memory (nothing is shared between waves but the end).
// Its weights go in as two bf16 pieces (16 bits): where the cache's bytes or the launches
// are what is waited for that costs nothing (the two cases below 231 -> 230 and 11.8 -> 11.7
// us with the host's part; error 2.31e-3 -> 1.65e-3, the rounding of the result).
// Bound by the cache's bytes: 32 windows of 1,000 to 16,384 keys, 8 key heads of 128,
// 230 us, 3.9 TB/s of the 4.9 of a copy; short ones by the launches (8 windows of 60 to
// 1,000: 7 us one after another in a graph, with the join).
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256) void k_packed_few(FewArgs fa) {
  using L = Tile<T, DP>;
  const FwdArgs& a = fa.f;
  constexpr int kTileBytes = 32 * L::kRow;
  constexpr int kJoin = 36;  // floats per row of the join's buffer
  constexpr int kBytes = 4 * kTileBytes > 4 * 32 * kJoin * 4 ? 4 * kTileBytes : 4 * 32 * kJoin * 4;
  __shared__ __align__(16) char buf[kBytes];
  __shared__ float ml[4][32][2];
  extern __shared__ float tabs[];  // [group][kTable] with a bias
  const int tid = tid_x(), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = wave_id();
  const int bid = wg_x();
  const int kvh = bid % a.Hkv, split = (bid / a.Hkv) % fa.splits, w = bid / (a.Hkv * fa.splits);
  const int G = a.H / a.Hkv;
  const int64_t q0 = a.q_start[w], k0 = a.k_start[w];
  const int nq = static_cast<int>(a.q_start[w + 1] - q0);
  const int nk = static_cast<int>(a.k_start[w + 1] - k0);
  if (nq == 0) return;
  const int rows = nq * G;
  const int r = min(l32, rows - 1), grp = r / nq, qi = r - grp * nq, h = kvh * G + grp;
  const int lim = a.causal ? min(qi + nk - nq, nk - 1) : nk - 1;
  const int first_lim = a.causal ? min(nk - nq, nk - 1) : nk - 1;
  const int tiles = (nk + 31) >> 5;
  const int t_begin = static_cast<int>(int64_t(tiles) * split / fa.splits);
  const int t_end = static_cast<int>(int64_t(tiles) * (split + 1) / fa.splits);
  const T* kb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.k) + k0 * a.sk) +
                int64_t(kvh) * a.d;
  const T* vb = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.v) + k0 * a.sv) +
                int64_t(kvh) * a.d;
  RowFrag<T, DP> q;
  q.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(a.q) + (q0 + qi) * a.sq) +
             int64_t(h) * a.d,
         l32 < rows, a.d, half);
  const int ld = (nk + 63) & ~63;
  const uint8_t* ids = nullptr;
  const float* tab = nullptr;
  if constexpr (BIAS) {
    for (int g = 0; g < G; ++g)
      load_table<T>(tabs + g * kTable, a.table, a.table_f32, a.n_buckets, a.H, kvh * G + g, tid,
                    256);
    ids = a.ids + a.b_start[w];
    tab = tabs + grp * kTable;
    __syncthreads();
  }
  const float s2 = a.scale * kLog2e;
  RowSoftmax<BIAS> sm(BIAS ? 1.f : s2, BIAS ? 1.f / s2 : 1.f);
  f32x16 acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = fill16(0.f);
  char* vs = buf + wave * kTileBytes;

  Stage<T, DP, 32, 64> pv(a.sv, a.d, lane);
  u32x4 pk[L::kChunks][L::kRaw];
  u32x4 idw = {0u, 0u, 0u, 0u};
  const int k_at = L::a_row(l32) * static_cast<int>(a.sk);
  const Buffer id_buf = make_buffer(ids, int64_t(nq) * ld);
  const int id_at = qi * ld + 16 * half;
  auto fetch = [&](int t) {
    const int kt = 32 * t;
    const Buffer kbuf = make_buffer(reinterpret_cast<const char*>(kb) + int64_t(kt) * a.sk,
                                    int64_t(nk - kt - 1) * a.sk + a.d * L::kEs);
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
      for (int i = 0; i < L::kRaw; ++i) {
        const int at = ((2 * c + half) * L::kRaw + i) * 16;
        pk[c][i] = read16(kbuf, at < a.d * L::kEs ? k_at + at : kNowhere);
      }
    pv.load(vb, a.sv, kt, nk, a.d);
    if constexpr (BIAS) idw = read16(id_buf, id_at + kt);
  };
  int t = t_begin + wave;
  if (t < t_end) fetch(t);
  while (t < t_end) {
    const int kt = 32 * t;
    f32x16 bias;
    if constexpr (BIAS) bias = look_up(tab, idw);
    f32x16 x[1] = {sm.start};
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c) x[0] = L::mma(L::op_of(pk[c]), q.w[c], x[0]);
    if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[0][i] = fmaf(x[0][i], s2, bias[i]);
    }
    pv.store(vs, lane);
    t += 4;
    if (t < t_end) fetch(t);
    if (kt + 31 > first_lim) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kt + 16 * half + i > lim) x[0][i] = -INFINITY;
    }
    sm.weights(x, acc);
    // the wave's own tile: its writes above, then its reads
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    L::template mma_cols<true>(vs, 0, x[0], acc, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // join the four waves, in wave order
  float base, l;
  sm.finish(base, l);
  if (half == 0) {
    ml[wave][l32][0] = base;
    ml[wave][l32][1] = l;
  }
  __syncthreads();
  const int jr = tid >> 3, jd = (tid & 7) * 4;
  float top = -INFINITY, f[4], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i][jr][0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = ml[i][jr][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i][jr][0] - top);
    sum += ml[i][jr][1] * f[i];
  }
  const int64_t slot = (int64_t(w) * a.Hkv + kvh) * fa.splits + split;
  const int jg = jr / nq, jq = jr - jg * nq, jh = kvh * G + jg;
  const float inv = fa.splits > 1 ? 1.f : inverse(sum);
  float* jb = reinterpret_cast<float*>(buf);
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) {
    if (c) __syncthreads();
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4(jb + (wave * 32 + l32) * kJoin + 8 * g + 4 * half, acc[c][4 * g], acc[c][4 * g + 1],
             acc[c][4 * g + 2], acc[c][4 * g + 3]);
    __syncthreads();
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(jb + (i * 32 + jr) * kJoin + jd);
      if (f[i] != 0.f) {
        o[0] = fmaf(y.x, f[i], o[0]);
        o[1] = fmaf(y.y, f[i], o[1]);
        o[2] = fmaf(y.z, f[i], o[2]);
        o[3] = fmaf(y.w, f[i], o[3]);
      }
    }
    const int at = 32 * c + jd;
    if (jr < rows) {
      if (fa.splits > 1) {
        store4(fa.part_acc + (slot * 32 + jr) * (32 * L::kCols) + at, o[0], o[1], o[2], o[3]);
      } else if (at < a.d) {
        const int64_t row = ((q0 + jq) * a.H + jh) * int64_t(a.d) + at;
        store4(reinterpret_cast<T*>(a.out) + row, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
        if (a.out32) store4(a.out32 + row, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      }
    }
  }
  if (jr < rows && jd == 0) {
    if (fa.splits > 1) {
      fa.part_ml[(slot * 32 + jr) * 2] = top;
      fa.part_ml[(slot * 32 + jr) * 2 + 1] = sum;
    } else if (a.lse) {
      store_lse(a, int64_t(jh) * a.n_q + q0 + jq, top, sum);
    }
  }
}

// Joins the splits of k_packed_few, in split order: 8 threads a row.
template <typename T, int DP>
__global__ __launch_bounds__(256) void k_packed_few_join(FewArgs fa) {
  const FwdArgs& a = fa.f;
  const int tid = tid_x(), jr = tid >> 3, jd = (tid & 7) * 4;
  const int kvh = wg_x() % a.Hkv, w = wg_x() / a.Hkv, G = a.H / a.Hkv;
  const int64_t q0 = a.q_start[w];
  const int nq = static_cast<int>(a.q_start[w + 1] - q0);
  if (nq == 0 || jr >= nq * G) return;
  const int jg = jr / nq, jq = jr - jg * nq, jh = kvh * G + jg;
  const int64_t slot = (int64_t(w) * a.Hkv + kvh) * fa.splits;
  constexpr int kCols = Tile<T, DP>::kCols;
  float top = -INFINITY, sum = 0.f, o[4 * kCols];
#pragma unroll
  for (int i = 0; i < 4 * kCols; ++i) o[i] = 0.f;
  const int last = fa.splits - 1;
  const float* ml = fa.part_ml + (slot * 32 + jr) * 2;
  const float* acc = fa.part_acc + (slot * 32 + jr) * (32 * kCols) + jd;
  for (int s = 0; s < fa.splits; s += 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, ml[min(s + i, last) * 64]);
  }
  // kAtOnce splits' reads under way together
  constexpr int kAtOnce = kCols > 2 ? 4 : 8;
  for (int s = 0; s < fa.splits; s += kAtOnce) {
    float2 x[kAtOnce];
    float4 y[kAtOnce][kCols];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = min(s + i, last);
      x[i] = *reinterpret_cast<const float2*>(ml + at * 64);
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        y[i][c] = *reinterpret_cast<const float4*>(acc + at * (32 * 32 * kCols) + 32 * c);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      // (a split that saw nothing has written no sums)
      if (s + i > last || x[i].x == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(x[i].x - top);
      sum = fmaf(x[i].y, f, sum);
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        o[4 * c] = fmaf(y[i][c].x, f, o[4 * c]);
        o[4 * c + 1] = fmaf(y[i][c].y, f, o[4 * c + 1]);
        o[4 * c + 2] = fmaf(y[i][c].z, f, o[4 * c + 2]);
        o[4 * c + 3] = fmaf(y[i][c].w, f, o[4 * c + 3]);
      }
    }
  }
  const float inv = inverse(sum);
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int at = 32 * c + jd;
    if (at >= a.d) continue;
    const int64_t row = ((q0 + jq) * a.H + jh) * int64_t(a.d) + at;
    store4(reinterpret_cast<T*>(a.out) + row, o[4 * c] * inv, o[4 * c + 1] * inv,
           o[4 * c + 2] * inv, o[4 * c + 3] * inv);
    if (a.out32)
      store4(a.out32 + row, o[4 * c] * inv, o[4 * c + 1] * inv, o[4 * c + 2] * inv,
             o[4 * c + 3] * inv);
  }
  if (a.lse && jd == 0) store_lse(a, int64_t(jh) * a.n_q + q0 + jq, top, sum);
}

// The windows' bucket ids as the kernels read them: one byte a pair, rows padded
// to 64 with 255, by queries and by keys.  One block: 64 queries of a window and
// every gridDim.y-th 64 of its keys (3 windows of 1,000 to 3,333, 16 M pairs: 21 us,
// with all of the keys in one block 215; about twice a copy of its bytes, no unit busy for
// more than 19 % of it: a block waits for a tile's ids before it turns them).
template <typename I>
__global__ __launch_bounds__(256) void k_packed_buckets(const I* __restrict__ ids,
                                                        const int64_t* __restrict__ q_start,
                                                        const int64_t* __restrict__ k_start,
                                                        const int64_t* __restrict__ p_start,
                                                        const int64_t* __restrict__ b_start,
                                                        const int64_t* __restrict__ bt_start,
                                                        const int2* __restrict__ items,
                                                        int steps, uint8_t* __restrict__ out,
                                                        uint8_t* __restrict__ out_t) {
  __shared__ uint8_t t[64][68];
  const int tid = tid_x();
  const int2 item = items[wg_x()];
  const int nq = static_cast<int>(q_start[item.x + 1] - q_start[item.x]);
  const int nk = static_cast<int>(k_start[item.x + 1] - k_start[item.x]);
  const int ldq = (nk + 63) & ~63, ldk = (nq + 63) & ~63;
  const I* src = ids + p_start[item.x];
  uint8_t* dst = out + b_start[item.x];
  uint8_t* dst_t = out_t + bt_start[item.x];
  for (int kt = 64 * __builtin_amdgcn_workgroup_id_y(); kt < ldq; kt += 64 * steps) {
    __syncthreads();
#pragma unroll
    for (int e = tid; e < 64 * 64; e += 256) {
      const int r = e >> 6, c = e & 63;
      int64_t x = 255;
      if (item.y + r < nq && kt + c < nk) x = int64_t(src[int64_t(item.y + r) * nk + kt + c]);
      t[r][c] = static_cast<uint8_t>(x < 0 || x > 255 ? 255 : x);
    }
    __syncthreads();
    const int r = tid >> 2, c0 = (tid & 3) * 16;
    uint32_t w[4], wt[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = wt[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[i] |= uint32_t(t[r][c0 + 4 * i + j]) << (8 * j);
        wt[i] |= uint32_t(t[c0 + 4 * i + j][r]) << (8 * j);
      }
    }
    if (item.y + r < nq)
      *reinterpret_cast<u32x4*>(dst + int64_t(item.y + r) * ldq + kt + c0) =
          u32x4{w[0], w[1], w[2], w[3]};
    if (kt + r < nk)
      *reinterpret_cast<u32x4*>(dst_t + int64_t(kt + r) * ldk + item.y + c0) =
          u32x4{wt[0], wt[1], wt[2], wt[3]};
  }
}

// ------------------------------------------------------------------ host side
constexpr int kTargetBlocks = 512;  // two blocks for each of the 256 compute units
constexpr int kSimds = 1024;
constexpr int64_t kMostThreads = 0xffffffff;  // of a launch
constexpr size_t kLds = 160 * 1024;
constexpr int kMostIds = 1 << 23;      // of a window with a bias
constexpr int32_t kMostRows = 1 << 28;  // of a window

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

inline int list_of(Shape s) { return s.rw == 4 ? 2 : s.rw == 2 ? 1 : 0; }

// The block's shape.  Row waves: as many as the longest window fills, up to 4.
// Sets: a wave's path is the stages it passes through, `path` for the longest
// window; with `steps` of them over all waves a SIMD's share is steps / 1024, and
// a path of more than 0.7 of that share leaves the chip waiting for the longest
// blocks: then 2 or 4 sets take turns.  (us, 1 / 2 / 4 sets: dK/dV of 6 causal
// windows up to 4,096, 4 heads a group, path 2.5 shares, 340 / 265 / 181; fp32, 9
// windows up to 1,777, 8 heads of 16, 0.85 shares, 233 / 209 / 249 for the three
// passes; 3,001 rows, 8 heads of 8, 1.4 shares, 366 / 297 / 344; causal forward of the 6
// windows, 0.64 shares, 87 / 106 / 153.)  Two sets go with four row waves where that
// gives every compute unit at most one block (192 blocks 297, with two 347) and
// with two where there are more (448 blocks 225, with two 209).
// blocks: of four row waves; stage: LDS bytes of 64 rows of both tiles; wave: bytes of
// each wave beside them.
Shape pick_shape(int32_t longest, int64_t path, int64_t steps, int64_t blocks, size_t stage,
                 size_t wave, int most) {
  if (longest <= 32) return Shape{1, 1};
  Shape s{longest <= 64 ? 2 : 4, 1};
  auto over = [&](int ks) { return path * 10 * kSimds > 7 * ks * steps && ks * 2 <= path; };
  if (most >= 2 && over(1)) s = Shape{s.rw == 4 && blocks <= kTargetBlocks / 2 ? 4 : 2, 2};
  if (most >= 4 && s.ks == 2 && over(2)) s = Shape{2, 4};
  auto bytes = [&] {
    return std::max(s.ks * stage, size_t(s.ks - 1) * s.rw * 4096) + size_t(s.rw) * s.ks * wave + 6 * 1024;
  };
  while (bytes() > kLds && s.ks > 1) s = Shape{2, s.ks / 2};
  while (bytes() > kLds && s.rw > 1) s.rw /= 2;
  return s;
}

struct FewPlan {
  bool use;
  int splits;
  size_t acc, total;
};
FewPlan few_plan(const ngt_packed_windows& w, int H, int Hkv, int dp) {
  FewPlan p{};
  // all heads of a group and all queries of a window in one 32-row tile, and
  // keys enough for four waves
  p.use = int64_t(w.max_q) * (H / Hkv) <= 32 && w.max_k > 128;
  if (!p.use) return p;
  const int64_t blocks = int64_t(w.n_windows) * Hkv;
  const int tiles = (w.max_k + 31) / 32;
  // Two blocks for each compute unit, of two tiles a wave or more; many splits cost the
  // join (us, 8 heads of 16, one window of 16,000 keys: 62 splits 16.8, 31 12.7, 15 12.1;
  // 4,000: 15 8.0, 7 8.0, 3 10.5; 1,000: 3 6.9, 1 7.0), and none saves its launch (600 keys:
  // 2 splits 7.2, 1 5.7).
  if (tiles < 24) {
    p.splits = 1;
  } else {
    const int most = std::min({64, tiles / 8, std::max(16, tiles / 32)});
    p.splits = static_cast<int>(
        std::min<int64_t>((kTargetBlocks + blocks - 1) / blocks, most));
  }
  if (p.splits > 1) {
    const size_t rows = size_t(blocks) * p.splits * 32;
    p.acc = align256(rows * 8);
    p.total = p.acc + align256(rows * std::max(dp, 32) * 4);
  }
  return p;
}

int dp_of(int d) { return d <= 16 ? 16 : d <= 32 ? 32 : d <= 64 ? 64 : 128; }

int check_call(const char* fn, int dtype, const ngt_packed_windows* w, int H, int Hkv, int d,
               float scale, const void* table, int n_buckets, const uint8_t* ids) {
  if (!w) return set_error(NGT_ERR_ARG, "%s: null windows", fn);
  if (dtype != NGT_F32 && dtype != NGT_BF16)
    return set_error(NGT_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
  if (H < 1 || Hkv < 1 || H > 65535 || H % Hkv)
    return set_error(NGT_ERR_ARG, "%s: %d heads over %d key heads", fn, H, Hkv);
  if (d < 8 || d > 128 || d % 8)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: head_dim=%d (a multiple of 8 up to 128)", fn, d);
  // A base or lse of up to kFar is divided by scale log2(e), and scores are multiplied by
  // it: inside this range neither leaves fp32 (at 1e-40 a bias gave NaN, at 1e-38 bf16
  // lost its gradients).
  if (!(scale >= 0x1p-100f) || !(scale <= 0x1p100f))
    return set_error(NGT_ERR_ARG, "%s: scale must lie in [2^-100, 2^100]", fn);
  if (w->n_windows < 0 || w->n_q < 0 || w->n_k < 0 || w->max_q < 0 || w->max_k < 0 || w->steps_q < 0 ||
      w->steps_k < 0)
    return set_error(NGT_ERR_ARG, "%s: bad windows", fn);
  for (int i = 0; i < 3; ++i)
    if (w->n_items_q[i] < 0 || w->n_items_k[i] < 0 ||
        int64_t(std::max(w->n_items_q[i], w->n_items_k[i])) * H > 0x7fffffff)
      return set_error(NGT_ERR_UNSUPPORTED, "%s: too many rows for one launch", fn);
  if ((table != nullptr) != (ids != nullptr))
    return set_error(NGT_ERR_ARG, "%s: a bias takes a table and bucket ids", fn);
  if (table && (n_buckets < 1 || n_buckets > 255))
    return set_error(NGT_ERR_ARG, "%s: n_buckets=%d (1 to 255)", fn, n_buckets);
  // 32-bit offsets within a block's rows
  if (table && (w->max_q > kMostIds || w->max_k > kMostIds))
    return set_error(NGT_ERR_UNSUPPORTED, "%s: a bias over windows of more than %d rows", fn,
                     kMostIds);
  if (int64_t(H) * d * (dtype == NGT_F32 ? 4 : 2) > kMostRowBytes)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: %d heads of %d", fn, H, d);
  if (table && !(w->b_start && w->bt_start))
    return set_error(NGT_ERR_ARG, "%s: null bucket offsets", fn);
  return NGT_OK;
}

int check_stride(const char* fn, const char* name, const void* p, int64_t stride, int heads, int d,
                 int es) {
  if (stride > kMostRowBytes / es)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: %s rows more than 8 MB apart", fn, name);
  if (stride < int64_t(heads) * d || (stride * es) % 16 || reinterpret_cast<uintptr_t>(p) % 16)
    return set_error(NGT_ERR_ARG,
                     "%s: %s rows must be at least heads * head_dim apart and 16-byte aligned", fn,
                     name);
  return NGT_OK;
}

template <typename T, int DP, bool BIAS>
int run_fwd(const ngt_packed_windows& w, const FewPlan& fp, FwdArgs a, void* ws, hipStream_t st) {
  if (fp.use) {
    FewArgs fa{a, fp.splits, nullptr, nullptr};
    if (fp.splits > 1) {
      fa.part_ml = static_cast<float*>(ws);
      fa.part_acc = reinterpret_cast<float*>(static_cast<char*>(ws) + fp.acc);
    }
    const int64_t blocks = int64_t(w.n_windows) * a.Hkv;
    {
      KernelTimer timer_("packed_few", st);
      hipLaunchKernelGGL((k_packed_few<T, DP, BIAS>), dim3(unsigned(blocks * fp.splits)), dim3(256),
                         BIAS ? (a.H / a.Hkv) * kTable * sizeof(float) : 0, st, fa);
      NGT_HIP_CHECK(hipGetLastError());
    }
    if (fp.splits > 1) {
      KernelTimer timer_("packed_few_join", st);
      hipLaunchKernelGGL((k_packed_few_join<T, DP>), dim3(unsigned(blocks)), dim3(256), 0, st, fa);
      NGT_HIP_CHECK(hipGetLastError());
    }
    return NGT_OK;
  }
  constexpr int kMost = most_sets(Tile<T, DP>::kRow, false);
  const Shape shape =
      pick_shape(w.max_q, (w.max_k + 63) / 64, w.steps_q * a.H, int64_t(w.n_items_q[2]) * a.H,
                 128 * Tile<T, DP>::kRow, 512, kMost);
  const int i = list_of(shape);
  const int64_t blocks = int64_t(w.n_items_q[i]) * a.H;
  if (!blocks) return NGT_OK;
  if (blocks * 64 * shape.rw * shape.ks > kMostThreads)
    return set_error(NGT_ERR_UNSUPPORTED, "ngt_packed_fwd: too many rows and heads for one launch");
  a.items = reinterpret_cast<const int2*>(w.items_q[i]);
  KernelTimer timer_("packed_fwd", st);
  return with_shape<kMost>(shape, [&](auto rw, auto ks) {
    hipLaunchKernelGGL((k_packed_fwd<T, DP, BIAS, rw.value, ks.value>), dim3(unsigned(blocks)),
                       dim3(64 * rw.value * ks.value), 0, st, a);
    NGT_HIP_CHECK(hipGetLastError());
    return int(NGT_OK);
  });
}

template <typename T>
int run_fwd_d(int dp, const ngt_packed_windows& w, const FewPlan& fp, const FwdArgs& a, void* ws,
              hipStream_t st) {
  if (a.table)
    return dp == 16   ? run_fwd<T, 16, true>(w, fp, a, ws, st)
           : dp == 32 ? run_fwd<T, 32, true>(w, fp, a, ws, st)
           : dp == 64 ? run_fwd<T, 64, true>(w, fp, a, ws, st)
                      : run_fwd<T, 128, true>(w, fp, a, ws, st);
  return dp == 16   ? run_fwd<T, 16, false>(w, fp, a, ws, st)
         : dp == 32 ? run_fwd<T, 32, false>(w, fp, a, ws, st)
         : dp == 64 ? run_fwd<T, 64, false>(w, fp, a, ws, st)
                    : run_fwd<T, 128, false>(w, fp, a, ws, st);
}

struct BwdLayout {
  size_t part, total;
  Shape dq, dkv;
};
BwdLayout bwd_layout(int dtype, const ngt_packed_windows& w, int H, int Hkv, int d, int n_buckets) {
  BwdLayout L{};
  const int dp = dp_of(d);  // bytes of a tile's row in LDS:
  static_assert(Tile<bf16_t, 16>::kRow == 32 && Tile<float, 16>::kRow == 96 &&
                    Tile<float, 128>::kRow == 512, "row below");
  const int row = dtype != NGT_F32 ? 2 * dp : dp == 128 ? 4 * dp : 6 * dp;
  const size_t sums = size_t(8) << hist_shift(dtype == NGT_F32, n_buckets);
  L.dq = pick_shape(w.max_q, (w.max_k + 63) / 64, w.steps_q * H, int64_t(w.n_items_q[2]) * H,
                    size_t(128) * row,
                    n_buckets ? size_t(n_buckets + 1) * sums : 0, most_sets(row, false));
  L.dkv = pick_shape(w.max_k, int64_t((w.max_q + 63) / 64) * (H / Hkv), w.steps_k * H,
                     int64_t(w.n_items_k[2]) * Hkv, size_t(128) * row, 0, most_sets(row, true));
  L.part = align256(size_t(w.n_q) * H * 4);
  L.total = L.part + align256(size_t(w.n_items_q[list_of(L.dq)]) * H * n_buckets * 4);
  return L;
}

// The plan's arrays, in the order in which they lie in its buffer.
struct PlanLayout {
  int64_t items[2][3];
  size_t start[5], list[2][3], total;
};
PlanLayout plan_layout(int32_t n, const int32_t* q_len, const int32_t* k_len) {
  PlanLayout L{};
  for (int32_t w = 0; w < n; ++w)
    for (int i = 0; i < 3; ++i) {
      L.items[0][i] += (int64_t(q_len[w]) + (32 << i) - 1) / (32 << i);
      L.items[1][i] += (int64_t(k_len[w]) + (32 << i) - 1) / (32 << i);
    }
  size_t at = 0;
  for (int s = 0; s < 5; ++s) L.start[s] = at, at += align256((size_t(n) + 1) * 8);
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < 3; ++i) L.list[o][i] = at, at += align256(size_t(L.items[o][i]) * 8);
  L.total = at;
  return L;
}

int check_lengths(const char* fn, int32_t n, const int32_t* q_len, const int32_t* k_len) {
  if (n < 0 || (n > 0 && (!q_len || !k_len)))
    return set_error(NGT_ERR_ARG, "%s: bad window count or null lengths", fn);
  int64_t tq = 0, tk = 0;
  for (int32_t w = 0; w < n; ++w) {
    if (q_len[w] < 0 || k_len[w] < 0)
      return set_error(NGT_ERR_ARG, "%s: window %d has a negative length", fn, w);
    if (q_len[w] > kMostRows || k_len[w] > kMostRows)
      return set_error(NGT_ERR_UNSUPPORTED, "%s: window %d is longer than 2^28", fn, w);
    tq += (q_len[w] + 31) / 32;
    tk += (k_len[w] + 31) / 32;
  }
  if (tq > 0x7fffffff || tk > 0x7fffffff)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: too many rows", fn);
  return NGT_OK;
}

}  // namespace
}  // namespace packed
}  // namespace ngt

using namespace ngt;
using namespace ngt::packed;

extern "C" int ngt_packed_plan_bytes(int32_t n_windows, const int32_t* q_len, const int32_t* k_len,
                                     size_t* bytes) {
  NGT_CHECK_OK(check_lengths("ngt_packed_plan_bytes", n_windows, q_len, k_len));
  if (!bytes) return set_error(NGT_ERR_ARG, "ngt_packed_plan_bytes: null bytes");
  *bytes = plan_layout(n_windows, q_len, k_len).total;
  return NGT_OK;
}

extern "C" int ngt_packed_plan(int32_t n_windows, const int32_t* q_len, const int32_t* k_len,
                               int32_t causal, void* host, size_t bytes, void* device,
                               ngt_packed_windows* out) {
  NGT_CHECK_OK(check_lengths("ngt_packed_plan", n_windows, q_len, k_len));
  if (!out) return set_error(NGT_ERR_ARG, "ngt_packed_plan: null windows");
  const PlanLayout L = plan_layout(n_windows, q_len, k_len);
  if (!host || !device || bytes < L.total)
    return set_error(NGT_ERR_WORKSPACE, "ngt_packed_plan: buffer %zu < %zu", bytes, L.total);
  char* base = static_cast<char*>(host);
  char* dev = static_cast<char*>(device);
  memset(out, 0, sizeof(*out));
  memset(base, 0, L.total);
  out->n_windows = n_windows;
  out->causal = causal != 0;
  int64_t* s[5];
  for (int i = 0; i < 5; ++i) s[i] = reinterpret_cast<int64_t*>(base + L.start[i]);
  for (int32_t w = 0; w < n_windows; ++w) {
    const int64_t nq = q_len[w], nk = k_len[w];
    s[0][w + 1] = s[0][w] + nq;
    s[1][w + 1] = s[1][w] + nk;
    s[2][w + 1] = s[2][w] + nq * nk;
    s[3][w + 1] = s[3][w] + nq * ((nk + 63) & ~int64_t(63));
    s[4][w + 1] = s[4][w] + nk * ((nq + 63) & ~int64_t(63));
    out->max_q = std::max(out->max_q, q_len[w]);
    out->max_k = std::max(out->max_k, k_len[w]);
  }
  out->n_q = s[0][n_windows];
  out->n_k = s[1][n_windows];
  out->n_pairs = s[2][n_windows];
  out->bucket_bytes_q = s[3][n_windows];
  out->bucket_bytes_k = s[4][n_windows];
  out->q_start = reinterpret_cast<const int64_t*>(dev + L.start[0]);
  out->k_start = reinterpret_cast<const int64_t*>(dev + L.start[1]);
  out->p_start = reinterpret_cast<const int64_t*>(dev + L.start[2]);
  out->b_start = reinterpret_cast<const int64_t*>(dev + L.start[3]);
  out->bt_start = reinterpret_cast<const int64_t*>(dev + L.start[4]);
  try {
    // the work lists, the items with the most rows on the other side first (a
    // counting sort by 64-row steps): the last blocks to start are short ones
    for (int o = 0; o < 2; ++o)
      for (int i = 0; i < 3; ++i) {
        const int rows = 32 << i;
        int32_t* list = reinterpret_cast<int32_t*>(base + L.list[o][i]);
        auto steps = [&](int32_t w, int32_t row) {
          const int64_t nq = q_len[w], nk = k_len[w], mine = o ? nk : nq, other = o ? nq : nk;
          int64_t seen = other;
          if (causal) {
            const int64_t last = std::min<int64_t>(row + rows, mine);
            seen = o ? nq - std::max<int64_t>(0, row - (nk - nq)) : std::min(last + nk - nq, nk);
          }
          return std::max<int64_t>(0, std::min(seen, other) + 63) / 64;
        };
        const int64_t top = ((o ? out->max_q : out->max_k) + 63) / 64;
        std::vector<int64_t> at(size_t(top) + 2, 0);
        for (int32_t w = 0; w < n_windows; ++w)
          for (int32_t r = 0; r < (o ? k_len[w] : q_len[w]); r += rows) {
          ++at[size_t(top - steps(w, r)) + 1];
          if (i == 0) (o ? out->steps_k : out->steps_q) += steps(w, r);
        }
        for (size_t j = 1; j < at.size(); ++j) at[j] += at[j - 1];
        for (int32_t w = 0; w < n_windows; ++w)
          for (int32_t r = 0; r < (o ? k_len[w] : q_len[w]); r += rows) {
            const int64_t j = at[size_t(top - steps(w, r))]++;
            list[2 * j] = w;
            list[2 * j + 1] = r;
          }
        const int32_t* d = reinterpret_cast<const int32_t*>(dev + L.list[o][i]);
        if (o) out->n_items_k[i] = static_cast<int32_t>(L.items[1][i]), out->items_k[i] = d;
        else out->n_items_q[i] = static_cast<int32_t>(L.items[0][i]), out->items_q[i] = d;
      }
  } catch (const std::bad_alloc&) {
    return set_error(NGT_ERR_HIP, "ngt_packed_plan: out of host memory");
  }
  return NGT_OK;
}

extern "C" int ngt_packed_buckets(const ngt_packed_windows* w, const void* ids, int32_t id_bytes,
                                  uint8_t* buckets_q, uint8_t* buckets_k, void* stream) {
  if (!w) return set_error(NGT_ERR_ARG, "ngt_packed_buckets: null windows");
  if (id_bytes != 1 && id_bytes != 4 && id_bytes != 8)
    return set_error(NGT_ERR_ARG, "ngt_packed_buckets: ids of %d bytes (1, 4 or 8)", id_bytes);
  if (w->n_pairs == 0) return NGT_OK;
  if (!ids || !buckets_q || !buckets_k)
    return set_error(NGT_ERR_ARG, "ngt_packed_buckets: null ids or buckets");
  hipStream_t st = static_cast<hipStream_t>(stream);
  KernelTimer timer_("packed_buckets", st);
  const int n = std::max(w->n_items_q[1], 1), most = 4096 / n;
  if (int64_t(n) * 256 > kMostThreads)
    return set_error(NGT_ERR_UNSUPPORTED, "ngt_packed_buckets: too many rows for one launch");
  const int steps = most < 1 ? 1 : most > 64 ? 64 : most;
  auto run = [&](auto kernel, auto* p) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(n), unsigned(steps)), dim3(256), 0, st, p,
                       w->q_start, w->k_start, w->p_start, w->b_start, w->bt_start,
                       reinterpret_cast<const int2*>(w->items_q[1]), steps, buckets_q, buckets_k);
  };
  if (id_bytes == 1) run(k_packed_buckets<uint8_t>, static_cast<const uint8_t*>(ids));
  else if (id_bytes == 4) run(k_packed_buckets<int32_t>, static_cast<const int32_t*>(ids));
  else run(k_packed_buckets<int64_t>, static_cast<const int64_t*>(ids));
  NGT_HIP_CHECK(hipGetLastError());
  return NGT_OK;
}

extern "C" int ngt_packed_workspace_bytes(int dtype, const ngt_packed_windows* w, int32_t n_heads,
                                          int32_t n_kv_heads, int32_t head_dim, int32_t n_buckets,
                                          size_t* fwd_bytes, size_t* bwd_bytes) {
  dtype &= ~NGT_TABLE_F32;
  NGT_CHECK_OK(check_call("ngt_packed_workspace_bytes", dtype, w, n_heads, n_kv_heads, head_dim,
                          1.f, nullptr, 0, nullptr));
  if (n_buckets < 0 || n_buckets > 255)
    return set_error(NGT_ERR_ARG, "ngt_packed_workspace_bytes: n_buckets=%d", n_buckets);
  if (fwd_bytes) *fwd_bytes = few_plan(*w, n_heads, n_kv_heads, dp_of(head_dim)).total;
  if (bwd_bytes)
    *bwd_bytes = bwd_layout(dtype, *w, n_heads, n_kv_heads, head_dim, n_buckets).total;
  return NGT_OK;
}

extern "C" int ngt_packed_fwd(int dtype, const void* q, const void* k, const void* v,
                              int64_t q_stride, int64_t k_stride, int64_t v_stride,
                              const ngt_packed_windows* w, int32_t n_heads, int32_t n_kv_heads,
                              int32_t head_dim, float scale, const void* table, int32_t n_buckets,
                              const uint8_t* buckets_q, void* out, float* out_f32, float* lse,
                              void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "ngt_packed_fwd";
  const int table_f32 = dtype & NGT_TABLE_F32;
  dtype &= ~NGT_TABLE_F32;
  NGT_CHECK_OK(check_call(fn, dtype, w, n_heads, n_kv_heads, head_dim, scale, table, n_buckets,
                          buckets_q));
  if (w->n_q == 0) return NGT_OK;
  const int es = dtype == NGT_F32 ? 4 : 2;
  if (!q || !out) return set_error(NGT_ERR_ARG, "%s: null q or out", fn);
  if (w->n_k > 0 && (!k || !v)) return set_error(NGT_ERR_ARG, "%s: null k or v", fn);
  NGT_CHECK_OK(check_stride(fn, "q", q, q_stride, n_heads, head_dim, es));
  if (w->n_k > 0) {
    NGT_CHECK_OK(check_stride(fn, "k", k, k_stride, n_kv_heads, head_dim, es));
    NGT_CHECK_OK(check_stride(fn, "v", v, v_stride, n_kv_heads, head_dim, es));
  }
  const int dp = dp_of(head_dim);
  const FewPlan fp = few_plan(*w, n_heads, n_kv_heads, dp);
  if (fp.total && (!workspace || workspace_bytes < fp.total))
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu", fn, workspace_bytes, fp.total);
  if (fp.use && int64_t(w->n_windows) * n_kv_heads * fp.splits * 256 > kMostThreads)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: too many windows for one launch", fn);
  FwdArgs a{w->q_start, w->k_start, w->b_start, nullptr, n_heads, n_kv_heads, head_dim, w->causal,
            n_buckets, table_f32, scale, q_stride * es, k_stride * es, v_stride * es, q, k, v, table,
            buckets_q, out, out_f32, lse, w->n_q};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == NGT_F32 ? run_fwd_d<float>(dp, *w, fp, a, workspace, st)
                          : run_fwd_d<bf16_t>(dp, *w, fp, a, workspace, st);
}

extern "C" int ngt_packed_bwd(int dtype, const void* q, const void* k, const void* v,
                              int64_t q_stride, int64_t k_stride, int64_t v_stride,
                              const float* out_f32, const void* grad_out, const float* lse,
                              const ngt_packed_windows* w, int32_t n_heads, int32_t n_kv_heads,
                              int32_t head_dim, float scale, const void* table, int32_t n_buckets,
                              const uint8_t* buckets_q, const uint8_t* buckets_k, void* grad_q,
                              void* grad_k, void* grad_v, void* grad_table, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* fn = "ngt_packed_bwd";
  const int table_f32 = dtype & NGT_TABLE_F32;
  dtype &= ~NGT_TABLE_F32;
  NGT_CHECK_OK(check_call(fn, dtype, w, n_heads, n_kv_heads, head_dim, scale, table, n_buckets,
                          buckets_q));
  const int es = dtype == NGT_F32 ? 4 : 2;
  if (table && !buckets_k) return set_error(NGT_ERR_ARG, "%s: null buckets_k", fn);
  if (grad_table && !table) return set_error(NGT_ERR_ARG, "%s: grad_table without a table", fn);
  if (w->n_q > 0 && (!q || !out_f32 || !grad_out || !lse || !grad_q))
    return set_error(NGT_ERR_ARG, "%s: null query-side pointer", fn);
  if (w->n_k > 0 && (!k || !v || !grad_k || !grad_v))
    return set_error(NGT_ERR_ARG, "%s: null key-side pointer", fn);
  if (w->n_q > 0) NGT_CHECK_OK(check_stride(fn, "q", q, q_stride, n_heads, head_dim, es));
  if (w->n_k > 0) {
    NGT_CHECK_OK(check_stride(fn, "k", k, k_stride, n_kv_heads, head_dim, es));
    NGT_CHECK_OK(check_stride(fn, "v", v, v_stride, n_kv_heads, head_dim, es));
  }
  const int hist = grad_table ? n_buckets : 0;
  const BwdLayout L = bwd_layout(dtype, *w, n_heads, n_kv_heads, head_dim, hist);
  if (L.total && (!workspace || workspace_bytes < L.total))
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu", fn, workspace_bytes, L.total);
  char* ws = static_cast<char*>(workspace);
  BwdArgs a{};
  a.q_start = w->q_start, a.k_start = w->k_start, a.b_start = w->b_start, a.bt_start = w->bt_start;
  a.H = n_heads, a.Hkv = n_kv_heads, a.d = head_dim, a.causal = w->causal, a.n_buckets = n_buckets;
  a.table_f32 = table_f32;
  a.scale = scale, a.sq = q_stride * es, a.sk = k_stride * es, a.sv = v_stride * es, a.n_q = w->n_q;
  a.q = q, a.k = k, a.v = v, a.go = grad_out, a.out32 = out_f32, a.lse = lse;
  a.dsum = reinterpret_cast<float*>(ws);
  a.table = table, a.ids = buckets_q, a.ids_t = buckets_k;
  a.part_table = reinterpret_cast<float*>(ws + L.part);
  a.gq = grad_q, a.gk = grad_k, a.gv = grad_v, a.grad_table = grad_table;
  a.hist_shift = hist_shift(dtype == NGT_F32, n_buckets);
  BwdPlan p{};
  p.dq = L.dq, p.dkv = L.dkv;
  p.items_q = reinterpret_cast<const int2*>(w->items_q[list_of(L.dq)]);
  p.items_k = reinterpret_cast<const int2*>(w->items_k[list_of(L.dkv)]);
  p.n_items_q = w->n_items_q[list_of(L.dq)];
  p.dq_blocks = int64_t(p.n_items_q) * n_heads;
  p.dkv_blocks = int64_t(w->n_items_k[list_of(L.dkv)]) * n_kv_heads;
  if (p.dq_blocks * 64 * L.dq.rw * L.dq.ks > kMostThreads ||
      p.dkv_blocks * 64 * L.dkv.rw * L.dkv.ks > kMostThreads)
    return set_error(NGT_ERR_UNSUPPORTED, "%s: too many rows and heads for one launch", fn);
  return packed_bwd(dtype, p, a, static_cast<hipStream_t>(stream));
}
