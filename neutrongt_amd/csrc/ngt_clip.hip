// The 2-norm over many gradients and their scaling to a largest norm:
//   norm = sqrt(sum g^2),  g <- g min(1, max_norm / norm).
// Bound by memory: all gradients are read once for the norm and, where they are to be
// scaled, read and written once more.  Their addresses go in the launch's arguments, so a
// captured graph holds them and no table is copied.
// Squares and sums are fp64: exact squares of fp32, no overflow, and a sum over any
// number of elements that does not depend on how they are cut.
// us of norm and scaling, by rocprofv3: 42.6 M fp32 (170 MB, 198 tensors) into fp32 28 + 57, 6.0
// TB/s with what the last-level cache keeps; 303 M bf16 (606 MB) into fp32 153 + 370, 4.0 and 4.9
// TB/s; 66 M fp32 below the limit 41 + 5; the slim preset's 70 tensors 4 + 4.  With the library's
// timer, which adds 2 to 3 us a launch, the 42.6 M in place 29 + 56, in 198 allocations 30 + 57;
// into results that lie apart 31 + 60, and 49 + 68 where one element before them leaves no run aligned
// to 16 bytes: such a run goes element by element.
#include "ngt_common.h"

#include <new>
#include <type_traits>
#include <vector>

namespace ngt {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;      // elements of a run that a block takes at a time
constexpr int kBlocks = 2048;     // most of a launch
// Partial sums that every block of k_scale adds by itself: a launch less (about 3 us), for 0.5 (14
// parts) to 1.7 us (2,023) in it.
constexpr int kJoined = 2048;
constexpr int kFlight = 4;        // 16-byte reads of a thread under way at a time

// The runs of memory of one launch, in its arguments (below 4 KB): gradients that lie back to
// back in one buffer, like their results, are one run.
template <int RUNS, bool OUT>
struct Table {
  void* x[RUNS];
  void* out[OUT ? RUNS : 1];  // (not OUT: x)
  int32_t first[RUNS + 1];    // chunks before a run's
  uint16_t tail[RUNS];        // elements of its last chunk
  uint8_t kind[RUNS];         // bits 0, 1: x, out is bf16; bit 2: both 16-byte aligned
  int32_t count;
};
constexpr int kRuns = 250, kRunsOut = 165;
using TableIn = Table<kRuns, false>;
using TableOut = Table<kRunsOut, true>;
static_assert(sizeof(TableIn) <= 4000 && sizeof(TableOut) <= 4000, "a launch's arguments");

struct Part {
  int run;
  int64_t from, to;  // elements
};
template <typename T>
__device__ __forceinline__ Part part_of(const T& t, int chunk) {
  int lo = 0, hi = t.count;  // the last run whose first chunk is not behind it
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  const int64_t from = int64_t(chunk - t.first[lo]) * kChunk;
  return {lo, from, from + (chunk + 1 == t.first[lo + 1] ? t.tail[lo] : kChunk)};
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double* red) {
  for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / kWave; ++i) v += red[i];
  return v;
}

// 16 bytes as floats
template <typename T>
struct Piece {
  static constexpr int V = 16 / static_cast<int>(sizeof(T));
  float v[V];
};
template <typename T>
__device__ __forceinline__ Piece<T> piece_of(const uint4& w) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  Piece<T> p;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p.v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p.v[2 * i] = __uint_as_float(u[i] << 16);
      p.v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  return p;
}

// f(i, 16 bytes from element i) for the whole pieces of [from, to), kFlight reads under way at a
// time; the first element that is in none.
template <typename T, typename F>
__device__ __forceinline__ int64_t pieces(const T* __restrict__ x, int64_t from, int64_t to, F f) {
  constexpr int V = Piece<T>::V, kStep = kThreads * V;
  const int64_t end = from + (to - from) / V * V;
  int64_t i = from + threadIdx.x * V;
  for (; i + (kFlight - 1) * kStep < end; i += kFlight * kStep) {
    uint4 w[kFlight];
#pragma unroll
    for (int t = 0; t < kFlight; ++t) w[t] = *reinterpret_cast<const uint4*>(x + i + t * kStep);
#pragma unroll
    for (int t = 0; t < kFlight; ++t) f(i + t * kStep, w[t]);
  }
  for (; i < end; i += kStep) f(i, *reinterpret_cast<const uint4*>(x + i));
  return end;
}

template <typename T>
__device__ __forceinline__ double squares(const void* base, const Part& p, bool wide) {
  const T* x = static_cast<const T*>(base);
  double s[2] = {0.0, 0.0};
  int64_t i = p.from;
  if (wide)
    i = pieces(x, p.from, p.to, [&](int64_t, const uint4& w) {
      const Piece<T> v = piece_of<T>(w);
#pragma unroll
      for (int k = 0; k < Piece<T>::V; ++k) s[k & 1] = fma(double(v.v[k]), double(v.v[k]), s[k & 1]);
    });
  for (i += threadIdx.x; i < p.to; i += kThreads) {
    const double v = elem<T>::load(x + i);
    s[0] = fma(v, v, s[0]);
  }
  return s[0] + s[1];
}

// part[block]: the sum of the squares of the block's chunks.
__global__ __launch_bounds__(kThreads) void k_squares(const TableIn t, double* __restrict__ part) {
  __shared__ double red[kThreads / kWave];
  double s = 0.0;
  for (int chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
    const Part p = part_of(t, chunk);
    s += t.kind[p.run] & 1 ? squares<bf16_t>(t.x[p.run], p, t.kind[p.run] & 4)
                           : squares<float>(t.x[p.run], p, t.kind[p.run] & 4);
  }
  s = block_sum<kThreads>(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// What the gradients are scaled by: `by`, and where that would be below fp32's normal range a
// power of two more (its numbers there have fewer bits, or are 0).  An element times a `by` of
// 2^-120 does not overflow, and where it loses bits the result is below 2^-126 too.
struct Factor {
  float by;
  int32_t shift;
  __device__ __forceinline__ float operator()(float x) const { return ldexpf(x * by, shift); }
};
// 1 where the norm, as the caller gets it, is not finite.
__device__ __forceinline__ Factor factor_of(double norm, double max_norm) {
  if (!(static_cast<float>(norm) < INFINITY && norm > max_norm)) return {1.f, 0};
  const double f = max_norm / norm;
  if (f >= 0x1p-126 || f == 0.0) return {static_cast<float>(f), 0};
  int e;
  const double m = frexp(f, &e);
  return {static_cast<float>(ldexp(m, -120)), e + 120};
}

// The norm and the factor, of more parts than k_scale adds by itself or of a norm alone.
__global__ __launch_bounds__(1024) void k_norm(const double* __restrict__ part, int32_t n,
                                               double max_norm, float* __restrict__ norm,
                                               Factor* __restrict__ factor) {
  __shared__ double red[1024 / kWave];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
  s = sqrt(block_sum<1024>(s, red));
  if (threadIdx.x != 0) return;
  *norm = static_cast<float>(s);
  *factor = factor_of(s, max_norm);
}

template <typename T, typename O>
__device__ __forceinline__ void scaled(const void* base, void* result, const Part& p, bool wide,
                                       const Factor& by) {
  const T* x = static_cast<const T*>(base);
  O* o = static_cast<O*>(result);
  int64_t i = p.from;
  if (wide)
    i = pieces(x, p.from, p.to, [&](int64_t at, const uint4& w) {
      Piece<T> v = piece_of<T>(w);
#pragma unroll
      for (int k = 0; k < Piece<T>::V; ++k) v.v[k] = by(v.v[k]);
      if constexpr (sizeof(T) == 4 && sizeof(O) == 2)
        *reinterpret_cast<uint2*>(o + at) = make_uint2(pack2_bf16(v.v[0], v.v[1]), pack2_bf16(v.v[2], v.v[3]));
      else
        store_row<O, Piece<T>::V>(o + at, v.v);
    });
  for (i += threadIdx.x; i < p.to; i += kThreads) elem<O>::store(o + i, by(elem<T>::load(x + i)));
}

// parts > 0: the factor from so many sums, which all blocks add in the same order (the first
// one writes the norm); else *factor.  The chunks in the opposite order to k_squares', so that
// what it read last, which the last-level cache still holds, comes first.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_scale(const T t, const double* __restrict__ part,
                                                    int32_t parts, double max_norm,
                                                    float* __restrict__ norm,
                                                    const Factor* __restrict__ factor) {
  constexpr bool kOut = std::is_same_v<T, TableOut>;
  __shared__ double red[kThreads / kWave];
  Factor by;
  if (parts > 0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    s = sqrt(block_sum<kThreads>(s, red));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(s);
    by = factor_of(s, max_norm);
  } else {
    by = *factor;
  }
  if (!kOut && by.by == 1.f) return;  // left alone
  for (int chunk = t.first[t.count] - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const Part p = part_of(t, chunk);
    const bool wide = t.kind[p.run] & 4;
    void* out = kOut ? t.out[p.run] : t.x[p.run];
    switch (t.kind[p.run] & 3) {
      case 0: scaled<float, float>(t.x[p.run], out, p, wide, by); break;
      case 1: scaled<bf16_t, float>(t.x[p.run], out, p, wide, by); break;
      case 2: scaled<float, bf16_t>(t.x[p.run], out, p, wide, by); break;
      default: scaled<bf16_t, bf16_t>(t.x[p.run], out, p, wide, by); break;
    }
  }
}

bool bad_dtype(int32_t d) { return d != NGT_F32 && d != NGT_BF16; }

int check(const char* fn, const ngt_gradient* g, int32_t n) {
  if (n < 0 || (n > 0 && !g)) return set_error(NGT_ERR_ARG, "%s: n_tensors=%d", fn, n);
  for (int32_t i = 0; i < n; ++i) {
    if (g[i].n < 0 || g[i].n > int64_t(1) << 40)
      return set_error(NGT_ERR_ARG, "%s: tensor %d has %lld elements", fn, i,
                       static_cast<long long>(g[i].n));
    if (bad_dtype(g[i].dtype) || (g[i].out && bad_dtype(g[i].out_dtype)))
      return set_error(NGT_ERR_ARG, "%s: tensor %d: dtype", fn, i);
    if (g[i].n > 0 && !g[i].x) return set_error(NGT_ERR_ARG, "%s: tensor %d is null", fn, i);
    if (g[i].out == g[i].x && g[i].out && g[i].out_dtype != g[i].dtype)
      return set_error(NGT_ERR_ARG, "%s: tensor %d: another type in its own memory", fn, i);
    auto es = [](int32_t d) { return d == NGT_F32 ? 4 : 2; };
    if (reinterpret_cast<uintptr_t>(g[i].x) % es(g[i].dtype) ||
        (g[i].out && reinterpret_cast<uintptr_t>(g[i].out) % es(g[i].out_dtype)))
      return set_error(NGT_ERR_ARG, "%s: tensor %d is not aligned to its type", fn, i);
  }
  return NGT_OK;
}

// The gradients' runs of memory, in their order.
struct Run {
  char* x;
  char* out;  // null: x
  int64_t n;
  int32_t dtype, out_dtype;
};
int64_t size_of(int32_t dtype) { return dtype == NGT_F32 ? 4 : 2; }
std::vector<Run> runs_of(const ngt_gradient* g, int32_t n) {
  std::vector<Run> runs;
  runs.reserve(n);
  for (int32_t i = 0; i < n; ++i) {
    if (g[i].n == 0) continue;
    const Run r{static_cast<char*>(g[i].x), static_cast<char*>(g[i].out), g[i].n, g[i].dtype,
                g[i].out ? g[i].out_dtype : g[i].dtype};
    if (!runs.empty()) {
      Run& l = runs.back();
      if (l.dtype == r.dtype && l.out_dtype == r.out_dtype && l.x + l.n * size_of(l.dtype) == r.x &&
          (l.out ? l.out + l.n * size_of(l.out_dtype) == r.out : !r.out)) {
        l.n += r.n;
        continue;
      }
    }
    runs.push_back(r);
  }
  return runs;
}

// The tables of the launches over the runs, one after another: f(table, chunks).
template <int RUNS, bool OUT, typename F>
int each_launch(const std::vector<Run>& runs, F f) {
  Table<RUNS, OUT> t;
  t.count = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (t.count == 0) return NGT_OK;
    t.first[t.count] = static_cast<int32_t>(chunks);
    const int rc = f(t, static_cast<int32_t>(chunks));
    t.count = 0, chunks = 0;
    return rc;
  };
  for (const Run& r : runs) {
    const int64_t mine = (r.n + kChunk - 1) / kChunk;
    if (t.count == RUNS || chunks + mine > INT32_MAX / 2) NGT_CHECK_OK(flush());
    const int c = t.count++;
    char* out = r.out ? r.out : r.x;
    t.x[c] = r.x;
    if constexpr (OUT) t.out[c] = out;
    t.first[c] = static_cast<int32_t>(chunks);
    t.tail[c] = static_cast<uint16_t>(r.n - (mine - 1) * kChunk);
    const bool wide = !((reinterpret_cast<uintptr_t>(r.x) | (OUT ? reinterpret_cast<uintptr_t>(out) : 0)) & 15);
    t.kind[c] = static_cast<uint8_t>((r.dtype == NGT_BF16) | (r.out_dtype == NGT_BF16) << 1 | wide << 2);
    chunks += mine;
  }
  return flush();
}

// As many blocks as share the chunks evenly.
int32_t blocks_of(int32_t chunks) {
  const int32_t rounds = (chunks + kBlocks - 1) / kBlocks;
  return (chunks + rounds - 1) / rounds;
}

int32_t parts_of(const std::vector<Run>& runs) {
  int32_t parts = 0;
  each_launch<kRuns, false>(runs, [&](const TableIn&, int32_t chunks) {
    parts += blocks_of(chunks);
    return NGT_OK;
  });
  return parts;
}

}  // namespace
}  // namespace ngt

using namespace ngt;

extern "C" int ngt_clip_workspace_bytes(const ngt_gradient* tensors, int32_t n_tensors,
                                        size_t* bytes) try {
  const char* fn = "ngt_clip_workspace_bytes";
  NGT_CHECK_OK(check(fn, tensors, n_tensors));
  if (!bytes) return set_error(NGT_ERR_ARG, "%s: null bytes", fn);
  *bytes = 16 + parts_of(runs_of(tensors, n_tensors)) * sizeof(double);
  return NGT_OK;
} catch (const std::bad_alloc&) {
  return set_error(NGT_ERR_ARG, "ngt_clip_workspace_bytes: out of host memory");
}

extern "C" int ngt_clip_gradients(const ngt_gradient* tensors, int32_t n_tensors, double max_norm,
                                  float* norm, void* workspace, size_t workspace_bytes,
                                  void* stream) try {
  const char* fn = "ngt_clip_gradients";
  NGT_CHECK_OK(check(fn, tensors, n_tensors));
  if (max_norm != max_norm) return set_error(NGT_ERR_ARG, "%s: max_norm is not a number", fn);
  if (!norm) return set_error(NGT_ERR_ARG, "%s: null norm", fn);
  const std::vector<Run> runs = runs_of(tensors, n_tensors);
  const int32_t parts = parts_of(runs);
  const size_t need = 16 + parts * sizeof(double);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu or not 16-byte aligned", fn,
                     workspace_bytes, need);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto* factor = static_cast<Factor*>(workspace);
  double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
  int32_t done = 0;
  NGT_CHECK_OK((each_launch<kRuns, false>(runs, [&](const TableIn& t, int32_t chunks) -> int {
    KernelTimer timer_("clip_squares", st);
    const int32_t blocks = blocks_of(chunks);
    hipLaunchKernelGGL(k_squares, dim3(unsigned(blocks)), dim3(kThreads), 0, st, t, part + done);
    NGT_HIP_CHECK(hipGetLastError());
    done += blocks;
    return NGT_OK;
  })));
  const bool apart = max_norm < 0.0 || parts > kJoined || parts == 0;
  if (apart) {
    KernelTimer timer_("clip_norm", st);
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(1024), 0, st, part, parts,
                       max_norm < 0.0 ? INFINITY : max_norm, norm, factor);
    NGT_HIP_CHECK(hipGetLastError());
  }
  if (max_norm < 0.0) return NGT_OK;
  bool first = true;
  auto scale = [&](const auto& t, int32_t chunks) -> int {
    using T = std::decay_t<decltype(t)>;
    KernelTimer timer_("clip_scale", st);
    hipLaunchKernelGGL(k_scale<T>, dim3(unsigned(blocks_of(chunks))), dim3(kThreads), 0, st, t, part,
                       apart ? 0 : parts, max_norm, first && !apart ? norm : nullptr, factor);
    NGT_HIP_CHECK(hipGetLastError());
    first = false;
    return NGT_OK;
  };
  // in place and apart from it
  std::vector<Run> in, out;
  for (const Run& r : runs) (r.out && r.out != r.x ? out : in).push_back(r);
  NGT_CHECK_OK((each_launch<kRunsOut, true>(out, scale)));
  return each_launch<kRuns, false>(in, scale);
} catch (const std::bad_alloc&) {
  return set_error(NGT_ERR_ARG, "ngt_clip_gradients: out of host memory");
}
