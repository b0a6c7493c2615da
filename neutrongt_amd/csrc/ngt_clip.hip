// The 2-norm over many gradients and their scaling to a largest norm:
//   norm = sqrt(sum g^2),  g <- g min(1, max_norm / norm).
// Bound by memory: all gradients are read once for the norm and, where they are to be
// scaled, read and written once more.  The tensors' addresses go in the launch's arguments
// (kTensors a launch), so a captured graph holds them and no table is copied.
// Squares and sums are fp64: exact squares of fp32, no overflow, and a sum over any
// number of elements that does not depend on how they are cut.
#include "ngt_common.h"

namespace ngt {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 96;      // a launch
constexpr int kChunk = 16384;     // elements of a tensor that a block takes at a time
constexpr int kBlocks = 1024;     // most of a launch

struct Table {
  void* x[kTensors];
  void* out[kTensors];
  int64_t n[kTensors];
  int32_t first[kTensors + 1];  // chunks before a tensor's
  uint8_t kind[kTensors];       // bits 0, 1: x, out is bf16; bit 2: 16-byte accesses
  int32_t count;
};

// The tensor of a chunk: the last whose first chunk is not behind it.
__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v, double* red) {
  for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < int(blockDim.x) / kWave; ++i) v += red[i];
  return v;
}

template <typename T>
__device__ __forceinline__ double squares(const void* base, int64_t from, int64_t to, bool wide) {
  const T* x = static_cast<const T*>(base);
  double s = 0.0;
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  int64_t i = from;
  if (wide) {
    for (i += threadIdx.x * V; i + V <= to; i += kThreads * V) {
      float v[V];
      load_row<T, V>(x + i, v);
#pragma unroll
      for (int k = 0; k < V; ++k) s = fma(double(v[k]), double(v[k]), s);
    }
    i = to - (to - from) % V;  // what is left, an element a thread
  }
  for (i += threadIdx.x; i < to; i += kThreads) {
    const double v = elem<T>::load(x + i);
    s = fma(v, v, s);
  }
  return s;
}

// part[block]: the sum of the squares of the block's chunks.
__global__ __launch_bounds__(kThreads) void k_squares(const Table t, double* __restrict__ part) {
  __shared__ double red[kThreads / kWave];
  double s = 0.0;
  for (int chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
    const int i = tensor_of(t, chunk);
    const int64_t from = int64_t(chunk - t.first[i]) * kChunk;
    const int64_t to = from + kChunk < t.n[i] ? from + kChunk : t.n[i];
    const bool wide = t.kind[i] & 4;
    s += t.kind[i] & 1 ? squares<bf16_t>(t.x[i], from, to, wide)
                       : squares<float>(t.x[i], from, to, wide);
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm, and the factor of the gradients.
__global__ __launch_bounds__(1024) void k_norm(const double* __restrict__ part, int32_t n,
                                               double max_norm, float* __restrict__ norm,
                                               float* __restrict__ factor) {
  __shared__ double red[1024 / kWave];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
  s = sqrt(block_sum(s, red));
  if (threadIdx.x != 0) return;
  *norm = static_cast<float>(s);
  const bool finite = s < INFINITY;
  *factor = finite && s > max_norm ? static_cast<float>(max_norm / s) : 1.f;
}

template <typename T, typename O>
__device__ __forceinline__ void scaled(const void* base, void* result, int64_t from, int64_t to,
                                       bool wide, float by) {
  const T* x = static_cast<const T*>(base);
  O* o = static_cast<O*>(result);
  constexpr int V = sizeof(T) == 2 && sizeof(O) == 2 ? 8 : 4;
  int64_t i = from;
  if (wide) {
    for (i += threadIdx.x * V; i + V <= to; i += kThreads * V) {
      float v[V];
      if constexpr (sizeof(T) == 2 && V == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(x + i);
        v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xffff0000u);
      } else {
        load_row<T, V>(x + i, v);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] *= by;
      if constexpr (sizeof(O) == 2 && V == 4)
        *reinterpret_cast<uint2*>(o + i) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
      else
        store_row<O, V>(o + i, v);
    }
    i = to - (to - from) % V;
  }
  for (i += threadIdx.x; i < to; i += kThreads) elem<O>::store(o + i, elem<T>::load(x + i) * by);
}

__global__ __launch_bounds__(kThreads) void k_scale(const Table t, const float* __restrict__ factor) {
  const float by = *factor;
  for (int chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
    const int i = tensor_of(t, chunk);
    if (by == 1.f && t.out[i] == t.x[i]) continue;
    const int64_t from = int64_t(chunk - t.first[i]) * kChunk;
    const int64_t to = from + kChunk < t.n[i] ? from + kChunk : t.n[i];
    const bool wide = t.kind[i] & 4;
    switch (t.kind[i] & 3) {
      case 0: scaled<float, float>(t.x[i], t.out[i], from, to, wide, by); break;
      case 1: scaled<bf16_t, float>(t.x[i], t.out[i], from, to, wide, by); break;
      case 2: scaled<float, bf16_t>(t.x[i], t.out[i], from, to, wide, by); break;
      default: scaled<bf16_t, bf16_t>(t.x[i], t.out[i], from, to, wide, by); break;
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

// The tables of the launches, one after another: f(table, chunks).
template <typename F>
int each_launch(const ngt_gradient* g, int32_t n, F f) {
  Table t;
  t.count = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (t.count == 0) return NGT_OK;
    t.first[t.count] = static_cast<int32_t>(chunks);
    const int rc = f(t, static_cast<int32_t>(chunks));
    t.count = 0, chunks = 0;
    return rc;
  };
  for (int32_t i = 0; i < n; ++i) {
    if (g[i].n == 0) continue;
    const int64_t mine = (g[i].n + kChunk - 1) / kChunk;
    if (t.count == kTensors || chunks + mine > INT32_MAX / 2) NGT_CHECK_OK(flush());
    const int c = t.count++;
    t.x[c] = g[i].x;
    t.out[c] = g[i].out ? g[i].out : g[i].x;
    t.n[c] = g[i].n;
    t.first[c] = static_cast<int32_t>(chunks);
    const int32_t od = g[i].out ? g[i].out_dtype : g[i].dtype;
    const bool wide = !((reinterpret_cast<uintptr_t>(t.x[c]) | reinterpret_cast<uintptr_t>(t.out[c])) & 15);
    t.kind[c] = static_cast<uint8_t>((g[i].dtype == NGT_BF16) | (od == NGT_BF16) << 1 | wide << 2);
    chunks += mine;
  }
  return flush();
}

int32_t blocks_of(int32_t chunks) { return chunks < kBlocks ? chunks : kBlocks; }

size_t bytes_of(const ngt_gradient* g, int32_t n) {
  size_t parts = 0;
  each_launch(g, n, [&](const Table&, int32_t chunks) {
    parts += blocks_of(chunks);
    return NGT_OK;
  });
  return 16 + parts * sizeof(double);
}

}  // namespace
}  // namespace ngt

using namespace ngt;

extern "C" int ngt_clip_workspace_bytes(const ngt_gradient* tensors, int32_t n_tensors,
                                        size_t* bytes) {
  const char* fn = "ngt_clip_workspace_bytes";
  NGT_CHECK_OK(check(fn, tensors, n_tensors));
  if (!bytes) return set_error(NGT_ERR_ARG, "%s: null bytes", fn);
  *bytes = bytes_of(tensors, n_tensors);
  return NGT_OK;
}

extern "C" int ngt_clip_gradients(const ngt_gradient* tensors, int32_t n_tensors, double max_norm,
                                  float* norm, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const char* fn = "ngt_clip_gradients";
  NGT_CHECK_OK(check(fn, tensors, n_tensors));
  if (max_norm != max_norm) return set_error(NGT_ERR_ARG, "%s: max_norm is not a number", fn);
  if (!norm) return set_error(NGT_ERR_ARG, "%s: null norm", fn);
  const size_t need = bytes_of(tensors, n_tensors);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(NGT_ERR_WORKSPACE, "%s: workspace %zu < %zu or not 16-byte aligned", fn,
                     workspace_bytes, need);
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* factor = static_cast<float*>(workspace);
  double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
  int32_t parts = 0;
  NGT_CHECK_OK(each_launch(tensors, n_tensors, [&](const Table& t, int32_t chunks) -> int {
    KernelTimer timer_("clip_squares", st);
    const int32_t blocks = blocks_of(chunks);
    hipLaunchKernelGGL(k_squares, dim3(unsigned(blocks)), dim3(kThreads), 0, st, t, part + parts);
    NGT_HIP_CHECK(hipGetLastError());
    parts += blocks;
    return NGT_OK;
  }));
  {
    KernelTimer timer_("clip_norm", st);
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(1024), 0, st, part, parts,
                       max_norm < 0.0 ? INFINITY : max_norm, norm, factor);
    NGT_HIP_CHECK(hipGetLastError());
  }
  if (max_norm < 0.0) return NGT_OK;
  return each_launch(tensors, n_tensors, [&](const Table& t, int32_t chunks) -> int {
    KernelTimer timer_("clip_scale", st);
    hipLaunchKernelGGL(k_scale, dim3(unsigned(blocks_of(chunks))), dim3(kThreads), 0, st, t, factor);
    NGT_HIP_CHECK(hipGetLastError());
    return NGT_OK;
  });
}
