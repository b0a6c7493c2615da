// What the linear kernels share: the normal distribution of GELU, and 8-element
// pieces of bf16 rows of any length and alignment.
#pragma once

#include "ngt_packed.h"

namespace ngt {
namespace {

using packed::u32x4;

// gelu(z) = z Phi(z), gelu'(z) = Phi(z) + z phi(z).  For z < 0, without cancellation,
//   Phi(z) = erfc(x) / 2 = (a1 t + .. + a8 t^8) e^(-x^2), x = |z| / sqrt 2, t = 1 / (1 + p x)
// and 1 - Phi(-z) above.  p and a1 .. a8 are the minimax fit of the RELATIVE error over x in
// [0, 9.6] (Remez exchange): 8.2e-8, and with the roundings 5e-7 down to z = -1, 3e-6 to -8
// and 8e-6 to -13, where a half step of a bf16 result is 2^-8 of it.  (A form with 1.5e-7 of
// ABSOLUTE error was off by 1.6e-3 of the result at z = -5, 1e-2 at -8 and 3.7e-2 at -13.)
// Below -13.2 the exponential underflows and the result is 0.
struct Normal {
  float cdf, pdf;  // pdf times sqrt(2 pi)
};
__device__ __forceinline__ Normal normal(float z) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.33f, x, 1.f));
  const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  float p = fmaf(-0.06796437f, t, 0.23134395f);
  p = fmaf(p, t, -0.1777192f);
  p = fmaf(p, t, 0.20627058f);
  p = fmaf(p, t, 0.022505442f);
  p = fmaf(p, t, 0.10096188f);
  p = fmaf(p, t, 0.09141863f);
  p = fmaf(p, t, 0.093183056f);
  const float h = p * t * e;
  return {z < 0.f ? h : 1.f - h, e};
}

struct __attribute__((packed, aligned(2))) Loose16 {
  u32x4 w;
};

// 8 elements at column c of a row of n: whole pieces in one access (any 2-byte
// alignment without ALIGNED), what is behind the row as zeros.
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load8(const uint16_t* __restrict__ row, int c, int n) {
  if constexpr (ALIGNED) {
    if (c < n) return *reinterpret_cast<const u32x4*>(row + c);
    return u32x4{0u, 0u, 0u, 0u};
  } else {
    if (c + 8 <= n) return reinterpret_cast<const Loose16*>(row + c)->w;
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) v[i / 2] |= uint32_t(row[c + i]) << (16 * (i & 1));
    return v;
  }
}

__device__ __forceinline__ float half_of(const u32x4& v, int i) {
  const uint32_t w = v[i / 2];
  return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
}

// 64 pieces of a wave from memory to LDS, one after another from `at`.
__device__ __forceinline__ void to_lds(packed::Buffer b, int offset, char* at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      b, (__attribute__((address_space(3))) void*)at, 16, offset, 0, 0, 0);
}
// Until at most N of this wave's reads from memory are under way.
template <int N>
__device__ __forceinline__ void wait_for_all_but() {
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace ngt
