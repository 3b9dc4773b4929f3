// 8-element vector accesses and base-2 exponentials shared by the
// memory-bound kernels.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace msb {
namespace {

template <typename T>
struct alignas(16) Pack8 {
  T v[8];
};

// 2^x on the special-function unit; e^x = 2^(x * log2(e))
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / x to 1 unit in the last place
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that is NaN where either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// two fp32 operations in one instruction
__device__ __forceinline__ unsigned long long bits_of(float2 v) {
  return (unsigned long long)__float_as_uint(v.y) << 32 | __float_as_uint(v.x);
}
__device__ __forceinline__ float2 pair_of(unsigned long long b) {
  return make_float2(__uint_as_float((unsigned)b), __uint_as_float((unsigned)(b >> 32)));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
  return pair_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(d);
}

// 8-element accesses: one 16-byte transaction when the address allows it,
// element-wise otherwise.  Parameters are views into a flat arena at
// arbitrary element offsets, so weights and biases need not be aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    Pack8<T> r = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = to_f32(r.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = to_f32(p[k]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    Pack8<T> r;
#pragma unroll
    for (int k = 0; k < 8; ++k) r.v[k] = from_f32<T>(f[k]);
    *reinterpret_cast<Pack8<T>*>(p) = r;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) p[k] = from_f32<T>(f[k]);
  }
}

// 8 16-bit values as one 16-byte quad of registers, unpacked and packed two
// at a time (a bf16 is the upper half of an fp32; element 0 is the low half
// of the first word), so packed rows take 4 registers per 8 values.
template <typename T>
__device__ __forceinline__ void unpack_u4(const uint4& r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * q] = __uint_as_float(w[q] << 16);
      f[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[q]));
      f[2 * q] = v.x;
      f[2 * q + 1] = v.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack_u4(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * q], f[2 * q + 1]);
      w[q] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
      w[q] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// n / d for 0 <= n < 2^31 by a multiplication: m = ceil(2^p / d) with
// p = 31 + ceil(log2 d) gives floor(n m / 2^p) = floor(n / d) there (Granlund
// and Montgomery 1994).  A 64-bit division costs more than the rest of a
// streaming kernel's loop.
struct FastDiv {
  unsigned d, m, s;
  explicit FastDiv(unsigned d_) : d(d_), m(0), s(0) {
    while ((1u << s) < d) ++s;
    if (s > 0) m = (unsigned)(((1ull << (31 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ unsigned div(unsigned n) const {
    return s == 0 ? n : __umulhi(n, m) >> (s - 1);
  }
};

}  // namespace
}  // namespace msb
