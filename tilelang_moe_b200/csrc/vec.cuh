// Vector accesses of element types that the memory-bound kernels share: V bytes at a time as one load or store, elements
// as fp32 in registers; division by a number known on the host.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace moe {

template <int V> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<1> { using type = uint8_t; };
template <int V> using Raw = typename RawOf<V>::type;

template <class T> __device__ __forceinline__ float2 halves(uint32_t w);
template <> __device__ __forceinline__ float2 halves<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 halves<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <class T> __device__ __forceinline__ uint32_t join(float a, float b);
template <> __device__ __forceinline__ uint32_t join<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t join<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// the V / sizeof(T) elements of one vector
template <class T, int V>
__device__ __forceinline__ void unpack(const Raw<V>& r, float (&x)[V / sizeof(T)]) {
  if constexpr (V == 2) {
    x[0] = halves<T>(r).x;
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = halves<T>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
}
template <class T, int V>
__device__ __forceinline__ Raw<V> pack(const float (&x)[V / sizeof(T)]) {
  Raw<V> r;
  if constexpr (V == 2) {
    r = (uint16_t)join<T>(x[0], 0.f);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(x[i]);
      else w[i] = join<T>(x[2 * i], x[2 * i + 1]);
    }
  }
  return r;
}

// widest access (16, 8, 4, 2 or 1 bytes) that these addresses, strides and lengths, ORed together, allow
static inline int vec_bytes(uintptr_t all) {
  int v = 16;
  while (v > 1 && (all & (uintptr_t)(v - 1))) v >>= 1;
  return v;
}

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, PLDI 1994)
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t div) : d(div) {
    for (s = 0; s < 31 && (1u << s) < d; ++s) {}
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

}  // namespace moe
