// N elements of fp32, bf16 or fp16 as they lie in memory, moved by one access and widened where they are used.  Held as 32-bit words: an array of 16-bit elements
// would be taken apart into a register per element as soon as it is loaded.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace q38 {

template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T, int N> struct alignas(N * sizeof(T)) Pack { uint32_t w[N * sizeof(T) / 4]; };
template <> struct Pack<__nv_bfloat16, 1> { __nv_bfloat16 v; };
template <> struct Pack<__half, 1> { __half v; };

template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, N>*>(p); }
template <typename T, int N> __device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& v) { *reinterpret_cast<Pack<T, N>*>(p) = v; }

template <typename T, int N> __device__ __forceinline__ void unpack(const Pack<T, N>& p, float (&v)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(p.w[i]);
  } else if constexpr (N == 1) {
    v[0] = to_float(p.v);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) { v[2 * i] = __uint_as_float(p.w[i] << 16); v[2 * i + 1] = __uint_as_float(p.w[i] & 0xffff0000u); }
      else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p.w[i])); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
  }
}
// Rounded to nearest, ties to even
template <typename T, int N> __device__ __forceinline__ Pack<T, N> pack(const float (&v)[N]) {
  Pack<T, N> p;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) p.w[i] = __float_as_uint(v[i]);
  } else if constexpr (N == 1) {
    p.v = from_float<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) { const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); p.w[i] = *reinterpret_cast<const uint32_t*>(&h); }
      else { const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]); p.w[i] = *reinterpret_cast<const uint32_t*>(&h); }
    }
  }
  return p;
}

// Hides from the compiler that `p` is what it was: without this it keeps the widened values from one use to the next, which takes the registers that packing saves.
template <typename T, int N> __device__ __forceinline__ void forget(Pack<T, N>& p) {
  if constexpr (N > 1) {
#pragma unroll
    for (int i = 0; i < int(N * sizeof(T) / 4); ++i) asm volatile("" : "+r"(p.w[i]));
  }
}

}  // namespace q38
