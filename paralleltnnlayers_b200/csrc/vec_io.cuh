// Values of float, bfloat16 and float16 in groups, as fp32 in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace b200cp {

template <typename T, int N>
struct alignas(sizeof(T) * N) Group {
  T v[N];
};
template <typename T>
__device__ __forceinline__ float to_float(T x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return x;
}
template <typename T, int N>
__device__ __forceinline__ Group<T, N> pack(const float (&x)[N]) {
  Group<T, N> g;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(g.v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __half2 p = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) g.v[i] = from_float<T>(x[i]);
  }
  return g;
}
// (bfloat16 by words: one operation a value, where a value by itself takes two)
template <typename T, int N>
__device__ __forceinline__ void unpack(const Group<T, N>& g, float (&x)[N]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value && N % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(g.v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(g.v[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ Group<T, N> load_group(const T* p) { return *reinterpret_cast<const Group<T, N>*>(p); }
template <typename T, int N>
__device__ __forceinline__ void store_group(T* p, const Group<T, N>& g) { *reinterpret_cast<Group<T, N>*>(p) = g; }

// values of a type that 16 bytes hold
template <typename T>
constexpr int kPerLoad = 16 / (int)sizeof(T);
// whether rows of n values from p on can be read 16 bytes at a time
template <typename T>
inline bool rows_of_16(const void* p, long long n) { return !(reinterpret_cast<uintptr_t>(p) & 15) && n % kPerLoad<T> == 0; }

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

}  // namespace b200cp
