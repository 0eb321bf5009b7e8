// kd_float16.hpp -- the 16-bit float types of the surface-embedding kernels, their conversions and
// small aligned packs for vector loads and stores.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kd {

typedef _Float16 half_t;
typedef __bf16 bfloat_t;

// the type in which products and sums of T are held
template <typename T>
struct Wide {
  using type = float;
};
template <>
struct Wide<double> {
  using type = double;
};

template <typename T>
__device__ __forceinline__ typename Wide<T>::type to_wide(T x) {
  return (typename Wide<T>::type)x;
}
template <typename T>
__device__ __forceinline__ T from_wide(typename Wide<T>::type x) {
  return (T)x;  // to nearest, ties to even
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

}  // namespace kd
