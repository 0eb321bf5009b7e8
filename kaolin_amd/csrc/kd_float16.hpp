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

// N elements at any element's address: 16-byte loads and stores here need no alignment.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[N];
};

// the first `n` of N elements (n < N only at the end of a row)
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p, int n) {
  if (n >= N) return *(const Pack<T, N> *)p;
  Pack<T, N> x;
#pragma unroll
  for (int j = 0; j < N; ++j) x.v[j] = j < n ? p[j] : (T)0.f;
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &x, int n) {
  if (n >= N) {
    *(Pack<T, N> *)p = x;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = x.v[j];
  }
}

}  // namespace kd
