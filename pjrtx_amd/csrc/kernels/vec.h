// Vector loads and stores of tensor elements as floats. Rows of any length
// start at any element, so a vector is aligned to its element only (global
// memory takes 16 bytes at any address).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pjrtx {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// kVec elements of T are 16 bytes.
template <typename T>
constexpr int kVecElems = 16 / (int)sizeof(T);

template <typename T>
struct Vec {
  typedef T type __attribute__((ext_vector_type(kVecElems<T>)));
  typedef type unaligned __attribute__((aligned(sizeof(T))));
};

// Tensors of at least this size are read and written past the caches' lines
// that others use (kStream below): they do not stay in an L2 anyway.
constexpr int64_t kStreamBytes = int64_t(32) << 20;

// Elements [0, n) of the vector at p, the others `fill`. n >= kVecElems is the
// common case: one load.
template <typename T, bool kStream = false>
__device__ __forceinline__ typename Vec<T>::type load_vec(const T* p, int64_t n, T fill) {
  if (n >= kVecElems<T>) {
    const auto* at = reinterpret_cast<const typename Vec<T>::unaligned*>(p);
    if constexpr (kStream) return __builtin_nontemporal_load(at);
    else return *at;
  }
  typename Vec<T>::type v;
#pragma unroll
  for (int e = 0; e < kVecElems<T>; ++e) v[e] = e < n ? p[e] : fill;
  return v;
}

template <typename T, bool kStream = false>
__device__ __forceinline__ void store_vec(T* p, int64_t n, const typename Vec<T>::type& v) {
  if (n >= kVecElems<T>) {
    auto* at = reinterpret_cast<typename Vec<T>::unaligned*>(p);
    if constexpr (kStream) __builtin_nontemporal_store(v, at);
    else *at = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < kVecElems<T>; ++e)
    if (e < n) p[e] = v[e];
}

// N dwords at p, which is aligned to an element only, and not a byte past them:
// a vector of 3 may be read as one of 4, and the last row's ends the memory.
template <int N>
__host__ __device__ __forceinline__ void load_words(const void* p, uint32_t* w) {
  typedef uint32_t one __attribute__((aligned(2)));
  if constexpr (N == 1) {
    w[0] = *static_cast<const one*>(p);
  } else if constexpr (N == 3) {
    load_words<2>(p, w);
    load_words<1>(static_cast<const one*>(p) + 2, w + 2);
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(N)));
    typedef words unaligned __attribute__((aligned(2)));
    static_assert(sizeof(words) == 4 * N, "as many bytes as words");
    const words v = *static_cast<const unaligned*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = v[i];
  }
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) x += __shfl_xor(x, k);
  return x;
}
// NaN where any lane's is.
__device__ __forceinline__ float wave_max_nan(float x) {
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) x = __builtin_elementwise_maximum(x, __shfl_xor(x, k));
  return x;
}

}  // namespace pjrtx
