// lowp.h -- what the layer norm and the 8-bit block kernels share: storage types, row access, reductions.
#pragma once
#include "common.h"

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// storage type -> arithmetic type: sums, statistics and products are never held in fewer than 32 bits
template <typename T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

// Launches with T = the storage type of dtype code `code`
#define LOWP_DISPATCH(code, what, T, ...)                                                            \
  do {                                                                                               \
    if ((code) == VMF_F32) { using T = float; __VA_ARGS__; }                                         \
    else if ((code) == VMF_F16) { using T = f16_t; __VA_ARGS__; }                                    \
    else if ((code) == VMF_BF16) { using T = bf16_t; __VA_ARGS__; }                                  \
    else { vmf_set_error(what ": dtype %d is not VMF_F32/VMF_F16/VMF_BF16", (int)(code)); return VMF_ERR_DTYPE; } \
  } while (0)

// N consecutive elements at any address that is a multiple of the element size.  The hardware takes 16-byte accesses at
// such addresses, so rows of an odd width go the same way as aligned ones.
template <typename T, int N> struct Pack {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T> struct Pack<T, 1> { typedef T type; };

template <int N, typename T, typename A>
__device__ __forceinline__ void load_pack(const T* p, A* out) {
  if constexpr (N == 1) {
    out[0] = (A)p[0];
  } else {
    const typename Pack<T, N>::type v = *reinterpret_cast<const typename Pack<T, N>::type*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (A)v[i];
  }
}
template <int N, typename T, typename A>
__device__ __forceinline__ void store_pack(T* p, const A* in) {
  if constexpr (N == 1) {
    p[0] = (T)in[0];
  } else {
    typename Pack<T, N>::type v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)in[i];
    *reinterpret_cast<typename Pack<T, N>::type*>(p) = v;
  }
}
// the first `left` of N elements (left may be <= 0 or >= N); the others read as `fill`
template <int N, typename T, typename A>
__device__ __forceinline__ void load_some(const T* p, int64_t left, A fill, A* out) {
  if (left >= N) {
    load_pack<N>(p, out);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = i < left ? (A)p[i] : fill;
  }
}
template <int N, typename T, typename A>
__device__ __forceinline__ void store_some(T* p, int64_t left, const A* in) {
  if (left >= N) {
    store_pack<N>(p, in);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (T)in[i];
  }
}

// sum over groups of G consecutive lanes (G a power of two <= 64), the same value in every lane
template <int G, typename A>
__device__ __forceinline__ A lane_sum(A v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int G, typename A>
__device__ __forceinline__ A lane_max(A v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const A u = __shfl_xor(v, o, 64);
    v = u > v ? u : v;
  }
  return v;
}
