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

// Reductions over groups of G consecutive lanes (G a power of two, 16 .. 64), the same bits in every lane, in the vector
// unit: inside 16 lanes by rotations (a rotation by half the distance left pairs every lane with one whose sum is over the
// complementary lanes), across them by swaps of 16 and of 32 lanes.
template <int N, typename A>
__device__ __forceinline__ A rotated16(A v) {
  if constexpr (sizeof(A) == 4) {
    union {
      A a;
      int i;
    } u;
    u.a = v;
    u.i = __builtin_amdgcn_update_dpp(0, u.i, 0x120 + N, 0xf, 0xf, true);
    return u.a;
  } else {
    union {
      A a;
      int i[2];
    } u;
    u.a = v;
    u.i[0] = __builtin_amdgcn_update_dpp(0, u.i[0], 0x120 + N, 0xf, 0xf, true);
    u.i[1] = __builtin_amdgcn_update_dpp(0, u.i[1], 0x120 + N, 0xf, 0xf, true);
    return u.a;
  }
}
// The values of the lower and the upper N lanes (N: 16 or 32) of each 2 N: both of them in all 2 N lanes.
template <int N>
__device__ __forceinline__ void halves32(uint32_t v, uint32_t& lower, uint32_t& upper) {
  typedef unsigned pair __attribute__((ext_vector_type(2)));
  pair r;
  if constexpr (N == 16) r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  else r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  lower = r[0];
  upper = r[1];
}
template <int N, typename A>
__device__ __forceinline__ void halves(A v, A& lower, A& upper) {
  constexpr int W = (int)sizeof(A) / 4;
  union {
    A a;
    uint32_t w[W];
  } in, lo, hi;
  in.a = v;
#pragma unroll
  for (int i = 0; i < W; ++i) halves32<N>(in.w[i], lo.w[i], hi.w[i]);
  lower = lo.a;
  upper = hi.a;
}
template <int G, typename A>
__device__ __forceinline__ A lane_sum(A v) {
  v += rotated16<8>(v);
  v += rotated16<4>(v);
  v += rotated16<2>(v);
  v += rotated16<1>(v);
  A lower, upper;
  if constexpr (G > 16) {
    halves<16>(v, lower, upper);
    v = lower + upper;
  }
  if constexpr (G > 32) {
    halves<32>(v, lower, upper);
    v = lower + upper;
  }
  return v;
}
template <typename A>
__device__ __forceinline__ A larger(A a, A b) { return b > a ? b : a; }
template <int G, typename A>
__device__ __forceinline__ A lane_max(A v) {
  v = larger(v, rotated16<8>(v));
  v = larger(v, rotated16<4>(v));
  v = larger(v, rotated16<2>(v));
  v = larger(v, rotated16<1>(v));
  A lower, upper;
  if constexpr (G > 16) {
    halves<16>(v, lower, upper);
    v = larger(lower, upper);
  }
  if constexpr (G > 32) {
    halves<32>(v, lower, upper);
    v = larger(lower, upper);
  }
  return v;
}
