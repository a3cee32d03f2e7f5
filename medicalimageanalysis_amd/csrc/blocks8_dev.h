// blocks8_dev.h -- the 8-bit block format on the device.
//
// A block is 128 consecutive elements of a row (or, for a weight matrix, a tile of 128 x 128): 8-bit e4m3 values and
// one exponent e, kept as the byte e + 127; an element is value * 2^e.  e is the smallest integer with
// 448 * 2^e >= the largest finite magnitude, inside [-110, 119]: with the lower end every element is a normal bf16 and
// fp32 number (the smallest value is 2^-9), with the upper end none overflows.  A power-of-two scale makes the scaling
// exact, in the quantiser, in the conversion back and in the matrix instruction, which takes the byte as it is.
// NaN and infinities are kept as NaN and take no part in the exponent; a block of zeros has e = 0.
// Values: row-major bytes, rows padded with zeros to a multiple of 128.  Exponents: [block column][row].
#pragma once
#include <utility>

#include "lowp.h"

constexpr int B8 = 128;
constexpr int B8_EMIN = -110, B8_EMAX = 119;

__device__ __forceinline__ float b8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// the stored byte is the exponent field of 2^e
__device__ __forceinline__ float b8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// top: a finite magnitude
__device__ __forceinline__ int b8_exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u == 0) return 0;
  // 448 = 1.75 * 2^8
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < B8_EMIN ? B8_EMIN : e > B8_EMAX ? B8_EMAX : e;
}
// two values already divided by 2^e -> two bytes (low half), round to nearest even; NaN stays NaN
__device__ __forceinline__ uint32_t b8_pack2(float a, float b) {
  const float ca = a != a ? a : __builtin_amdgcn_fmed3f(a, -448.0f, 448.0f);
  const float cb = b != b ? b : __builtin_amdgcn_fmed3f(b, -448.0f, 448.0f);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(ca, cb, 0, false) & 0xffffu;
}
// the four elements of a word
__device__ __forceinline__ void b8_unpack4(uint32_t w, float scale, float* out) {
  out[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale;
  out[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale;
  out[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale;
  out[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale;
}
// d softplus / dh from the kept a = softplus(h): sigmoid(beta h) = 1 - exp(-beta a)
__device__ __forceinline__ float b8_softplus_slope(float a, float beta) { return -expm1f(-beta * a); }

// f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>)
template <typename F, int... I>
__device__ __forceinline__ void static_for_(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_(f, std::make_integer_sequence<int, N>{});
}

// ---- host side -----------------------------------------------------------------------------------------------
static inline int64_t b8_blocks(int64_t width) { return (width + B8 - 1) / B8; }
int b8_check_shape(const char* what, int64_t rows, int64_t width);
