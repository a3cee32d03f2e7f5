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
// Two values already divided by the block's 2^e -> two bytes (low half), rounded to nearest even.  Nothing finite is
// above 448 (1 + 2^-20) then, which the conversion rounds to 448; infinities and NaN become NaN.  (e = 119, the largest,
// is the exception: b8_pack2_top cuts what is above 448.)
__device__ __forceinline__ uint32_t b8_pack2(float a, float b) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
__device__ __forceinline__ float b8_cut(float a) {
  return fabsf(a) < __builtin_inff() ? fminf(fmaxf(a, -448.0f), 448.0f) : __builtin_nanf("");
}
// four values into a word
__device__ __forceinline__ uint32_t b8_pack4(const float* v) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
}
// the largest finite magnitude of a block of rows' elements: its bits as an integer, which order as the numbers do.
// Anything at or above the bits of infinity counts as 0.
__device__ __forceinline__ uint32_t b8_size(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t B8_INF = 0x7f800000u;

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
// vmf_blocks8_quantize of x (m, k) and vmf_blocks8_quantize_tiles of w (n, k), in one launch where both are small
int b8_quantize_both(const void* x, int64_t x_stride, uint8_t* values, uint8_t* exponents, int64_t exp_pitch, int64_t m,
                     int64_t k, int activation, double beta, int dtype, const void* w, int64_t w_stride,
                     uint8_t* w_values, uint8_t* w_exponents, uint8_t* wt_values, uint8_t* wt_exponents, int64_t n,
                     int w_dtype, vmf_stream_t stream);
