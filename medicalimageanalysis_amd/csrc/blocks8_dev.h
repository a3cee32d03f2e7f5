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

// top: a finite magnitude.  448 = 1.75 * 2^8: a mantissa above 0x600000 carries into the exponent field.
__device__ __forceinline__ int b8_exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = (int)((u + 0x1fffffu) >> 23) - 127 - 8;
  return u == 0 ? 0 : e < B8_EMIN ? B8_EMIN : e > B8_EMAX ? B8_EMAX : e;
}
// Two values already divided by the block's 2^e -> two bytes (low half), rounded to nearest even.  Nothing finite is above 448
// then but a bound of softplus8, by a few 2^-20, which the conversion rounds to 448, and with e = 119, the largest, where
// b8_cut brings it down first; infinities and NaN become NaN.
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
// ---- softplus into blocks -----------------------------------------------------------------------------------------

// In 32 bits: log(1 + u), u = exp(-|t|) from the hardware's exponential (1 unit in the last place), as u times a polynomial
// of degree 7 in u: the best one on [0, 1] by relative error (an exchange fit), 2e-7, with its roundings 3.4e-7.
// beta, t = beta h and t log2(e) are rounded, 3 * 2^-24 |t| in the exponential's argument, which counts in full for
// negative t only (for positive t its share is |t| exp(-t) <= 0.37 of that).  With the exponential's 1.2e-7 and the
// roundings of 1 / beta, its product and the bounds (2^-24 each) the result is off by less than softplus_margin relative to
// its value: 8e-7 + 2e-7 |t|.  (Over all floats with |t| < 87 and five betas it is off by 4.0e-7 + 1.2e-7 |t|.)  Results of
// exponentials below 2^-126 are 0.
__device__ __forceinline__ float softplus32(float h, float beta, float inv_beta) {
  const float t = beta * h;
  const float u = __builtin_amdgcn_exp2f(-fabsf(t) * 1.44269504f);
  float s = -0.00853920821f;
  s = fmaf(s, u, 0.044089634f);
  s = fmaf(s, u, -0.107681714f);
  s = fmaf(s, u, 0.177452415f);
  s = fmaf(s, u, -0.244954631f);
  s = fmaf(s, u, 0.332754791f);
  s = fmaf(s, u, -0.499974042f);
  s = fmaf(s, u, 0.999999821f);
  return fmaf(u, s, __builtin_amdgcn_fmed3f(t, 0.0f, __builtin_inff())) * inv_beta;  // (a NaN is in u)
}
// (below t = -88 there is nothing left to be off, down to -inf, the fill of short rows)
__device__ __forceinline__ float softplus_margin(float h, float beta) {
  return fmaf(__builtin_amdgcn_fmed3f(-beta * h, 0.0f, 88.0f), 2e-7f, 8e-7f);
}

// exp in 64 bits, t <= 1: t = n ln 2 + r, |r| <= 0.35, and the power series of exp(r) to r^13 (the next term is under
// 5e-18).  Below -1000, down to -inf, it is 0; n ln 2 would leave no digits of r there.
__device__ __forceinline__ double exp64(double t) {
  t = ::fmax(t, -1000.0);
  const double n = ::rint(t * 1.4426950408889634);
  const double r = ::fma(-n, 2.3190468138462996e-17, ::fma(-n, 0.69314718055994531, t));
  double s = 1.0 / 6227020800.0;
  s = ::fma(s, r, 1.0 / 479001600.0);
  s = ::fma(s, r, 1.0 / 39916800.0);
  s = ::fma(s, r, 1.0 / 3628800.0);
  s = ::fma(s, r, 1.0 / 362880.0);
  s = ::fma(s, r, 1.0 / 40320.0);
  s = ::fma(s, r, 1.0 / 5040.0);
  s = ::fma(s, r, 1.0 / 720.0);
  s = ::fma(s, r, 1.0 / 120.0);
  s = ::fma(s, r, 1.0 / 24.0);
  s = ::fma(s, r, 1.0 / 6.0);
  s = ::fma(s, r, 0.5);
  s = ::fma(s, r, 1.0);
  s = ::fma(s, r, 1.0);
  return ::ldexp(s, (int)n);
}
// softplus to 40 bits and more, for the few values that lie next to a rounding border (see softplus8).
// l = log(1 + u), u = exp(-|t|): for small u its series; else from the 32-bit l0, with d = (1 + u) exp(-l0) - 1 under 1e-5,
// l = l0 + log(1 + d) = l0 + d - d^2 / 2 + d^3 / 3.
static __device__ __noinline__ double softplus64(double h, double beta) {
  const double t = beta * h;
  const double u = exp64(-::fabs(t));
  double l;
  if (u < 1.0 / 4096) {
    l = u * ::fma(u, ::fma(u, ::fma(u, -0.25, 1.0 / 3), -0.5), 1.0);
  } else {
    const double l0 = (double)(0.69314718f * __builtin_amdgcn_logf((float)(1.0 + u)));
    const double d = ::fma(1.0 + u, exp64(-l0), -1.0);
    l = l0 + d * ::fma(d, ::fma(d, 1.0 / 3, -0.5), 1.0);
  }
  return ((t > 0 ? t : 0) + l) / beta;
}

// a double in [0, 448] -> the float from which a second rounding to fewer bits gives what one rounding of the double
// would: truncated, with the last bit set if anything was cut off
__device__ __forceinline__ float round_to_odd(double d) {
  float f = (float)d;
  if ((double)f != d) {
    uint32_t u = __float_as_uint(f);
    if ((double)f > d) --u;
    f = __uint_as_float(u | 1u);
  }
  return f;
}

// the exponent and the scaled elements of a block that sixteen lanes hold, 8 elements each
__device__ __forceinline__ int scale8(float (&h)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = larger(top, b8_size(h[i]));
  top = lane_max<16>(top);
  if (top >= B8_INF) {  // some are not finite: the largest of the others
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = b8_size(h[i]) < B8_INF ? larger(top, b8_size(h[i])) : top;
    top = lane_max<16>(top);
  }
  const int e = b8_exponent(__uint_as_float(top));
  const float inv = b8_pow2(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] *= inv;
  if (e == B8_EMAX) {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = b8_cut(h[i]);
  }
  return e;
}

// One element the exact way: softplus(x) / 2^e, ready for the conversion
static __device__ __noinline__ float softplus_scaled(float x, double beta, int e) {
  if (!(x < __builtin_inff())) return __builtin_nanf("");
  return round_to_odd(::fmin(softplus64((double)x, beta) * ::ldexp(1.0, -e), 448.0));
}

// The block of softplus(h).  Which of two neighbouring 8-bit values is nearest to softplus(h) can hang on its last bits,
// so a value is computed in 32 bits, and once more in 64 where its 32-bit error could change the result (some twenty of
// a million; of 16-bit inputs, which repeat, it can be more): the bytes are those of the softplus computed in 64 bits.  (A
// large h is its own softplus, and as the middle of two 8-bit values goes to either: beta h / beta is h but for its last
// bit.)
__device__ __forceinline__ uint2 softplus8(const float (&h)[8], float beta, float inv_beta, double beta64, int& e_out) {
  constexpr float INF = __builtin_inff();
  // softplus grows with h: the block's largest comes from the largest h.  As integers the bits of floats order like them
  // from zero up; if none is there, the largest is the negative one with the smallest bits.
  int most = INT32_MIN;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = larger(most, __float_as_int(h[i]));
  most = lane_max<16>(most);
  float top = __int_as_float(most);
  if (most < 0 || most >= (int)B8_INF) {
    top = -INF;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = h[i] < INF && h[i] > top ? h[i] : top;  // (neither infinity nor NaN)
    top = lane_max<16>(top);
  }
  float at = softplus32(top, beta, inv_beta);
  if (beta > 1.0f && !(at < INF)) at = top;  // beta h is beyond 32 bits, softplus(h) is h to its last bit
  const float mt = softplus_margin(top, beta);
  const float most32 = 3.4e38f;
  int e = b8_exponent(at < most32 ? at * (1.0f - mt) : most32);
  const int above = b8_exponent(at < most32 ? at * (1.0f + mt) : most32);
  if (e != above && softplus64((double)top, beta64) > 448.0 * ::ldexp(1.0, e)) e = above;
  if (top == -INF) e = 0;
  e_out = e;
  const float scale = inv_beta * b8_pow2(-e);
  // With a beta above 1 beta h, with one below 2^-17 2^-e / beta may be beyond 32 bits where the elements are not.  (beta is
  // the launch's: the usual ones skip the test.)
  bool exact = e == B8_EMAX;
  if (beta > 1.0f || beta < 0x1p-17f) exact |= !(larger(beta * top, scale) < INF);
  float lo[8], hi[8], least = h[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) least = fminf(least, h[i]);
  const float m = softplus_margin(least, beta);  // (the largest of the eight)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = softplus32(h[i], beta, scale);
    lo[i] = fmaf(a, -m, a);
    hi[i] = fmaf(a, m, a);
  }
  uint32_t w[2] = {b8_pack4(lo), b8_pack4(lo + 4)};
  const uint32_t x[2] = {w[0] ^ b8_pack4(hi), w[1] ^ b8_pack4(hi + 4)};
  if ((x[0] | x[1]) != 0 || exact) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = 8 * (i & 3);
      if ((x[i >> 2] >> at & 0xff) != 0 || exact) {
        const float v = softplus_scaled(h[i], beta64, e);
        w[i >> 2] = (w[i >> 2] & ~(0xffu << at)) | (b8_pack2(v, v) & 0xff) << at;
      }
    }
  }
  return uint2{w[0], w[1]};
}

// d softplus / dh from the kept a = softplus(h): sigmoid(beta h) = 1 - exp(-z), z = beta a.  For small z a series, else
// from the hardware's exponential (a unit in the last place is 2^-24).  For 32-bit results the series runs to z^8 under
// 1/2 (the rest is under 2e-8 of it) and the difference is at least 0.39; SHORT, for results of 11 bits and fewer: to z^4
// under 1/16 (2e-7), the difference at least 0.06 (1e-6 off at most).
template <bool SHORT>
__device__ __forceinline__ float b8_softplus_slope(float a, float beta) {
  const float z = beta * a;
  float s = 1.0f / 24;
  if constexpr (!SHORT) {
    s = fmaf(z, -1.0f / 40320, 1.0f / 5040);
    s = fmaf(z, -s, 1.0f / 720);
    s = fmaf(z, -s, 1.0f / 120);
    s = fmaf(z, -s, 1.0f / 24);
  }
  s = fmaf(z, -s, 1.0f / 6);
  s = fmaf(z, -s, 0.5f);
  s = fmaf(z, -s, 1.0f);
  return z < (SHORT ? 0.0625f : 0.5f) ? z * s : 1.0f - __builtin_amdgcn_exp2f(z * -1.44269504f);
}

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
