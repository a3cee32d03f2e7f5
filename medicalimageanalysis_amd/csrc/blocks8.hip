// blocks8.hip -- into and out of 8-bit blocks: quantisation of rows (of x or of softplus(x)) and of weight tiles,
// conversion back, the gradient through a softplus whose result was kept in blocks.  All are HBM streams.
#include "blocks8_dev.h"

namespace {

// softplus in 64 bits, for the few values that lie next to a rounding border (see below)
__device__ __noinline__ double softplus64(double h, double beta) {
  const double t = beta * h;
  return ((t > 0 ? t : 0) + ::log1p(::exp(-::fabs(t)))) / beta;
}
// In 32 bits: off by at most softplus_margin relative to the value.  exp and log1p of the library are within 2 units in
// the last place, the sum and the product add one each, and beta and t = beta h are rounded: 2 * 2^-24 * |t| in the
// argument of exp, which counts in full for negative t only (for positive t its share is |t| exp(-t) <= 0.37 of that).
__device__ __forceinline__ float softplus32(float h, float beta, float inv_beta) {
  const float t = beta * h;
  return (fmaxf(t, 0.0f) + log1pf(expf(-fabsf(t)))) * inv_beta;
}
__device__ __forceinline__ float softplus_margin(float h, float beta) { return 2e-6f + 3e-7f * fmaxf(-beta * h, 0.0f); }

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

// Sixteen lanes hold a block, 8 elements each.  ACT: the elements are softplus(h).  Which of two neighbouring 8-bit
// values is nearest to softplus(h) can hang on its last bits, so a value is computed in 32 bits, and once more in 64 where
// its 32-bit error could change the result (a few of a million): the bytes are those of the exactly computed softplus.
template <bool ACT>
__device__ __forceinline__ uint2 quantize8(float (&h)[8], float beta, float inv_beta, double beta64, int& e_out) {
  constexpr float INF = __builtin_inff();
  int e;
  if constexpr (!ACT) {
    float top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(h[i]);
      top = a < INF ? fmaxf(top, a) : top;  // false for NaN
    }
    e = b8_exponent(lane_max<16>(top));
    const float inv = b8_pow2(-e);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = fabsf(h[i]) < INF ? h[i] * inv : __builtin_nanf("");
    e_out = e;
    return uint2{b8_pack2(h[0], h[1]) | b8_pack2(h[2], h[3]) << 16, b8_pack2(h[4], h[5]) | b8_pack2(h[6], h[7]) << 16};
  } else {
    float top = -INF;  // softplus grows with h: the block's largest comes from the largest h
#pragma unroll
    for (int i = 0; i < 8; ++i) top = h[i] < INF ? fmaxf(top, h[i]) : top;
    top = lane_max<16>(top);
    const float at = softplus32(top, beta, inv_beta), mt = softplus_margin(top, beta);
    if (at < INF) {
      e = b8_exponent(at * (1.0f - mt));
      const int above = b8_exponent(fminf(at * (1.0f + mt), 3.4e38f));
      if (e != above && softplus64((double)top, beta64) > 448.0 * ::ldexp(1.0, e)) e = above;
    } else {
      e = B8_EMAX;
    }
    if (top == -INF) e = 0;
    const float inv = b8_pow2(-e);
    uint32_t r[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      float lo[2], hi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = h[2 * p + i];
        const float a = softplus32(x, beta, inv_beta) * inv, m = x == -INF ? 0.0f : softplus_margin(x, beta);
        lo[i] = x < INF ? a * (1.0f - m) : __builtin_nanf("");
        hi[i] = x < INF ? a * (1.0f + m) : __builtin_nanf("");
      }
      r[p] = b8_pack2(lo[0], lo[1]);
      if (r[p] != b8_pack2(hi[0], hi[1])) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = h[2 * p + i];
          v[i] = x < INF ? round_to_odd(::fmin(softplus64((double)x, beta64) * ::ldexp(1.0, -e), 448.0))
                         : __builtin_nanf("");
        }
        r[p] = b8_pack2(v[0], v[1]);
      }
    }
    e_out = e;
    return uint2{r[0] | r[1] << 16, r[2] | r[3] << 16};
  }
}

// A workgroup has 16 groups of 16 lanes: 1 << row_bits of them side by side in rows (so that the exponent bytes of
// neighbouring rows, which lie side by side, leave together), the others in block columns.
template <typename T, bool ACT>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t x_stride,
                                                       uint8_t* __restrict__ values, int64_t pitch,
                                                       uint8_t* __restrict__ exponents, int64_t exp_pitch, int64_t rows,
                                                       int64_t width, int64_t blocks, int row_bits, double beta) {
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t row = ((int64_t)blockIdx.x << row_bits) + (group & ((1 << row_bits) - 1));
  if (row >= rows) return;
  const int side = 16 >> row_bits;
  const float b32 = (float)beta, ib32 = (float)(1.0 / beta);
  for (int64_t kb = (int64_t)blockIdx.y * side + (group >> row_bits); kb < blocks; kb += (int64_t)gridDim.y * side) {
    const int64_t col = kb * B8 + lane * 8;
    float h[8];
    load_some<8>(x + row * x_stride + col, width - col, ACT ? -__builtin_inff() : 0.0f, h);
    int e;
    const uint2 v = quantize8<ACT>(h, b32, ib32, beta, e);
    *reinterpret_cast<uint2*>(values + row * pitch + col) = v;
    if (lane == 0) exponents[kb * exp_pitch + row] = (uint8_t)(e + 127);
  }
}

// One workgroup per 128 x 128 tile of a matrix (n rows, k columns): the tile's bytes in the matrix's order and, through
// LDS, in the transpose's.
template <typename T>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(const T* __restrict__ w, int64_t w_stride,
                                                             uint8_t* __restrict__ values, uint8_t* __restrict__ exps,
                                                             uint8_t* __restrict__ values_t,
                                                             uint8_t* __restrict__ exps_t, int64_t n, int64_t k) {
  __shared__ float red[4];
  __shared__ uint8_t tile[B8 * (B8 + 4)];
  const int64_t nt = blockIdx.y, kt = blockIdx.x;
  const int64_t n_tiles = gridDim.y, k_tiles = gridDim.x;
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  float h[8][8];
  float top = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t row = nt * B8 + r * 16 + group, col = kt * B8 + lane * 8;
    load_some<8>(w + row * w_stride + col, row < n ? k - col : 0, 0.0f, h[r]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(h[r][i]);
      top = a < __builtin_inff() ? fmaxf(top, a) : top;
    }
  }
  top = lane_max<64>(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  const int e = b8_exponent(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  const float inv = b8_pow2(-e);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t row = nt * B8 + r * 16 + group;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[r][i] = fabsf(h[r][i]) < __builtin_inff() ? h[r][i] * inv : __builtin_nanf("");
    const uint32_t lo = b8_pack2(h[r][0], h[r][1]) | b8_pack2(h[r][2], h[r][3]) << 16;
    const uint32_t hi = b8_pack2(h[r][4], h[r][5]) | b8_pack2(h[r][6], h[r][7]) << 16;
    if (row < n)
      *reinterpret_cast<uint2*>(values + row * (k_tiles * B8) + kt * B8 + lane * 8) = uint2{lo, hi};
    uint32_t* t = reinterpret_cast<uint32_t*>(tile + (r * 16 + group) * (B8 + 4) + lane * 8);
    t[0] = lo;
    t[1] = hi;
  }
  if (threadIdx.x == 0) {
    exps[kt * n_tiles + nt] = (uint8_t)(e + 127);
    if (exps_t) exps_t[nt * k_tiles + kt] = (uint8_t)(e + 127);
  }
  if (!values_t) return;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t row = kt * B8 + r * 16 + group;  // of the transpose
    uint32_t v[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i >> 2] |= (uint32_t)tile[(lane * 8 + i) * (B8 + 4) + r * 16 + group] << (8 * (i & 3));
    if (row < k) *reinterpret_cast<uint2*>(values_t + row * (n_tiles * B8) + nt * B8 + lane * 8) = uint2{v[0], v[1]};
  }
}

// out = value * 2^e (GRAD: out = g * slope of the softplus at the kept value)
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void from_blocks_kernel(const T* __restrict__ g, int64_t g_stride,
                                                          const uint8_t* __restrict__ values, int64_t pitch,
                                                          const uint8_t* __restrict__ exponents, int64_t exp_pitch,
                                                          int exp_shift, T* __restrict__ out, int64_t rows,
                                                          int64_t width, int64_t blocks, int row_bits, float beta) {
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t row = ((int64_t)blockIdx.x << row_bits) + (group & ((1 << row_bits) - 1));
  if (row >= rows) return;
  const int side = 16 >> row_bits;
  for (int64_t kb = (int64_t)blockIdx.y * side + (group >> row_bits); kb < blocks; kb += (int64_t)gridDim.y * side) {
    const int64_t col = kb * B8 + lane * 8;
    const uint2 v = *reinterpret_cast<const uint2*>(values + row * pitch + col);
    const float scale = b8_scale(exponents[kb * exp_pitch + (row >> exp_shift)]);
    float a[8];
    b8_unpack4(v.x, scale, a);
    b8_unpack4(v.y, scale, a + 4);
    if constexpr (GRAD) {
      float gv[8];
      load_some<8>(g + row * g_stride + col, width - col, 0.0f, gv);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = gv[i] * b8_softplus_slope(a[i], beta);
    }
    store_some<8>(out + row * width + col, width - col, a);
  }
}

struct Shape {
  dim3 grid;
  int row_bits;
};
// as many rows side by side as there are, up to 16; block columns are walked in a loop once there are enough groups
Shape shape_for(int64_t rows, int64_t blocks) {
  Shape s;
  s.row_bits = 0;
  while (s.row_bits < 4 && (1 << s.row_bits) < rows) ++s.row_bits;
  const int64_t gx = (rows + (1 << s.row_bits) - 1) >> s.row_bits;
  const int64_t most = (blocks + (16 >> s.row_bits) - 1) / (16 >> s.row_bits);
  int64_t gy = (8192 + gx - 1) / gx;
  if (gy > most) gy = most;
  s.grid = dim3((unsigned)gx, (unsigned)(gy < 1 ? 1 : gy > 65535 ? 65535 : gy));
  return s;
}

}  // namespace

int b8_check_shape(const char* what, int64_t rows, int64_t width) {
  VMF_REQUIRE(rows >= 0 && width >= 1, VMF_ERR_BAD_ARG, "%s: %lld rows of %lld columns", what, (long long)rows,
              (long long)width);
  VMF_REQUIRE(rows <= VMF_BLOCKS8_MAX_ROWS && width <= VMF_BLOCKS8_MAX_WIDTH, VMF_ERR_UNSUPPORTED,
              "%s: more than %lld rows or %lld columns", what, (long long)VMF_BLOCKS8_MAX_ROWS,
              (long long)VMF_BLOCKS8_MAX_WIDTH);
  return VMF_OK;
}

extern "C" int vmf_blocks8_quantize(const void* x, int64_t x_stride, uint8_t* values, uint8_t* exponents,
                                    int64_t exp_pitch, int64_t rows, int64_t width, int activation, double beta,
                                    int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_quantize");
  int rc = b8_check_shape("vmf_blocks8_quantize", rows, width);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(activation == VMF_ACT_NONE || activation == VMF_ACT_SOFTPLUS, VMF_ERR_BAD_ARG,
              "vmf_blocks8_quantize: activation %d", activation);
  VMF_REQUIRE(activation == VMF_ACT_NONE || (beta > 0 && beta <= 1e30 && beta >= 1e-30), VMF_ERR_BAD_ARG,
              "vmf_blocks8_quantize: beta %g", beta);
  VMF_REQUIRE(x_stride >= 0 && exp_pitch >= rows, VMF_ERR_BAD_ARG, "vmf_blocks8_quantize: strides");
  if (rows == 0) return VMF_OK;
  VMF_REQUIRE(x && values && exponents, VMF_ERR_BAD_ARG, "vmf_blocks8_quantize: null pointer");
  VMF_REQUIRE(((uintptr_t)values & 15) == 0, VMF_ERR_BAD_ARG, "vmf_blocks8_quantize: values must be 16-byte aligned");
  const int64_t blocks = b8_blocks(width);
  const Shape s = shape_for(rows, blocks);
  hipStream_t st = (hipStream_t)stream;
  LOWP_DISPATCH(dtype, "vmf_blocks8_quantize", T, {
    if (activation == VMF_ACT_SOFTPLUS)
      quantize_kernel<T, true><<<s.grid, 256, 0, st>>>((const T*)x, x_stride, values, blocks * B8, exponents, exp_pitch,
                                                       rows, width, blocks, s.row_bits, beta);
    else
      quantize_kernel<T, false><<<s.grid, 256, 0, st>>>((const T*)x, x_stride, values, blocks * B8, exponents,
                                                        exp_pitch, rows, width, blocks, s.row_bits, 1.0);
  });
  return vmf_check_launch("vmf_blocks8_quantize");
}

extern "C" int vmf_blocks8_quantize_tiles(const void* w, int64_t w_stride, uint8_t* values, uint8_t* exponents,
                                          uint8_t* values_t, uint8_t* exponents_t, int64_t rows, int64_t width,
                                          int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_quantize_tiles");
  int rc = b8_check_shape("vmf_blocks8_quantize_tiles", rows, width);
  if (rc != VMF_OK) return rc;
  rc = b8_check_shape("vmf_blocks8_quantize_tiles", width, rows < 1 ? 1 : rows);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(w_stride >= 0, VMF_ERR_BAD_ARG, "vmf_blocks8_quantize_tiles: negative row stride");
  VMF_REQUIRE(!values_t == !exponents_t, VMF_ERR_BAD_ARG,
              "vmf_blocks8_quantize_tiles: values_t and exponents_t go together");
  if (rows == 0) return VMF_OK;
  VMF_REQUIRE(w && values && exponents, VMF_ERR_BAD_ARG, "vmf_blocks8_quantize_tiles: null pointer");
  VMF_REQUIRE((((uintptr_t)values | (uintptr_t)values_t) & 15) == 0, VMF_ERR_BAD_ARG,
              "vmf_blocks8_quantize_tiles: values must be 16-byte aligned");
  const int64_t n_tiles = b8_blocks(rows);
  VMF_REQUIRE(n_tiles <= 65535, VMF_ERR_UNSUPPORTED, "vmf_blocks8_quantize_tiles: %lld rows", (long long)rows);
  hipStream_t st = (hipStream_t)stream;
  LOWP_DISPATCH(dtype, "vmf_blocks8_quantize_tiles", T,
                (quantize_tiles_kernel<T><<<dim3((unsigned)b8_blocks(width), (unsigned)n_tiles), 256, 0, st>>>(
                    (const T*)w, w_stride, values, exponents, values_t, exponents_t, rows, width)));
  return vmf_check_launch("vmf_blocks8_quantize_tiles");
}

static int from_blocks(const char* what, const void* g, int64_t g_stride, const uint8_t* values,
                       const uint8_t* exponents, int64_t exp_pitch, int tiled, void* out, int64_t rows, int64_t width,
                       double beta, int grad, int dtype, vmf_stream_t stream) {
  int rc = b8_check_shape(what, rows, width);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(g_stride >= 0 && exp_pitch >= (tiled ? b8_blocks(rows) : rows), VMF_ERR_BAD_ARG, "%s: strides", what);
  VMF_REQUIRE(!grad || (beta > 0 && beta <= 1e30 && beta >= 1e-30), VMF_ERR_BAD_ARG, "%s: beta %g", what, beta);
  if (rows == 0) return VMF_OK;
  VMF_REQUIRE(values && exponents && out && (g || !grad), VMF_ERR_BAD_ARG, "%s: null pointer", what);
  VMF_REQUIRE(((uintptr_t)values & 15) == 0, VMF_ERR_BAD_ARG, "%s: values must be 16-byte aligned", what);
  const int64_t blocks = b8_blocks(width);
  const Shape s = shape_for(rows, blocks);
  hipStream_t st = (hipStream_t)stream;
  LOWP_DISPATCH(dtype, "vmf_blocks8", T, {
    if (grad)
      from_blocks_kernel<T, true><<<s.grid, 256, 0, st>>>((const T*)g, g_stride, values, blocks * B8, exponents,
                                                          exp_pitch, tiled ? 7 : 0, (T*)out, rows, width, blocks,
                                                          s.row_bits, (float)beta);
    else
      from_blocks_kernel<T, false><<<s.grid, 256, 0, st>>>(nullptr, 0, values, blocks * B8, exponents, exp_pitch,
                                                           tiled ? 7 : 0, (T*)out, rows, width, blocks, s.row_bits,
                                                           1.0f);
  });
  return vmf_check_launch(what);
}

extern "C" int vmf_blocks8_dequantize(const uint8_t* values, const uint8_t* exponents, int64_t exp_pitch, int tiled,
                                      void* out, int64_t rows, int64_t width, int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_dequantize");
  return from_blocks("vmf_blocks8_dequantize", nullptr, 0, values, exponents, exp_pitch, tiled, out, rows, width, 1.0,
                     0, dtype, stream);
}

extern "C" int vmf_blocks8_softplus_grad(const void* g, int64_t g_stride, const uint8_t* values,
                                         const uint8_t* exponents, int64_t exp_pitch, void* out, int64_t rows,
                                         int64_t width, double beta, int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_softplus_grad");
  return from_blocks("vmf_blocks8_softplus_grad", g, g_stride, values, exponents, exp_pitch, 0, out, rows, width, beta,
                     1, dtype, stream);
}
