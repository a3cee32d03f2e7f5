// blocks8.hip -- into and out of 8-bit blocks: quantisation of rows (of x or of softplus(x)) and of weight tiles,
// conversion back, the gradient through a softplus whose result was kept in blocks.  All are HBM streams.
#include "blocks8_dev.h"

namespace {

// A workgroup has 16 groups of 16 lanes: 1 << row_bits of them side by side in rows (so that the exponent bytes of
// neighbouring rows, which lie side by side, leave together), the others in block columns.
// Measured: 1048576x784 fp32 0.79 ms (5.2 TB/s), of softplus 0.79; bf16 0.47 ms (5.2), of softplus 0.64, bound by the vector
// work (some 25 instructions to an element).
struct RowArgs {
  const void* x;
  int64_t x_stride;
  uint8_t* values;
  uint8_t* exponents;
  int64_t exp_pitch, rows, width, blocks;
  int row_bits, gx, gy;  // workgroups along the rows and along the block columns
  double beta;
  float beta32, inv_beta;
};
template <typename T, bool ACT>
__device__ __forceinline__ void quantize_rows(const RowArgs& p, int bx, int by) {
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t row = ((int64_t)bx << p.row_bits) + (group & ((1 << p.row_bits) - 1));
  if (row >= p.rows) return;
  const int side = 16 >> p.row_bits;
  const T* x = (const T*)p.x + row * p.x_stride;
  for (int64_t kb = (int64_t)by * side + (group >> p.row_bits); kb < p.blocks; kb += (int64_t)p.gy * side) {
    const int64_t col = kb * B8 + lane * 8;
    float h[8];
    load_some<8>(x + col, p.width - col, ACT ? -__builtin_inff() : 0.0f, h);
    int e;
    uint2 v;
    if constexpr (ACT) {
      v = softplus8(h, p.beta32, p.inv_beta, p.beta, e);
    } else {
      e = scale8(h);
      v = uint2{b8_pack4(h), b8_pack4(h + 4)};
    }
    *reinterpret_cast<uint2*>(p.values + row * (p.blocks * B8) + col) = v;
    if (lane == 0) p.exponents[kb * p.exp_pitch + row] = (uint8_t)(e + 127);
  }
}
template <typename T, bool ACT>
__global__ __launch_bounds__(256) void quantize_kernel(RowArgs p) {
  quantize_rows<T, ACT>(p, blockIdx.x, blockIdx.y);
}

// One workgroup per 128 x 128 tile of a matrix (n rows, k columns): the tile's bytes in the matrix's order and, through
// LDS, in the transpose's (4096x4096 fp32 18 us, 5.6 TB/s).
struct TileArgs {
  const void* w;
  int64_t w_stride;
  uint8_t* values;
  uint8_t* exps;
  uint8_t* values_t;
  uint8_t* exps_t;
  int64_t n, k, n_tiles, k_tiles;
};
template <typename T>
__device__ __forceinline__ void quantize_tile(const TileArgs& p, int64_t id) {
  __shared__ uint32_t red[4];
  __shared__ uint8_t tile[B8 * (B8 + 4)];
  const int64_t n_tiles = p.n_tiles, k_tiles = p.k_tiles;
  const int64_t nt = id / k_tiles, kt = id - nt * k_tiles;
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  float h[8][8];
  uint32_t top = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t row = nt * B8 + r * 16 + group, col = kt * B8 + lane * 8;
    load_some<8>((const T*)p.w + row * p.w_stride + col, row < p.n ? p.k - col : 0, 0.0f, h[r]);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = b8_size(h[r][i]) < B8_INF ? larger(top, b8_size(h[r][i])) : top;
  }
  top = lane_max<64>(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  const int e = b8_exponent(__uint_as_float(larger(larger(red[0], red[1]), larger(red[2], red[3]))));
  const float inv = b8_pow2(-e);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t row = nt * B8 + r * 16 + group;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[r][i] = e == B8_EMAX ? b8_cut(h[r][i] * inv) : h[r][i] * inv;
    const uint32_t lo = b8_pack4(h[r]), hi = b8_pack4(h[r] + 4);
    if (row < p.n)
      *reinterpret_cast<uint2*>(p.values + row * (k_tiles * B8) + kt * B8 + lane * 8) = uint2{lo, hi};
    uint32_t* t = reinterpret_cast<uint32_t*>(tile + (r * 16 + group) * (B8 + 4) + lane * 8);
    t[0] = lo;
    t[1] = hi;
  }
  if (threadIdx.x == 0) {
    p.exps[kt * n_tiles + nt] = (uint8_t)(e + 127);
    if (p.exps_t) p.exps_t[nt * k_tiles + kt] = (uint8_t)(e + 127);
  }
  if (!p.values_t) return;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t row = kt * B8 + r * 16 + group;  // of the transpose
    uint32_t v[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i >> 2] |= (uint32_t)tile[(lane * 8 + i) * (B8 + 4) + r * 16 + group] << (8 * (i & 3));
    if (row < p.k) *reinterpret_cast<uint2*>(p.values_t + row * (n_tiles * B8) + nt * B8 + lane * 8) = uint2{v[0], v[1]};
  }
}
template <typename T>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(TileArgs p) {
  quantize_tile<T>(p, blockIdx.x);
}
// both in one launch: the tiles' workgroups first
template <typename T, bool ACT, typename TW>
__global__ __launch_bounds__(256) void quantize_both_kernel(RowArgs r, TileArgs t) {
  const int tiles = (int)(t.n_tiles * t.k_tiles), id = (int)blockIdx.x;
  if (id < tiles) {
    quantize_tile<TW>(t, id);
  } else {
    const int by = (id - tiles) / r.gx;
    quantize_rows<T, ACT>(r, id - tiles - by * r.gx, by);
  }
}

// out = value * 2^e (GRAD: out = g * slope of the softplus at the kept value).  A lane has as many elements as fill the 16
// bytes of a store: 8 of 16 bits and, so that the lanes' stores lie side by side, 4 of 32 (1048576x784 fp32 0.81 ms,
// 5.0 TB/s, with 8 to a lane 1.30; bf16 0.56 ms; GRAD bf16 0.96 ms, 4.3 TB/s).
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void from_blocks_kernel(const T* __restrict__ g, int64_t g_stride,
                                                          const uint8_t* __restrict__ values, int64_t pitch,
                                                          const uint8_t* __restrict__ exponents, int64_t exp_pitch,
                                                          int exp_shift, T* __restrict__ out, int64_t rows,
                                                          int64_t width, int64_t blocks, int row_bits, float beta) {
  constexpr int E = 16 / (int)sizeof(T), LANES = B8 / E, GROUPS = 256 / LANES;
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int64_t row = ((int64_t)blockIdx.x << row_bits) + (group & ((1 << row_bits) - 1));
  if (row >= rows) return;
  const int side = GROUPS >> row_bits;
  for (int64_t kb = (int64_t)blockIdx.y * side + (group >> row_bits); kb < blocks; kb += (int64_t)gridDim.y * side) {
    const int64_t col = kb * B8 + lane * E;
    const float scale = b8_scale(exponents[kb * exp_pitch + (row >> exp_shift)]);
    const uint32_t* v = reinterpret_cast<const uint32_t*>(values + row * pitch + col);
    uint32_t w[E / 4];
    float a[E];
    if constexpr (E == 8) {
      const uint2 both = *reinterpret_cast<const uint2*>(v);
      w[0] = both.x;
      w[1] = both.y;
    } else {
      w[0] = *v;
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) b8_unpack4(w[i], scale, a + 4 * i);
    if constexpr (GRAD) {
      float gv[E];
      load_some<E>(g + row * g_stride + col, width - col, 0.0f, gv);
#pragma unroll
      for (int i = 0; i < E; ++i) a[i] = gv[i] * b8_softplus_slope<sizeof(T) == 2>(a[i], beta);
    }
    store_some<E>(out + row * width + col, width - col, a);
  }
}

struct Shape {
  dim3 grid;
  int row_bits;
};
// A workgroup's 1 << group_bits groups: as many rows side by side as there are; block columns are walked in a loop once
// there are enough workgroups
Shape shape_for(int64_t rows, int64_t blocks, int group_bits) {
  Shape s;
  s.row_bits = 0;
  while (s.row_bits < group_bits && (1 << s.row_bits) < rows) ++s.row_bits;
  const int64_t gx = rows > 0 ? (rows + (1 << s.row_bits) - 1) >> s.row_bits : 1;
  const int64_t side = (1 << group_bits) >> s.row_bits, most = (blocks + side - 1) / side;
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

namespace {

int row_args(const char* what, const void* x, int64_t x_stride, uint8_t* values, uint8_t* exponents, int64_t exp_pitch,
             int64_t rows, int64_t width, int activation, double beta, RowArgs* out) {
  int rc = b8_check_shape(what, rows, width);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(activation == VMF_ACT_NONE || activation == VMF_ACT_SOFTPLUS, VMF_ERR_BAD_ARG, "%s: activation %d", what,
              activation);
  VMF_REQUIRE(activation == VMF_ACT_NONE || (beta > 0 && beta <= 1e30 && beta >= 1e-30), VMF_ERR_BAD_ARG,
              "%s: beta %g", what, beta);
  VMF_REQUIRE(x_stride >= 0 && exp_pitch >= rows, VMF_ERR_BAD_ARG, "%s: strides", what);
  if (rows > 0) {
    VMF_REQUIRE(x && values && exponents, VMF_ERR_BAD_ARG, "%s: null pointer", what);
    VMF_REQUIRE(((uintptr_t)values & 15) == 0, VMF_ERR_BAD_ARG, "%s: values must be 16-byte aligned", what);
  }
  if (activation == VMF_ACT_NONE) beta = 1.0;
  const int64_t blocks = b8_blocks(width);
  const Shape s = shape_for(rows, blocks, 4);
  *out = RowArgs{x, x_stride, values, exponents, exp_pitch, rows, width, blocks, s.row_bits, (int)s.grid.x,
                 (int)s.grid.y, beta, (float)beta, (float)(1.0 / beta)};
  return VMF_OK;
}

int tile_args(const char* what, const void* w, int64_t w_stride, uint8_t* values, uint8_t* exponents,
              uint8_t* values_t, uint8_t* exponents_t, int64_t rows, int64_t width, TileArgs* out) {
  int rc = b8_check_shape(what, rows, width);
  if (rc != VMF_OK) return rc;
  rc = b8_check_shape(what, width, rows < 1 ? 1 : rows);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(w_stride >= 0, VMF_ERR_BAD_ARG, "%s: negative row stride", what);
  VMF_REQUIRE(!values_t == !exponents_t, VMF_ERR_BAD_ARG, "%s: values_t and exponents_t go together", what);
  if (rows > 0) {
    VMF_REQUIRE(w && values && exponents, VMF_ERR_BAD_ARG, "%s: null pointer", what);
    VMF_REQUIRE((((uintptr_t)values | (uintptr_t)values_t) & 15) == 0, VMF_ERR_BAD_ARG,
                "%s: values must be 16-byte aligned", what);
  }
  *out = TileArgs{w, w_stride, values, exponents, values_t, exponents_t, rows, width, b8_blocks(rows), b8_blocks(width)};
  // (a launch has fewer than 2^32 threads)
  VMF_REQUIRE(out->n_tiles * out->k_tiles < (1 << 24), VMF_ERR_UNSUPPORTED, "%s: %lld x %lld", what, (long long)rows,
              (long long)width);
  return VMF_OK;
}

int launch_rows(const RowArgs& r, int activation, int dtype, hipStream_t st) {
  LOWP_DISPATCH(dtype, "vmf_blocks8_quantize", T, {
    if (activation == VMF_ACT_SOFTPLUS) quantize_kernel<T, true><<<dim3(r.gx, r.gy), 256, 0, st>>>(r);
    else quantize_kernel<T, false><<<dim3(r.gx, r.gy), 256, 0, st>>>(r);
  });
  return vmf_check_launch("vmf_blocks8_quantize");
}

int launch_tiles(const TileArgs& t, int dtype, hipStream_t st) {
  LOWP_DISPATCH(dtype, "vmf_blocks8_quantize_tiles", T,
                (quantize_tiles_kernel<T><<<(unsigned)(t.n_tiles * t.k_tiles), 256, 0, st>>>(t)));
  return vmf_check_launch("vmf_blocks8_quantize_tiles");
}

template <typename T, typename TW>
void launch_both(const RowArgs& r, const TileArgs& t, int activation, hipStream_t st) {
  const unsigned grid = (unsigned)(t.n_tiles * t.k_tiles + (int64_t)r.gx * r.gy);
  if (activation == VMF_ACT_SOFTPLUS) quantize_both_kernel<T, true, TW><<<grid, 256, 0, st>>>(r, t);
  else quantize_both_kernel<T, false, TW><<<grid, 256, 0, st>>>(r, t);
}

}  // namespace

extern "C" int vmf_blocks8_quantize(const void* x, int64_t x_stride, uint8_t* values, uint8_t* exponents,
                                    int64_t exp_pitch, int64_t rows, int64_t width, int activation, double beta,
                                    int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_quantize");
  RowArgs r;
  int rc = row_args("vmf_blocks8_quantize", x, x_stride, values, exponents, exp_pitch, rows, width, activation, beta, &r);
  if (rc != VMF_OK || rows == 0) return rc;
  return launch_rows(r, activation, dtype, (hipStream_t)stream);
}

extern "C" int vmf_blocks8_quantize_tiles(const void* w, int64_t w_stride, uint8_t* values, uint8_t* exponents,
                                          uint8_t* values_t, uint8_t* exponents_t, int64_t rows, int64_t width,
                                          int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_quantize_tiles");
  TileArgs t;
  int rc = tile_args("vmf_blocks8_quantize_tiles", w, w_stride, values, exponents, values_t, exponents_t, rows, width, &t);
  if (rc != VMF_OK || rows == 0) return rc;
  return launch_tiles(t, dtype, (hipStream_t)stream);
}

int b8_quantize_both(const void* x, int64_t x_stride, uint8_t* values, uint8_t* exponents, int64_t exp_pitch, int64_t m,
                     int64_t k, int activation, double beta, int dtype, const void* w, int64_t w_stride,
                     uint8_t* w_values, uint8_t* w_exponents, uint8_t* wt_values, uint8_t* wt_exponents, int64_t n,
                     int w_dtype, vmf_stream_t stream) {
  const char* what = "vmf_blocks8_linear_fwd";
  RowArgs r;
  TileArgs t;
  int rc = row_args(what, x, x_stride, values, exponents, exp_pitch, m, k, activation, beta, &r);
  if (rc != VMF_OK) return rc;
  rc = tile_args(what, w, w_stride, w_values, w_exponents, wt_values, wt_exponents, n, k, &t);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(w_dtype == dtype || w_dtype == VMF_F32, VMF_ERR_DTYPE, "%s: the weight's dtype is x's or VMF_F32, got %d",
              what, w_dtype);
  hipStream_t st = (hipStream_t)stream;
  // One launch saves its own microseconds and lets the rows start beside the tiles (a layer's forward pass in fp32 with
  // softplus, 16384x128x784: 27.5 us, in two launches 30.9; 16384x2048x2048 in bf16 100.9 and 103); with many more rows
  // those do better without the tiles' registers and LDS (1048576x128x784 in bf16: 1247 us, in two launches 1141).
  constexpr int64_t MOST = 1 << 25;
  if (m == 0 || m * k > MOST || n * k > MOST) {
    rc = launch_tiles(t, w_dtype, st);
    return rc != VMF_OK || m == 0 ? rc : launch_rows(r, activation, dtype, st);
  }
  LOWP_DISPATCH(dtype, "vmf_blocks8_linear_fwd", T, {
    if (w_dtype == VMF_F32) launch_both<T, float>(r, t, activation, st);
    else launch_both<T, T>(r, t, activation, st);
  });
  return vmf_check_launch(what);
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
  const Shape s = shape_for(rows, blocks, dtype == VMF_F32 ? 3 : 4);
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
