// layer_norm.hip -- layer norm over the last dimension, forward and backward.
//
//   xhat = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xhat w + b
//   h = gy w,  gx = rstd (h - mean(h) - xhat mean(h xhat)),  gw = sum_rows gy xhat,  gb = sum_rows gy
//
// Both directions are streams of HBM: the forward pass reads x and writes y, the backward pass reads x and gy and
// writes gx, about 8 and 20 operations per element against 8 and 12 bytes (fp32).  A row is held in the registers of
// TPR lanes, so it is read once and the variance is summed from centred values (no difference of large squares).
// Statistics, sums and the partial gradients are 32-bit (64-bit for double rows).
// Measured (a large copy: 5.2 TB/s): 1048576x784 fp32 forward 1.22 ms (5.4 TB/s), backward 1.88 ms (5.2); bf16 0.69 ms (4.7)
// and 1.14 ms (4.3), where the vector work of 16-bit rows takes as long; 16384x1001 bf16 16 and 28 us.
#include "lowp.h"

namespace {

constexpr int THREADS = 256;

template <typename T> struct LnVec { static constexpr int value = 16 / (int)sizeof(T); };

// sum over the TPR threads that share a row; `red` holds one value per wave and a second set alternates with it, so
// that one barrier per sum is enough (a wave can only be one sum ahead of the others)
template <int TPR, typename A>
__device__ __forceinline__ A row_sum(A v, A* red, int& flip) {
  if constexpr (TPR <= 64) {
    return lane_sum<TPR>(v);
  } else {
    constexpr int WAVES = TPR / 64;
    v = lane_sum<64>(v);
    A* r = red + flip * WAVES;
    flip ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    A s = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) s += r[i];
    return s;
  }
}

// Whether a workgroup keeps weight and bias in registers and has its next row's loads under way while it works on one.  For
// 16-bit rows, whose loads are half as many (1048576x784 bf16 0.95 -> 0.69 ms, 65536x8192 0.60 -> 0.54); fp32 rows keep the
// memory busy without (1048576x784 1.22 ms, with it 1.35), and 1024 lanes to a row have no registers left for it.
template <typename T, int TPR> constexpr bool ahead() { return sizeof(T) == 2 && TPR <= THREADS; }

template <typename T, typename W, int TPR, int NCH>
__global__ __launch_bounds__(TPR > THREADS ? TPR : THREADS) void ln_fwd_kernel(
    const T* __restrict__ x, int64_t x_stride, const W* __restrict__ w, const W* __restrict__ b, T* __restrict__ y,
    typename AccOf<T>::type* __restrict__ mean_out, typename AccOf<T>::type* __restrict__ rstd_out, int64_t n,
    int width, double eps) {
  using A = typename AccOf<T>::type;
  constexpr int V = LnVec<T>::value;
  constexpr int NT = TPR > THREADS ? TPR : THREADS;
  constexpr int ROWS = NT / TPR;
  constexpr bool AHEAD = ahead<T, TPR>();
  constexpr int KEPT = AHEAD ? NCH : 1;
  __shared__ A red[2 * (TPR > 64 ? TPR / 64 : 1)];
  int flip = 0;
  const int lane = threadIdx.x % TPR;
  const A inv = (A)1 / (A)width;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  A v[NCH][V], next[KEPT][V], wv[KEPT][V], bv[KEPT][V];
  auto load_row = [&](int64_t row, auto& to) {
    const T* xr = x + row * x_stride;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + lane) * V;
      load_some<V>(xr + col, (int64_t)width - col, (A)0, to[c]);
    }
  };
  auto load_affine = [&](int c, int to) {
    const int col = (c * TPR + lane) * V;
    if (w) load_some<V>(w + col, (int64_t)width - col, (A)0, wv[to]);
    if (b) load_some<V>(b + col, (int64_t)width - col, (A)0, bv[to]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!w) wv[to][i] = (A)1;
      if (!b) bv[to][i] = (A)0;
    }
  };
  int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  if constexpr (AHEAD) {
    if (row < n) load_row(row, next);
#pragma unroll
    for (int c = 0; c < NCH; ++c) load_affine(c, c);
  }
  for (; row < n; row += step) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] = next[c][i];
      if (row + step < n) load_row(row + step, next);
    } else {
      load_row(row, v);
    }
    A s = 0;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[c][i];
    const A mean = row_sum<TPR>(s, red, flip) * inv;
    s = 0;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int left = width - (c * TPR + lane) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[c][i] -= mean;
        s += i < left ? v[c][i] * v[c][i] : (A)0;
      }
    }
    const A rstd = (A)1 / M<A>::sqrt(row_sum<TPR>(s, red, flip) * inv + (A)eps);
    if (lane == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    T* yr = y + row * (int64_t)width;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + lane) * V, at = AHEAD ? c : 0;
      if constexpr (!AHEAD) load_affine(c, 0);
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] = v[c][i] * rstd * wv[at][i] + bv[at][i];
      store_some<V>(yr + col, (int64_t)width - col, v[c]);
    }
  }
}

// Rows that do not fit the registers (more than 32768 elements): the same sums over three reads of the row, the second and
// third out of the L2 (16384x40000 fp32 1.45 ms, 3.6 TB/s counting one read).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, int64_t x_stride,
                                                           const W* __restrict__ w, const W* __restrict__ b,
                                                           T* __restrict__ y,
                                                           typename AccOf<T>::type* __restrict__ mean_out,
                                                           typename AccOf<T>::type* __restrict__ rstd_out, int64_t n,
                                                           int64_t width, double eps) {
  using A = typename AccOf<T>::type;
  constexpr int V = LnVec<T>::value;
  __shared__ A red[32];
  int flip = 0;
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const T* xr = x + row * x_stride;
    A v[V], s = 0;
    for (int64_t col = (int64_t)threadIdx.x * V; col < width; col += 1024 * V) {
      load_some<V>(xr + col, width - col, (A)0, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[i];
    }
    const A mean = row_sum<1024>(s, red, flip) / (A)width;
    s = 0;
    for (int64_t col = (int64_t)threadIdx.x * V; col < width; col += 1024 * V) {
      load_some<V>(xr + col, width - col, mean, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += (v[i] - mean) * (v[i] - mean);
    }
    const A rstd = (A)1 / M<A>::sqrt(row_sum<1024>(s, red, flip) / (A)width + (A)eps);
    if (threadIdx.x == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    for (int64_t col = (int64_t)threadIdx.x * V; col < width; col += 1024 * V) {
      A wv[V], bv[V];
      load_some<V>(xr + col, width - col, (A)0, v);
      if (w) load_some<V>(w + col, width - col, (A)0, wv);
      if (b) load_some<V>(b + col, width - col, (A)0, bv);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (v[i] - mean) * rstd * (w ? wv[i] : (A)1) + (b ? bv[i] : (A)0);
      store_some<V>(y + row * width + col, width - col, v);
    }
  }
}

// The backward pass of the rows that a workgroup of NT threads takes (TPR to a row, the workgroup's rows `step` apart).
// A lane keeps the same columns for every row it sees, so gw and gb grow in its registers (SUMS); at the end the rows
// side by side are added in LDS, in order, into one partial row of each per workgroup.
template <typename T, typename W, int NT, int TPR, int NCH, bool SUMS>
__device__ __forceinline__ void ln_bwd_rows(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ gy,
                                            int64_t gy_stride, const W* __restrict__ w,
                                            const typename AccOf<T>::type* __restrict__ mean_in,
                                            const typename AccOf<T>::type* __restrict__ rstd_in, T* __restrict__ gx,
                                            typename AccOf<T>::type* __restrict__ partial, int64_t n, int width,
                                            int64_t first, int64_t step) {
  using A = typename AccOf<T>::type;
  constexpr int V = LnVec<T>::value;
  constexpr int ROWS = NT / TPR;
  __shared__ A red[2 * (TPR > 64 ? TPR / 64 : 1)];
  __shared__ A side[SUMS && ROWS > 1 ? (ROWS - 1) * TPR * V : 1];
  int flip = 0;
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const A inv = (A)1 / (A)width;
  A wv[NCH][V], gw[NCH][V], gb[NCH][V];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * TPR + lane) * V;
    if (w) load_some<V>(w + col, (int64_t)width - col, (A)0, wv[c]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!w) wv[c][i] = (A)1;
      gw[c][i] = gb[c][i] = 0;
    }
  }
  for (int64_t row = first + sub; row < n; row += step) {
    const T* xr = x + row * x_stride;
    const T* gr = gy + row * gy_stride;
    const A mean = mean_in[row], rstd = rstd_in[row];
    A xh[NCH][V], h[NCH][V];
    A s1 = 0, s2 = 0;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + lane) * V;
      load_some<V>(xr + col, (int64_t)width - col, mean, xh[c]);
      load_some<V>(gr + col, (int64_t)width - col, (A)0, h[c]);
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[c][i] = (xh[c][i] - mean) * rstd;
        if constexpr (SUMS) {
          gw[c][i] += h[c][i] * xh[c][i];
          gb[c][i] += h[c][i];
        }
        h[c][i] *= wv[c][i];
        s1 += h[c][i];
        s2 += h[c][i] * xh[c][i];
      }
    if (gx) {
      s1 = row_sum<TPR>(s1, red, flip) * inv;
      s2 = row_sum<TPR>(s2, red, flip) * inv;
      T* out = gx + row * (int64_t)width;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (c * TPR + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) h[c][i] = (h[c][i] - s1 - xh[c][i] * s2) * rstd;
        store_some<V>(out + col, (int64_t)width - col, h[c]);
      }
    }
  }
  if constexpr (SUMS) {
    if (!partial) return;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        A(&g)[V] = which ? gb[c] : gw[c];
        if constexpr (ROWS > 1) {
          __syncthreads();
          if (sub > 0)
#pragma unroll
            for (int i = 0; i < V; ++i) side[((sub - 1) * TPR + lane) * V + i] = g[i];
          __syncthreads();
          if (sub == 0)
            for (int r = 0; r < ROWS - 1; ++r)
#pragma unroll
              for (int i = 0; i < V; ++i) g[i] += side[(r * TPR + lane) * V + i];
        }
        const int col = (c * TPR + lane) * V;
        if (sub == 0) store_some<V>(partial + (int64_t)which * width + col, (int64_t)width - col, g);
      }
  }
}
// One partial row of gw and gb per workgroup; ln_reduce_kernel adds them in order: the same bits on every run.
template <typename T, typename W, int NT, int TPR, int NCH>
__global__ __launch_bounds__(NT) void ln_bwd_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ gy,
                                                    int64_t gy_stride, const W* __restrict__ w,
                                                    const typename AccOf<T>::type* __restrict__ mean_in,
                                                    const typename AccOf<T>::type* __restrict__ rstd_in,
                                                    T* __restrict__ gx, typename AccOf<T>::type* __restrict__ partial,
                                                    int64_t n, int width) {
  constexpr int ROWS = NT / TPR;
  ln_bwd_rows<T, W, NT, TPR, NCH, true>(x, x_stride, gy, gy_stride, w, mean_in, rstd_in, gx,
                                        partial ? partial + (int64_t)blockIdx.x * 2 * width : nullptr, n, width,
                                        (int64_t)blockIdx.x * ROWS, (int64_t)gridDim.x * ROWS);
}
// Few rows: both results in one launch and without partials.  The first workgroups take the rows, the others 16 columns
// each, which 16 threads share; x and gy are read twice, the second time out of the L2.
template <typename T, typename W, int TPR, int NCH>
__global__ __launch_bounds__(THREADS) void ln_bwd_few_kernel(const T* __restrict__ x, int64_t x_stride,
                                                             const T* __restrict__ gy, int64_t gy_stride,
                                                             const W* __restrict__ w,
                                                             const typename AccOf<T>::type* __restrict__ mean_in,
                                                             const typename AccOf<T>::type* __restrict__ rstd_in,
                                                             T* __restrict__ gx, W* __restrict__ gw,
                                                             W* __restrict__ gb, int n, int width, int row_groups) {
  using A = typename AccOf<T>::type;
  constexpr int ROWS = THREADS / TPR;
  if ((int)blockIdx.x < row_groups) {
    ln_bwd_rows<T, W, THREADS, TPR, NCH, false>(x, x_stride, gy, gy_stride, w, mean_in, rstd_in, gx, nullptr, n, width,
                                                (int64_t)blockIdx.x * ROWS, (int64_t)row_groups * ROWS);
    return;
  }
  __shared__ A sums[2][16][17];
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int col = ((int)blockIdx.x - row_groups) * 16 + c;
  A a = 0, b = 0;
  if (col < width)
#pragma unroll 4
    for (int r = r0; r < n; r += 16) {
      const A g = (A)gy[r * gy_stride + col];
      a += g * (((A)x[r * x_stride + col] - mean_in[r]) * rstd_in[r]);
      b += g;
    }
  sums[0][r0][c] = a;
  sums[1][r0][c] = b;
  __syncthreads();
  if (threadIdx.x < 32 && col < width) {  // threads 0 - 15: gw, 16 - 31: gb
    const int which = threadIdx.x >> 4;
    A s = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += sums[which][r][c];
    W* out = which ? gb : gw;
    if (out) out[col] = (W)s;
  }
}

// Rows that do not fit (more than 16384 elements): gx alone, a workgroup per row, ...
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(
    const T* __restrict__ x, int64_t x_stride, const T* __restrict__ gy, int64_t gy_stride, const W* __restrict__ w,
    const typename AccOf<T>::type* __restrict__ mean_in, const typename AccOf<T>::type* __restrict__ rstd_in,
    T* __restrict__ gx, int64_t n, int64_t width) {
  using A = typename AccOf<T>::type;
  constexpr int V = LnVec<T>::value;
  __shared__ A red[32];
  int flip = 0;
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const T* xr = x + row * x_stride;
    const T* gr = gy + row * gy_stride;
    const A mean = mean_in[row], rstd = rstd_in[row];
    A xv[V], hv[V], wv[V], s1 = 0, s2 = 0;
    for (int64_t col = (int64_t)threadIdx.x * V; col < width; col += 1024 * V) {
      load_some<V>(xr + col, width - col, mean, xv);
      load_some<V>(gr + col, width - col, (A)0, hv);
      if (w) load_some<V>(w + col, width - col, (A)0, wv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const A h = w ? hv[i] * wv[i] : hv[i];
        s1 += h;
        s2 += h * ((xv[i] - mean) * rstd);
      }
    }
    s1 = row_sum<1024>(s1, red, flip) / (A)width;
    s2 = row_sum<1024>(s2, red, flip) / (A)width;
    for (int64_t col = (int64_t)threadIdx.x * V; col < width; col += 1024 * V) {
      load_some<V>(xr + col, width - col, mean, xv);
      load_some<V>(gr + col, width - col, (A)0, hv);
      if (w) load_some<V>(w + col, width - col, (A)0, wv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const A h = w ? hv[i] * wv[i] : hv[i];
        hv[i] = (h - s1 - (xv[i] - mean) * rstd * s2) * rstd;
      }
      store_some<V>(gx + row * width + col, width - col, hv);
    }
  }
}
// ... and gw, gb by columns: a workgroup takes 256 columns and one slice of the rows (together 16384x40000 fp32 2.96 ms)
template <typename T>
__global__ __launch_bounds__(256) void ln_cols_kernel(const T* __restrict__ x, int64_t x_stride,
                                                      const T* __restrict__ gy, int64_t gy_stride,
                                                      const typename AccOf<T>::type* __restrict__ mean_in,
                                                      const typename AccOf<T>::type* __restrict__ rstd_in,
                                                      typename AccOf<T>::type* __restrict__ partial, int64_t n,
                                                      int64_t width) {
  using A = typename AccOf<T>::type;
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= width) return;
  A gw = 0, gb = 0;
  for (int64_t row = blockIdx.y; row < n; row += gridDim.y) {
    const A g = (A)gy[row * gy_stride + col];
    gw += g * (((A)x[row * x_stride + col] - mean_in[row]) * rstd_in[row]);
    gb += g;
  }
  partial[((int64_t)blockIdx.y * 2) * width + col] = gw;
  partial[((int64_t)blockIdx.y * 2 + 1) * width + col] = gb;
}

// gw / gb from `parts` partial rows of 2 * width values: a workgroup takes 16 columns, 32 threads share one
constexpr int REDUCE_SHARE = 32;
template <typename A, typename W>
__global__ __launch_bounds__(16 * REDUCE_SHARE) void ln_reduce_kernel(const A* __restrict__ partial, W* __restrict__ gw,
                                                        W* __restrict__ gb, int parts, int64_t width) {
  __shared__ A red[16 * REDUCE_SHARE];
  const int64_t col = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);  // 0 .. 2 width
  A s = 0;
  if (col < 2 * width)
#pragma unroll 8
    for (int p = threadIdx.x >> 4; p < parts; p += REDUCE_SHARE) s += partial[(int64_t)p * 2 * width + col];
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 16 && col < 2 * width) {
#pragma unroll
    for (int r = 1; r < REDUCE_SHARE; ++r) s += red[r * 16 + threadIdx.x];
    if (col < width) {
      if (gw) gw[col] = (W)s;
    } else if (gb) {
      gb[col - width] = (W)s;
    }
  }
}

// lanes per row by the width in vectors of 16 bytes: as few as hold the row in at most `chunks` registers' worth each
int lanes_for(int64_t vectors, int chunks) {
  for (int tpr = 16; tpr <= 1024; tpr *= tpr == 64 ? 4 : tpr == 256 ? 4 : 2)
    if (vectors <= (int64_t)tpr * chunks) return tpr;
  return 0;
}

template <typename T, typename W, int TPR, int NCH>
void launch_fwd(const void* x, int64_t xs, const void* w, const void* b, void* y, void* mean, void* rstd, int64_t n,
                int64_t width, double eps, hipStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int NT = TPR > THREADS ? TPR : THREADS;
  // (four workgroups to a compute unit where a workgroup gains from going on: 65536x4096 bf16 0.20 ms, with 65536 0.26)
  const int grid = vmf_grid_for(n, NT / TPR, ahead<T, TPR>() ? 1024 : 1 << 16);
  ln_fwd_kernel<T, W, TPR, NCH><<<grid, NT, 0, st>>>((const T*)x, xs, (const W*)w, (const W*)b, (T*)y, (A*)mean,
                                                      (A*)rstd, n, (int)width, eps);
}
template <typename T, typename W>
void run_fwd(const void* x, int64_t xs, const void* w, const void* b, void* y, void* mean, void* rstd, int64_t n,
             int64_t width, double eps, hipStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int V = LnVec<T>::value;
  // The fewest lanes that hold the row in 32 values each, and for them the shortest of these rows: 65536x128 bf16 with 16
  // lanes 8.1 us, with 32 13.5, with 64 22.6; 65536x784 bf16 in two vectors to a lane 45 us, in four 75; 16384x4096 bf16 in
  // 256 lanes 47 us, in four vectors to a lane 83, in 1024 lanes 398 (all without the rows ahead).  (64 values in one wave
  // instead of 16 in four: 65536x4096 bf16 0.36 ms against 0.26.)
  constexpr int MAXC = 32 / V;
  const int64_t vectors = (width + V - 1) / V;
#define LN_FWD(TPR, NCH) \
  if (vectors <= (int64_t)(TPR) * (NCH)) return launch_fwd<T, W, TPR, NCH>(x, xs, w, b, y, mean, rstd, n, width, eps, st)
  LN_FWD(16, 1);
  LN_FWD(32, 1);
  LN_FWD(64, 1);
  LN_FWD(64, 2);
  LN_FWD(64, MAXC / 2 < 2 ? 2 : MAXC / 2);
  LN_FWD(64, MAXC);
  LN_FWD(256, MAXC / 2 < 2 ? 2 : MAXC / 2);
  LN_FWD(256, MAXC);
  LN_FWD(1024, MAXC);
#undef LN_FWD
  ln_fwd_long_kernel<T, W><<<vmf_grid_for(n, 1, 1 << 16), 1024, 0, st>>>((const T*)x, xs, (const W*)w, (const W*)b,
                                                                         (T*)y, (A*)mean, (A*)rstd, n, width, eps);
}

template <typename T> constexpr int bwd_chunks() { return 16 / LnVec<T>::value; }  // 16 values per lane

// How the backward pass is launched (host arithmetic shared with the workspace query).
struct BwdPlan {
  int tpr;      // lanes per row; 0: rows that do not fit the registers
  int threads;  // of a workgroup
  int parts;    // workgroups, each leaving a partial row of gw and gb; 0: none are left (few rows)
};
// Few rows (up to 1024, rows of up to 256 lanes): one launch (128x128 fp32 3.1 us, with partials 8.9; 1024x784 7.8 and 8.6;
// 1536x784 12.7 and 9.5; wide rows: 128x4096 3.5 and 9.8, 512x4096 10.1 and 15.8, 1024x4096 19.1 and 18.3, in bf16 14.3 and
// 19.9).
// Otherwise two workgroups for each of 256 compute units (1048576x784 fp32, a wave to a row, 1.88 ms, with four 2.00), four
// where the other waves have more to fill: rows of 16 bits, whose loads are half as many (1048576x784 bf16 1.14 ms, with two
// 1.88), and rows of four waves, which wait at barriers (65536x4096 bf16 0.33 ms, with two 0.50).  No more than have 32
// rows each, since each leaves 2 * width values that are written and read again; 16 where a wave or more works on one row
// (16384x4096 bf16 98 us, with 32 136; 8192x128 bf16, 16 lanes to a row, 8.2 us, with 32 7.8).
template <typename T>
BwdPlan bwd_plan(int64_t n, int64_t width) {
  constexpr int V = LnVec<T>::value;
  BwdPlan p;
  p.tpr = lanes_for((width + V - 1) / V, bwd_chunks<T>());
  p.threads = p.tpr == 0 ? 256 : p.tpr > THREADS ? p.tpr : THREADS;
  const int64_t most = sizeof(T) == 2 || p.tpr == THREADS ? 1024 : 512;
  if (p.tpr == 0) {
    // (its launch has a workgroup for each 256 columns of a part: more parts only where those do not fill the chip, since
    // wide parts are large: 16 rows of 2^22 fp32 leave one of 34 MB, where one for each row takes 2.79 ms for 2.52)
    const int64_t columns = (width + 255) / 256;
    int64_t g = (n + 15) / 16;
    if (g * columns < 1024) g = (1024 + columns - 1) / columns < n ? (1024 + columns - 1) / columns : n;
    p.parts = (int)(g < 1 ? 1 : g > most ? most : g);
    return p;
  }
  if (p.tpr != 0 && p.tpr <= THREADS && n <= 1024) {
    p.parts = 0;
    return p;
  }
  // rows to a workgroup: those, or as many as it has side by side, or fewer where that leaves compute units without one
  const int64_t at_once = p.threads / p.tpr;
  const int64_t few = p.tpr >= 64 ? 16 : 32, rows = at_once > few ? at_once : few;
  int64_t g = (n + rows - 1) / rows;
  if (g < 256) g = (n + at_once - 1) / at_once < 256 ? (n + at_once - 1) / at_once : 256;
  p.parts = (int)(g < 1 ? 1 : g > most ? most : g);
  return p;
}

template <typename T, typename W>
int run_bwd(const void* x, int64_t xs, const void* gy, int64_t gs, const void* w, const void* mean, const void* rstd,
            void* gx, void* gw, void* gb, void* ws, int64_t n, int64_t width, hipStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int V = LnVec<T>::value;
  constexpr int C = bwd_chunks<T>();
  const BwdPlan pl = bwd_plan<T>(n, width);
  A* partial = gw || gb ? (A*)ws : nullptr;
  const int64_t vectors = (width + V - 1) / V;
  if (pl.tpr != 0 && pl.parts == 0) {
    const int rows = THREADS / pl.tpr;
    const int row_groups = gx ? (int)((n + rows - 1) / rows) : 0;
    const int grid = row_groups + (gw || gb ? (int)((width + 15) / 16) : 0);
#define LN_FEW(TPR, NCH)                                                                                      \
  ln_bwd_few_kernel<T, W, TPR, NCH><<<grid, THREADS, 0, st>>>((const T*)x, xs, (const T*)gy, gs, (const W*)w, \
                                                              (const A*)mean, (const A*)rstd, (T*)gx, (W*)gw, \
                                                              (W*)gb, (int)n, (int)width, row_groups)
    if (grid > 0) {
      if (pl.tpr == 16) LN_FEW(16, C);
      else if (pl.tpr == 32) LN_FEW(32, C);
      else if (pl.tpr == 64) LN_FEW(64, C);
      else LN_FEW(256, C);
    }
#undef LN_FEW
    return vmf_check_launch("vmf_layer_norm_bwd");
  }
#define LN_BWD(NT, TPR, NCH)                                                                                    \
  ln_bwd_kernel<T, W, NT, TPR, NCH><<<pl.parts, NT, 0, st>>>((const T*)x, xs, (const T*)gy, gs, (const W*)w,      \
                                                             (const A*)mean, (const A*)rstd, (T*)gx, partial, n, \
                                                             (int)width)
  if (pl.tpr == 16) {
    if (vectors <= 16) LN_BWD(THREADS, 16, 1);
    else LN_BWD(THREADS, 16, C);
  } else if (pl.tpr == 32) {
    LN_BWD(THREADS, 32, C);
  } else if (pl.tpr == 64) {
    LN_BWD(THREADS, 64, C);
  } else if (pl.tpr == 256) {
    LN_BWD(256, 256, C);
  } else if (pl.tpr == 1024) {
    LN_BWD(1024, 1024, C);
  } else {
    if (gx)
      ln_bwd_long_kernel<T, W><<<vmf_grid_for(n, 1, 1 << 16), 1024, 0, st>>>(
          (const T*)x, xs, (const T*)gy, gs, (const W*)w, (const A*)mean, (const A*)rstd, (T*)gx, n, width);
    if (partial)
      ln_cols_kernel<T><<<dim3((unsigned)((width + 255) / 256), (unsigned)pl.parts), 256, 0, st>>>(
          (const T*)x, xs, (const T*)gy, gs, (const A*)mean, (const A*)rstd, partial, n, width);
  }
#undef LN_BWD
  int rc = vmf_check_launch("vmf_layer_norm_bwd");
  if (rc != VMF_OK || !partial) return rc;
  ln_reduce_kernel<A, W><<<(unsigned)((2 * width + 15) / 16), 16 * REDUCE_SHARE, 0, st>>>(partial, (W*)gw, (W*)gb,
                                                                                         pl.parts, width);
  return vmf_check_launch("vmf_layer_norm_bwd sums");
}

int check_common(const char* what, int64_t n, int64_t width, int64_t stride, int dtype, int wdtype) {
  VMF_REQUIRE(n >= 0, VMF_ERR_BAD_ARG, "%s: n < 0", what);
  VMF_REQUIRE(width >= 1, VMF_ERR_BAD_ARG, "%s: width must be at least 1", what);
  VMF_REQUIRE(width <= VMF_LAYER_NORM_MAX_WIDTH, VMF_ERR_UNSUPPORTED, "%s: width > %lld", what,
              (long long)VMF_LAYER_NORM_MAX_WIDTH);
  VMF_REQUIRE(stride >= 0, VMF_ERR_BAD_ARG, "%s: negative row stride", what);
  VMF_REQUIRE(dtype >= VMF_F32 && dtype <= VMF_BF16, VMF_ERR_DTYPE, "%s: dtype %d", what, dtype);
  VMF_REQUIRE(wdtype == dtype || (wdtype == VMF_F32 && dtype != VMF_F64), VMF_ERR_DTYPE,
              "%s: the weight's dtype is the rows' or VMF_F32, got %d", what, wdtype);
  return VMF_OK;
}

}  // namespace

// (T, W) pairs: weights in the rows' type, or fp32 ones with 16-bit rows
#define LN_DISPATCH(dtype, wdtype, CALL)                                   \
  do {                                                                     \
    if ((dtype) == VMF_F32) { using T = float; using W = float; CALL; }    \
    else if ((dtype) == VMF_F64) { using T = double; using W = double; CALL; } \
    else if ((dtype) == VMF_F16) {                                         \
      using T = f16_t;                                                     \
      if ((wdtype) == VMF_F32) { using W = float; CALL; } else { using W = f16_t; CALL; } \
    } else {                                                               \
      using T = bf16_t;                                                    \
      if ((wdtype) == VMF_F32) { using W = float; CALL; } else { using W = bf16_t; CALL; } \
    }                                                                      \
  } while (0)

extern "C" int vmf_layer_norm_fwd(const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                                  void* mean_out, void* rstd_out, int64_t n, int64_t width, double eps, int dtype,
                                  int weight_dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_layer_norm_fwd");
  int rc = check_common("vmf_layer_norm_fwd", n, width, x_stride, dtype, weight_dtype);
  if (rc != VMF_OK) return rc;
  if (n == 0) return VMF_OK;
  VMF_REQUIRE(x && y, VMF_ERR_BAD_ARG, "vmf_layer_norm_fwd: null pointer");
  VMF_REQUIRE(!mean_out == !rstd_out, VMF_ERR_BAD_ARG, "vmf_layer_norm_fwd: mean_out and rstd_out go together");
  hipStream_t st = (hipStream_t)stream;
  LN_DISPATCH(dtype, weight_dtype,
              (run_fwd<T, W>(x, x_stride, weight, bias, y, mean_out, rstd_out, n, width, eps, st)));
  return vmf_check_launch("vmf_layer_norm_fwd");
}

extern "C" int vmf_layer_norm_bwd_workspace(int64_t n, int64_t width, int dtype, int64_t* bytes_out) {
  int rc = check_common("vmf_layer_norm_bwd_workspace", n, width, 0, dtype, dtype);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(bytes_out, VMF_ERR_BAD_ARG, "vmf_layer_norm_bwd_workspace: null pointer");
  int parts;
  if (dtype == VMF_F32) parts = bwd_plan<float>(n, width).parts;
  else if (dtype == VMF_F64) parts = bwd_plan<double>(n, width).parts;
  else parts = bwd_plan<f16_t>(n, width).parts;
  *bytes_out = (int64_t)parts * 2 * width * (dtype == VMF_F64 ? 8 : 4);
  return VMF_OK;
}

extern "C" int vmf_layer_norm_bwd(const void* x, int64_t x_stride, const void* gy, int64_t gy_stride,
                                  const void* weight, const void* mean, const void* rstd, void* gx, void* gweight,
                                  void* gbias, int64_t n, int64_t width, void* workspace, int64_t workspace_bytes,
                                  int dtype, int weight_dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_layer_norm_bwd");
  int rc = check_common("vmf_layer_norm_bwd", n, width, x_stride < gy_stride ? x_stride : gy_stride, dtype,
                        weight_dtype);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(n == 0 || (x && gy && mean && rstd), VMF_ERR_BAD_ARG, "vmf_layer_norm_bwd: null pointer");
  if (gweight || gbias) {
    int64_t need = 0;
    vmf_layer_norm_bwd_workspace(n, width, dtype, &need);
    VMF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VMF_ERR_BAD_ARG,
                "vmf_layer_norm_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  } else if (!gx || n == 0) {
    return VMF_OK;
  }
  hipStream_t st = (hipStream_t)stream;
  LN_DISPATCH(dtype, weight_dtype, (rc = run_bwd<T, W>(x, x_stride, gy, gy_stride, weight, mean, rstd, gx, gweight,
                                                       gbias, workspace, n, width, st)));
  return rc;
}
