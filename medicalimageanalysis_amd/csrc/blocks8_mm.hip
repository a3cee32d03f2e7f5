// blocks8_mm.hip -- products of 8-bit blocks.
//
//   out[m][n] = sum over block columns of 2^(ea + eb) sum_k a[m][k] b[n][k]  (+ bias[n]) (* softplus slope at gate[m][n])
//   gweight[n][k] = sum_m gy[m][n] a[m][k],  gbias[n] = sum_m gy[m][n]
//
// Both are bound by the matrix instructions for large sizes and by the bytes of the operands for few rows.
//
// The 8-bit matrix instruction takes a whole block column (K = 128) and both exponent bytes, so the scales cost no vector
// work.  Its sums are not 32-bit: it adds the products in eights (consecutive k), and of each cuts off what is below 2^-13 of
// the largest one's power of two; the eights' sums are then added with the bits of fp32.  So a result is off by at most
// 7 * 2^-13 = 8.5e-4 of the sum of its terms' magnitudes.  Measured: of normal values 1.3e-5, of the results' norm as of the
// sum of magnitudes, for K = 128 as for K = 8192; of values whose sizes spread like exp(2 normal) inside a block up to
// 2.6e-4 of the sum of magnitudes.  Half a step is 3.9e-3 in bf16, 4.9e-4 in fp16: the 1.3e-5 are a 300th and a 37th of that,
// and 1 % of bf16 results, 7 % of fp16 ones, are rounded to the other neighbour.  It is used for 16-bit results, since it
// takes half the time (16384x4096x4096 224 - 260 us against 500) and what the operands lost to their 3 bits of mantissa is
// far more.  A 32-bit result is computed with the bf16 instruction instead: an element of a block is exact in bf16, so are
// the products, and the sums are 32-bit (4e-8 at K = 1024).
#include <type_traits>

#include "blocks8_dev.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v8i_at16 __attribute__((ext_vector_type(8), aligned(16)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

#define LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))
#define GLOBAL_PTR(p) ((__attribute__((address_space(1))) const void*)(p))

struct Operand {
  const uint8_t* values;
  const uint8_t* exps;
  int64_t pitch, exp_pitch;  // bytes
  int64_t rows;
  int tiled;  // one exponent per 128 rows
};
struct MmArgs {
  Operand a, b, gate;  // gate.values null: none
  const void* bias;
  void* out;
  float* partial;  // split over the block columns: [split][m][n]
  int64_t m, n;
  int blocks, blocks_per_split;
  int mt, nt;  // tiles
  int bias_code;
  float beta;
};

// F exponent bytes of the rows row0 + F * (lane & 15) + 0..F-1, in one word.  Rows behind the last one get some byte of
// the array (their products are dropped).  A tile's one byte is repeated by spread_exps, later: an operation on the loaded
// value would wait for every load before it, the next stage's among them.
template <int F>
__device__ __forceinline__ int load_exps(const Operand& o, int64_t kb, int64_t row0, int lane) {
  const uint8_t* e = o.exps + kb * o.exp_pitch;
  if (o.tiled) {
    int64_t r = row0 >> 7;
    r = r < o.exp_pitch ? r : o.exp_pitch - 1;
    return e[r];
  }
  int64_t r = row0 + F * (lane & 15);
  const int64_t last = o.exp_pitch - F;
  r = r < last ? r : last;
  if constexpr (F == 4) return *reinterpret_cast<const int*>(e + r);
  if constexpr (F == 2) return *reinterpret_cast<const uint16_t*>(e + r);
  return e[r];
}
__device__ __forceinline__ int spread_exps(const Operand& o, int raw) { return o.tiled ? raw * 0x01010101 : raw; }

// acc += A B for one block column of a 16 x 16 tile; IA, IB: which byte of the exponent words
template <int IA, int IB>
__device__ __forceinline__ v4f mm_step(v8i a, v8i b, v4f acc, int ea, int eb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, IA, ea, IB, eb);
}
// the 32 values of a lane as four bf16 operands, scaled (exact: 4 bits times a power of two)
__device__ __forceinline__ void to_bf16(v8i v, float scale, v8b* out) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v2b lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * q + h], scale, false);
      const v2b hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * q + h], scale, true);
      out[q][4 * h] = lo[0];
      out[q][4 * h + 1] = lo[1];
      out[q][4 * h + 2] = hi[0];
      out[q][4 * h + 3] = hi[1];
    }
}
__device__ __forceinline__ v4f mm_step_bf16(const v8b* a, const v8b* b, v4f acc) {
#pragma unroll
  for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[q], b[q], acc, 0, 0, 0);
  return acc;
}

__device__ __forceinline__ float load_bias(const void* bias, int code, int64_t i) {
  return code == VMF_F32 ? ((const float*)bias)[i]
                         : code == VMF_F16 ? (float)((const f16_t*)bias)[i] : (float)((const bf16_t*)bias)[i];
}

// bias, gate and rounding of one element
template <typename OUT>
__device__ __forceinline__ void finish1(const MmArgs& p, int64_t row, int64_t col, float v) {
  if (p.bias) v += load_bias(p.bias, p.bias_code, col);
  if (p.gate.values) {
    float a[4];
    b8_unpack4(p.gate.values[row * p.gate.pitch + col], b8_scale(p.gate.exps[(col >> 7) * p.gate.exp_pitch + row]), a);
    v *= b8_softplus_slope<sizeof(OUT) == 2>(a[0], p.beta);
  }
  ((OUT*)p.out)[row * p.n + col] = (OUT)v;
}

// Workgroup b of `all` runs on XCD b % 8: the place of b where each XCD has a contiguous run
__device__ __forceinline__ int xcd_run(int b, int all) {
  const int q = all >> 3, r = all & 7, x = b & 7;
  return x * q + (x < r ? x : r) + (b >> 3);
}
// Each XCD gets a contiguous run of tiles, and the run is walked in columns of 8 row tiles, so that the rows and columns
// in use at a time fit its L2.
__device__ __forceinline__ void tile_of(const MmArgs& p, int id, int& mt, int& nt) {
  id = xcd_run(id, p.mt * p.nt);
  const int group = id / (8 * p.nt), first = group * 8, high = p.mt - first < 8 ? p.mt - first : 8;
  const int in_group = id - group * 8 * p.nt;
  mt = first + in_group % high;
  nt = in_group / high;
}
// The row of an operand whose 16-byte pieces lie at place `at` of a stage's part for it (F: row tiles that share an
// exponent word), and the piece that lies there.
template <int F>
__device__ __forceinline__ int row_at(int at) {
  const int tile = at >> 4;
  return tile / F * (16 * F) + F * (at & 15) + tile % F;
}
// Where piece c of row q (of 16 side by side, 128 bytes each) lies in the row: c ^ swizzle(q).  A 16-byte LDS read is served
// in groups of 16 lanes, which measured are lanes 0 - 3, 12 - 15 and 20 - 27 of each 32 and the others: the 16 rows, once
// each, with piece c in rows 0 - 3 and 12 - 15 and c ^ 2 in rows 4 - 11.  Two rows fill the banks once, so the eight pairs of
// rows have to read eight different places.
__device__ __forceinline__ int swizzle(int q) {
  const int h = q >> 1;
  return h ^ (((h + 2) >> 1) & 2);
}
// a 16-row operand tile from LDS: lane l gets row l % 16, the 32 bytes of quarter l / 16
__device__ __forceinline__ v8i operand(const uint8_t* tile, int lane) {
  const int q = lane & 15, c = (lane >> 4) * 2;
  const v4i lo = *reinterpret_cast<const v4i*>(tile + q * B8 + ((c ^ swizzle(q)) << 4));
  const v4i hi = *reinterpret_cast<const v4i*>(tile + q * B8 + (((c + 1) ^ swizzle(q)) << 4));
  return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
// What a wave holds of the result: lane l has the rows 4 FM * (l / 16) + t (t = FM * r + i: element r of row tile i) and
// the columns FN * (l % 16) + 0 .. FN - 1 of each group of 16 FM rows and 16 FN columns.  GATE: the 4 FM rows' kept
// values are all asked for before the first is used.
template <int FM, int FN, int GM, int GN, bool GATE, typename OUT>
__device__ __forceinline__ void write_tile(const MmArgs& p, const v4f (&acc)[GM * FM][GN * FN], int64_t row0, int64_t col0,
                                           int lane) {
  constexpr int R = 4 * FM;
  const bool whole = row0 + GM * 16 * FM <= p.m && col0 + GN * 16 * FN <= p.n;
#pragma unroll
  for (int h = 0; h < GN; ++h) {
    const int64_t col = col0 + h * 16 * FN + FN * (lane & 15);
    if (!whole && col >= p.n) continue;
    const int left = whole || p.n - col >= FN ? FN : (int)(p.n - col);
    float bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) bias[j] = p.bias && !p.partial && j < left ? load_bias(p.bias, p.bias_code, col + j) : 0.0f;
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      const int64_t row = row0 + g * 16 * FM + R * (lane >> 4);
      const int rows = whole || p.m - row >= R ? R : (int)(p.m - row);
      if (rows <= 0) continue;
      uint32_t code[GATE ? R : 1], ex[GATE ? R / 4 : 1];
      if constexpr (GATE) {
        const uint8_t* q = p.gate.values + row * p.gate.pitch + col;
#pragma unroll
        for (int t = 0; t < R; ++t) {
          const uint8_t* at = q + (t < rows ? t : rows - 1) * p.gate.pitch;
          code[t] = FN == 4 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
        }
        // (the exponents of rows come in sixteens, so these words are all there)
        const uint32_t* e = reinterpret_cast<const uint32_t*>(p.gate.exps + (col >> 7) * p.gate.exp_pitch + row);
#pragma unroll
        for (int t = 0; t < R / 4; ++t) ex[t] = e[t];
      }
      OUT* out = (OUT*)p.out + row * p.n + col;
      float* part = p.partial + ((int64_t)blockIdx.y * p.m + row) * p.n + col;
#pragma unroll
      for (int t = 0; t < R; ++t) {
        if (t < rows) {
          float v[FN];
#pragma unroll
          for (int j = 0; j < FN; ++j) v[j] = acc[g * FM + t % FM][h * FN + j][t / FM];
          if (p.partial) {
            store_some<FN>(part, left, v);
          } else {
#pragma unroll
            for (int j = 0; j < FN; ++j) v[j] += bias[j];
            if constexpr (GATE) {
              float a[4];
              b8_unpack4(code[t], b8_scale(ex[t / 4] >> (8 * (t % 4)) & 0xff), a);
#pragma unroll
              for (int j = 0; j < FN; ++j) v[j] *= b8_softplus_slope<sizeof(OUT) == 2>(a[j], p.beta);
            }
            store_some<FN>(out, left, v);
          }
        }
        out += p.n;
        part += p.n;
      }
    }
  }
}

// Tile of BM x BN over the block columns, waves of WM x WN side by side.
//   LDS: two stages of the tile's rows of 128 bytes, filled by loads that go from global memory straight into LDS; while
//   one stage is multiplied the next is on its way, one barrier per block column.
//   A 16-row operand tile takes the rows F * (lane & 15) + i (i = 0 .. F - 1 the tile's number): the exponents of a
//   lane's F tiles are then one word, and a lane's results are F consecutive columns of a row.
//   In LDS the 16 rows of an operand tile lie side by side, their pieces swizzled (see swizzle).
// Measured: WIDE (fp32) 16384x4096x4096 500 us (1.1 PFLOP/s of bf16 instructions, whose number bounds it), 16384x784x128
// 17 us; 37x785x1000 7.4 us, a matter of latency.
template <int BM, int BN, int WM, int WN, bool WIDE, bool GATE, typename OUT>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void mm_kernel(MmArgs p) {
  constexpr int WAVES_N = BN / WN, WAVES = (BM / WM) * WAVES_N;
  constexpr int FM = WM / 16 < 4 ? WM / 16 : 4, FN = WN / 16 < 4 ? WN / 16 : 4;  // tiles that share an exponent word
  constexpr int GM = WM / (16 * FM), GN = WN / (16 * FN);
  constexpr int STAGE = (BM + BN) * B8;
  constexpr int LOADS = (BM + BN) / 8 / WAVES;  // one fills eight rows
  static_assert((BM + BN) % (8 * WAVES) == 0, "every wave loads the same number of rows");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int mt, nt;
  tile_of(p, (int)blockIdx.x, mt, nt);
  const int64_t m0 = (int64_t)mt * BM, n0 = (int64_t)nt * BN;
  const int kb0 = (int)blockIdx.y * p.blocks_per_split;
  const int kb1 = kb0 + p.blocks_per_split < p.blocks ? kb0 + p.blocks_per_split : p.blocks;

  // where this lane's loads read: row (clamped to the last one) and 16-byte piece
  const uint8_t* src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r8 = wave * LOADS + i;  // eight rows of the stage: first A's, then B's
    const bool is_b = r8 >= BM / 8;
    const int at = (is_b ? r8 - BM / 8 : r8) * 8 + (lane >> 3), q = at & 15;  // the row's place in LDS
    const int r = is_b ? row_at<FN>(at) : row_at<FM>(at);
    const int piece = (lane & 7) ^ swizzle(q);
    const Operand& o = is_b ? p.b : p.a;
    int64_t row = (is_b ? n0 : m0) + r;
    row = row < o.rows ? row : o.rows - 1;
    src[i] = o.values + row * o.pitch + piece * 16;
  }
  const int wm = (wave / WAVES_N) * WM, wn = (wave % WAVES_N) * WN;

  v4f acc[GM * FM][GN * FN];
#pragma unroll
  for (int i = 0; i < GM * FM; ++i)
#pragma unroll
    for (int j = 0; j < GN * FN; ++j) acc[i][j] = v4f{0, 0, 0, 0};

  int ea[2][GM], eb[2][GN];
  auto fetch = [&](int kb, int stage) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      __builtin_amdgcn_global_load_lds(GLOBAL_PTR(src[i] + (int64_t)kb * B8),
                                       LDS_PTR(void, lds + stage * STAGE + (wave * LOADS + i) * 1024), 16, 0, 0);
  };
  auto fetch_exps = [&](int kb, int slot) {
#pragma unroll
    for (int g = 0; g < GM; ++g) ea[slot][g] = load_exps<FM>(p.a, kb, m0 + wm + g * 16 * FM, lane);
#pragma unroll
    for (int g = 0; g < GN; ++g) eb[slot][g] = load_exps<FN>(p.b, kb, n0 + wn + g * 16 * FN, lane);
  };
  auto multiply = [&](int stage, const int* xa, const int* xb, auto&& then) {
    const uint8_t* A = lds + stage * STAGE;
    const uint8_t* B = A + BM * B8;
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      if constexpr (!WIDE) {
        v8i a[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) a[i] = operand(A + (wm + (g * FM + i) * 16) * B8, lane);
        if (g == 0) then();
#pragma unroll
        for (int h = 0; h < GN; ++h)
          static_for<FN>([&](auto J) {
            constexpr int j = decltype(J)::value;
            const v8i b = operand(B + (wn + (h * FN + j) * 16) * B8, lane);
            static_for<FM>([&](auto I) {
              constexpr int i = decltype(I)::value;
              v4f& c = acc[g * FM + i][h * FN + j];
              c = mm_step<i, j>(a[i], b, c, xa[g], xb[h]);
            });
          });
      } else {
        v8b a[FM][4], b[4];
#pragma unroll
        for (int i = 0; i < FM; ++i)
          to_bf16(operand(A + (wm + (g * FM + i) * 16) * B8, lane), b8_scale((xa[g] >> (8 * i)) & 0xff), a[i]);
        if (g == 0) then();
#pragma unroll
        for (int h = 0; h < GN; ++h)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            to_bf16(operand(B + (wn + (h * FN + j) * 16) * B8, lane), b8_scale((xb[h] >> (8 * j)) & 0xff), b);
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[g * FM + i][h * FN + j] = mm_step_bf16(a[i], b, acc[g * FM + i][h * FN + j]);
          }
      }
    }
  };

  if (kb0 < kb1) {
    fetch(kb0, 0);
    fetch_exps(kb0, 0);
  }
  for (int kb = kb0; kb < kb1; kb += 2) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (kb + half < kb1) {
        // this wave's share of the stage has arrived; after the barrier everyone's has, and the other stage is free
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        int xa[GM], xb[GN];
#pragma unroll
        for (int g = 0; g < GM; ++g) xa[g] = spread_exps(p.a, ea[half][g]);
#pragma unroll
        for (int g = 0; g < GN; ++g) xb[g] = spread_exps(p.b, eb[half][g]);
        multiply(half, xa, xb, [&] {  // (behind the first operand reads, which would wait in the queue otherwise)
          if (kb + half + 1 < kb1) {
            fetch(kb + half + 1, half ^ 1);
            fetch_exps(kb + half + 1, half ^ 1);
          }
        });
      }
    }
  }

  write_tile<FM, FN, GM, GN, GATE, OUT>(p, acc, m0 + wm, n0 + wn, lane);
}

// The same for large 16-bit results: tile of 256 x 256, eight waves of 128 x 64, a block column's 32 products per wave in
// four phases of two row tiles and all four column tiles.  What a phase multiplies was read from LDS in the phase before,
// also across block columns: the barrier that makes the next stage readable, and the stage read last writable, stands
// before the last phase's products, whose operands are in registers by then.  The loads into LDS are spread over three
// phases, so that they do not stand before the operand reads in the queue.
// Bound: 2048 clocks of matrix instructions per block column and CU, against 768 + 512 clocks of LDS reads and writes; and the
// clock itself, which falls to 1.8 - 2.0 GHz under them.  16384x4096x4096 bf16: 224 us by itself (2.45 PFLOP/s), 235 - 260 us
// in a row of calls, GATE 260 - 275; 8192^3 2.5 PFLOP/s.
// a by rows, b by tiles, as a layer has them.
template <bool GATE, typename OUT>
__global__ __launch_bounds__(512, 2) void mm_large_kernel(MmArgs p) {
  constexpr int BM = 256, BN = 256, STAGE = (BM + BN) * B8;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int mt, nt;
  tile_of(p, (int)blockIdx.x, mt, nt);
  const int64_t m0 = (int64_t)mt * BM, n0 = (int64_t)nt * BN;
  const int kb0 = (int)blockIdx.y * p.blocks_per_split;
  const int kb1 = kb0 + p.blocks_per_split < p.blocks ? kb0 + p.blocks_per_split : p.blocks;
  const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;

  // waves 0 - 3 load A's rows, 4 - 7 B's, 64 each; offsets from the tile's first row fit 32 bits (rows of up to 2^22)
  const Operand& mine = wave < 4 ? p.a : p.b;
  const int64_t first = wave < 4 ? m0 : n0;
  const uint8_t* base = mine.values + first * mine.pitch;
  const int64_t last = mine.rows - 1 - first;
  uint32_t off[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = (wave & 3) * 64 + i * 8 + (lane >> 3), r = row_at<4>(at);
    off[i] = (uint32_t)((r < last ? r : last) * mine.pitch) + (((lane & 7) ^ swizzle(at & 15)) << 4);
  }
  auto load = [&](int kb, int stage, int i) {
    __builtin_amdgcn_global_load_lds(GLOBAL_PTR(base + (int64_t)kb * B8 + off[i]),
                                     LDS_PTR(void, lds + stage * STAGE + (wave * 8 + i) * 1024), 16, 0, 0);
  };
  // the exponents of this lane's 8 row tiles, in two words, and the byte of the wave's column tile
  struct Exps {
    int a0, a1, b;
  };
  const int64_t end = p.a.exp_pitch - 4, r0 = m0 + wm + 4 * (lane & 15), r1 = r0 + 64;
  const uint8_t* ea0 = p.a.exps + (r0 < end ? r0 : end);
  const uint8_t* ea1 = p.a.exps + (r1 < end ? r1 : end);
  const int64_t ct = (n0 + wn) >> 7;
  const uint8_t* eb = p.b.exps + (ct < p.b.exp_pitch ? ct : p.b.exp_pitch - 1);
  auto load_exps_of = [&](int kb) {
    return Exps{*reinterpret_cast<const int*>(ea0 + kb * p.a.exp_pitch),
                *reinterpret_cast<const int*>(ea1 + kb * p.a.exp_pitch), eb[kb * p.b.exp_pitch]};
  };

  v4f acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  v8i a[2][2], b[4];
  auto read_a = [&](int stage, int pair, v8i(&to)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) to[i] = operand(lds + stage * STAGE + (wm + (2 * pair + i) * 16) * B8, lane);
  };
  auto read_b = [&](int stage, int j) { b[j] = operand(lds + stage * STAGE + (BM + wn + j * 16) * B8, lane); };
  // row tiles 2 PAIR, 2 PAIR + 1 with column tile J
  auto multiply = [&](const v8i(&row)[2], auto PAIR, auto J, const Exps& e) {
    constexpr int j = decltype(J)::value, t = 2 * decltype(PAIR)::value;
    const int xa = t < 4 ? e.a0 : e.a1;
    acc[t][j] = mm_step<t % 4, j>(row[0], b[j], acc[t][j], xa, e.b);
    acc[t + 1][j] = mm_step<t % 4 + 1, j>(row[1], b[j], acc[t + 1][j], xa, e.b);
  };

  // One block column.  MORE: how many follow (2: at least two).  No branch inside: products and reads keep their order.
  Exps now, raw;
  auto step = [&](int kb, int stage, auto MORE) {
    constexpr int more = decltype(MORE)::value;
    static_for<3>([&](auto P) {
      constexpr int ph = decltype(P)::value;
      __builtin_amdgcn_sched_barrier(0);
      multiply(a[ph & 1], P, std::integral_constant<int, 0>{}, now);
      __builtin_amdgcn_sched_barrier(0);
      read_a(stage, ph + 1, a[(ph + 1) & 1]);
      if constexpr (more > 0 && ph < 2) {
#pragma unroll
        for (int i = 0; i < 3; ++i) load(kb + 1, stage ^ 1, 2 + 3 * ph + i);
      }
      __builtin_amdgcn_sched_barrier(0);
      static_for<3>([&](auto J) { multiply(a[ph & 1], P, std::integral_constant<int, decltype(J)::value + 1>{}, now); });
    });
    __builtin_amdgcn_sched_barrier(0);
    Exps then = now;
    if constexpr (more > 0) {
      // this wave's share of the next stage has arrived; after the barrier everyone's has, and everyone has read the
      // last of this stage
      // (the exponents pass through the wait, so that their first use does not bring one of its own)
      asm volatile("s_waitcnt vmcnt(0)" : "+v"(raw.a0), "+v"(raw.a1), "+v"(raw.b) : : "memory");
      __syncthreads();
      then = Exps{raw.a0, raw.a1, raw.b * 0x01010101};
      if constexpr (more > 1) {
        raw = load_exps_of(kb + 2);
        load(kb + 2, stage, 0);
        load(kb + 2, stage, 1);
      }
      read_a(stage ^ 1, 0, a[0]);
    }
    static_for<4>([&](auto J) {
      __builtin_amdgcn_sched_barrier(0);
      multiply(a[1], std::integral_constant<int, 3>{}, J, now);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (more > 0) read_b(stage ^ 1, decltype(J)::value);
    });
    __builtin_amdgcn_sched_barrier(0);
    now = then;
  };
  if (kb0 < kb1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) load(kb0, 0, i);
    now = load_exps_of(kb0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    now.b *= 0x01010101;
    read_a(0, 0, a[0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) read_b(0, j);
    int kb = kb0;
    if (kb + 1 < kb1) {
      raw = load_exps_of(kb0 + 1);
      load(kb0 + 1, 1, 0);
      load(kb0 + 1, 1, 1);
      for (; kb + 2 < kb1; ++kb) step(kb, (kb - kb0) & 1, std::integral_constant<int, 2>{});
      step(kb, (kb - kb0) & 1, std::integral_constant<int, 1>{});
      ++kb;
    }
    step(kb, (kb - kb0) & 1, std::integral_constant<int, 0>{});
  }
  write_tile<4, 4, 2, 1, GATE, OUT>(p, acc, m0 + wm, n0 + wn, lane);
}

// the eight waves' sums of 16 rows and 16 columns, added in their order
template <typename OUT>
__device__ __forceinline__ void few_result(const MmArgs& p, float (&sums)[8][16][17], v4f acc, int64_t n0, int lane,
                                           int wave) {
#pragma unroll
  for (int r = 0; r < 4; ++r) sums[wave][4 * (lane >> 4) + r][lane & 15] = acc[r];
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int64_t row = threadIdx.x >> 4, col = n0 + (threadIdx.x & 15);
  if (row >= p.m || col >= p.n) return;
  float v = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) v += sums[w][threadIdx.x >> 4][threadIdx.x & 15];
  if (p.partial) {
    p.partial[((int64_t)blockIdx.y * p.m + row) * p.n + col] = v;
  } else {
    finish1<OUT>(p, row, col, v);
  }
}

// Up to 16 rows: the weight's bytes are what there is to move.  A workgroup takes 16 columns, its eight waves share the
// block columns and read both operands straight into registers; their sums are added through LDS (1x4096x4096 4.5 us,
// 3.7 TB/s of the weight).
template <bool WIDE, typename OUT>
__global__ __launch_bounds__(512) void mm_few_kernel(MmArgs p) {
  __shared__ float sums[8][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int kb0 = (int)blockIdx.y * p.blocks_per_split;
  const int kb1 = kb0 + p.blocks_per_split < p.blocks ? kb0 + p.blocks_per_split : p.blocks;
  const int64_t ra = (lane & 15) < p.m ? (lane & 15) : p.m - 1;
  const int64_t rb = n0 + (lane & 15) < p.n ? n0 + (lane & 15) : p.n - 1;
  const uint8_t* A = p.a.values + ra * p.a.pitch + (lane >> 4) * 32;
  const uint8_t* B = p.b.values + rb * p.b.pitch + (lane >> 4) * 32;
  const uint8_t* ea = p.a.exps + (p.a.tiled ? ra >> 7 : ra);
  const uint8_t* eb = p.b.exps + (p.b.tiled ? rb >> 7 : rb);
  v4f acc = {0, 0, 0, 0};
  for (int kb = kb0 + wave; kb < kb1; kb += 8) {
    const v8i a = *reinterpret_cast<const v8i_at16*>(A + (int64_t)kb * B8);
    const v8i b = *reinterpret_cast<const v8i_at16*>(B + (int64_t)kb * B8);
    const int xa = ea[(int64_t)kb * p.a.exp_pitch], xb = eb[(int64_t)kb * p.b.exp_pitch];
    if constexpr (!WIDE) {
      acc = mm_step<0, 0>(a, b, acc, xa, xb);
    } else {
      v8b aw[4], bw[4];
      to_bf16(a, b8_scale(xa), aw);
      to_bf16(b, b8_scale(xb), bw);
      acc = mm_step_bf16(aw, bw, acc);
    }
  }
  few_result<OUT>(p, sums, acc, n0, lane, wave);
}

// The same in one launch with x's quantisation, for a row or a few through a weight that was laid out before (and no
// blocks of x to keep): every workgroup quantises its rows for itself into LDS, at most two blocks per 16 lanes, while
// the weight's bytes are on their way into registers.
constexpr int FEW_AHEAD = 4;        // block columns of the weight that a wave asks for in advance
constexpr int FEW_MAX_BLOCKS = 64;  // blocks of x per workgroup
struct FewArgs {
  const void* x;
  int64_t x_stride, width;
  float beta, inv_beta;
  double beta64;
};
template <typename T, bool ACT>
__global__ __launch_bounds__(512) void linear_few_kernel(MmArgs p, FewArgs f) {
  constexpr bool WIDE = std::is_same<T, float>::value;
  constexpr int PAD = 16;  // after every row: the rows of an operand lie in different banks
  __shared__ float sums[8][16][17];
  __shared__ __attribute__((aligned(16))) uint8_t rows[FEW_MAX_BLOCKS * B8 + 16 * PAD];
  __shared__ uint8_t exps[FEW_MAX_BLOCKS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int kb0 = (int)blockIdx.y * p.blocks_per_split;
  const int kb1 = kb0 + p.blocks_per_split < p.blocks ? kb0 + p.blocks_per_split : p.blocks;
  const int count = kb1 - kb0, pitch = count * B8 + PAD;
  const int64_t rb = n0 + (lane & 15) < p.n ? n0 + (lane & 15) : p.n - 1;
  const uint8_t* B = p.b.values + rb * p.b.pitch + (lane >> 4) * 32;
  const uint8_t* eb = p.b.exps + (p.b.tiled ? rb >> 7 : rb);
  v8i b[FEW_AHEAD];
  int xb[FEW_AHEAD];
#pragma unroll
  for (int i = 0; i < FEW_AHEAD; ++i) {
    const int kb = kb0 + wave + 8 * i;
    if (kb < kb1) {
      b[i] = *reinterpret_cast<const v8i_at16*>(B + (int64_t)kb * B8);
      xb[i] = eb[(int64_t)kb * p.b.exp_pitch];
    }
  }
  {  // x's blocks: 32 groups of 16 lanes
    const int group = threadIdx.x >> 4, part = threadIdx.x & 15;
    for (int id = group; id < (int)p.m * count; id += 32) {
      const int row = id / count, c = id - row * count;
      const int64_t col = (int64_t)(kb0 + c) * B8 + part * 8;
      float h[8];
      load_some<8>((const T*)f.x + row * f.x_stride + col, f.width - col, ACT ? -__builtin_inff() : 0.0f, h);
      int e;
      uint2 v;
      if constexpr (ACT) {
        v = softplus8(h, f.beta, f.inv_beta, f.beta64, e);
      } else {
        e = scale8(h);
        v = uint2{b8_pack4(h), b8_pack4(h + 4)};
      }
      *reinterpret_cast<uint2*>(rows + row * pitch + c * B8 + part * 8) = v;
      if (part == 0) exps[id] = (uint8_t)(e + 127);
    }
  }
  __syncthreads();
  const int ra = (lane & 15) < p.m ? (lane & 15) : (int)p.m - 1;
  const uint8_t* A = rows + ra * pitch + (lane >> 4) * 32;
  v4f acc = {0, 0, 0, 0};
  auto product = [&](int kb, v8i bv, int be) {
    const v8i a = *reinterpret_cast<const v8i_at16*>(A + (kb - kb0) * B8);
    const int ae = exps[ra * count + kb - kb0];
    if constexpr (!WIDE) {
      acc = mm_step<0, 0>(a, bv, acc, ae, be);
    } else {
      v8b aw[4], bw[4];
      to_bf16(a, b8_scale(ae), aw);
      to_bf16(bv, b8_scale(be), bw);
      acc = mm_step_bf16(aw, bw, acc);
    }
  };
#pragma unroll
  for (int i = 0; i < FEW_AHEAD; ++i) {
    const int kb = kb0 + wave + 8 * i;
    if (kb < kb1) product(kb, b[i], xb[i]);
  }
  for (int kb = kb0 + wave + 8 * FEW_AHEAD; kb < kb1; kb += 8)
    product(kb, *reinterpret_cast<const v8i_at16*>(B + (int64_t)kb * B8), eb[(int64_t)kb * p.b.exp_pitch]);
  few_result<T>(p, sums, acc, n0, lane, wave);
}

// the splits' sums in their order, then what the tile would have done
template <typename OUT>
__global__ __launch_bounds__(256) void mm_join_kernel(MmArgs p, int splits) {
  const int64_t total = p.m * p.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float v = 0;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) v += p.partial[s * total + i];
    const int64_t row = i / p.n, col = i - row * p.n;
    finish1<OUT>(p, row, col, v);
  }
}

enum MmKind { MM_FEW, MM_64, MM_128, MM_256 };
struct MmPlan {
  MmKind kind;
  int splits, per_split, mt, nt;
};
// Up to 16 rows: mm_few_kernel (1 x 4096 x 4096 bf16 4.7 us, in 64 x 64 tiles 8.2; 16 x 4096 x 4096 6.0 and 9.2).
// Else the largest tile that still gives the 256 compute units enough workgroups:
//   256 x 256 (`large`: a 16-bit result of rows and tiles) from 256 of them on: 4096 x 4096 x 1024 21.9 us, 128 x 128 29.4,
//     64 x 64 36.7; at 128 of them (4096 x 2048 x 2048) 43.0 us against 25.5;
//   128 x 128 from 384 on: at 400 (2560 x 2560 x 2048) 24.4 us, 64 x 64 27.8; at 256 (2048^3) 19.2 and 16.9.
// Where even the smallest tile leaves compute units without one the block columns are split, at least 4 to a split
// (256 x 256 x 4096 7.4 us, 8 to a split 8.9, unsplit 13.2), and none up to 16 of them (256 x 1024 x 1024 6.0 us, split in
// two 7.9); up to 16 rows at least 8 (16 x 512 x 8192 5.1 us, 16 to a split 6.8, unsplit 9.1), and none up to 32
// (1 x 128 x 4096 4.1 us, split in two 5.1).
MmPlan mm_plan(int64_t m, int64_t n, int64_t blocks, bool large) {
  MmPlan p;
  auto tiles = [&](int64_t t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
  int64_t groups;
  if (m <= 16) {
    p.kind = MM_FEW;
    p.mt = 1;
    p.nt = (int)((n + 15) / 16);
    groups = p.nt;
  } else {
    const int t = large && tiles(256) >= 256 ? 256 : tiles(128) >= 384 ? 128 : 64;
    p.kind = t == 256 ? MM_256 : t == 128 ? MM_128 : MM_64;
    p.mt = (int)((m + t - 1) / t);
    p.nt = (int)((n + t - 1) / t);
    groups = (int64_t)p.mt * p.nt;
  }
  const int64_t least = p.kind == MM_FEW ? (blocks > 32 ? 8 : blocks) : blocks > 16 ? 4 : blocks;
  int64_t s = (256 + groups - 1) / groups;
  if (s > blocks / least) s = blocks / least;
  if (s < 1) s = 1;
  p.per_split = (int)((blocks + s - 1) / s);
  p.splits = (int)((blocks + p.per_split - 1) / p.per_split);
  return p;
}

template <bool WIDE, bool GATE, typename OUT>
void mm_launch_tiles(const MmPlan& pl, const MmArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(pl.mt * pl.nt), (unsigned)pl.splits);
  if (pl.kind == MM_64) mm_kernel<64, 64, 32, 32, WIDE, GATE, OUT><<<grid, 256, 0, st>>>(a);
  else if (pl.kind == MM_128) mm_kernel<128, 128, 64, 64, WIDE, GATE, OUT><<<grid, 256, 0, st>>>(a);
  else if constexpr (!WIDE) mm_large_kernel<GATE, OUT><<<grid, 512, 0, st>>>(a);
}
template <bool WIDE, typename OUT>
void mm_launch(const MmPlan& pl, const MmArgs& a, hipStream_t st) {
  if (pl.kind == MM_FEW) mm_few_kernel<WIDE, OUT><<<dim3((unsigned)pl.nt, (unsigned)pl.splits), 512, 0, st>>>(a);
  else if (a.gate.values && !a.partial) mm_launch_tiles<WIDE, true, OUT>(pl, a, st);
  else mm_launch_tiles<WIDE, false, OUT>(pl, a, st);
  if (a.partial) mm_join_kernel<OUT><<<vmf_grid_for(a.m * a.n, 256, 1 << 14), 256, 0, st>>>(a, pl.splits);
}

// ---- weight gradient ---------------------------------------------------------------------------------------------

// A value of gy as bf16 terms whose sum is the value: 8 bits each, so 1 term for bf16, 2 for fp16 (11 bits), 3 for fp32.
// Cut off, not rounded: no term overflows.  NaN and infinity stay in the first term.  (Of fp32 values below 2^-110 digits
// under 2^-133, the smallest bf16, are lost: 1.2e-36 is off by 2e-5.)
template <typename T> struct Terms;
template <> struct Terms<bf16_t> { static constexpr int count = 1; };
template <> struct Terms<f16_t> { static constexpr int count = 2; };
template <> struct Terms<float> { static constexpr int count = 3; };
__device__ __forceinline__ uint32_t cut(float& v) {  // the upper 16 bits; v becomes the rest
  uint32_t u = __float_as_uint(v) & 0xffff0000u;
  if (!(fabsf(v) < __builtin_inff())) {
    if (v != v) u = 0x7fc00000u;
    v = 0;
  } else {
    v -= __uint_as_float(u);
  }
  return u >> 16;
}

// the same of two finite values, in one word; `more`: their rests are wanted
__device__ __forceinline__ uint32_t cut_finite(float& a, float& b, bool more) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  if (more) {
    a -= __uint_as_float(x & 0xffff0000u);
    b -= __uint_as_float(y & 0xffff0000u);
  }
  return __builtin_amdgcn_perm(y, x, 0x07060302u);
}

struct WgArgs {
  const void* gy;
  int64_t gy_stride;
  Operand a;
  void* gw;
  void* gb;
  float* partial;  // [split][n][k] then [split][n]; null with one split
  uint8_t* q;      // gy's blocks by rows (null: not wanted)
  uint8_t* q_exps;
  int64_t q_pitch, q_exp_pitch;
  int64_t m, n, k;
  int64_t rows_per_split;
  int nt, kt, splits;
  bool gb32;  // gb is float whatever gw is
};

// 32 columns of the 16 rows that start at `rows`, as the operand of a 32 x 32 x 16 product: lane l gets column l % 32 of
// rows 8 * (l / 32) .. + 7.  `at(row)` is where the row's 32 columns start.
template <typename F>
__device__ __forceinline__ v8b transposed(int lane, F&& at) {
  const int q = lane & 15, grp = lane >> 4;
  const int row = (grp >> 1) * 8 + (q >> 2), col = ((grp & 1) * 16 + (q & 3) * 4) * 2;
  union {
    v4s h[2];
    v8b v;
  } u;
  u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(v4s, at(row) + col));
  u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(v4s, at(row + 4) + col));
  return u.v;
}
// a wave's part of the result: D of a product has column (k) lane % 32, rows (n) (e & 3) + 8 (e >> 2) + 4 (lane / 32)
template <typename W, int FN, int FK>
__device__ __forceinline__ void write_wgrad(const WgArgs& p, const v16f (&acc)[FN][FK], int split, int64_t n0, int64_t k0,
                                            int lane) {
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FK; ++j) {
      const int64_t k = k0 + j * 32 + (lane & 31);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t n = n0 + i * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
        if (n < p.n && k < p.k) {
          if (p.partial) p.partial[((int64_t)split * p.n + n) * p.k + k] = acc[i][j][e];
          else ((W*)p.gw)[n * p.k + k] = (W)acc[i][j][e];
        }
      }
    }
}
// gbias: SHARE threads have sums of the same BN columns (thread: row `share`, E columns from `col`); added in order
template <typename W, int BN, int SHARE, int E>
__device__ __forceinline__ void write_gbias(const WgArgs& p, uint8_t* lds, const float (&sum)[E], int share, int col,
                                            int split, int64_t n0) {
  float* red = reinterpret_cast<float*>(lds);  // SHARE * BN floats
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; ++i) red[share * BN + col + i] = sum[i];
  __syncthreads();
  if (threadIdx.x < BN) {
    float s = 0;
#pragma unroll
    for (int q = 0; q < SHARE; ++q) s += red[q * BN + threadIdx.x];
    const int64_t n = n0 + threadIdx.x;
    if (n < p.n) {
      if (p.partial) p.partial[(int64_t)p.splits * p.n * p.k + (int64_t)split * p.n + n] = s;
      else if (p.gb32) ((float*)p.gb)[n] = s;
      else ((W*)p.gb)[n] = (W)s;
    }
  }
}
// E consecutive elements of gy's row `row` from column `col`, of a block that 128 / E neighbouring lanes hold: into gy's
// 8-bit blocks.  `in`: the row is one of the batch.  top: the largest of the lane's sizes.
template <int E>
__device__ __forceinline__ void write_gy_block(const WgArgs& p, float (&v)[E], uint32_t top, int64_t row, int64_t col,
                                               bool in) {
  top = lane_max<B8 / E>(top);
  if (top >= B8_INF) {
    top = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) top = b8_size(v[j]) < B8_INF ? larger(top, b8_size(v[j])) : top;
    top = lane_max<B8 / E>(top);
  }
  const int e = b8_exponent(__uint_as_float(top));
  const float inv = b8_pow2(-e);
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] *= inv;
  if (e == B8_EMAX)
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = b8_cut(v[j]);
  if (in && col < p.q_pitch) {
    uint8_t* q = p.q + row * p.q_pitch + col;
    if constexpr (E == 8) *reinterpret_cast<uint2*>(q) = uint2{b8_pack4(v), b8_pack4(v + 4)};
    else *reinterpret_cast<uint32_t*>(q) = b8_pack4(v);
    if ((col & (B8 - 1)) == 0) p.q_exps[(col >> 7) * p.q_exp_pitch + row] = (uint8_t)(e + 127);
  }
}
// 16 elements of a as bf16
__device__ __forceinline__ void expand16(v4i a, uint32_t exp_byte, uint4* out) {
  const float scale = b8_scale(exp_byte);
  union {
    v2b h[8];
    uint4 w[2];
  } u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    u.h[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[j], scale, false);
    u.h[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[j], scale, true);
  }
  out[0] = u.w[0];
  out[1] = u.w[1];
}

// Tile of BN (n) x BK (k) over the batch's rows, 32 at a time; waves of WN x WK.
//   gy's terms and a's values lie in LDS as bf16 rows and are read back transposed (the rows are the products' inner
//   dimension).  Each half of a step's products has its operands read while the half before it is multiplied, across the
//   step's one barrier as well; the next step's rows go from registers into the other stage between, and the rows after
//   that are asked for.
//   WHOLE: gy comes in whole aligned 16-byte pieces (n, the row stride and the address are multiples of them).
//   The workgroups of the first k tile also add up gbias.  gy's 8-bit blocks (what the input gradient's product reads) are
//   written on the way too, the k tiles' workgroups taking turns.
// Bound: per step and CU the 256 x 256 tile (bf16) takes 1024 clocks of matrix instructions against 900 of LDS reads and
// writes; the 128 x 256 tile 1024 (fp16) and 1536 (fp32), where the vector work of taking gy apart comes next, which
// is why this tile is wide in k.  16384x4096x4096: bf16 475 - 495 us (1.15 PFLOP/s; matrix instructions 55 % of the clocks, at
// 1.9 GHz), fp16 920 us, fp32 1.29 ms; 16384x784x128 20, 25, 28 us.
constexpr int WG_ROWS = 32;

template <typename T, typename W, int BN, int BK, int WN, int WK, bool WHOLE>
__global__ __launch_bounds__((BN / WN) * (BK / WK) * 64, 2) void wgrad_kernel(WgArgs p) {
  constexpr int WAVES_K = BK / WK, THREADS = (BN / WN) * WAVES_K * 64;
  constexpr int NT = Terms<T>::count;
  constexpr int E = 16 / (int)sizeof(T);                     // elements of gy in a 16-byte piece
  constexpr int GP = BN / E, GROWS = THREADS / GP;           // pieces per row, rows per pass of the workgroup
  constexpr int GN = WG_ROWS / GROWS;                        // passes
  constexpr int FN = WN / 32, FK = WK / 32;
  // bytes; 64 more than the row: the four rows of a transposed read lie in different banks
  constexpr int PITCH_G = 2 * BN + 64, PITCH_A = 2 * BK + 64;
  constexpr int PLANE = WG_ROWS * PITCH_G, STAGE = NT * PLANE + WG_ROWS * PITCH_A;
  static_assert(THREADS % GP == 0 && GN >= 1 && THREADS == WG_ROWS * (BK / 16), "whole pieces");
  static_assert(GROWS * BN * 4 <= 2 * STAGE, "gbias's sums fit the stages");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroup b runs on XCD b % 8: the tiles of a split, which read the same rows, on the same one
  const int tiles = p.nt * p.kt;
  const int id = xcd_run((int)blockIdx.x, tiles * p.splits), split = id / tiles, tile = id - split * tiles;
  const int nt = tile / p.kt, kt = tile - nt * p.kt;
  const int64_t n0 = (int64_t)nt * BN, k0 = (int64_t)kt * BK;
  const int64_t m0 = (int64_t)split * p.rows_per_split;
  const int rows = (int)(m0 + p.rows_per_split < p.m ? p.rows_per_split : p.m - m0);
  const int steps = (rows + WG_ROWS - 1) / WG_ROWS;
  const int wn = wave / WAVES_K * WN, wk = wave % WAVES_K * WK;

  // gy: the E values from gc of rows gr, gr + GROWS ... of a step; a: the 16 values from ac of row ar.  Where a tile
  // reaches behind the last column other ones are read instead, or none (their results are dropped).
  const int gr = threadIdx.x / GP, gc = threadIdx.x % GP * E;
  const int ar = threadIdx.x / (BK / 16), ac = threadIdx.x % (BK / 16) * 16;
  // No piece reaches behind its row: a column behind the last whole piece reads that, and where the row ends inside the
  // piece (not WHOLE) it is moved into place by g_back elements.
  const bool g_in = n0 + gc < p.n, a_in = k0 + ac < p.a.pitch;
  const bool ragged = !WHOLE && n0 + BN > p.n, tiny = !WHOLE && p.n < E;
  const int64_t g_col = tiny ? 0 : n0 + gc + E > p.n ? p.n - E : n0 + gc;
  const int g_back = g_in ? (int)(n0 + gc - g_col) : 0;
  const uint8_t* gsrc = (const uint8_t*)p.gy + ((m0 + gr) * p.gy_stride + g_col) * (int64_t)sizeof(T);
  const uint8_t* asrc = p.a.values + (m0 + ar) * p.a.pitch + k0 + (a_in ? ac : 0);
  const uint8_t* esrc = p.a.exps + ((k0 + (a_in ? ac : 0)) >> 7) * p.a.exp_pitch + m0 + ar;
  const int64_t g_pass = GROWS * p.gy_stride * (int64_t)sizeof(T), g_step = GN * g_pass, a_step = WG_ROWS * p.a.pitch;
  v4i g[GN], av;
  uint32_t ae;
  auto load_piece = [&](const uint8_t* src) -> v4i {
    if constexpr (WHOLE) {
      return *reinterpret_cast<const v4i*>(src);
    } else {
      union {
        T e[E];
        typename Pack<T, E>::type w;
        v4i v;
      } u;
      if (!tiny) {
        u.w = *reinterpret_cast<const typename Pack<T, E>::type*>(src);
      } else {  // fewer columns than a piece has
        u.v = v4i{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (g_in && j < p.n) u.e[j] = reinterpret_cast<const T*>(src)[j];
      }
      return u.v;
    }
  };
  auto place = [&] {  // what has arrived, in a tile that reaches behind the last column
    if (ragged && !tiny) {
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        union {
          v4i v;
          unsigned __int128 bits;
        } u;
        u.v = g[i];
        u.bits = g_in ? u.bits >> (8 * (int)sizeof(T) * g_back) : 0;
        g[i] = u.v;
      }
    }
  };
  // the next step's rows; ALL: all 32 are there, else `left` of them
  auto load = [&](auto ALL, int left) {
    if constexpr (decltype(ALL)::value) {
#pragma unroll
      for (int i = 0; i < GN; ++i) g[i] = load_piece(gsrc + i * g_pass);
      av = *reinterpret_cast<const v4i*>(asrc);
      ae = *esrc;
    } else {
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        g[i] = v4i{0, 0, 0, 0};
        if (gr + i * GROWS < left) g[i] = load_piece(gsrc + i * g_pass);
      }
      av = v4i{0, 0, 0, 0};
      ae = 127;
      if (ar < left) {
        av = *reinterpret_cast<const v4i*>(asrc);
        ae = *esrc;
      }
    }
    gsrc += g_step;
    asrc += a_step;
    esrc += WG_ROWS;
  };
  auto unpack = [&](v4i piece, float(&v)[E]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = __int_as_float(piece[j]);
    } else {
      union {
        v4i i;
        T e[E];
      } u;
      u.i = piece;
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = (float)u.e[j];
    }
  };
  uint8_t* const g_to = lds + gr * PITCH_G + gc * 2;
  uint8_t* const a_to = lds + NT * PLANE + ar * PITCH_A + ac * 2;
  auto put = [&](int stage) {
    uint8_t* to = g_to + stage * STAGE;
    if constexpr (NT == 1) {
#pragma unroll
      for (int i = 0; i < GN; ++i) *reinterpret_cast<v4i*>(to + i * GROWS * PITCH_G) = g[i];
    } else {
      float v[GN][E];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        unpack(g[i], v[i]);
#pragma unroll
        for (int j = 0; j < E; ++j) top = larger(top, b8_size(v[i][j]));
      }
      auto write = [&](int t, int i, const uint32_t(&w)[E / 2]) {
        uint8_t* d = to + t * PLANE + i * GROWS * PITCH_G;
        if constexpr (E == 8) *reinterpret_cast<uint4*>(d) = uint4{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<uint2*>(d) = uint2{w[0], w[1]};
      };
      if (__all(top < B8_INF)) {
#pragma unroll
        for (int i = 0; i < GN; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t w[E / 2];
#pragma unroll
            for (int j = 0; j < E / 2; ++j) w[j] = cut_finite(v[i][2 * j], v[i][2 * j + 1], t < NT - 1);
            write(t, i, w);
          }
      } else {
#pragma unroll
        for (int i = 0; i < GN; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t w[E / 2];
#pragma unroll
            for (int j = 0; j < E / 2; ++j) {
              const uint32_t lo = cut(v[i][2 * j]), hi = cut(v[i][2 * j + 1]);
              w[j] = lo | hi << 16;
            }
            write(t, i, w);
          }
      }
    }
    expand16(av, ae, reinterpret_cast<uint4*>(a_to + stage * STAGE));
  };
  // gbias and gy's blocks, from the rows in registers (those of step t)
  const bool sums = kt == 0 && p.gb;
  float gsum[E];
#pragma unroll
  for (int i = 0; i < E; ++i) gsum[i] = 0;
  int turn = 0;  // which k tile's workgroup writes the blocks of this step
  auto side = [&](int t) {
    const bool blocks = p.q && turn == kt;
    turn = turn + 1 == p.kt ? 0 : turn + 1;
    if (!sums && !blocks) return;
#pragma unroll
    for (int i = 0; i < GN; ++i) {
      float v[E];
      uint32_t top = 0;
      unpack(g[i], v);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (WHOLE && !g_in) v[j] = 0;
        gsum[j] += v[j];
        top = larger(top, b8_size(v[j]));
      }
      const int r = t * WG_ROWS + gr + i * GROWS;
      if (blocks) write_gy_block<E>(p, v, top, m0 + r, n0 + gc, r < rows);
    }
  };

  struct Half {
    v8b g[NT * FN], a[FK];
  };
  auto read_half = [&](int stage, int s, Half& h) {
    const uint8_t* G = lds + stage * STAGE + s * PITCH_G + wn * 2;
    const uint8_t* A = lds + stage * STAGE + NT * PLANE + s * PITCH_A + wk * 2;
#pragma unroll
    for (int j = 0; j < FK; ++j) h.a[j] = transposed(lane, [&](int r) { return A + r * PITCH_A + j * 64; });
#pragma unroll
    for (int i = 0; i < NT * FN; ++i)  // the smallest terms first
      h.g[i] = transposed(lane, [&](int r) { return G + (NT - 1 - i / FN) * PLANE + r * PITCH_G + i % FN * 64; });
  };
  v16f acc[FN][FK];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FK; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  auto multiply = [&](const Half& h, int from, int to) {
#pragma unroll
    for (int i = from; i < to; ++i)
#pragma unroll
      for (int j = 0; j < FK; ++j)
        acc[i % FN][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(h.g[i], h.a[j], acc[i % FN][j], 0, 0, 0);
  };

  Half h0, h1;
  // MORE: how many steps follow (3: at least three)
  auto step = [&](int t, auto MORE) {
    constexpr int more = decltype(MORE)::value;
    const int stage = t & 1;
    if constexpr (more > 0) {
      place();
      side(t + 1);
    }
    read_half(stage, 16, h1);
    multiply(h0, 0, NT * FN / 2);
    if constexpr (more > 0) put(stage ^ 1);
    if constexpr (more > 2) load(std::true_type{}, 0);
    if constexpr (more == 2) load(std::false_type{}, rows - (t + 2) * WG_ROWS);
    multiply(h0, NT * FN / 2, NT * FN);
    // between two products: operand reads, the vector work of the next rows, their writes, the loads of those after
#pragma unroll
    for (int q = 0; q < NT * FN * FK; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instruction
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // vector instructions
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // load
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (more > 0) {
      __syncthreads();  // the next step's rows are there, and this step's have been read
      read_half(stage ^ 1, 0, h0);
    }
    multiply(h1, 0, NT * FN);
#pragma unroll
    for (int q = 0; q < NT * FN * FK; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 1);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (steps > 0) {
    load(std::false_type{}, rows);
    place();
    side(0);
    put(0);
    if (steps > 1) load(std::false_type{}, rows - WG_ROWS);
    __syncthreads();
    read_half(0, 0, h0);
    int t = 0;
    for (; t + 3 < steps; ++t) step(t, std::integral_constant<int, 3>{});
    if (t + 2 < steps) step(t++, std::integral_constant<int, 2>{});
    if (t + 1 < steps) step(t++, std::integral_constant<int, 1>{});
    step(t, std::integral_constant<int, 0>{});
  }
  write_wgrad<W, FN, FK>(p, acc, split, n0 + wn, k0 + wk, lane);
  if (sums) write_gbias<W, BN, GROWS, E>(p, lds, gsum, gr, gc, split, n0);
}

// The splits' sums in a fixed order: gweight and gbias in fours, which PARTS threads of a workgroup share (each adds every
// PARTS-th split, the results are added in LDS).  A sum is a chain of loads that wait for memory: with one thread to a four,
// 36 splits of 128 x 784 took as long as the product itself (16384x128x784 fp32 with eight threads 27.8 us, with one 34.2).
// One does where there are many fours and few splits (16384x1024x2048 fp32, 8 splits: 172.7 us, with eight threads 177).
template <typename W, int PARTS>
__global__ __launch_bounds__(256) void wgrad_join_kernel(const float* __restrict__ partial, W* __restrict__ gw,
                                                         void* __restrict__ gb, bool gb32, int splits, int64_t nk,
                                                         int64_t n) {
  constexpr int FOURS = 256 / PARTS;
  __shared__ float red[PARTS > 1 ? PARTS : 1][FOURS][4];
  const int at = threadIdx.x % FOURS, part = threadIdx.x / FOURS;
  const int64_t w_fours = (nk + 3) / 4, total = w_fours + (gb ? (n + 3) / 4 : 0);
  for (int64_t first = (int64_t)blockIdx.x * FOURS; first < total; first += (int64_t)gridDim.x * FOURS) {
    int64_t i = first + at, size = nk;
    const float* src = partial;
    W* out = gw;
    const bool bias = i >= w_fours;
    if (bias) {
      i -= w_fours;
      src += splits * nk;
      size = n;
      out = (W*)gb;
    }
    const int64_t left = first + at < total ? size - 4 * i : 0;
    float s[4] = {0, 0, 0, 0};
    if (left > 0) {
#pragma unroll 8
      for (int q = part; q < splits; q += PARTS) {
        float v[4];
        load_some<4>(src + q * size + 4 * i, left, 0.0f, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += v[j];
      }
    }
    if constexpr (PARTS > 1) {
      __syncthreads();  // (the last round's sums have been read)
#pragma unroll
      for (int j = 0; j < 4; ++j) red[part][at][j] = s[j];
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int q = 1; q < PARTS; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[j] += red[q][at][j];
      }
    }
    if (part == 0) {
      if (bias && gb32) store_some<4>((float*)gb + 4 * i, left, s);
      else store_some<4>(out + 4 * i, left, s);
    }
  }
}

// gbias by itself.  A workgroup takes 128 columns of its split's rows, in the lanes and the order that the weight gradient's
// tiles have; the splits are joined as theirs are.  A read of gy: 16384x4096 bf16 24 us (5.6 TB/s), 16384x784 fp32 17 us.
template <typename T, typename W>
__global__ __launch_bounds__(256) void bias_grad_kernel(const T* __restrict__ gy, int64_t gy_stride, W* __restrict__ gb,
                                                        float* __restrict__ partial, int64_t m, int64_t n,
                                                        int64_t rows_per_split) {
  constexpr int E = 16 / (int)sizeof(T), GP = 128 / E, GROWS = 256 / GP;
  __shared__ float red[GROWS][128];
  const int gr = threadIdx.x / GP, gc = threadIdx.x % GP * E;
  const int64_t n0 = (int64_t)blockIdx.x * 128, left = n - n0 - gc;
  const int64_t m0 = (int64_t)blockIdx.y * rows_per_split, end = m0 + rows_per_split < m ? m0 + rows_per_split : m;
  const T* p = gy + n0 + gc;
  float s[E];
#pragma unroll
  for (int i = 0; i < E; ++i) s[i] = 0;
  if (left > 0) {
#pragma unroll 8
    for (int64_t r = m0 + gr; r < end; r += GROWS) {
      float v[E];
      load_some<E>(p + r * gy_stride, left, 0.0f, v);
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) red[gr][gc + i] = s[i];
  __syncthreads();
  if (threadIdx.x >= 128 || n0 + threadIdx.x >= n) return;
  float v = 0;
#pragma unroll
  for (int q = 0; q < GROWS; ++q) v += red[q][threadIdx.x];
  if (partial) partial[(int64_t)blockIdx.y * n + n0 + threadIdx.x] = v;
  else gb[n0 + threadIdx.x] = (W)v;
}
// four workgroups to a compute unit, at least 256 rows to a split
struct BiasPlan {
  int nt, splits;
  int64_t per_split;
};
BiasPlan bias_plan(int64_t m, int64_t n) {
  BiasPlan p;
  p.nt = (int)((n + 127) / 128);
  int64_t s = 1024 / p.nt;
  if (s > m / 256) s = m / 256;
  if (s < 1) s = 1;
  p.per_split = ((m + s - 1) / s + WG_ROWS - 1) / WG_ROWS * WG_ROWS;
  p.splits = p.per_split > 0 ? (int)((m + p.per_split - 1) / p.per_split) : 1;
  return p;
}

struct WgPlan {
  int splits, nt, kt, bn, bk;
  int64_t per_split;
};
// The large tile is 256 x 256 for bf16, 128 x 256 for fp16 and fp32, whose two and three terms take the registers and LDS.
// It reads less for a product but fills a compute unit by itself, where two workgroups of the 128 x 128 tile hide each
// other's start, barriers and end: it is taken above 2^33 products (bf16: 65536x512x512 53.7 us, small 57.4; 16384x512x512
// 33.8 and 27.7; 4096^3 126 and 173), for the others above 2^30 (fp32: 16384x128x784 24.5 us, small 27.8; 4096^3 328 and
// 391; 1024^3 25.4 and 24.2).
// The batch is split until every compute unit has a workgroup, at least 256 rows to a split (fp32 16384x512x512 36 us,
// unsplit over 500; bf16 4096x256x256 13.0 us, with 64 rows 17.9), in up to 16 splits 128 rows (fp32 1000x257x257 15.1 us,
// with 256 19.9); the small tile until there are two for each, at least 512 rows to a split and in up to 128 splits (bf16
// 16384x512x512 27.7 us, with one 30.8; 2048x1024x1024, where that is 256 rows, 26.5 and 23.7; 262144x128x128, where that is
// 512 splits, 43.0 and 37.2).
WgPlan wg_plan(int64_t m, int64_t n, int64_t k, int dtype) {
  WgPlan p;
  const bool bf16 = dtype == VMF_BF16;
  const bool large = (double)m * n * k > (bf16 ? 0x1p33 : 0x1p30) && k > 128 && (!bf16 || n > 128);
  p.bk = large ? 256 : 128;
  p.bn = large && bf16 ? 256 : 128;
  p.nt = (int)((n + p.bn - 1) / p.bn);
  p.kt = (int)((k + p.bk - 1) / p.bk);
  const int64_t tiles = (int64_t)p.nt * p.kt;
  auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  int64_t s = least(256 / tiles, m / 256 > 16 ? m / 256 : least(m / 128, 16));
  const int64_t two = least(least(512 / tiles, m / 512), 128);
  if (!large && two > s) s = two;
  if (s < 1) s = 1;
  p.per_split = ((m + s - 1) / s + WG_ROWS - 1) / WG_ROWS * WG_ROWS;
  p.splits = p.per_split > 0 ? (int)((m + p.per_split - 1) / p.per_split) : 1;
  return p;
}

template <typename T, typename W, bool WHOLE>
void wgrad_launch_tiles(const WgPlan& pl, const WgArgs& p, hipStream_t st) {
  const unsigned grid = (unsigned)(pl.nt * pl.kt * pl.splits);
  if constexpr (std::is_same<T, bf16_t>::value) {
    if (pl.bn == 256) wgrad_kernel<T, W, 256, 256, 128, 64, WHOLE><<<grid, 512, 0, st>>>(p);
    else wgrad_kernel<T, W, 128, 128, 64, 64, WHOLE><<<grid, 256, 0, st>>>(p);
  } else {
    if (pl.bk == 256) wgrad_kernel<T, W, 128, 256, 64, 64, WHOLE><<<grid, 512, 0, st>>>(p);
    else wgrad_kernel<T, W, 128, 128, 64, 64, WHOLE><<<grid, 256, 0, st>>>(p);
  }
}
template <typename T, typename W>
void wgrad_launch(const WgPlan& pl, const WgArgs& p, hipStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  if (p.n % E == 0 && p.gy_stride % E == 0 && ((uintptr_t)p.gy & 15) == 0) wgrad_launch_tiles<T, W, true>(pl, p, st);
  else wgrad_launch_tiles<T, W, false>(pl, p, st);
}

int check_operand(const char* what, const char* name, const uint8_t* values, const uint8_t* exps, int64_t exp_pitch,
                  int tiled, int64_t rows) {
  VMF_REQUIRE(values && exps, VMF_ERR_BAD_ARG, "%s: %s is null", what, name);
  VMF_REQUIRE(((uintptr_t)values & 15) == 0 && (tiled || ((uintptr_t)exps & 3) == 0), VMF_ERR_BAD_ARG,
              "%s: %s is not aligned", what, name);
  VMF_REQUIRE(tiled ? exp_pitch >= b8_blocks(rows) : exp_pitch >= rows && exp_pitch % 16 == 0, VMF_ERR_BAD_ARG,
              "%s: exponent pitch %lld of %s", what, (long long)exp_pitch, name);
  return VMF_OK;
}

}  // namespace

extern "C" int vmf_blocks8_matmul_workspace(int64_t m, int64_t n, int64_t k, int out_dtype, int64_t* bytes_out) {
  int rc = b8_check_shape("vmf_blocks8_matmul_workspace", m, k);
  if (rc != VMF_OK) return rc;
  rc = b8_check_shape("vmf_blocks8_matmul_workspace", n, k);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(bytes_out, VMF_ERR_BAD_ARG, "vmf_blocks8_matmul_workspace: null pointer");
  *bytes_out = 0;
  if (m == 0 || n == 0) return VMF_OK;
  // (no kind of operand makes a difference where the block columns are split)
  const MmPlan pl = mm_plan(m, n, b8_blocks(k), false);
  if (pl.splits > 1) *bytes_out = (int64_t)pl.splits * m * n * 4;
  return VMF_OK;
}

// vmf_blocks8_matmul; few: not null, a are the rows there, quantised by the same launch (one that few_fits)
static int matmul(const FewArgs* few, int activation, const uint8_t* a, const uint8_t* a_exponents,
                  int64_t a_exp_pitch, int a_tiled, const uint8_t* b, const uint8_t* b_exponents, int64_t b_exp_pitch,
                  int b_tiled, const void* bias, int bias_dtype, const uint8_t* gate, const uint8_t* gate_exponents,
                  int64_t gate_exp_pitch, double beta, void* out, int64_t m, int64_t n, int64_t k, void* workspace,
                  int64_t workspace_bytes, int out_dtype, vmf_stream_t stream) {
  const char* what = "vmf_blocks8_matmul";
  int64_t need = 0;
  int rc = vmf_blocks8_matmul_workspace(m, n, k, out_dtype, &need);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(out_dtype == VMF_F32 || out_dtype == VMF_F16 || out_dtype == VMF_BF16, VMF_ERR_DTYPE,
              "%s: out dtype %d is not VMF_F32/VMF_F16/VMF_BF16", what, out_dtype);
  VMF_REQUIRE(!bias || bias_dtype == VMF_F32 || bias_dtype == VMF_F16 || bias_dtype == VMF_BF16, VMF_ERR_DTYPE,
              "%s: bias dtype %d", what, bias_dtype);
  if (m == 0 || n == 0) return VMF_OK;
  if (!few && (rc = check_operand(what, "a", a, a_exponents, a_exp_pitch, a_tiled, m)) != VMF_OK) return rc;
  if ((rc = check_operand(what, "b", b, b_exponents, b_exp_pitch, b_tiled, n)) != VMF_OK) return rc;
  if (gate) {
    if ((rc = check_operand(what, "gate", gate, gate_exponents, gate_exp_pitch, 0, m)) != VMF_OK) return rc;
    VMF_REQUIRE(n <= VMF_BLOCKS8_MAX_WIDTH, VMF_ERR_UNSUPPORTED, "%s: n", what);
    VMF_REQUIRE(beta > 0 && beta <= 1e30 && beta >= 1e-30, VMF_ERR_BAD_ARG, "%s: beta %g", what, beta);
  }
  VMF_REQUIRE(out, VMF_ERR_BAD_ARG, "%s: null pointer", what);
  VMF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VMF_ERR_BAD_ARG,
              "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  const int64_t blocks = b8_blocks(k);
  const MmPlan pl = mm_plan(m, n, blocks, out_dtype != VMF_F32 && !a_tiled && b_tiled);
  // (a launch has fewer than 2^32 threads)
  VMF_REQUIRE((int64_t)pl.mt * pl.nt < (1 << 23), VMF_ERR_UNSUPPORTED, "%s: %lld x %lld results", what, (long long)m,
              (long long)n);
  MmArgs p;
  p.a = Operand{a, a_exponents, blocks * B8, a_exp_pitch, m, a_tiled};
  p.b = Operand{b, b_exponents, blocks * B8, b_exp_pitch, n, b_tiled};
  p.gate = Operand{gate, gate_exponents, b8_blocks(n) * B8, gate_exp_pitch, m, 0};
  p.bias = bias;
  p.bias_code = bias_dtype;
  p.out = out;
  p.partial = need ? (float*)workspace : nullptr;
  p.m = m;
  p.n = n;
  p.blocks = (int)blocks;
  p.blocks_per_split = pl.per_split;
  p.mt = pl.mt;
  p.nt = pl.nt;
  p.beta = (float)beta;
  hipStream_t st = (hipStream_t)stream;
  if (few) {
    const dim3 grid((unsigned)pl.nt, (unsigned)pl.splits);
    LOWP_DISPATCH(out_dtype, "vmf_blocks8_linear_fwd", T, {
      if (activation == VMF_ACT_SOFTPLUS) linear_few_kernel<T, true><<<grid, 512, 0, st>>>(p, *few);
      else linear_few_kernel<T, false><<<grid, 512, 0, st>>>(p, *few);
      if (p.partial) mm_join_kernel<T><<<vmf_grid_for(m * n, 256, 1 << 14), 256, 0, st>>>(p, pl.splits);
    });
    return vmf_check_launch("vmf_blocks8_linear_fwd");
  }
  if (out_dtype == VMF_F32) mm_launch<true, float>(pl, p, st);
  else if (out_dtype == VMF_F16) mm_launch<false, f16_t>(pl, p, st);
  else mm_launch<false, bf16_t>(pl, p, st);
  return vmf_check_launch(what);
}

extern "C" int vmf_blocks8_matmul(const uint8_t* a, const uint8_t* a_exponents, int64_t a_exp_pitch, int a_tiled,
                                  const uint8_t* b, const uint8_t* b_exponents, int64_t b_exp_pitch, int b_tiled,
                                  const void* bias, int bias_dtype, const uint8_t* gate,
                                  const uint8_t* gate_exponents, int64_t gate_exp_pitch, double beta, void* out,
                                  int64_t m, int64_t n, int64_t k, void* workspace, int64_t workspace_bytes,
                                  int out_dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_matmul");
  return matmul(nullptr, VMF_ACT_NONE, a, a_exponents, a_exp_pitch, a_tiled, b, b_exponents, b_exp_pitch, b_tiled, bias,
                bias_dtype, gate, gate_exponents, gate_exp_pitch, beta, out, m, n, k, workspace, workspace_bytes,
                out_dtype, stream);
}

extern "C" int vmf_blocks8_weight_grad_workspace(int64_t m, int64_t n, int64_t k, int dtype, int64_t* bytes_out) {
  int rc = b8_check_shape("vmf_blocks8_weight_grad_workspace", m, k);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(bytes_out && n >= 0 && n <= VMF_BLOCKS8_MAX_WIDTH, VMF_ERR_BAD_ARG,
              "vmf_blocks8_weight_grad_workspace: n = %lld or a null pointer", (long long)n);
  *bytes_out = 0;
  if (n == 0) return VMF_OK;
  const WgPlan pl = wg_plan(m, n, k, dtype);
  if (pl.splits > 1) *bytes_out = (int64_t)pl.splits * n * (k + 1) * 4;
  return VMF_OK;
}

extern "C" int vmf_blocks8_weight_grad(const void* gy, int64_t gy_stride, const uint8_t* a, const uint8_t* a_exponents,
                                       int64_t a_exp_pitch, void* gweight, void* gbias, uint8_t* gy_values,
                                       uint8_t* gy_exponents, int64_t gy_exp_pitch, int64_t m, int64_t n, int64_t k,
                                       void* workspace, int64_t workspace_bytes, int dtype, int out_dtype,
                                       vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_weight_grad");
  const char* what = "vmf_blocks8_weight_grad";
  const bool gb32 = out_dtype & VMF_GBIAS_F32;
  out_dtype &= ~VMF_GBIAS_F32;
  int64_t need = 0;
  int rc = vmf_blocks8_weight_grad_workspace(m, n, k, dtype, &need);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(out_dtype == VMF_F32 || out_dtype == dtype, VMF_ERR_DTYPE, "%s: out dtype %d", what, out_dtype);
  VMF_REQUIRE(gy_stride >= 0, VMF_ERR_BAD_ARG, "%s: negative row stride", what);
  if (n == 0) return VMF_OK;
  VMF_REQUIRE(gweight && (m == 0 || gy), VMF_ERR_BAD_ARG, "%s: null pointer", what);
  if (m > 0 && (rc = check_operand(what, "a", a, a_exponents, a_exp_pitch, 0, m)) != VMF_OK) return rc;
  if (gy_values && (rc = check_operand(what, "gy's blocks", gy_values, gy_exponents, gy_exp_pitch, 0, m)) != VMF_OK)
    return rc;
  VMF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VMF_ERR_BAD_ARG,
              "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  const WgPlan pl = wg_plan(m, n, k, dtype);
  VMF_REQUIRE((int64_t)pl.nt * pl.kt * pl.splits < (1 << 23), VMF_ERR_UNSUPPORTED, "%s: %lld x %lld results", what,
              (long long)n, (long long)k);
  WgArgs p;
  p.gy = gy;
  p.gy_stride = gy_stride;
  p.a = Operand{a, a_exponents, b8_blocks(k) * B8, a_exp_pitch, m, 0};
  p.gw = gweight;
  p.gb = gbias;
  p.partial = need ? (float*)workspace : nullptr;
  p.q = gy_values;
  p.q_exps = gy_exponents;
  p.q_pitch = b8_blocks(n) * B8;
  p.q_exp_pitch = gy_exp_pitch;
  p.m = m;
  p.n = n;
  p.k = k;
  p.rows_per_split = pl.per_split;
  p.nt = pl.nt;
  p.kt = pl.kt;
  p.splits = pl.splits;
  p.gb32 = gb32;
  hipStream_t st = (hipStream_t)stream;
  LOWP_DISPATCH(dtype, "vmf_blocks8_weight_grad", T, {
    if (out_dtype == VMF_F32) wgrad_launch<T, float>(pl, p, st);
    else wgrad_launch<T, T>(pl, p, st);
  });
  rc = vmf_check_launch(what);
  if (rc != VMF_OK || !need) return rc;
  const int64_t fours = (n * k + 3) / 4 + (n + 3) / 4;
  LOWP_DISPATCH(out_dtype, "vmf_blocks8_weight_grad", W, {
    if (pl.splits > 8 || fours <= 1 << 16)
      wgrad_join_kernel<W, 8><<<vmf_grid_for(fours, 32, 1 << 13), 256, 0, st>>>(p.partial, (W*)gweight, gbias, gb32,
                                                                               pl.splits, n * k, n);
    else
      wgrad_join_kernel<W, 1><<<vmf_grid_for(fours, 256, 1 << 13), 256, 0, st>>>(p.partial, (W*)gweight, gbias, gb32,
                                                                                pl.splits, n * k, n);
  });
  return vmf_check_launch(what);
}

extern "C" int vmf_blocks8_bias_grad_workspace(int64_t m, int64_t n, int dtype, int64_t* bytes_out) {
  int rc = b8_check_shape("vmf_blocks8_bias_grad_workspace", m, n);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(bytes_out, VMF_ERR_BAD_ARG, "vmf_blocks8_bias_grad_workspace: null pointer");
  const BiasPlan pl = bias_plan(m, n);
  *bytes_out = pl.splits > 1 ? (int64_t)pl.splits * n * 4 : 0;
  return VMF_OK;
}

extern "C" int vmf_blocks8_bias_grad(const void* gy, int64_t gy_stride, void* gbias, int64_t m, int64_t n, void* workspace,
                                     int64_t workspace_bytes, int dtype, int out_dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_bias_grad");
  const char* what = "vmf_blocks8_bias_grad";
  int64_t need = 0;
  int rc = vmf_blocks8_bias_grad_workspace(m, n, dtype, &need);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(out_dtype == VMF_F32 || out_dtype == dtype, VMF_ERR_DTYPE, "%s: out dtype %d", what, out_dtype);
  VMF_REQUIRE(gy_stride >= 0, VMF_ERR_BAD_ARG, "%s: negative row stride", what);
  VMF_REQUIRE(gbias && (m == 0 || gy), VMF_ERR_BAD_ARG, "%s: null pointer", what);
  VMF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VMF_ERR_BAD_ARG,
              "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  const BiasPlan pl = bias_plan(m, n);
  float* partial = need ? (float*)workspace : nullptr;
  const dim3 grid((unsigned)pl.nt, (unsigned)pl.splits);
  hipStream_t st = (hipStream_t)stream;
  LOWP_DISPATCH(dtype, "vmf_blocks8_bias_grad", T, {
    if (out_dtype == VMF_F32)
      bias_grad_kernel<T, float><<<grid, 256, 0, st>>>((const T*)gy, gy_stride, (float*)gbias, partial, m, n, pl.per_split);
    else
      bias_grad_kernel<T, T><<<grid, 256, 0, st>>>((const T*)gy, gy_stride, (T*)gbias, partial, m, n, pl.per_split);
  });
  rc = vmf_check_launch(what);
  if (rc != VMF_OK || !need) return rc;
  LOWP_DISPATCH(out_dtype, "vmf_blocks8_bias_grad", W, {
    wgrad_join_kernel<W, 8><<<vmf_grid_for((n + 3) / 4, 32, 1 << 13), 256, 0, st>>>(partial, nullptr, gbias, false,
                                                                                   pl.splits, 0, n);
  });
  return vmf_check_launch(what);
}

// ---- a layer's two directions --------------------------------------------------------------------------------------

namespace {
int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
int64_t exp_rows(int64_t rows) { return rows < 16 ? 16 : up16(rows); }
int64_t row_block_bytes(int64_t rows, int64_t width) { return b8_blocks(width) * (rows * B8 + exp_rows(rows)); }
int64_t tile_bytes(int64_t rows, int64_t width) { return up16(b8_blocks(width) * (rows * B8 + b8_blocks(rows))); }
}  // namespace

// Whether linear_few_kernel pays: at most 64 blocks for a workgroup to quantise (two per 16 lanes, about a microsecond, as
// long as the weight's bytes take to come) and at most two workgroups for a compute unit, since every one does it again.
// bf16, softplus, the launches one after the other: 1 x 4096 x 4096 6.5 us, in two launches 7.8; 4 x 1024 x 1024 5.2 and 6.2;
// 1 x 8192 x 4096 11.1 and 10.2 (where a call alone still gains the launch, 3 us); 1 x 16384 x 4096 26.8 and 21.0.
static bool few_fits(int64_t m, int64_t n, int64_t k) {
  if (m < 1 || m > 16) return false;
  const MmPlan pl = mm_plan(m, n, b8_blocks(k), false);
  return m * pl.per_split <= FEW_MAX_BLOCKS && (int64_t)pl.nt * pl.splits <= 512;
}

extern "C" int vmf_blocks8_linear_fwd_workspace(int64_t m, int64_t n, int64_t k, int laid_out, int kept, int dtype,
                                                int64_t* bytes_out) {
  int rc = vmf_blocks8_matmul_workspace(m, n, k, dtype, bytes_out);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(n >= 1, VMF_ERR_BAD_ARG, "vmf_blocks8_linear_fwd_workspace: n = %lld", (long long)n);
  *bytes_out = up16(*bytes_out);
  if (!laid_out) *bytes_out += tile_bytes(n, k);
  if (!kept && !(laid_out && few_fits(m, n, k))) *bytes_out += row_block_bytes(m, k);
  return VMF_OK;
}

extern "C" int vmf_blocks8_linear_fwd(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                      int weight_dtype, const uint8_t* w_values, const uint8_t* w_exponents,
                                      uint8_t* wt_values, uint8_t* wt_exponents, const void* bias, int bias_dtype,
                                      int activation, double beta, uint8_t* a_values, uint8_t* a_exponents,
                                      int64_t a_exp_pitch, void* y, int64_t m, int64_t n, int64_t k, void* workspace,
                                      int64_t workspace_bytes, int dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_linear_fwd");
  const char* what = "vmf_blocks8_linear_fwd";
  int64_t all = 0, need = 0;
  int rc = vmf_blocks8_linear_fwd_workspace(m, n, k, weight == nullptr, a_values != nullptr, dtype, &all);
  if (rc != VMF_OK) return rc;
  vmf_blocks8_matmul_workspace(m, n, k, dtype, &need);
  VMF_REQUIRE(all == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= all), VMF_ERR_BAD_ARG,
              "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)all);
  uint8_t* at = (uint8_t*)workspace + up16(need);
  if (!a_values && !weight && few_fits(m, n, k)) {
    VMF_REQUIRE(x && x_stride >= 0, VMF_ERR_BAD_ARG, "%s: x", what);
    VMF_REQUIRE(activation == VMF_ACT_NONE || activation == VMF_ACT_SOFTPLUS, VMF_ERR_BAD_ARG, "%s: activation %d", what,
                activation);
    if (activation == VMF_ACT_NONE) beta = 1.0;
    VMF_REQUIRE(beta > 0 && beta <= 1e30 && beta >= 1e-30, VMF_ERR_BAD_ARG, "%s: beta %g", what, beta);
    const FewArgs f{x, x_stride, k, (float)beta, (float)(1.0 / beta), beta};
    return matmul(&f, activation, nullptr, nullptr, 0, 0, w_values, w_exponents, b8_blocks(n), 1, bias, bias_dtype,
                  nullptr, nullptr, 0, 1.0, y, m, n, k, workspace, need, dtype, stream);
  }
  if (!a_values) {
    a_values = at;
    a_exponents = at + m * b8_blocks(k) * B8;
    a_exp_pitch = exp_rows(m);
    at += row_block_bytes(m, k);
  }
  if (weight) {
    uint8_t* e = at + n * b8_blocks(k) * B8;
    rc = b8_quantize_both(x, x_stride, a_values, a_exponents, a_exp_pitch, m, k, activation, beta, dtype, weight,
                          weight_stride, at, e, wt_values, wt_exponents, n, weight_dtype, stream);
    w_values = at;
    w_exponents = e;
  } else {
    rc = vmf_blocks8_quantize(x, x_stride, a_values, a_exponents, a_exp_pitch, m, k, activation, beta, dtype, stream);
  }
  if (rc != VMF_OK) return rc;
  return vmf_blocks8_matmul(a_values, a_exponents, a_exp_pitch, 0, w_values, w_exponents, b8_blocks(n), 1, bias,
                            bias_dtype, nullptr, nullptr, 0, 1.0, y, m, n, k, workspace, need, dtype, stream);
}

extern "C" int vmf_blocks8_linear_bwd_workspace(int64_t m, int64_t n, int64_t k, int dtype, int64_t* bytes_out) {
  int64_t mm = 0, wg = 0;
  int rc = n >= 1 ? vmf_blocks8_matmul_workspace(m, k, n, dtype, &mm) : VMF_ERR_BAD_ARG;
  VMF_REQUIRE(n >= 1, VMF_ERR_BAD_ARG, "vmf_blocks8_linear_bwd_workspace: n = %lld", (long long)n);
  if (rc != VMF_OK) return rc;
  rc = vmf_blocks8_weight_grad_workspace(m, n, k, dtype, &wg);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(bytes_out, VMF_ERR_BAD_ARG, "vmf_blocks8_linear_bwd_workspace: null pointer");
  *bytes_out = up16(mm > wg ? mm : wg) + row_block_bytes(m, n);
  return VMF_OK;
}

extern "C" int vmf_blocks8_linear_bwd(const void* gy, int64_t gy_stride, const uint8_t* a_values,
                                      const uint8_t* a_exponents, int64_t a_exp_pitch, const uint8_t* wt_values,
                                      const uint8_t* wt_exponents, int activation, double beta, void* gx, void* gweight,
                                      void* gbias, int64_t m, int64_t n, int64_t k, void* workspace,
                                      int64_t workspace_bytes, int dtype, int weight_dtype, vmf_stream_t stream) {
  VMF_RANGE("vmf_blocks8_linear_bwd");
  const char* what = "vmf_blocks8_linear_bwd";
  int64_t need = 0;
  int rc = vmf_blocks8_linear_bwd_workspace(m, n, k, dtype, &need);
  if (rc != VMF_OK) return rc;
  VMF_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need, VMF_ERR_BAD_ARG,
              "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  VMF_REQUIRE(gweight || !gbias, VMF_ERR_BAD_ARG, "%s: gbias comes with gweight", what);
  VMF_REQUIRE(!gx || wt_values, VMF_ERR_BAD_ARG, "%s: gx needs the transposed weight", what);
  VMF_REQUIRE(activation == VMF_ACT_NONE || activation == VMF_ACT_SOFTPLUS, VMF_ERR_BAD_ARG, "%s: activation %d", what,
              activation);
  const bool gate = gx && activation == VMF_ACT_SOFTPLUS;
  VMF_REQUIRE(!gate || m == 0 || (a_values && a_exponents), VMF_ERR_BAD_ARG, "%s: the softplus gradient needs x's blocks",
              what);
  // gy's blocks lie in front, what the products add up in parts behind them: one after the other, on one stream
  uint8_t* q = (uint8_t*)workspace;
  uint8_t* q_exps = q + m * b8_blocks(n) * B8;
  uint8_t* parts = q + row_block_bytes(m, n);
  const int64_t left = workspace_bytes - row_block_bytes(m, n);
  if (gweight)
    rc = vmf_blocks8_weight_grad(gy, gy_stride, a_values, a_exponents, a_exp_pitch, gweight, gbias, gx ? q : nullptr,
                                 q_exps, exp_rows(m), m, n, k, parts, left, dtype, weight_dtype, stream);
  else if (gx)
    rc = vmf_blocks8_quantize(gy, gy_stride, q, q_exps, exp_rows(m), m, n, VMF_ACT_NONE, 1.0, dtype, stream);
  if (rc != VMF_OK || !gx) return rc;
  return vmf_blocks8_matmul(q, q_exps, exp_rows(m), 0, wt_values, wt_exponents, b8_blocks(k), 1, nullptr, 0,
                            gate ? a_values : nullptr, a_exponents, a_exp_pitch, beta, gx, m, k, n, parts, left, dtype,
                            stream);
}
