// Activation rows in 8 bits (float8.h): one pass over the rows, which it is bound by reading.
//   float8_rows   [rows][width] bfloat16 or float32 -> blocks of 16 rows x 128 k of e4m3 and a word of exponents for each 512 k of a row;
//                 of rows [gate | up] the activation act(gate) * up, in 32 bits until it is rounded once
//   float8_norm   the RMSNorm of float32 rows, x / sqrt(mean(x^2) + eps) * w, of float32 or of the bfloat16 that it is elsewhere
//
// 16 lanes hold a stretch of 128 values, 8 each (16 bytes of bfloat16), a wave four stretches of a row: its largest magnitude takes four
// steps between neighbouring lanes, the exponents of the four stretches make one word.  A block's runs of 256 bytes are written by its 16 rows in pieces of 8
// bytes: from 4,096 pieces of 512 columns on a workgroup takes a row, and the 16 rows of a block run on one XCD, so that the pieces meet in one L2.
// Measured, us, in brackets with four rows a wave in workgroups of a block: 512 x 4,096 bfloat16 3.1 (4.0), 2,048 x 4,096 6.5 (7.2), 8,160 x 4,096 22.4 (26.7, 4.5 TB/s), 8,192 x
// 12,288 64.6 (80); few rows that way 2.7, in pieces of four rows 2.3 (45 x 12,288).
#include "float8.h"

namespace {

// 8 neighbouring values of a row from `k` on, zeros beyond its width.  WHOLE: they are all there, on an address of 16 bytes.
template <typename T, bool WHOLE>
__device__ inline void load_eight(const T* __restrict__ row, int k, int width, float v[8]) {
  if constexpr (WHOLE) {
    if (k < width) {
      const float4 a = load_four(row + k), b = load_four(row + k + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < width ? to_f32(row[k + i]) : 0.f;
  }
}

// v with the lanes of a group of 16 turned by N.
template <int N>
__device__ inline uint32_t turned(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N /* row_ror */, 0xf, 0xf, true);
}

// A lane's eight values of a row from column k on, in 8 bits; 64 lanes hold 512 neighbouring columns, a word of exponents.
__device__ inline void eight_in_8(const float (&v)[8], long row, int k, int stretches, int padded, int in_rows, uint8_t* __restrict__ data,
                                  uint32_t* __restrict__ exponents) {
  const int lane = threadIdx.x % 64, stretch = k / F8_K;
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) largest = f8_larger(largest, v[j]);
  largest = max(largest, turned<8>(largest));
  largest = max(largest, turned<4>(largest));
  largest = max(largest, turned<2>(largest));
  largest = max(largest, turned<1>(largest));
  const uint32_t exponent = f8_exponent(largest);
  const float scale = f8_scale(exponent);
  if (stretch < stretches) {
    const uint2 eight = make_uint2(f8_four(v[0], v[1], v[2], v[3], scale), f8_four(v[4], v[5], v[6], v[7], scale));
    const long at = in_rows ? (row * stretches + stretch) * F8_K + k % F8_K
                            : (row / 16 * stretches + stretch) * F8_BLOCK + f8_place((int)(row % 16), k % F8_K);
    *reinterpret_cast<uint2*>(data + at) = eight;
  }
  const uint32_t word = f8_over_rows(exponent << (8 * (lane / 16)), [](uint32_t a, uint32_t b) { return a | b; });
  if (lane == 0) exponents[(long)(k / 512) * padded + row] = word;
}

// SPREAD false: grid (ceil(rows / 4), ceil(width / 512)), 512 columns of four rows a workgroup.  True: grid (whole rounds of rows, ceil(width / 4,096)), up to
// 4,096 columns of a row a workgroup, the 16 rows of a block on one XCD.
// `in_rows`: row after row instead, each of whole stretches (what the experts' products pick their rows from).
template <typename T, bool GATED, bool WHOLE, bool SPREAD>
__global__ __launch_bounds__(512) void float8_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ data, uint32_t* __restrict__ exponents,
                                                          int rows, int width, int in_rows, GateForm form) {
  const int stretches = (width + F8_K - 1) / F8_K, padded = (rows + 15) / 16 * 16;
  const int row = SPREAD ? bh_row_of_block<true>() : (int)(blockIdx.x * 4 + threadIdx.x / 64);
  const int k = SPREAD ? (int)(blockIdx.y * blockDim.x + threadIdx.x) * 8 : (int)(blockIdx.y * 512 + threadIdx.x % 64 * 8);
  if (row >= rows || k / 512 * 512 >= width) return;      // the whole wave
  const T* from = x + (size_t)row * (GATED ? 2L * width : (long)width);
  float v[8];
  load_eight<T, WHOLE>(from, k, width, v);
  if constexpr (GATED) {
    float u[8];
    load_eight<T, WHOLE>(from + width, k, width, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f8_gate_mul(v[j], u[j], form);
  }
  eight_in_8(v, row, k, stretches, padded, in_rows, data, exponents);
}

template <typename T>
void launch(const void* x, uint8_t* data, uint32_t* exponents, int rows, int width, int in_rows, int gate, hipStream_t stream) {
  const bool whole = width % 8 == 0 && (uintptr_t)x % 16 == 0;
  const int pieces = (width + 511) / 512, waves = pieces < 8 ? pieces : 8;
  const bool few = (long)rows * pieces < 16L * bh_compute_units();
  const GateForm form = bh_gate_form(gate);
  const dim3 grid = few ? dim3((rows + 3) / 4, pieces) : dim3(((unsigned)rows + BH_ROWS_ROUND - 1) / BH_ROWS_ROUND * BH_ROWS_ROUND, (pieces + waves - 1) / waves);
#define BH_F8_ROWS(GATED, WHOLE)                                                                                                                              \
  do {                                                                                                                                                        \
    if (few) float8_rows_kernel<T, GATED, WHOLE, false><<<grid, 256, 0, stream>>>((const T*)x, data, exponents, rows, width, in_rows, form);                   \
    else float8_rows_kernel<T, GATED, WHOLE, true><<<grid, waves * 64, 0, stream>>>((const T*)x, data, exponents, rows, width, in_rows, form);                 \
  } while (0)
  if (gate) {
    if (whole) BH_F8_ROWS(true, true);
    else BH_F8_ROWS(true, false);
  } else if (whole) BH_F8_ROWS(false, true);
  else BH_F8_ROWS(false, false);
#undef BH_F8_ROWS
}

// A row is a workgroup's, 512 columns a wave's, read once.  The 16 rows of a block, whose pieces of 8 bytes share lines, are the work of one XCD.
// Measured, us, in brackets the norm to bfloat16 and then its 8 bits: 32 rows of 4,096 3.1 (5.5), 512 4.2 (10.5), 2,048 9.8 (18.6), 8,192 35
// (58, 4.8 TB/s of its own bytes).
// `through_bf16`: a norm is rounded to bfloat16 first, so that a row has the same 8 bits as among few rows, which products quantise from bfloat16.
template <typename TW, bool WHOLE>
__global__ __launch_bounds__(1024) void float8_norm_kernel(const float* __restrict__ x, const TW* __restrict__ w, float eps, int through_bf16, uint8_t* __restrict__ data,
                                                           uint32_t* __restrict__ exponents, int rows, int width) {
  __shared__ float of_wave[16];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64, row = bh_row_of_block<true>();
  if (row >= rows) return;      // the whole workgroup
  const int k = threadIdx.x * 8, stretches = (width + F8_K - 1) / F8_K, padded = (rows + 15) / 16 * 16;
  float v[8], g[8];
  load_eight<float, WHOLE>(x + (size_t)row * width, k, width, v);
  if (w) load_eight<TW, WHOLE>(w, k, width, g);
  else
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = 1.f;
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
  ss = wave_sum(ss);
  if (lane == 0) of_wave[wave] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < waves; ++i) ss += of_wave[i];
  const float inv = 1.0f / sqrtf(ss / (float)width + eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = k + j < width ? v[j] * inv * g[j] : 0.f;
    if (through_bf16) v[j] = to_f32(from_f32<bf16_t>(v[j]));
  }
  eight_in_8(v, row, k, stretches, padded, 0, data, exponents);
}

template <typename TW>
void launch_norm(const float* x, const void* w, float eps, int through_bf16, uint8_t* data, uint32_t* exponents, int rows, int width, hipStream_t stream) {
  const bool whole = width % 8 == 0 && ((uintptr_t)x | (uintptr_t)w) % 16 == 0;
  const unsigned grid = ((unsigned)rows + BH_ROWS_ROUND - 1) / BH_ROWS_ROUND * BH_ROWS_ROUND, threads = (width + 511) / 512 * 64;
  if (whole) float8_norm_kernel<TW, true><<<grid, threads, 0, stream>>>(x, (const TW*)w, eps, through_bf16, data, exponents, rows, width);
  else float8_norm_kernel<TW, false><<<grid, threads, 0, stream>>>(x, (const TW*)w, eps, through_bf16, data, exponents, rows, width);
}

}  // namespace

int float8_rows_launch(const void* x, int dtype, uint8_t* data, uint32_t* exponents, int rows, int width, int in_rows, int gate, hipStream_t stream) {
  BH_REQUIRE(rows > 0 && width > 0 && width <= (1 << 24), "float8_rows: %d rows of %d values", rows, width);
  BH_REQUIRE(gate == 0 || gate == BH_GATE_SILU || gate == BH_GATE_GELU_TANH, "float8_rows: unknown gate %d", gate);
  BH_REQUIRE(((uintptr_t)data | (uintptr_t)exponents) % 16 == 0, "float8_rows: the 8-bit rows must be 16-byte aligned");
  if (dtype == BH_F32) launch<float>(x, data, exponents, rows, width, in_rows, gate, stream);
  else if (dtype == BH_BF16) launch<bf16_t>(x, data, exponents, rows, width, in_rows, gate, stream);
  else return bh_fail("float8_rows: unknown dtype %d", dtype);
  return bh_check_launch("float8_rows");
}

extern "C" int bh_float8_rows(const void* x, int dtype, void* data, void* exponents, int rows, int width, int in_rows, int gate, hipStream_t stream) {
  return float8_rows_launch(x, dtype, (uint8_t*)data, (uint32_t*)exponents, rows, width, in_rows, gate, stream);
}

// Up to so many columns.
extern "C" int bh_float8_norm_columns() { return 8192; }
// x float32 [rows][width], w null (all ones) or [width] of `w_dtype`; blocks and words as float8_rows leaves them.
extern "C" int bh_float8_norm(const float* x, const void* w, int w_dtype, float eps, int through_bf16, void* data, void* exponents, int rows, int width, hipStream_t stream) {
  BH_REQUIRE(rows > 0 && width > 0 && width <= bh_float8_norm_columns(), "float8_norm: rows of 1 to %d values, got %d of %d", bh_float8_norm_columns(), rows, width);
  BH_REQUIRE(((uintptr_t)data | (uintptr_t)exponents) % 16 == 0, "float8_norm: the 8-bit rows must be 16-byte aligned");
  if (w_dtype == BH_F32) launch_norm<float>(x, w, eps, through_bf16, (uint8_t*)data, (uint32_t*)exponents, rows, width, stream);
  else if (w_dtype == BH_BF16) launch_norm<bf16_t>(x, w, eps, through_bf16, (uint8_t*)data, (uint32_t*)exponents, rows, width, stream);
  else return bh_fail("float8_norm: unknown dtype %d", w_dtype);
  return bh_check_launch("float8_norm");
}
