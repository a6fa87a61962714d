// Rows of bfloat16 or float32 that a product of few rows brings into 8 bits itself, a stretch of 128 k of 16 rows a wave.
#pragma once
#include "float8.h"

// The largest over the four lanes of a row (lane % 16).
__device__ inline uint32_t f8_largest_of_row(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}

// A lane's 32 values of a stretch of one row: k 16 q .. + 15 and 64 + 16 q .. + 15.
template <typename T>
struct F8Stretch;
template <>
struct F8Stretch<bf16_t> {
  f8_u32x4_t v[4];
  __device__ inline f8_operand_t quantised(float* scale) const {
    uint32_t pair = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) pair = f8_larger_pair(pair, v[i][j]);
    *scale = f8_scale(f8_exponent(f8_largest_of_row(f8_of_pair(pair))));
    f8_operand_t out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (int)f8_four(v[i / 2][i % 2 * 2], v[i / 2][i % 2 * 2 + 1], *scale);
    return out;
  }
};
template <>
struct F8Stretch<float> {
  f8_u32x4_t v[8];
  __device__ inline f8_operand_t quantised(float* scale) const {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) largest = max(largest, v[i][j] & 0x7fffffffu);
    *scale = f8_scale(f8_exponent(f8_largest_of_row(largest)));
    f8_operand_t out;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      out[i] = (int)f8_four(__builtin_bit_cast(float, (uint32_t)v[i][0]), __builtin_bit_cast(float, (uint32_t)v[i][1]), __builtin_bit_cast(float, (uint32_t)v[i][2]),
                            __builtin_bit_cast(float, (uint32_t)v[i][3]), *scale);
    return out;
  }
};

// WHOLE: rows on addresses of 16 bytes whose K is a multiple of 8; otherwise value by value.
template <typename T, bool WHOLE>
__device__ inline void f8_load_stretch(F8Stretch<T>& to, const T* __restrict__ row, bool there, int k0, int K) {
  constexpr int PIECE = 16 / sizeof(T), PIECES = 32 / PIECE;      // values of a load, loads of a lane
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int k = k0 + (i / (PIECES / 2)) * 64 + (i % (PIECES / 2)) * PIECE;
    f8_u32x4_t piece = {0u, 0u, 0u, 0u};
    if constexpr (WHOLE) {
      if (there && k < K) piece = *reinterpret_cast<const f8_u32x4_t*>(row + k);
    } else if (there) {
#pragma unroll
      for (int j = 0; j < PIECE; ++j)
        if (k + j < K) {
          if constexpr (sizeof(T) == 4) piece[j] = __builtin_bit_cast(uint32_t, (float)row[k + j]);
          else piece[j / 2] |= (uint32_t)row[k + j].bits << (16 * (j % 2));
        }
    }
    to.v[i] = piece;
  }
}
