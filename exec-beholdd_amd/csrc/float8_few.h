// Rows of bfloat16 or float32 that a product of few rows brings into 8 bits itself, a stretch of 128 k of 16 rows a wave.
#pragma once
#include "float8.h"

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

// Rows that are in 8 bits already, in blocks.
template <>
struct F8Stretch<uint8_t> {
  f8_u32x4_t v[2];
  uint32_t exponent;
  __device__ inline f8_operand_t quantised(float* scale) const {
    *scale = f8_scale(exponent);
    return f8_operand(v[0], v[1]);
  }
};

// How a row's values are loaded.  EVEN: rows on addresses of 16 bytes, of whole stretches; a lane without a row of its own loads another
// row's, whose outputs nobody stores.  PIECES: rows on addresses of 16 bytes whose K is a multiple of 8.  VALUES: any.
enum F8Load { F8_VALUES = 0, F8_PIECES = 1, F8_EVEN = 2 };
template <typename T, int LOAD>
__device__ inline void f8_load_stretch(F8Stretch<T>& to, const T* __restrict__ row, bool there, int k0, int K) {
  constexpr int PIECE = 16 / sizeof(T), PIECES = 32 / PIECE;      // values of a load, loads of a lane
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int k = k0 + (i / (PIECES / 2)) * 64 + (i % (PIECES / 2)) * PIECE;
    if constexpr (LOAD == F8_EVEN) {
      to.v[i] = *reinterpret_cast<const f8_u32x4_t*>(row + k);
    } else {
      f8_u32x4_t piece = {0u, 0u, 0u, 0u};
      if constexpr (LOAD == F8_PIECES) {
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
}
inline int f8_load_of(const void* rows, int K) { return (uintptr_t)rows % 16 != 0 || K % 8 != 0 ? F8_VALUES : K % F8_K == 0 ? F8_EVEN : F8_PIECES; }
