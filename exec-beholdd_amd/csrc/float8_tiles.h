// A wave's walk over k for a tile of 16 XB rows x 16 YB weight rows in 8 bits, operands straight from memory with the next stretch's on
// their way: what the tiled products of gemm_float8.hip and experts_float8.hip have in common.
#pragma once
#include "float8.h"

// ap: a lane's address of its row's first stretch; a stretch is A_STEP bytes further, an operand's second half A_HALF.  xp: its row's word of
// exponents of the first four stretches, the next four `exponents_step` words further.  wp, ws: a lane's address in each block of 16 weight
// rows, and the block's scales.
template <bool FULL, int XB, int YB, int A_STEP, int A_HALF>
__device__ inline void f8_walk(const uint8_t* const (&ap)[XB], const uint32_t* const (&xp)[XB], long exponents_step, const uint8_t* const (&wp)[YB],
                               const float* const (&ws)[YB], int first, int end, f8_f32x4_t (&acc)[XB][YB]) {
  f8_u32x4_t av[2][XB][2], wv[2][YB][2];
  float xs[2][XB], wsv[2][YB];
  auto ask = [&](int u, int j) {
#pragma unroll
    for (int x = 0; x < XB; ++x) {
      const uint8_t* from = ap[x] + (size_t)j * A_STEP;
      av[u][x][0] = *reinterpret_cast<const f8_u32x4_t*>(from), av[u][x][1] = *reinterpret_cast<const f8_u32x4_t*>(from + A_HALF);
      xs[u][x] = f8_scale((xp[x][(j / 4) * exponents_step] >> (8 * (j % 4))) & 0xffu);
    }
#pragma unroll
    for (int y = 0; y < YB; ++y) {
      const f8_u32x4_t* from = reinterpret_cast<const f8_u32x4_t*>(wp[y] + (size_t)j * F8_BLOCK);
      wv[u][y][0] = from[0], wv[u][y][1] = from[64];
      wsv[u][y] = ws[y][j];
    }
  };
  auto multiply = [&](int u) {
    F8Operand<FULL> xo[XB];
#pragma unroll
    for (int x = 0; x < XB; ++x) xo[x].set(f8_operand(av[u][x][0], av[u][x][1]));
#pragma unroll
    for (int y = 0; y < YB; ++y) {
      F8Operand<FULL> wo;
      wo.set(f8_operand(wv[u][y][0], wv[u][y][1]));
#pragma unroll
      for (int x = 0; x < XB; ++x) {
        const f8_f32x4_t sum = f8_stretch(wo, xo[x]);
        const float s = xs[u][x] * wsv[u][y];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][y][e] = fmaf(sum[e], s, acc[x][y][e]);
      }
    }
  };
  if (first < end) ask(0, first);
  for (int j = first; j < end; j += 2) {
    if (j + 1 < end) ask(1, j + 1);
    multiply(0);
    if (j + 2 < end) ask(0, j + 2);
    if (j + 1 < end) multiply(1);
  }
}
