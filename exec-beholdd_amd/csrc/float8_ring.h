// The walk over k of a workgroup of WM x WN waves with a tile of 16 XB WM rows x 16 YB WN weight rows in 8 bits (float8.h), in steps of 128,
// the k of one 8-bit MFMA and of one scale.  Global memory hands a step's operands to LDS directly, in pieces of 1 KB (16 rows x 64 k in
// lane order), into a ring of R steps.  While step j is multiplied, the wave reads the rows of step j + 1 from LDS into its other set of
// registers and the weights of step j one block ahead of their MFMAs, and asks for the rows of step j + R, whose place those of step j have
// left when it begins, and for the weights of step j + R - 1, whose place those of step j - 1 have left.  So both are on their way for R - 1
// steps.  One barrier a step.  A stretch's sums leave the matrix cores into one of three sets of registers and are multiplied by their scales
// two MFMAs later, while those run.
#pragma once
#include "float8.h"
#include <type_traits>

// s_waitcnt of gfx9 (vmcnt in bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8): all LDS reads are back, and at most `vm` of the wave's
// global loads are still on their way.
#define F8_WAIT(vm) __builtin_amdgcn_s_waitcnt(((vm) & 15) | (((vm) >> 4) << 14) | (7 << 4) | (0 << 8))
// Every wave has waited for its loads.  Nothing may be moved across it by the compiler.
#define F8_MEET()                         \
  do {                                    \
    __builtin_amdgcn_sched_barrier(0);    \
    __builtin_amdgcn_s_barrier();         \
    __builtin_amdgcn_sched_barrier(0);    \
  } while (0)

#define F8_BUFFER 0x00020000      // a buffer of bytes; the addresses are checked by the launch

// FULL: float8.h.  G: matrices that a wave's weight rows are of (2: gate rows, then as many up rows).  DIRECT: a wave loads its rows of the
// next step from memory into its other set of registers itself, and only the weights go through LDS.  LINES: rows lie one after the other, and a piece is 8 rows x 128 k, whole lines of memory, rather than
// 16 rows x 64; the 16 bytes c of its row r lie at place c ^ r, so that 8 rows' are in different banks.
template <bool FULL_, int XB_, int YB_, int WM_, int WN_, int R_, int G_, bool DIRECT_ = false, bool LINES_ = false>
struct F8Ring {
  static constexpr bool FULL = FULL_, DIRECT = DIRECT_, LINES = LINES_;
  static constexpr int XB = XB_, YB = YB_, WM = WM_, WN = WN_, R = R_, G = G_;
  static constexpr int WAVES = WM * WN, A_PIECES = DIRECT ? 0 : 2 * XB * WM, W_PIECES = 2 * YB * WN, PIECES = A_PIECES + W_PIECES;
  static constexpr int A_EACH = A_PIECES / WAVES, W_EACH = W_PIECES / WAVES, EACH = A_EACH + W_EACH, HALF = YB / G;
  static constexpr int ROW_PARTS = DIRECT ? XB : A_EACH;      // addresses of rows that a wave has: of its blocks, or of its pieces
  static constexpr int ROWS = 16 * XB * WM, OUTS = 16 * HALF * WN;
  static_assert(A_PIECES % WAVES == 0 && W_PIECES % WAVES == 0 && R >= 2 && EACH * (R - 2) < 64 && (!DIRECT || R >= 3), "every wave brings as many pieces, and their count fits s_waitcnt");
  static_assert(F8_K % (16 * HALF) == 0, "a wave's blocks of a matrix have one scale");
  static_assert(YB % 2 == 0 && YB % G == 0, "the first weights of a step lie in the first set");

  // Where a wave's operands come from: the first ROW_PARTS addresses are those of rows, `row_step` bytes a step, the others those of its pieces
  // of the weights; row_at: a lane's own offset (16 * lane for rows in blocks), x_at: that of its row's word of exponents, four stretches
  // `exponents_step` words behind the four before, from stretch `first` on (the other addresses are those of stretch `first`).  All of an address but the lane's offset is the same for the wave: buffer loads take it from
  // scalar registers, of which there are enough.  DIRECT takes rows in blocks.
  // acc[x][y][i]: row 16 (XB wm + x) + lane % 16 of the tile, weight row 16 y + 4 (lane / 16) + i of the wave's.
  __device__ static inline void walk(f8_u32x4_t* __restrict__ ring, const uint8_t* const (&from)[ROW_PARTS + W_EACH], const uint32_t (&row_at)[ROW_PARTS],
                                     int row_step, const uint32_t* exponents, const uint32_t (&x_at)[XB], uint32_t exponents_step,
                                     const float* const (&ws)[G], int first, int steps, f8_f32x4_t (&acc)[XB][YB]) {
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN, wn = wave % WN;
    __amdgpu_buffer_rsrc_t buffer[ROW_PARTS + W_EACH];
#pragma unroll
    for (int i = 0; i < ROW_PARTS + W_EACH; ++i) buffer[i] = __builtin_amdgcn_make_buffer_rsrc((void*)from[i], 0, -1, F8_BUFFER);
    const __amdgpu_buffer_rsrc_t words_buffer = __builtin_amdgcn_make_buffer_rsrc((void*)exponents, 0, -1, F8_BUFFER);
    auto ask_piece = [&](int i, int step, int place) {
      const int piece = i < A_EACH ? wave * A_EACH + i : A_PIECES + wave * W_EACH + i - A_EACH;
      __attribute__((address_space(3))) void* to = (__attribute__((address_space(3))) void*)&ring[(place * PIECES + piece) * 64];
      if (i < A_EACH) __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer[i], to, 16, row_at[i < A_EACH ? i : 0], step * row_step, 0, 0);
      else __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer[ROW_PARTS + i - A_EACH], to, 16, lane * 16, step * F8_BLOCK, 0, 0);
    };
    auto ask_rows = [&](int step, int place) {
#pragma unroll
      for (int i = 0; i < A_EACH; ++i) ask_piece(i, step, place);
    };
    auto ask_weights = [&](int step, int place) {
#pragma unroll
      for (int i = A_EACH; i < EACH; ++i) ask_piece(i, step, place);
    };
#pragma unroll
    for (int x = 0; x < XB; ++x)
#pragma unroll
      for (int y = 0; y < YB; ++y) acc[x][y] = f8_f32x4_t{0.f, 0.f, 0.f, 0.f};
    f8_operand_t af[2][XB], wf[2];
    uint32_t words[XB];
    float wsv[G];
    auto load_a = [&](int step, int x) {
      return f8_operand(__builtin_amdgcn_raw_buffer_load_b128(buffer[x], row_at[x], step * row_step, 0),
                        __builtin_amdgcn_raw_buffer_load_b128(buffer[x], row_at[x] + 1024, step * row_step, 0));
    };
    auto read_a = [&](int place, int x) {
      if constexpr (LINES) {
        const f8_u32x4_t* block = &ring[(place * PIECES + 2 * (wm * XB + x)) * 64 + lane % 16 * 8];
        const int first_half = (lane / 16) ^ (lane % 8);
        return f8_operand(block[first_half], block[first_half ^ 4]);
      }
      const f8_u32x4_t* at = &ring[(place * PIECES + 2 * (wm * XB + x)) * 64 + lane];
      return f8_operand(at[0], at[64]);
    };
    auto read_w = [&](int place, int y) {
      const f8_u32x4_t* at = &ring[(place * PIECES + A_PIECES + 2 * (wn * YB + y)) * 64 + lane];
      return f8_operand(at[0], at[64]);
    };
    auto ask_scales = [&](int step) {
#pragma unroll
      for (int x = 0; x < XB; ++x) words[x] = __builtin_amdgcn_raw_buffer_load_b32(words_buffer, x_at[x] * 4, (uint32_t)((first + step) / 4) * exponents_step * 4, 0);
#pragma unroll
      for (int g = 0; g < G; ++g) wsv[g] = ws[g][step];
    };
    // The first step alone is waited for: its rows, then its weights, then what comes after.
    ask_scales(0);
    if (!DIRECT) ask_rows(0, 0);
    if (DIRECT) {
#pragma unroll
      for (int x = 0; x < XB; ++x) af[0][x] = load_a(0, x);
    }
    ask_weights(0, 0);
    for (int j = 1; j < R && j < steps; ++j) {
      if (!DIRECT) ask_rows(j, j);
      if (j < R - 1) ask_weights(j, j);
    }
    if (steps > R) F8_WAIT(EACH * (R - 2) + A_EACH);      // (all of them were asked for)
    else F8_WAIT(0);
    F8_MEET();
    if (!DIRECT) {
#pragma unroll
      for (int x = 0; x < XB; ++x) af[0][x] = read_a(0, x);
    }

    int place = 0;      // of the step that is multiplied
    // STEADY: the rows of step j + R and the weights of step j + R - 1 exist, and what was asked for in the last R - 2 steps may still be
    // on its way.
    auto multiply = [&](int j, auto odd, auto steady) {
      constexpr int U = decltype(odd)::value;
      constexpr bool STEADY = decltype(steady)::value;
      if (STEADY) F8_WAIT(EACH * (R - 2));      // (of the first step: its weights and the next rows, which were asked for before the others)
      else F8_WAIT(0);
      F8_MEET();
      wf[0] = read_w(place, 0);
      const int next = place == R - 1 ? 0 : place + 1, left = place == 0 ? R - 1 : place - 1;
      float s[G][XB];
#pragma unroll
      for (int x = 0; x < XB; ++x) {
        const float xs = f8_scale((words[x] >> (8 * ((first + j) % 4))) & 0xffu);
#pragma unroll
        for (int g = 0; g < G; ++g) s[g][x] = xs * wsv[g];
      }
      if (STEADY || j + 1 < steps) ask_scales(j + 1);      // (no branches while steady: sums would be kept across them and scaled behind all MFMAs)
      if (DIRECT && (STEADY || j + 1 < steps)) {
#pragma unroll
        for (int x = 0; x < XB; ++x) af[1 - U][x] = load_a(j + 1, x);
      }
      F8Operand<FULL> xo[XB];
#pragma unroll
      for (int x = 0; x < XB; ++x) xo[x].set(af[U][x]);
      f8_f32x4_t sum[3];
      auto scaled = [&](int t) {
        const int x = t % XB, y = t / XB;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][y][e] = fmaf(sum[t % 3][e], s[y / HALF][x], acc[x][y][e]);
      };
      if (!DIRECT && !STEADY && j + R < steps) ask_rows(j + R, place);
      if (!STEADY && j + R - 1 < steps) ask_weights(j + R - 1, left);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int y = 0; y < YB; ++y) {
        // (beyond the last step this reads what an earlier one has left there, and nobody uses it)
        if (y + 1 < YB) wf[(y + 1) % 2] = read_w(place, y + 1);
#pragma unroll
        for (int x = 0; x < XB; ++x)
          if (!DIRECT && x * YB / XB == y) af[1 - U][x] = read_a(next, x);
        if (STEADY) {
#pragma unroll
          for (int i = 0; i < EACH; ++i)
            if (i * YB / EACH == y) ask_piece(i, i < A_EACH ? j + R : j + R - 1, i < A_EACH ? place : left);
        }
        F8Operand<FULL> wo;
        wo.set(wf[y % 2]);
#pragma unroll
        for (int x = 0; x < XB; ++x) {
          const int t = y * XB + x;
          sum[t % 3] = f8_stretch(wo, xo[x]);
          __builtin_amdgcn_sched_barrier(0);      // the compiler would have every sum scaled behind its own MFMA, and wait for it
          if (t >= 2) scaled(t - 2);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      scaled(XB * YB - 2);
      scaled(XB * YB - 1);
      place = next;
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    int j = 0;
    for (; j + 1 + R < steps; j += 2) {
      multiply(j, even, std::true_type());
      multiply(j + 1, odd, std::true_type());
    }
    for (; j < steps; j += 2) {
      multiply(j, even, std::false_type());
      if (j + 1 < steps) multiply(j + 1, odd, std::false_type());
    }

  }
};
#undef F8_WAIT
#undef F8_MEET
