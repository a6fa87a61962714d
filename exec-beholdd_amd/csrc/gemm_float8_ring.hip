// Products of many rows with weights and activations in 8 bits (float8.h), C[M, N] (+)= A[M, K] * W[N, K]^T, from operands in blocks.
//
// A workgroup of WM x WN waves owns a tile of 16 XB WM rows x 16 YB WN weight rows and walks over k in steps of 128, the k of one 8-bit
// MFMA and of one scale.  Global memory hands a step's operands to LDS directly, in pieces of 1 KB (16 rows x 64 k in lane order), into a
// ring of R steps.  While step j is multiplied, the wave reads the rows of step j + 1 from LDS into its other set of registers and the
// weights of step j one block ahead of their MFMAs, and asks for the rows of step j + R, whose place those of step j have left when it
// begins, and for the weights of step j + R - 1, whose place those of step j - 1 have left.  So both are on their way for R - 1 steps.
// One barrier a step.  A stretch's sums leave the matrix cores into one of three sets of registers and are multiplied by their scales
// two MFMAs later, while those run.
#include "gemm_float8_ring.h"
#include <type_traits>

namespace {

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

// Workgroups go to the eight XCDs in turn, each with an L2 of its own: an XCD takes a run of neighbours in an order that goes through the
// tiles in blocks of BM row tiles x BN weight tiles, so that what walks over k there together asks that L2 for few different bytes.
template <int BM, int BN>
__device__ inline void tile_of_workgroup(int n_tiles, int m_tiles, int* tile_n, int* tile_m) {
  const int total = n_tiles * m_tiles, xcd = blockIdx.x % 8, each = total / 8, more = total % 8;
  int v = xcd * each + min(xcd, more) + blockIdx.x / 8;
  const int whole_columns = n_tiles / BN;
  int first_n = 0, columns = BN;
  if (v >= whole_columns * BN * m_tiles) {
    v -= whole_columns * BN * m_tiles;
    first_n = whole_columns * BN;
    columns = n_tiles - first_n;
  } else {
    first_n = (v / (BN * m_tiles)) * BN;
    v %= BN * m_tiles;
  }
  const int chunk = v / (BM * columns), within = v % (BM * columns);
  const int rows = min(BM, m_tiles - chunk * BM);
  *tile_m = chunk * BM + within % rows;
  *tile_n = first_n + within / rows;
}

// A tile that sticks out of the matrix repeats its last blocks and stores only what exists.
template <typename TC, bool GATED, bool FULL, int XB, int YB, int WM, int WN, int R, int BM, int BN>
__global__ __launch_bounds__(64 * WM * WN, 2) void float8_ring_kernel(const uint8_t* __restrict__ a, const uint32_t* __restrict__ exponents, F8Weight w,
                                                                     TC* __restrict__ c, int M, int ldc, int accumulate, GateForm form) {
  constexpr int WAVES = WM * WN, A_PIECES = 2 * XB * WM, W_PIECES = 2 * YB * WN, PIECES = A_PIECES + W_PIECES;
  constexpr int A_EACH = A_PIECES / WAVES, EACH = PIECES / WAVES, HALF = GATED ? YB / 2 : YB, ROWS = 16 * XB * WM, OUTS = 16 * HALF * WN, G = GATED ? 2 : 1;
  static_assert(A_PIECES % WAVES == 0 && W_PIECES % WAVES == 0 && R >= 2 && EACH * (R - 2) < 64, "every wave brings as many pieces, and their count fits s_waitcnt");
  static_assert(F8_K % (16 * HALF) == 0, "a wave's blocks of a matrix have one scale");
  __shared__ __attribute__((aligned(16))) f8_u32x4_t ring[R * PIECES * 64];      // [step in turn][A's pieces, then W's][lane]
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN, wn = wave % WN;
  const int N = w.rows, steps = w.stretches, blocks = w.blocks(), row_blocks = (M + 15) / 16, padded = row_blocks * 16;
  int tile_n, tile_m;
  tile_of_workgroup<BM, BN>((N + OUTS - 1) / OUTS, (M + ROWS - 1) / ROWS, &tile_n, &tile_m);

  // a wave's pieces of a step: A_EACH of the rows, the others of the weights
  const uint8_t* from[EACH];
  int to[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int piece = i < A_EACH ? wave * A_EACH + i : A_PIECES + wave * (EACH - A_EACH) + i - A_EACH, half = piece % 2;
    to[i] = piece * 64;
    if (i < A_EACH) {
      const int block = min(tile_m * (XB * WM) + piece / 2, row_blocks - 1);
      from[i] = a + (size_t)block * steps * F8_BLOCK + half * 1024;
    } else {
      const int b = (piece - A_PIECES) / 2, column = b / YB, y = b % YB;
      const int block = min((tile_n * WN + column) * HALF + y % HALF, blocks - 1);
      from[i] = w.data + ((size_t)(y / HALF) * blocks + block) * steps * F8_BLOCK + half * 1024;
    }
  }
  auto ask_piece = [&](int i, int step, int place) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from[i] + (size_t)step * F8_BLOCK + lane * 16),
                                     (__attribute__((address_space(3))) void*)&ring[place * PIECES * 64 + to[i]], 16, 0, 0);
  };
  auto ask_rows = [&](int step, int place) {
#pragma unroll
    for (int i = 0; i < A_EACH; ++i) ask_piece(i, step, place);
  };
  auto ask_weights = [&](int step, int place) {
#pragma unroll
    for (int i = A_EACH; i < EACH; ++i) ask_piece(i, step, place);
  };
  const uint32_t* xp[XB];
#pragma unroll
  for (int x = 0; x < XB; ++x) xp[x] = exponents + min(tile_m * (XB * WM) + wm * XB + x, row_blocks - 1) * 16 + lane % 16;
  const float* ws[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    ws[g] = w.scales + ((size_t)g * w.scale_rows() + min((tile_n * WN + wn) * HALF, blocks - 1) / 8) * steps;

  f8_f32x4_t acc[XB][YB];
#pragma unroll
  for (int x = 0; x < XB; ++x)
#pragma unroll
    for (int y = 0; y < YB; ++y) acc[x][y] = f8_f32x4_t{0.f, 0.f, 0.f, 0.f};
  f8_operand_t af[2][XB], wf[2];
  uint32_t words[XB];
  float wsv[G];
  auto read_a = [&](int place, int x) {
    const f8_u32x4_t* at = &ring[(place * PIECES + 2 * (wm * XB + x)) * 64 + lane];
    return f8_operand(at[0], at[64]);
  };
  auto read_w = [&](int place, int y) {
    const f8_u32x4_t* at = &ring[(place * PIECES + A_PIECES + 2 * (wn * YB + y)) * 64 + lane];
    return f8_operand(at[0], at[64]);
  };
  auto ask_scales = [&](int step) {
#pragma unroll
    for (int x = 0; x < XB; ++x) words[x] = xp[x][(size_t)(step / 4) * padded];
#pragma unroll
    for (int g = 0; g < G; ++g) wsv[g] = ws[g][step];
  };
  ask_scales(0);
  for (int j = 0; j < R && j < steps; ++j) {
    ask_rows(j, j);
    if (j < R - 1) ask_weights(j, j);
  }
  F8_WAIT(0);
  F8_MEET();
#pragma unroll
  for (int x = 0; x < XB; ++x) af[0][x] = read_a(0, x);

  int place = 0;      // of the step that is multiplied
  // STEADY: the rows of step j + R and the weights of step j + R - 1 exist, and what was asked for in the last R - 2 steps may still be
  // on its way.
  auto multiply = [&](int j, auto odd, auto steady) {
    constexpr int U = decltype(odd)::value;
    constexpr bool STEADY = decltype(steady)::value;
    if (STEADY) F8_WAIT(EACH * (R - 2));
    else F8_WAIT(0);
    F8_MEET();
    wf[0] = read_w(place, 0);
    const int next = place == R - 1 ? 0 : place + 1, left = place == 0 ? R - 1 : place - 1;
    float s[G][XB];
#pragma unroll
    for (int x = 0; x < XB; ++x) {
      const float xs = f8_scale((words[x] >> (8 * (j % 4))) & 0xffu);
#pragma unroll
      for (int g = 0; g < G; ++g) s[g][x] = xs * wsv[g];
    }
    if (j + 1 < steps) ask_scales(j + 1);
    F8Operand<FULL> xo[XB];
#pragma unroll
    for (int x = 0; x < XB; ++x) xo[x].set(af[U][x]);
    f8_f32x4_t sum[3];
    auto scaled = [&](int t) {
      const int x = t % XB, y = t / XB;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[x][y][e] = fmaf(sum[t % 3][e], s[y / HALF][x], acc[x][y][e]);
    };
    if (!STEADY && j + R < steps) ask_rows(j + R, place);
    if (!STEADY && j + R - 1 < steps) ask_weights(j + R - 1, left);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int y = 0; y < YB; ++y) {
      // (beyond the last step this reads what an earlier one has left there, and nobody uses it)
      if (y + 1 < YB) wf[(y + 1) % 2] = read_w(place, y + 1);
#pragma unroll
      for (int x = 0; x < XB; ++x)
        if (x * YB / XB == y) af[1 - U][x] = read_a(next, x);
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
        if (t >= 2) scaled(t - 2);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    scaled(XB * YB - 2);
    scaled(XB * YB - 1);
    place = next;
  };
  static_assert(YB % 2 == 0, "the first weights of a step lie in the first set");
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

  // acc[x][y][i]: row 16 (XB wm + x) + lane % 16 of the tile, weight row 16 (y % HALF) + 4 (lane / 16) + i of the wave's
  const bool fours = (N | ldc) % 4 == 0 && (uintptr_t)c % (4 * sizeof(TC)) == 0;
#pragma unroll
  for (int x = 0; x < XB; ++x) {
    const int row = tile_m * ROWS + (wm * XB + x) * 16 + lane % 16;
    if (row >= M) continue;
#pragma unroll
    for (int y = 0; y < HALF; ++y) {
      const int n = ((tile_n * WN + wn) * HALF + y) * 16 + 4 * (lane / 16);
      if (n >= N) continue;
      TC* at = c + (size_t)row * ldc + n;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = GATED ? gate_mul(acc[x][y][e], acc[x][y + (GATED ? HALF : 0)][e], form) : acc[x][y][e];
      if (fours) {
        if (accumulate) {
          const float4 old = load_four(at);
          v[0] += old.x, v[1] += old.y, v[2] += old.z, v[3] += old.w;
        }
        store_four(at, v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) at[e] = from_f32<TC>(accumulate ? v[e] + to_f32(at[e]) : v[e]);
      }
    }
  }
}
#undef F8_WAIT
#undef F8_MEET

struct TileShape {
  int rows, columns;      // of weight rows
};
constexpr TileShape SHAPES[] = {{128, 128}, {256, 128}};

template <typename TC, bool GATED, bool FULL>
void launch(int tile, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, TC* c, int accumulate, int M, int ldc, GateForm form, hipStream_t stream) {
  const int outs = SHAPES[tile].columns / (GATED ? 2 : 1), rows = SHAPES[tile].rows;
  const dim3 grid((unsigned)(((w.rows + outs - 1) / outs) * (long)((M + rows - 1) / rows)));
#define BH_F8_RING(XB, YB, WM, WN, R, BM, BN) \
  float8_ring_kernel<TC, GATED, FULL, XB, YB, WM, WN, R, BM, BN><<<grid, 64 * WM * WN, 0, stream>>>(a, exponents, w, c, M, ldc, accumulate, form)
  if (tile == 0) BH_F8_RING(4, 4, 2, 2, 2, 8, 8);
  else BH_F8_RING(4, 4, 4, 2, 3, 8, 4);
#undef BH_F8_RING
}

}  // namespace

int float8_ring_tile(int M, int N, int K, bool gated, bool full) {
  if (M <= 128 || K < 4 * F8_K) return -1;
  const long wide = (long)((M + 255) / 256) * ((N * (gated ? 2L : 1L) + 127) / 128);
  return wide >= bh_compute_units() ? 1 : 0;
}

int float8_ring_launch(int tile, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, void* c, int c_dtype, int accumulate, int M, int ldc,
                       int gated, int full, GateForm form, hipStream_t stream) {
#define BH_F8_RUN(TC, GATED, FULL) launch<TC, GATED, FULL>(tile, a, exponents, w, (TC*)c, accumulate, M, ldc, form, stream)
#define BH_F8_FULL(TC, GATED)               \
  do {                                      \
    if (full) BH_F8_RUN(TC, GATED, true);   \
    else BH_F8_RUN(TC, GATED, false);       \
  } while (0)
  if (gated) {
    if (c_dtype == BH_F32) BH_F8_FULL(float, true);
    else BH_F8_FULL(bf16_t, true);
  } else if (c_dtype == BH_F32) BH_F8_FULL(float, false);
  else BH_F8_FULL(bf16_t, false);
#undef BH_F8_FULL
#undef BH_F8_RUN
  return bh_check_launch("float8_ring");
}
