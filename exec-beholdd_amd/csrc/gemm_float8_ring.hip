// Products of many rows with weights and activations in 8 bits (float8.h), C[M, N] (+)= A[M, K] * W[N, K]^T, from operands in blocks.
//
// The tiles' walk over k is F8Ring's (float8_ring.h).
#include "gemm_float8_ring.h"
#include "float8_ring.h"

namespace {

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
template <typename TC, bool GATED, bool FULL, int XB, int YB, int WM, int WN, int R, bool DIRECT, int BM, int BN>
__global__ __launch_bounds__(64 * WM * WN, 2) void float8_ring_kernel(const uint8_t* __restrict__ a, const uint32_t* __restrict__ exponents, F8Weight w,
                                                                     TC* __restrict__ c, int M, int ldc, int accumulate, GateForm form) {
  using Ring = F8Ring<FULL, XB, YB, WM, WN, R, GATED ? 2 : 1, DIRECT>;
  constexpr int HALF = Ring::HALF, ROWS = Ring::ROWS, OUTS = Ring::OUTS;
  __shared__ __attribute__((aligned(16))) f8_u32x4_t ring[R * Ring::PIECES * 64];      // [step in turn][A's pieces, then W's][lane]
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN, wn = wave % WN;
  const int N = w.rows, steps = w.stretches, blocks = w.blocks(), row_blocks = (M + 15) / 16, padded = row_blocks * 16;
  int tile_n, tile_m;
  tile_of_workgroup<BM, BN>((N + OUTS - 1) / OUTS, (M + ROWS - 1) / ROWS, &tile_n, &tile_m);
  const uint8_t* from[Ring::ROW_PARTS + Ring::W_EACH];
  uint32_t row_at[Ring::ROW_PARTS];
#pragma unroll
  for (int i = 0; i < Ring::ROW_PARTS; ++i) {
    const int piece = DIRECT ? 2 * (wm * XB + i) : wave * Ring::A_EACH + i;
    from[i] = a + (size_t)min(tile_m * (XB * WM) + piece / 2, row_blocks - 1) * steps * F8_BLOCK + piece % 2 * 1024;
    row_at[i] = lane * 16;
  }
#pragma unroll
  for (int i = 0; i < Ring::W_EACH; ++i) {
    const int piece = wave * Ring::W_EACH + i, b = piece / 2, column = b / YB, y = b % YB;
    const int block = min((tile_n * WN + column) * HALF + y % HALF, blocks - 1);
    from[Ring::ROW_PARTS + i] = w.data + ((size_t)(y / HALF) * blocks + block) * steps * F8_BLOCK + piece % 2 * 1024;
  }
  uint32_t x_at[XB];
#pragma unroll
  for (int x = 0; x < XB; ++x) x_at[x] = min(tile_m * (XB * WM) + wm * XB + x, row_blocks - 1) * 16 + lane % 16;
  const float* ws[Ring::G];
#pragma unroll
  for (int g = 0; g < Ring::G; ++g)
    ws[g] = w.scales + ((size_t)g * w.scale_rows() + min((tile_n * WN + wn) * HALF, blocks - 1) / 8) * steps;
  f8_f32x4_t acc[XB][YB];
  Ring::walk(ring, from, row_at, F8_BLOCK, exponents, x_at, padded, ws, steps, acc);

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
        f8_store_four(at, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) at[e] = from_f32<TC>(accumulate ? v[e] + to_f32(at[e]) : v[e]);
      }
    }
  }
}

struct TileShape {
  int rows, columns;      // of weight rows
};
constexpr TileShape SHAPES[] = {{128, 128}, {256, 128}, {256, 256}};

template <typename TC, bool GATED, bool FULL>
void launch(int tile, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, TC* c, int accumulate, int M, int ldc, GateForm form, hipStream_t stream) {
  const int outs = SHAPES[tile].columns / (GATED ? 2 : 1), rows = SHAPES[tile].rows;
  const dim3 grid((unsigned)(((w.rows + outs - 1) / outs) * (long)((M + rows - 1) / rows)));
#define BH_F8_RING(FULL, XB, YB, WM, WN, R, DIRECT, BM, BN) \
  float8_ring_kernel<TC, GATED, FULL, XB, YB, WM, WN, R, DIRECT, BM, BN><<<grid, 64 * WM * WN, 0, stream>>>(a, exponents, w, c, M, ldc, accumulate, form)
  if (tile == 0) BH_F8_RING(FULL, 4, 4, 2, 2, 2, false, 8, 8);
  else if (tile == 1) BH_F8_RING(FULL, 4, 4, 4, 2, 3, false, 8, 4);
  else if constexpr (!FULL) BH_F8_RING(false, 4, 8, 4, 2, 3, true, 8, 4);
#undef BH_F8_RING
}

}  // namespace

int float8_ring_tile(int M, int N, int K, bool gated, bool full) {
  if (M <= 128 || K < 4 * F8_K) return -1;
  const long wide = (long)((M + 255) / 256) * ((N * (gated ? 2L : 1L) + 127) / 128);
  if (!full && wide >= 2L * bh_compute_units()) return 2;
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
