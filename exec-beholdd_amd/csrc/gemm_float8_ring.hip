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

// The gated outputs of a tile, a stretch of the next product's k, in 8 bits, in blocks and with their exponents: a row's largest is found between the
// waves that hold it.  `through_bf16`: they are rounded to bfloat16 first, as they would be on their way there.
template <typename Ring>
__device__ inline void leave_in_8(f8_u32x4_t* ring, f8_f32x4_t (&acc)[Ring::XB][Ring::YB], int tile_m, int tile_n, uint8_t* __restrict__ c,
                                  uint8_t* __restrict__ c_exponents, int M, int N, int through_bf16, const GateForm& form) {
  constexpr int XB = Ring::XB, HALF = Ring::HALF, ROWS = Ring::ROWS, OUTS = Ring::OUTS, WN = Ring::WN;
  static_assert(Ring::G == 2 && OUTS == F8_K, "a tile's outputs are a stretch");
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN, wn = wave % WN, padded = (M + 15) / 16 * 16;
  uint32_t* largest = reinterpret_cast<uint32_t*>(ring);      // [wave column][row]
  __syncthreads();      // every wave has read its last step
#pragma unroll
  for (int x = 0; x < XB; ++x) {
    uint32_t most = 0;
#pragma unroll
    for (int y = 0; y < HALF; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = tile_n * OUTS + (wn * HALF + y) * 16 + 4 * (lane / 16) + e;
        float v = n < N ? f8_gate_mul(acc[x][y][e], acc[x][y + HALF][e], form) : 0.f;
        if (through_bf16) v = to_f32(from_f32<bf16_t>(v));
        acc[x][y][e] = v;
        most = f8_larger(most, v);
      }
    most = f8_largest_of_row(most);
    if (lane < 16) largest[wn * ROWS + (wm * XB + x) * 16 + lane] = most;
  }
  __syncthreads();
  const int out_stretches = (N + F8_K - 1) / F8_K;
#pragma unroll
  for (int x = 0; x < XB; ++x) {
    const int r = (wm * XB + x) * 16 + lane % 16, row = tile_m * ROWS + r;
    uint32_t most = largest[r];
#pragma unroll
    for (int column = 1; column < WN; ++column) most = max(most, largest[column * ROWS + r]);
    const uint32_t exponent = f8_exponent(most);
    if (row >= M) continue;
    uint8_t* block = c + ((size_t)(row / 16) * out_stretches + tile_n) * F8_BLOCK;
#pragma unroll
    for (int y = 0; y < HALF; ++y)
      *reinterpret_cast<uint32_t*>(block + f8_place(row % 16, (wn * HALF + y) * 16 + 4 * (lane / 16))) =
          f8_four(acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3], f8_scale(exponent));
    if (wn == 0 && lane < 16) c_exponents[((size_t)(tile_n / 4) * padded + row) * 4 + tile_n % 4] = (uint8_t)exponent;
  }
}

// A tile that sticks out of the matrix repeats its last blocks and stores only what exists.
// With K in parts (PARTS, grid y) part p leaves its bare sums at c + p * M * width, width = N, or 2 N of a gated product (gate, then up).
// TC uint8_t: a gated product of 128 outputs a tile leaves them in 8 bits (leave_in_8; `accumulate` is its `through_bf16`).
template <typename TC, bool GATED, bool FULL, bool PARTS, int XB, int YB, int WM, int WN, int R, bool DIRECT, int BM, int BN>
__global__ __launch_bounds__(64 * WM * WN, 2) void float8_ring_kernel(const uint8_t* __restrict__ a, const uint32_t* __restrict__ exponents, F8Weight w,
                                                                     TC* __restrict__ c, uint8_t* __restrict__ c_exponents, int M, int ldc, int accumulate, GateForm form) {
  using Ring = F8Ring<FULL, XB, YB, WM, WN, R, GATED ? 2 : 1, DIRECT>;
  constexpr int HALF = Ring::HALF, ROWS = Ring::ROWS, OUTS = Ring::OUTS;
  __shared__ __attribute__((aligned(16))) f8_u32x4_t ring[R * Ring::PIECES * 64];      // [step in turn][A's pieces, then W's][lane]
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN, wn = wave % WN;
  const int N = w.rows, stretches = w.stretches, blocks = w.blocks(), row_blocks = (M + 15) / 16, padded = row_blocks * 16;
  const int first = PARTS ? (int)((long)stretches * blockIdx.y / gridDim.y) : 0;
  const int steps = PARTS ? (int)((long)stretches * (blockIdx.y + 1) / gridDim.y) - first : stretches;
  int tile_n, tile_m;
  tile_of_workgroup<BM, BN>((N + OUTS - 1) / OUTS, (M + ROWS - 1) / ROWS, &tile_n, &tile_m);
  const uint8_t* from[Ring::ROW_PARTS + Ring::W_EACH];
  uint32_t row_at[Ring::ROW_PARTS];
#pragma unroll
  for (int i = 0; i < Ring::ROW_PARTS; ++i) {
    const int piece = DIRECT ? 2 * (wm * XB + i) : wave * Ring::A_EACH + i;
    from[i] = a + ((size_t)min(tile_m * (XB * WM) + piece / 2, row_blocks - 1) * stretches + first) * F8_BLOCK + piece % 2 * 1024;
    row_at[i] = lane * 16;
  }
#pragma unroll
  for (int i = 0; i < Ring::W_EACH; ++i) {
    const int piece = wave * Ring::W_EACH + i, b = piece / 2, column = b / YB, y = b % YB;
    const int block = min((tile_n * WN + column) * HALF + y % HALF, blocks - 1);
    from[Ring::ROW_PARTS + i] = w.data + (((size_t)(y / HALF) * blocks + block) * stretches + first) * F8_BLOCK + piece % 2 * 1024;
  }
  uint32_t x_at[XB];
#pragma unroll
  for (int x = 0; x < XB; ++x) x_at[x] = min(tile_m * (XB * WM) + wm * XB + x, row_blocks - 1) * 16 + lane % 16;
  const float* ws[Ring::G];
#pragma unroll
  for (int g = 0; g < Ring::G; ++g)
    ws[g] = w.scales + ((size_t)g * w.scale_rows() + min((tile_n * WN + wn) * HALF, blocks - 1) / 8) * stretches + first;
  f8_f32x4_t acc[XB][YB];
  Ring::walk(ring, from, row_at, F8_BLOCK, exponents, x_at, padded, ws, first, steps, acc);

  if constexpr (sizeof(TC) == 1) {
    leave_in_8<Ring>(ring, acc, tile_m, tile_n, c, c_exponents, M, N, accumulate, form);
  } else {
    const bool fours = (N | ldc) % 4 == 0 && (uintptr_t)c % (4 * sizeof(TC)) == 0;
#pragma unroll
    for (int x = 0; x < XB; ++x) {
      const int row = tile_m * ROWS + (wm * XB + x) * 16 + lane % 16;
      if (row >= M) continue;
#pragma unroll
      for (int y = 0; y < (PARTS ? YB : HALF); ++y) {
        const int n = ((tile_n * WN + wn) * HALF + y % HALF) * 16 + 4 * (lane / 16);
        if (n >= N) continue;
        if constexpr (PARTS) {
          const size_t width = GATED ? 2 * (size_t)N : N;
          float* sums = reinterpret_cast<float*>(c) + ((size_t)blockIdx.y * M + row) * width + (size_t)(y / HALF) * N + n;
          if (N % 4 == 0) {
            store_four(sums, acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < N) sums[e] = acc[x][y][e];
          }
          continue;
        }
        TC* at = c + (size_t)row * ldc + n;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = GATED ? f8_gate_out<TC>(acc[x][y][e], acc[x][(y + (GATED ? HALF : 0)) % YB][e], form) : acc[x][y][e];
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
}

// A tile's sizes, how many of its workgroups share a compute unit, what a step of 128 k costs a compute unit that has one of them, two or three, and
// what their start and end cost, with the matrix cores' own sums and with full ones (us).  From the times of every tile and cut of K, and of few rows
// (gemm_float8.hip), for 12 products of 24 to 8,160 rows, 1,024 to 24,576 weight rows and k of 1,000 to 12,288 (220 sizes, 3,500 times): what is chosen there
// takes 2 % longer than the best of them on average, 22 % at most (300 rows of 1,024 x 1,024 7.0 / 5.8).  Where the tiles are ahead, us, 32 x 64 / 64 x 64 /
// 64 x 256 / 128 x 128 / 256 x 128 / 256 x 256: 256 rows of 2,048 x 2,048 6.4 / 7.9 / 13.6 / 16.3 / 18.1 / 24; 512 rows of 4,096 x 4,096 18.2 / 17.6 / 20.7 / 28.7 / 33 / 55; 2,048 rows of them
// from the third on 45.3 / 39.6 / 41.5 / 57, 4,096 rows 88 / 75.6 / 81.4 / 69.8; 200 rows of 4,096 x 12,288 in four parts of 64 x 256 26.3, in one 55.
struct TileShape {
  int rows, columns, share;
  double step[3], start_and_end, full_step[3], full_start_and_end;
};
constexpr TileShape SHAPES[] = {{128, 128, 2, {0.738, 1.101}, 3.94, {1.145, 1.761}, 6.24},
                                {256, 128, 1, {0.798}, 6.74, {1.610}, 8.36},
                                {256, 256, 1, {1.392}, 10.37, {}, 0.},
                                {64, 256, 1, {0.516}, 4.79, {0.959}, 5.50},
                                {128, 256, 1, {0.811}, 6.74, {1.577}, 8.99},
                                {64, 64, 3, {0.287, 0.432, 0.574}, 3.25, {0.462, 0.780, 0.860}, 3.78},
                                {32, 64, 3, {0.212, 0.294, 0.385}, 3.19, {0.334, 0.495, 0.557}, 3.55}};
constexpr int TILES = 7, MOST_PARTS = 8;

double cost_us(int tile, int parts, int M, int W, int K, bool full) {
  const TileShape& s = SHAPES[tile];
  const long units = bh_compute_units(), workgroups = (long)((M + s.rows - 1) / s.rows) * ((W + s.columns - 1) / s.columns) * parts;
  const double steps = ((K + F8_K - 1) / F8_K + parts - 1) / parts, ends = full ? s.full_start_and_end : s.start_and_end;
  const double* step = full ? s.full_step : s.step;
  // whole rounds of `share` a compute unit, then a last one of as many as are left, which take as long on some units as on all
  const long rounds = workgroups / (units * s.share), left = (workgroups % (units * s.share) + units - 1) / units;
  double t = rounds * (steps * step[s.share - 1] + ends);
  if (left > 0) t += steps * step[left - 1] + ends;
  const double read = ends + (double)W * K / 4.47e6;      // no sooner than the weights are there
  if (t < read) t = read;
  if (parts == 1) return t;
  return t + 2.7 + parts * (0.113 + (double)M * W * 8. / 7.42e6);      // the parts' sums on their way to memory and back, and a launch
}

template <typename TC, bool GATED, bool FULL, bool PARTS>
void launch(int tile, int parts, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, TC* c, uint8_t* c_exponents, int accumulate, int M, int ldc,
            GateForm form, hipStream_t stream) {
  const int outs = SHAPES[tile].columns / (GATED ? 2 : 1), rows = SHAPES[tile].rows;
  const dim3 grid((unsigned)(((w.rows + outs - 1) / outs) * (long)((M + rows - 1) / rows)), parts);
#define BH_F8_RING(FULL, XB, YB, WM, WN, R, DIRECT, BM, BN)                                                                             \
  float8_ring_kernel<TC, GATED, FULL, PARTS, XB, YB, WM, WN, R, DIRECT, BM, BN><<<grid, 64 * WM * WN, 0, stream>>>(a, exponents, w, c, \
                                                                                                                  c_exponents, M, ldc, accumulate, form)
  if (tile == 3) BH_F8_RING(FULL, 2, 4, 2, 4, 3, false, 8, 4);
  else if (tile == 4) BH_F8_RING(FULL, 4, 4, 2, 4, 3, false, 8, 4);
  else if (tile == 2) {
    if constexpr (!FULL && !PARTS) BH_F8_RING(false, 4, 8, 4, 2, 3, true, 8, 4);
  } else if constexpr (sizeof(TC) > 1) {
    if (tile == 0) BH_F8_RING(FULL, 4, 4, 2, 2, 2, false, 8, 8);
    else if (tile == 1) BH_F8_RING(FULL, 4, 4, 4, 2, 3, false, 8, 4);
    else if (tile == 5) BH_F8_RING(FULL, 2, 2, 2, 2, 3, false, 8, 8);
    else if (tile == 6) BH_F8_RING(FULL, 1, 2, 2, 2, 4, false, 8, 8);
  }
#undef BH_F8_RING
}

template <typename TC, bool GATED, bool FULL>
void launch_plan(const F8RingPlan& plan, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, TC* c, float* sums, int accumulate, int M, int ldc,
                 GateForm form, hipStream_t stream) {
  if (plan.parts == 1) launch<TC, GATED, FULL, false>(plan.tile, 1, a, exponents, w, c, nullptr, accumulate, M, ldc, form, stream);
  else launch<float, GATED, FULL, true>(plan.tile, plan.parts, a, exponents, w, sums, nullptr, 0, M, ldc, form, stream);
}

}  // namespace

F8RingPlan float8_ring_plan(int M, int N, int K, bool gated, bool full, bool in_stretches) {
  F8RingPlan plan = {0, 1, 0.};
  const int W = gated ? 2 * N : N, stretches = (K + F8_K - 1) / F8_K;
  for (int tile = 0; tile < TILES; ++tile) {
    if (tile == 2 && full) continue;      // (full sums have no registers for it)
    if (in_stretches && SHAPES[tile].columns != 2 * F8_K) continue;
    const long tiles = (long)((M + SHAPES[tile].rows - 1) / SHAPES[tile].rows) * ((W + SHAPES[tile].columns - 1) / SHAPES[tile].columns);
    const int most = tile == 2 || in_stretches || M > 65535 || tiles >= 2L * bh_compute_units() ? 1 : MOST_PARTS;
    for (int parts = 1; parts <= most && (parts == 1 || stretches >= 4 * parts); ++parts) {
      const double cost = cost_us(tile, parts, M, W, K, full);
      if (plan.us == 0. || cost < plan.us) plan = {tile, parts, cost};
    }
  }
  return plan;
}

int float8_ring_launch(const F8RingPlan& plan, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, void* c, int c_dtype, float* sums, int accumulate,
                       int M, int ldc, int gated, int full, GateForm form, hipStream_t stream) {
#define BH_F8_RUN(TC, GATED, FULL) launch_plan<TC, GATED, FULL>(plan, a, exponents, w, (TC*)c, sums, accumulate, M, ldc, form, stream)
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

// The outputs of a gated product in 8 bits, a tile's being a stretch.
int float8_ring_launch_in_8(const F8RingPlan& plan, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, uint8_t* c, uint8_t* c_exponents, int through_bf16,
                            int M, int full, GateForm form, hipStream_t stream) {
  if (full) launch<uint8_t, true, true, false>(plan.tile, 1, a, exponents, w, c, c_exponents, through_bf16, M, w.rows, form, stream);
  else launch<uint8_t, true, false, false>(plan.tile, 1, a, exponents, w, c, c_exponents, through_bf16, M, w.rows, form, stream);
  return bh_check_launch("float8_ring_in_8");
}
