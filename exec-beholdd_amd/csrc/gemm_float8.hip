// Matrix products with weights and activations in 8 bits (float8.h): C[M, N] (+)= x[M, K] * W[N, K]^T, plain or gated.
//   few     up to 16 rows straight from bfloat16 or float32 rows (a wave quantises the stretch it multiplies), up to 128 from rows in 8 bits where
//           an estimate says so
//   rings   more rows (gemm_float8_ring.hip), K in parts where the tiles alone leave compute units idle, and their sum
#include "float8_few.h"
#include "gemm_float8_ring.h"

namespace {

// ---- a few rows ------------------------------------------------------------------------------------------------
// Bound by reading W once, and for small W by the chain of a launch.  A workgroup owns `span` weight rows (gated: 16 pairs of gate and up);
// its eight waves take the stretches of k in turn, each with DEPTH of them on their way, and quantise the rows' stretch themselves (16 values
// a lane and half an operand, the largest of a stretch found between the four lanes of a row), or, from 17 rows on, read it in 8 bits.  The
// waves' sums are added through LDS in a fixed order.
// `span` is 16, a block of the layout; 24 where blocks of 16 are more than the compute units and fewer than twice as many, which would
// leave some with two blocks and the others with one; 8 where they are half of the compute units or fewer.
constexpr int FEW_WAVES = 8;

// grid (ceil(rows of W / span)).  MB: blocks of 16 rows.  NB: blocks of W that a span touches; MASKED: it is not the whole of one.  TC: the
// output's type.  T: the rows' type (uint8_t: in 8 bits, in blocks, with their exponents).
template <typename T, typename TC, int MB, int NB, bool GATED, bool FULL, int LOAD, bool MASKED, int DEPTH>
__global__ __launch_bounds__(FEW_WAVES * 64) void few_kernel(const T* __restrict__ x, const uint32_t* __restrict__ exponents, F8Weight w,
                                                             TC* __restrict__ c, int M, int K, int ldc, int accumulate, int span, GateForm form) {
  constexpr int TT = NB * (GATED ? 2 : 1);
  __shared__ float partial[FEW_WAVES][TT][MB][256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int i = lane % 16, q = lane / 16, blocks = w.blocks(), stretches = w.stretches, left = (stretches - wave + FEW_WAVES - 1) / FEW_WAVES;
  const int first_row = (int)blockIdx.x * span, first_block = first_row / 16;
  int lo[NB], hi[NB];      // the rows of each block that this workgroup owns
  int place[NB];           // a lane's place in it: where it has no row of its own that of the nearest, which brings no line more and is not stored
  const uint8_t* wp[TT];
  const float* ws[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int block = min(first_block + t % NB, blocks - 1), matrix = t / NB;      // (one beyond the last repeats it)
    wp[t] = w.data + ((size_t)matrix * blocks + block) * stretches * F8_BLOCK;
    ws[t] = w.scales + ((size_t)matrix * w.scale_rows() + block / 8) * stretches;
  }
#pragma unroll
  for (int t = 0; t < NB; ++t) {
    const int row = (first_block + t) * 16;
    lo[t] = MASKED ? max(first_row - row, 0) : 0;
    hi[t] = MASKED ? min(min(first_row + span, w.rows) - row, 16) : 16;
    place[t] = 16 * (MASKED ? 16 * q + max(min(i, hi[t] - 1), min(lo[t], 15)) : lane);
  }
  f8_f32x4_t acc[TT][MB];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[t][b] = f8_f32x4_t{0.f, 0.f, 0.f, 0.f};
  f8_u32x4_t wv[DEPTH][TT][2];
  float wsv[DEPTH][TT];
  F8Stretch<T> xv[DEPTH][MB];
  auto ask = [&](int u, int n) {      // the wave's n-th stretch
    const int j = wave + n * FEW_WAVES;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      if constexpr (sizeof(T) == 1) {
        const int row_blocks = (M + 15) / 16, block = min(b, row_blocks - 1);
        const f8_u32x4_t* from = reinterpret_cast<const f8_u32x4_t*>(x + ((size_t)block * stretches + j) * F8_BLOCK + lane * 16);
        xv[u][b].v[0] = from[0], xv[u][b].v[1] = from[64];
        xv[u][b].exponent = (exponents[(size_t)(j / 4) * (row_blocks * 16) + block * 16 + i] >> (8 * (j % 4))) & 0xffu;
      } else {
        f8_load_stretch<T, LOAD>(xv[u][b], x + (size_t)min(b * 16 + i, M - 1) * K, b * 16 + i < M, j * F8_K + 16 * q, K);
      }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const f8_u32x4_t* from = reinterpret_cast<const f8_u32x4_t*>(wp[t] + (size_t)j * F8_BLOCK + place[t % NB]);
      wv[u][t][0] = __builtin_nontemporal_load(from);
      wv[u][t][1] = __builtin_nontemporal_load(from + 64);
      wsv[u][t] = ws[t][j];
    }
  };
  auto multiply = [&](int u) {
    F8Operand<FULL> wo[TT], xo;
#pragma unroll
    for (int t = 0; t < TT; ++t) wo[t].set(f8_operand(wv[u][t][0], wv[u][t][1]));
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      float xs;
      xo.set(xv[u][b].quantised(&xs));
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const f8_f32x4_t sum = f8_stretch(wo[t], xo);
        const float s = xs * wsv[u][t];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][b][e] = fmaf(sum[e], s, acc[t][b][e]);
      }
    }
  };
#pragma unroll
  for (int u = 0; u < DEPTH; ++u)
    if (u < left) ask(u, u);
  for (int n = 0; n < left; n += DEPTH)
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (n + u < left) {
        multiply(u);
        if (n + u + DEPTH < left) ask(u, n + u + DEPTH);
      }
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b) *reinterpret_cast<f8_f32x4_t*>(&partial[wave][t][b][i * 16 + 4 * q]) = acc[t][b];
  __syncthreads();
  for (int e = threadIdx.x; e < MB * 256; e += FEW_WAVES * 64) {
    const int b = e / 256, m = b * 16 + (e % 256) / 16, column = e % 16;
    if (m >= M) continue;
#pragma unroll
    for (int t = 0; t < NB; ++t) {
      const int n = (first_block + t) * 16 + column;
      if (n >= w.rows || column < lo[t] || column >= hi[t]) continue;
      float sum[GATED ? 2 : 1];
#pragma unroll
      for (int g = 0; g < (GATED ? 2 : 1); ++g) {
        sum[g] = 0.f;
#pragma unroll
        for (int v = 0; v < FEW_WAVES; ++v) sum[g] += partial[v][g * NB + t][b][e % 256];
      }
      TC* at = c + (size_t)m * ldc + n;
      float value = GATED ? f8_gate_out<TC>(sum[0], sum[GATED ? 1 : 0], form) : sum[0];
      if (accumulate) value += to_f32(*at);
      *at = from_f32<TC>(value);
    }
  }
}

// ---- K in parts ------------------------------------------------------------------------------------------------
// The parts' sums in their order.  grid (ceil(N / 256), M).
template <typename TC, bool GATED>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ sums, TC* __restrict__ c, int parts, int N, int ldc, int accumulate,
                                                     GateForm form) {
  const int n = blockIdx.x * 256 + threadIdx.x, row = blockIdx.y, M = gridDim.y, width = GATED ? 2 * N : N;
  if (n >= N) return;
  float sum[GATED ? 2 : 1];
#pragma unroll
  for (int g = 0; g < (GATED ? 2 : 1); ++g) {
    sum[g] = 0.f;
    for (int p = 0; p < parts; ++p) sum[g] += sums[((size_t)p * M + row) * width + g * N + n];
  }
  TC* at = c + (size_t)row * ldc + n;
  float value = GATED ? f8_gate_out<TC>(sum[0], sum[GATED ? 1 : 0], form) : sum[0];
  if (accumulate) value += to_f32(*at);
  *at = from_f32<TC>(value);
}

// ---- which kernel ----------------------------------------------------------------------------------------------
constexpr int FEW_ROWS = 16, FEW_ROWS_ALWAYS = 48, FEW_ROWS_IN_8 = 128;      // `few`: the most rows as they are, in 8 bits always, and by an estimate
// (Steps of a model of 8 layers of 4,096 and 12,288 with rows as they are / in 8 bits, us: 17 sequences 791 / 732, 32 970 / 772: every workgroup quantises all rows.)

int span_of(int N, int K, bool gated) {
  if (gated) return 16;
  const int blocks = (N + 15) / 16, units = bh_compute_units();
  if (2 * blocks <= units && K >= 1536) return 8;
  if (blocks > units && blocks < 2 * units && (N + 23) / 24 <= units) return 24;
  return 16;
}

// The span that `few` runs with.  Plain bfloat16 rows and rows in 8 bits have other spans than 16 (float32 rows go in whole blocks: they are not what
// a step of few rows has as a rule).
int few_span(int N, int K, bool gated, size_t row_element, int load) {
  return row_element <= 2 && load == F8_EVEN ? span_of(N, K, gated) : 16;
}

// Blocks of 16 rows that the kernel for M rows is compiled for.
int few_row_blocks(int M) { return M <= 32 ? 2 : M <= 48 ? 3 : M <= 64 ? 4 : M <= 96 ? 6 : 8; }

// What `few` is estimated to take from rows in 8 bits (us): a start, and for a wave's every stretch the weights and the blocks of rows, which every
// workgroup reads whole from the L2.  From the times that SHAPES of gemm_float8_ring.hip comes from (64 rows of 1,333 x 1,000 4.7, on the rings 6.4; 128 rows of 4,096 x
// 4,096 12.1 and 10.6; 64 of 4,096 x 12,288 26.5 and 15.7).
double few_cost_us(int M, int N, int K, bool gated, bool full) {
  constexpr double STRETCH[2][3] = {{1.386, 1.800, 2.072}, {1.814, 2.243, 2.334}};      // of 4, 6 and 8 blocks of rows
  const int span = span_of(N, K, gated), stretches = (K + F8_K - 1) / F8_K;
  const double loads = (double)((N + span - 1) / span) * (gated ? 2. : span == 24 ? 1.5 : 1.) / bh_compute_units();
  const double walk = (stretches + FEW_WAVES - 1) / FEW_WAVES * (loads > 1. ? loads : 1.) * STRETCH[full][few_row_blocks(M) / 2 - 2];
  const double read = (double)(gated ? 2 : 1) * N * K / 4.47e6;
  return 3.2 + (walk > read ? walk : read);
}

// Whether a product from rows in 8 bits goes through `few`; else the rings' plan.  Up to 48 rows it does: weights that come from memory, and not from the
// caches as in the times behind the estimates, reach it sooner (steps of a model of 8 layers of 4,096 and 12,288, us, with the estimates alone / so: 32 rows 787 /
// 772, 40 978 / 931, 48 967 / 928; the other way round from there on, 64 rows 1,064 by the estimates, 1,080 through `few`, 128 rows 1,409 and 1,500).
bool few_takes(int M, int N, int K, bool gated, bool full, F8RingPlan* plan) {
  if (M <= FEW_ROWS_ALWAYS) return true;
  *plan = float8_ring_plan(M, N, K, gated, full);
  return M <= FEW_ROWS_IN_8 && few_cost_us(M, N, K, gated, full) <= plan->us;
}

template <typename T, typename TC, bool GATED, bool FULL, int MB>
void launch_few_blocks(const void* x, const uint32_t* exponents, const F8Weight& w, TC* c, int M, int K, int ldc, int accumulate, GateForm form, hipStream_t stream) {
  const int load = sizeof(T) == 1 ? (int)F8_EVEN : f8_load_of(x, K);
  constexpr bool SPANS = sizeof(T) <= 2 && !GATED;
  const int span = few_span(w.rows, K, GATED, sizeof(T), load);
  const dim3 grid((w.rows + span - 1) / span);
#define BH_F8_FEW(NB, LOAD, MASKED, DEPTH)                                                                                            \
  few_kernel<T, TC, MB, NB, GATED, FULL, LOAD, MASKED, DEPTH><<<grid, FEW_WAVES * 64, 0, stream>>>((const T*)x, exponents, w, c, M, K, \
                                                                                                   ldc, accumulate, span, form)
  constexpr int DEPTH = MB == 1 && !GATED ? 4 : MB <= 2 && sizeof(T) <= 2 ? 3 : MB <= 6 ? 2 : 1;
  if constexpr (SPANS) {
    if (span == 8) {
      BH_F8_FEW(1, F8_EVEN, true, DEPTH);
      return;
    }
    if (span == 24) {
      BH_F8_FEW(2, F8_EVEN, true, (MB == 1 ? 4 : MB <= 4 ? 2 : 1));
      return;
    }
  }
  if (load == F8_EVEN) BH_F8_FEW(1, F8_EVEN, false, DEPTH);
  else if constexpr (sizeof(T) != 1) {
    if (load == F8_PIECES) BH_F8_FEW(1, F8_PIECES, false, 2);
    else BH_F8_FEW(1, F8_VALUES, false, 2);
  }
#undef BH_F8_FEW
}

template <typename T, typename TC, bool GATED, bool FULL>
void launch_few(const void* x, const uint32_t* exponents, const F8Weight& w, TC* c, int M, int K, int ldc, int accumulate, GateForm form, hipStream_t stream) {
#define BH_F8_FEW(MB) launch_few_blocks<T, TC, GATED, FULL, MB>(x, exponents, w, c, M, K, ldc, accumulate, form, stream)
  if constexpr (sizeof(T) == 1) {
    const int row_blocks = few_row_blocks(M);
    if (row_blocks <= 2) BH_F8_FEW(2);
    else if (row_blocks == 3) BH_F8_FEW(3);
    else if (row_blocks == 4) BH_F8_FEW(4);
    else if (row_blocks == 6) BH_F8_FEW(6);
    else BH_F8_FEW(8);
  } else {
    BH_F8_FEW(1);
  }
#undef BH_F8_FEW
}

int fault_of(const void* w, const void* scales, const void* c, int c_dtype, int M, int N, int K, int ldc, int gate) {
  BH_REQUIRE(M > 0 && N > 0 && K > 0, "gemm_float8: sizes must be positive, got %d x %d x %d", M, N, K);
  BH_REQUIRE(K <= (1 << 24) && N <= (1 << 24) && ldc >= N, "gemm_float8: a product of %d outputs of %d inputs, rows %d apart", N, K, ldc);
  BH_REQUIRE((uintptr_t)w % 16 == 0 && scales != nullptr && c != nullptr, "gemm_float8: the weight must be 16-byte aligned");
  BH_REQUIRE(c_dtype == BH_F32 || c_dtype == BH_BF16, "gemm_float8: unknown output dtype %d", c_dtype);
  BH_REQUIRE(gate == 0 || gate == BH_GATE_SILU || gate == BH_GATE_GELU_TANH, "gemm_float8: unknown gate %d", gate);
  return 0;
}

}  // namespace

// Up to so many rows a product takes them as they are (`few`); more are brought into 8 bits first.
extern "C" int bh_gemm_float8_few_rows() { return FEW_ROWS; }
// Bytes of scratch memory of a product from rows in 8 bits.
extern "C" long bh_gemm_float8_scratch(int M, int N, int K, int gated, int full) {
  F8RingPlan plan;
  if (M <= 0 || N <= 0 || K <= 0 || few_takes(M, N, K, gated != 0, full != 0, &plan)) return 0;
  return plan.parts > 1 ? (long)plan.parts * M * N * (gated ? 2 : 1) * 4 : 0;
}

// Which kernel a product runs on, from rows of `dtype` on addresses of 16 bytes or (dtype -1) in 8 bits: kernel[0] blocks of 16 rows that `few` is
// compiled for and kernel[1] its span, or 0 and 0; kernel[2] the rings' tile and kernel[3] its parts, or -1 and 0.
extern "C" int bh_gemm_float8_kernel(int dtype, int M, int N, int K, int gated, int full, int* kernel) {
  BH_REQUIRE(M > 0 && N > 0 && K > 0 && kernel != nullptr, "gemm_float8: sizes must be positive, got %d x %d x %d", M, N, K);
  F8RingPlan plan = {-1, 0, 0.};
  const bool plain = dtype >= 0 && M <= FEW_ROWS, few = plain || few_takes(M, N, K, gated != 0, full != 0, &plan);
  kernel[0] = plain ? 1 : few ? few_row_blocks(M) : 0;
  kernel[1] = !few ? 0 : few_span(N, K, gated != 0, plain ? (dtype == BH_F32 ? 4 : 2) : 1, plain ? f8_load_of(nullptr, K) : F8_EVEN);
  kernel[2] = few ? -1 : plan.tile;
  kernel[3] = few ? 0 : plan.parts;
  return 0;
}

#define BH_F8_BY_TYPES(RUN)                                                                                        \
  do {                                                                                                             \
    if (gate) {                                                                                                    \
      if (c_dtype == BH_F32) { if (full) RUN(float, true, true); else RUN(float, true, false); }                   \
      else { if (full) RUN(bf16_t, true, true); else RUN(bf16_t, true, false); }                                   \
    } else if (c_dtype == BH_F32) { if (full) RUN(float, false, true); else RUN(float, false, false); }            \
    else { if (full) RUN(bf16_t, false, true); else RUN(bf16_t, false, false); }                                   \
  } while (0)

// N: the outputs; of a gated product `w` holds two matrices of N rows, gate then up.  ldc: elements from a row of C to the next.
extern "C" int bh_gemm_float8_few(const void* x, int dtype, const void* w, const void* scales, void* c, int c_dtype, int accumulate, int M, int N,
                                  int K, int ldc, int gate, int full, hipStream_t stream) {
  if (const int fault = fault_of(w, scales, c, c_dtype, M, N, K, ldc, gate)) return fault;
  BH_REQUIRE(M <= FEW_ROWS, "gemm_float8_few: up to %d rows, got %d", FEW_ROWS, M);
  BH_REQUIRE(dtype == BH_F32 || dtype == BH_BF16, "gemm_float8_few: unknown dtype %d", dtype);
  const F8Weight weight = {(const uint8_t*)w, (const float*)scales, N, (K + F8_K - 1) / F8_K};
  const GateForm form = bh_gate_form(gate);
#define BH_F8_RUN(TC, GATED, FULL)                                                                                     \
  do {                                                                                                                 \
    if (dtype == BH_F32) launch_few<float, TC, GATED, FULL>(x, nullptr, weight, (TC*)c, M, K, ldc, accumulate, form, stream);   \
    else launch_few<bf16_t, TC, GATED, FULL>(x, nullptr, weight, (TC*)c, M, K, ldc, accumulate, form, stream);                  \
  } while (0)
  BH_F8_BY_TYPES(BH_F8_RUN);
#undef BH_F8_RUN
  return bh_check_launch("gemm_float8_few");
}

extern "C" int bh_gemm_float8(const void* a, const void* exponents, const void* w, const void* scales, void* c, int c_dtype, int accumulate, int M,
                              int N, int K, int ldc, int gate, int full, void* scratch, hipStream_t stream) {
  if (const int fault = fault_of(w, scales, c, c_dtype, M, N, K, ldc, gate)) return fault;
  BH_REQUIRE(((uintptr_t)a | (uintptr_t)exponents) % 16 == 0, "gemm_float8: the rows must be 16-byte aligned");
  BH_REQUIRE((long)(M + 15) * ((K + 511) / 512) < (1L << 30), "gemm_float8: the exponents of %d rows of %d inputs do not lie within 4 GB", M, K);
  F8RingPlan plan;
  if (few_takes(M, N, K, gate != 0, full != 0, &plan)) {
    const F8Weight weight = {(const uint8_t*)w, (const float*)scales, N, (K + F8_K - 1) / F8_K};
    const GateForm form = bh_gate_form(gate);
#define BH_F8_RUN(TC, GATED, FULL) launch_few<uint8_t, TC, GATED, FULL>(a, (const uint32_t*)exponents, weight, (TC*)c, M, K, ldc, accumulate, form, stream)
    BH_F8_BY_TYPES(BH_F8_RUN);
#undef BH_F8_RUN
    return bh_check_launch("gemm_float8");
  }
  BH_REQUIRE(plan.parts == 1 || (scratch != nullptr && (uintptr_t)scratch % 16 == 0), "gemm_float8: a product in %d parts needs scratch memory", plan.parts);
  const F8Weight weight = {(const uint8_t*)w, (const float*)scales, N, (K + F8_K - 1) / F8_K};
  const GateForm form = bh_gate_form(gate);
  const int status = float8_ring_launch(plan, (const uint8_t*)a, (const uint32_t*)exponents, weight, c, c_dtype, (float*)scratch, accumulate, M, ldc, gate != 0, full,
                                        form, stream);
  if (status != 0 || plan.parts == 1) return status;
  const dim3 grid((N + 255) / 256, M);
  if (c_dtype == BH_F32) {
    if (gate) finish_kernel<float, true><<<grid, 256, 0, stream>>>((const float*)scratch, (float*)c, plan.parts, N, ldc, accumulate, form);
    else finish_kernel<float, false><<<grid, 256, 0, stream>>>((const float*)scratch, (float*)c, plan.parts, N, ldc, accumulate, form);
  } else if (gate) finish_kernel<bf16_t, true><<<grid, 256, 0, stream>>>((const float*)scratch, (bf16_t*)c, plan.parts, N, ldc, accumulate, form);
  else finish_kernel<bf16_t, false><<<grid, 256, 0, stream>>>((const float*)scratch, (bf16_t*)c, plan.parts, N, ldc, accumulate, form);
  return bh_check_launch("gemm_float8");
}

namespace {
long rounded(long bytes) { return (bytes + 511) / 512 * 512; }
long rows_bytes(int M, int K) { return rounded((M + 15L) / 16 * ((K + F8_K - 1) / F8_K) * F8_BLOCK); }
long exponents_bytes(int M, int K) { return rounded((M + 15L) / 16 * 16 * ((K + 511) / 512) * 4); }
}  // namespace

// The same from rows as they are, through their 8 bits in `working`: so many bytes.
extern "C" long bh_gemm_float8_working(int M, int N, int K, int gated, int full) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return rows_bytes(M, K) + exponents_bytes(M, K) + bh_gemm_float8_scratch(M, N, K, gated, full);
}
// x: null where `working` holds the rows in 8 bits already, from a product before with the same rows.
extern "C" int bh_gemm_float8_rows(const void* x, int dtype, void* working, const void* w, const void* scales, void* c, int c_dtype, int accumulate, int M,
                                   int N, int K, int ldc, int gate, int full, hipStream_t stream) {
  if (const int fault = fault_of(w, scales, c, c_dtype, M, N, K, ldc, gate)) return fault;
  BH_REQUIRE(working != nullptr && (uintptr_t)working % 16 == 0, "gemm_float8: rows in 8 bits need working memory");
  uint8_t* data = (uint8_t*)working;
  uint8_t* exponents = data + rows_bytes(M, K);
  if (x != nullptr) {
    if (const int status = float8_rows_launch(x, dtype, data, (uint32_t*)exponents, M, K, 0, 0, stream)) return status;
  }
  return bh_gemm_float8(data, exponents, w, scales, c, c_dtype, accumulate, M, N, K, ldc, gate, full, exponents + exponents_bytes(M, K), stream);
}

// Whether a gated product leaves its outputs in 8 bits itself: where its tiles take no longer than others and what would bring the outputs into 8 bits then, a
// launch and a pass over the outputs (so / in two, us, 2 x 12,288 x 4,096: 128 rows 23.9 / 27.3, 512 57.6 / 60.2, 2,048 185 / 201, 8,192 756 / 801; fewer rows are
// faster in two when weights come from memory, steps of 64 sequences of 8 such layers 1,068 / 1,019).
extern "C" int bh_gemm_float8_gives_8(int M, int N, int K, int full) {
  if (M < FEW_ROWS_IN_8 || N <= 0 || K <= 0) return 0;
  return float8_ring_plan(M, N, K, true, full != 0, true).us <= float8_ring_plan(M, N, K, true, full != 0).us + 2.5 + (double)M * N / 2.2e6;
}
// A gated product from rows in 8 bits to rows in 8 bits, both in blocks: N outputs, of matrices of N gate and N up rows.
extern "C" int bh_gemm_float8_gated_to_8(const void* a, const void* exponents, const void* w, const void* scales, void* c, void* c_exponents, int through_bf16,
                                         int M, int N, int K, int gate, int full, hipStream_t stream) {
  if (const int fault = fault_of(w, scales, c, BH_F32, M, N, K, N, gate)) return fault;
  BH_REQUIRE(gate != 0 && M >= FEW_ROWS_IN_8, "gemm_float8: gated products of %d rows or more give rows in 8 bits", FEW_ROWS_IN_8);
  BH_REQUIRE(((uintptr_t)a | (uintptr_t)exponents | (uintptr_t)c | (uintptr_t)c_exponents) % 16 == 0, "gemm_float8: the rows must be 16-byte aligned");
  BH_REQUIRE((long)(M + 15) * ((K + 511) / 512) < (1L << 30), "gemm_float8: the exponents of %d rows of %d inputs do not lie within 4 GB", M, K);
  const F8Weight weight = {(const uint8_t*)w, (const float*)scales, N, (K + F8_K - 1) / F8_K};
  return float8_ring_launch_in_8(float8_ring_plan(M, N, K, true, full != 0, true), (const uint8_t*)a, (const uint32_t*)exponents, weight, (uint8_t*)c,
                                 (uint8_t*)c_exponents, through_bf16, M, full, bh_gate_form(gate), stream);
}
