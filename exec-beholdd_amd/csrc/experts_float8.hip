// Routed experts whose matrices are kept in 8 bits (float8.h): for every (row, choice) pair p = row * top + j and its expert e = chosen[p]
//   inner[p] = act(Wg_e x[row], Wu_e x[row])     act(g, u) = g' / (1 + exp(-alpha g')) * (u' + shift), g' = min(g, limit), u' = clamp(u, +-limit)
//   y[p]     = Wd_e inner[p]                     inner in 32 bits, brought into 8 once
//   out[row] (+)= sum over j of weight[p] * y[p], j in order
// A sum that is not a number stays one behind a finite limit, as it does without: its inner value becomes e4m3's NaN, and its row's outputs NaN.
// Gate and up are summed in full (float8.h): they are rounded to 8 bits next, where each that falls on the other side of a border is a whole step off
// (4,096 rows of 4,096 to bfloat16: 2.6e-3 of the result with the 8-bit instruction's sums, 1.7e-3 so, of which 1.6e-3 are the output's own rounding).
// A pair's weight may multiply the expert's input instead (its gate and up sums).  A pair whose expert is none of the E gives nothing, or,
// with `through`, one numbered E or higher hands the row's input on.  Nothing here depends on the routing on the host.
//   one    the pairs of one row
//   few    an expert's pairs 16 at a time, brought into 8 bits by the workgroup that multiplies them
//   tiles  tiles of 64 or 128 pairs of an expert from rows in 8 bits, found from the experts' counts by every workgroup itself
#include "float8_few.h"
#include "float8_ring.h"

namespace {

struct ExpertGate {
  float limit, alpha, shift;
};
__device__ inline float activated(float g, float u, const ExpertGate& gate) {
  g = held_below(g, gate.limit);
  u = held_between(u, gate.limit);
  return f8_gated(g, gate.alpha * g) * (u + gate.shift);
}

// ---- few -------------------------------------------------------------------------------------------------------
// Bound by reading the matrices of the experts that have pairs.  A workgroup is one expert's and owns 8 / KS blocks of 16 outputs (gated: of
// gate and up rows); KS waves share a block and take its stretches of k in turn, their sums added through LDS in a fixed order.  The rows of
// up to 16 of the expert's pairs are brought into 8 bits once for the workgroup and kept in LDS, F8_SEGMENT stretches of k at a time, while
// the first weights are on their way.
constexpr int FEW_WAVES = 8, FEW_PAIRS = 1024;      // pairs of a call at most
constexpr int FEW_TOP = 32;                         // pairs of a row alone, at most
constexpr int SEGMENT = 32;                         // stretches of the rows that LDS holds

// grid (ceil(blocks / (8 / KS)), min(pairs, E)).  With at most E pairs a workgroup is a pair's, and the first pair of an expert does all of
// that expert's; otherwise it is an expert's.  The list of the expert's pairs is made here, in their order.
template <typename T, bool GATED, bool FULL, int LOAD, int KS, int DEPTH>
__global__ __launch_bounds__(FEW_WAVES * 64) void experts_few_kernel(const T* __restrict__ in, int in_div, const int32_t* __restrict__ chosen, int pairs,
                                                                    int E, F8Weight w, float* __restrict__ out, int K, ExpertGate gate,
                                                                    const float* __restrict__ in_weights) {
  constexpr int TT = GATED ? 2 : 1, OWN = FEW_WAVES / KS;
  extern __shared__ __attribute__((aligned(16))) f8_u32x4_t rows8[];      // [stretch of the segment][half][lane], then a scale for each stretch and row
  __shared__ float partial[KS > 1 ? FEW_WAVES : 1][TT][256];
  __shared__ int mine[FEW_PAIRS];
  __shared__ int of_wave[FEW_WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, i = lane % 16, q = lane / 16;
  const int expert = pairs <= E ? chosen[blockIdx.y] : (int)blockIdx.y;
  if (expert < 0 || expert >= E) return;      // the whole workgroup
  const int blocks = w.blocks(), stretches = w.stretches, block = (int)blockIdx.x * OWN + wave / KS, share = wave % KS;
  const uint8_t* wp[TT];
  const float* ws[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const size_t matrix = (size_t)expert * TT + t;
    const int b = min(block, blocks - 1);      // (one beyond the last repeats it and stores nothing)
    wp[t] = w.data + (matrix * blocks + b) * stretches * F8_BLOCK + lane * 16;
    ws[t] = w.scales + (matrix * w.scale_rows() + b / 8) * stretches;
  }
  f8_u32x4_t wv[DEPTH][TT][2];
  float wsv[DEPTH][TT];
  auto ask = [&](int u, int j) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const f8_u32x4_t* from = reinterpret_cast<const f8_u32x4_t*>(wp[t] + (size_t)j * F8_BLOCK);
      wv[u][t][0] = from[0], wv[u][t][1] = from[64];
      wsv[u][t] = ws[t][j];
    }
  };
  auto ask_first = [&](int j0) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (share + u * KS < min(stretches - j0, SEGMENT)) ask(u, j0 + share + u * KS);
  };
  ask_first(0);      // (the pairs are found while they are on their way)
  // the pairs in pieces of 64, FEW_PAIRS / 512 neighbouring pieces a wave
  constexpr int PIECES = FEW_PAIRS / 64 / FEW_WAVES;
  unsigned long long masks[PIECES];
  int own = 0;
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    const int p = (wave * PIECES + u) * 64 + lane;
    masks[u] = __ballot(p < pairs && chosen[min(p, pairs - 1)] == expert);
    own += __popcll(masks[u]);
  }
  if (lane == 0) of_wave[wave] = own;
  __syncthreads();
  int count = 0, at = 0;
#pragma unroll
  for (int v = 0; v < FEW_WAVES; ++v) {
    if (v < wave) at += of_wave[v];
    count += of_wave[v];
  }
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    if (masks[u] >> lane & 1ull) mine[at + __popcll(masks[u] & ((1ull << lane) - 1ull))] = (wave * PIECES + u) * 64 + lane;
    at += __popcll(masks[u]);
  }
  __syncthreads();
  if (count == 0 || (pairs <= E && mine[0] != (int)blockIdx.y)) return;

  const int segment = min(stretches, SEGMENT);
  float* const scales8 = reinterpret_cast<float*>(rows8 + segment * 128);
  for (int p0 = 0; p0 < count; p0 += 16) {
    const T* row = in + (size_t)(mine[min(p0 + i, count - 1)] / in_div) * K;
    f8_f32x4_t acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = f8_f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < stretches; j0 += SEGMENT) {
      const int here = min(stretches - j0, SEGMENT), left = (here - share + KS - 1) / KS;
      if (p0 || j0) {
        ask_first(j0);
        __syncthreads();      // everyone has read what stood there
      }
      for (int j = wave; j < here; j += FEW_WAVES) {
        F8Stretch<T> x;
        f8_load_stretch<T, LOAD>(x, row, true, (j0 + j) * F8_K + 16 * q, K);
        float scale;
        const f8_operand_t v = x.quantised(&scale);
        rows8[j * 128 + lane] = f8_u32x4_t{(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
        rows8[j * 128 + 64 + lane] = f8_u32x4_t{(uint32_t)v[4], (uint32_t)v[5], (uint32_t)v[6], (uint32_t)v[7]};
        if (q == 0) scales8[j * 16 + i] = scale;
      }
      __syncthreads();
      for (int n = 0; n < left; n += DEPTH)
#pragma unroll
        for (int u = 0; u < DEPTH; ++u)
          if (n + u < left) {
            const int j = share + (n + u) * KS;
            F8Operand<FULL> xo, wo;
            xo.set(f8_operand(rows8[j * 128 + lane], rows8[j * 128 + 64 + lane]));
            const float xs = scales8[j * 16 + i];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
              wo.set(f8_operand(wv[u][t][0], wv[u][t][1]));
              const f8_f32x4_t sum = f8_stretch(wo, xo);
              const float s = xs * wsv[u][t];
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(sum[e], s, acc[t][e]);
            }
            if (n + u + DEPTH < left) ask(u, j0 + j + DEPTH * KS);
          }
    }
    if constexpr (KS > 1) {
      __syncthreads();      // (the sums of the pairs before have been read)
#pragma unroll
      for (int t = 0; t < TT; ++t) *reinterpret_cast<f8_f32x4_t*>(&partial[wave][t][i * 16 + 4 * q]) = acc[t];
      __syncthreads();
    }
    if (share == 0 && block < blocks && p0 + i < count) {
      const int pair = mine[p0 + i];
      if constexpr (KS > 1) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
          for (int v = 1; v < KS; ++v) acc[t] += *reinterpret_cast<const f8_f32x4_t*>(&partial[wave + v][t][i * 16 + 4 * q]);
      }
      float v[4];
      const float wgt = GATED && in_weights ? in_weights[pair] : 1.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = GATED ? activated(acc[0][e] * wgt, acc[TT - 1][e] * wgt, gate) : acc[0][e];
      const int n = block * 16 + 4 * q;
      float* to = out + (size_t)pair * w.rows + n;
      if (w.rows % 4 == 0) {
        if (n < w.rows) store_four(to, v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < w.rows) to[e] = v[e];
      }
    }
  }
}

// ---- one row ---------------------------------------------------------------------------------------------------
// A step of one row is two trips to memory in a row (the choice, then the matrices) twice over: both products as short as that chain.
// The first product: a workgroup owns 16 outputs of a pair, its eight waves take the stretches of k in turn and bring the row into 8 bits
// themselves; the row does not wait for the choice.  grid (ceil(N / 16), top).  (As one of the workgroups of `few`, which look for the pairs of
// their expert first and keep its rows in LDS, 25 MB took 13.2 us, 8.0 so.)
template <typename T, int LOAD>
__global__ __launch_bounds__(FEW_WAVES * 64) void experts_one_kernel(const T* __restrict__ row, const int32_t* __restrict__ chosen, int E, F8Weight w,
                                                                    float* __restrict__ out, int K, ExpertGate gate, const float* __restrict__ in_weights) {
  constexpr int DEPTH = 2;
  __shared__ __attribute__((aligned(16))) float partial[FEW_WAVES][2][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, i = lane % 16, q = lane / 16;
  const int pair = blockIdx.y, block = blockIdx.x, blocks = w.blocks(), stretches = w.stretches, left = (stretches - wave + FEW_WAVES - 1) / FEW_WAVES;
  F8Stretch<T> xv[DEPTH];
  auto ask_row = [&](int u, int n) { f8_load_stretch<T, LOAD>(xv[u], row, true, (wave + n * FEW_WAVES) * F8_K + 16 * q, K); };
#pragma unroll
  for (int u = 0; u < DEPTH; ++u)
    if (u < left) ask_row(u, u);
  const int expert = chosen[pair];
  if (expert < 0 || expert >= E) return;      // the whole workgroup
  const float wgt = in_weights ? in_weights[pair] : 1.0f;
  const uint8_t* wp[2];
  const float* ws[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const size_t matrix = 2 * (size_t)expert + t;
    wp[t] = w.data + (matrix * blocks + block) * stretches * F8_BLOCK + lane * 16;
    ws[t] = w.scales + (matrix * w.scale_rows() + block / 8) * stretches;
  }
  f8_u32x4_t wv[DEPTH][2][2];
  float wsv[DEPTH][2];
  auto ask = [&](int u, int n) {
    const int j = wave + n * FEW_WAVES;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f8_u32x4_t* from = reinterpret_cast<const f8_u32x4_t*>(wp[t] + (size_t)j * F8_BLOCK);
      wv[u][t][0] = __builtin_nontemporal_load(from);
      wv[u][t][1] = __builtin_nontemporal_load(from + 64);
      wsv[u][t] = ws[t][j];
    }
  };
  f8_f32x4_t acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int u = 0; u < DEPTH; ++u)
    if (u < left) ask(u, u);
  for (int n = 0; n < left; n += DEPTH)
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (n + u < left) {
        F8Operand<true> xo, wo;
        float xs;
        xo.set(xv[u].quantised(&xs));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          wo.set(f8_operand(wv[u][t][0], wv[u][t][1]));
          const f8_f32x4_t sum = f8_stretch(wo, xo);
          const float s = xs * wsv[u][t];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(sum[e], s, acc[t][e]);
        }
        if (n + u + DEPTH < left) ask_row(u, n + u + DEPTH), ask(u, n + u + DEPTH);
      }
  if (i == 0) {      // (all rows of the operand are the row)
#pragma unroll
    for (int t = 0; t < 2; ++t) *reinterpret_cast<f8_f32x4_t*>(&partial[wave][t][4 * q]) = acc[t];
  }
  __syncthreads();
  const int n = block * 16 + threadIdx.x;
  if (threadIdx.x >= 16 || n >= w.rows) return;
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int v = 0; v < FEW_WAVES; ++v)
#pragma unroll
    for (int t = 0; t < 2; ++t) sum[t] += partial[v][t][threadIdx.x];
  out[(size_t)pair * w.rows + n] = activated(sum[0] * wgt, sum[1] * wgt, gate);
}

// The second product with the sum over the pairs: a workgroup owns 8 outputs, its sixteen waves share the pairs out between them, several
// waves a pair where there are few, each with half a block of its expert's matrix.  grid (ceil(D / 8)).  in float32 [top][K].
constexpr int ONE_WAVES = 16;
template <typename T, typename TC, bool FULL, int LOAD>
__global__ __launch_bounds__(ONE_WAVES * 64) void experts_one_sum_kernel(const float* __restrict__ in, const int32_t* __restrict__ chosen,
                                                                        const float* __restrict__ weights, const T* __restrict__ through, int E, F8Weight w,
                                                                        TC* __restrict__ out, int K, int top, int fresh) {
  constexpr int DEPTH = 2;
  __shared__ __attribute__((aligned(16))) float shares[FEW_TOP][ONE_WAVES][8];      // [pair][wave of the pair][output]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, i = lane % 16, q = lane / 16;
  const int D = w.rows, first = blockIdx.x * 8, block = first / 16, stretches = w.stretches;
  const int split = top >= ONE_WAVES ? 1 : ONE_WAVES / top, part = wave % split, at_once = ONE_WAVES / split;      // waves of a pair; pairs at a time
  const int left = (stretches - part + split - 1) / split;
  for (int j = wave / split; j < top && wave < split * at_once; j += at_once) {
    const float* from = in + (size_t)j * K;
    F8Stretch<float> xv[DEPTH];
    auto ask_row = [&](int u, int n) { f8_load_stretch<float, LOAD>(xv[u], from, true, (part + n * split) * F8_K + 16 * q, K); };
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (u < left) ask_row(u, u);
    const int expert = chosen[j];
    if (expert < 0 || expert >= E) continue;      // the wave
    const uint8_t* wp = w.data + ((size_t)expert * w.blocks() + block) * stretches * F8_BLOCK + (q * 16 + first % 16 + i % 8) * 16;      // (each of its rows twice)
    const float* ws = w.scales + ((size_t)expert * w.scale_rows() + block / 8) * stretches;
    f8_f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    f8_u32x4_t wv[DEPTH][2];
    float wsv[DEPTH];
    auto ask = [&](int u, int n) {
      const int s = part + n * split;
      const f8_u32x4_t* at = reinterpret_cast<const f8_u32x4_t*>(wp + (size_t)s * F8_BLOCK);
      wv[u][0] = __builtin_nontemporal_load(at);
      wv[u][1] = __builtin_nontemporal_load(at + 64);
      wsv[u] = ws[s];
    };
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (u < left) ask(u, u);
    for (int n = 0; n < left; n += DEPTH)
#pragma unroll
      for (int u = 0; u < DEPTH; ++u)
        if (n + u < left) {
          F8Operand<FULL> xo, wo;
          float xs;
          xo.set(xv[u].quantised(&xs));
          wo.set(f8_operand(wv[u][0], wv[u][1]));
          const f8_f32x4_t sum = f8_stretch(wo, xo);
          const float s = xs * wsv[u];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(sum[e], s, acc[e]);
          if (n + u + DEPTH < left) ask_row(u, n + u + DEPTH), ask(u, n + u + DEPTH);
        }
    if (i == 0 && q < 2) *reinterpret_cast<f8_f32x4_t*>(&shares[j][part][4 * q]) = acc;
  }
  // lane j of the first wave knows pair j's expert and weight before the shares are there
  const int own = chosen[min(lane, top - 1)];
  const float own_weight = weights ? weights[min(lane, top - 1)] : 1.0f;
  __syncthreads();
  if (wave) return;
  const int d = first + lane;
  float total = 0.f;
  for (int j = 0; j < top; ++j) {
    const int e = __builtin_amdgcn_readlane(own, j);
    const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, own_weight), j));
    if (e < 0 || (e >= E && through == nullptr) || lane >= 8 || d >= D) continue;
    float y = 0.f;
    if (e >= E) y = to_f32(through[d]);
    else
      for (int v = 0; v < split; ++v) y += shares[j][v][lane];
    total = fmaf(f, y, total);
  }
  if (lane >= 8 || d >= D) return;
  out[d] = from_f32<TC>(fresh ? total : to_f32(out[d]) + total);
}

// How many waves share a block: enough workgroups for every compute unit to have one, whatever the pairs.
int few_shares(int pairs, int E, int N, int stretches) {
  const long blocks = (long)((N + 15) / 16) * (pairs < E ? pairs : E);      // if no expert is chosen twice
  int shares = 1;
  while (shares < 8 && 2 * shares <= stretches && blocks * shares / 8 < 2L * bh_compute_units()) shares *= 2;
  return shares;
}

template <typename T, bool GATED, bool FULL, int LOAD>
void launch_few(const T* in, int in_div, const int32_t* chosen, int pairs, int E, const F8Weight& w, float* out, int K, const ExpertGate& gate,
                const float* in_weights, hipStream_t stream) {
  const int shares = few_shares(pairs, E, w.rows, w.stretches), segment = w.stretches < SEGMENT ? w.stretches : SEGMENT;
  const dim3 grid((w.blocks() * shares + 7) / 8, pairs < E ? pairs : E);
  const size_t lds = (size_t)segment * (F8_BLOCK + 64);
#define BH_F8_EXPERTS(KS)                                                                                                                   \
  do {                                                                                                                                      \
    bh_allow_lds<experts_few_kernel<T, GATED, FULL, LOAD, KS, (GATED ? 3 : 4)>>(lds);                                                       \
    experts_few_kernel<T, GATED, FULL, LOAD, KS, (GATED ? 3 : 4)><<<grid, FEW_WAVES * 64, lds, stream>>>(in, in_div, chosen, pairs, E, w, out, K, \
                                                                                                        gate, in_weights);                  \
  } while (0)
  switch (shares) {
    case 1: BH_F8_EXPERTS(1); break;
    case 2: BH_F8_EXPERTS(2); break;
    case 4: BH_F8_EXPERTS(4); break;
    default: BH_F8_EXPERTS(8);
  }
#undef BH_F8_EXPERTS
}

// ---- tiles -----------------------------------------------------------------------------------------------------
// A workgroup of 2 x 4 waves owns 32 XB pairs of one expert and 256 of its weight rows (gated: gate and up rows of the same 128 outputs), on
// the ring of float8_ring.h with rows picked through the expert's list.  The gated form's 128 outputs are a stretch of the next product's
// k: they are brought into 8 bits here, a pair's largest found between the four waves that hold its row.
// XB is 4 from 48 pairs an expert on, where the last tile of an expert goes as one of 64 if it has no more (us, 128 experts of 2,048 x 768, as
// tiles of 64 / so: 40 pairs each 194 / 208, 48 221 / 218, 62 238 / 233; 64 pairs each with whole last tiles 258, so 234, 128 each 348 / 336).
// a: rows in 8 bits, row after row; the input of pair p is row p / in_div.  out: float32 [pairs][N]; gated: rows in 8 bits, row after row,
// and their exponents, `out_padded` words a row of them.
template <bool GATED, bool FULL, int XB>
using ExpertsRing = F8Ring<FULL, XB, 4, 2, 4, 3, GATED ? 2 : 1, false, true>;

// The tile of pairs p0 .. and of weight rows tile_n.  (`ring` is not restrict: walk's own is, and within another the compiler has LDS reads wait for
// the loads that are on their way to other places of the ring.)
template <bool GATED, bool FULL, int XB>
__device__ __forceinline__ void experts_ring_tile(f8_u32x4_t* ring, const uint8_t* __restrict__ a, const uint32_t* __restrict__ exponents, int padded,
                                                  int in_div, const int32_t* __restrict__ pairs, int expert, int count, int p0, int tile_n, const F8Weight& w,
                                                  void* __restrict__ out, uint8_t* __restrict__ out_exponents, int out_padded, const ExpertGate& gate,
                                                  const float* __restrict__ in_weights) {
  using Ring = ExpertsRing<GATED, FULL, XB>;
  constexpr int YB = Ring::YB, HALF = Ring::HALF, ROWS = Ring::ROWS, OUTS = Ring::OUTS, WN = Ring::WN;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN, wn = wave % WN;
  const int N = w.rows, steps = w.stretches, blocks = w.blocks();
  const uint8_t* from[Ring::EACH];
  uint32_t row_at[Ring::ROW_PARTS];
#pragma unroll
  for (int i = 0; i < Ring::A_EACH; ++i) {
    const int piece = wave * Ring::A_EACH + i;
    from[i] = a;
    row_at[i] = (uint32_t)(pairs[min(p0 + piece * 8 + lane / 8, count - 1)] / in_div) * (steps * F8_K) + 16 * ((lane % 8) ^ (lane / 8));
  }
#pragma unroll
  for (int i = 0; i < Ring::W_EACH; ++i) {
    const int piece = wave * Ring::W_EACH + i, b = piece / 2, column = b / YB, y = b % YB;
    const int block = min((tile_n * WN + column) * HALF + y % HALF, blocks - 1);
    from[Ring::A_EACH + i] = w.data + (((size_t)expert * Ring::G + y / HALF) * blocks + block) * steps * F8_BLOCK + piece % 2 * 1024;
  }
  uint32_t x_at[XB];
#pragma unroll
  for (int x = 0; x < XB; ++x) x_at[x] = pairs[min(p0 + (wm * XB + x) * 16 + lane % 16, count - 1)] / in_div;
  const float* ws[Ring::G];
#pragma unroll
  for (int g = 0; g < Ring::G; ++g)
    ws[g] = w.scales + (((size_t)expert * Ring::G + g) * w.scale_rows() + min((tile_n * WN + wn) * HALF, blocks - 1) / 8) * steps;
  f8_f32x4_t acc[XB][YB];
  Ring::walk(ring, from, row_at, F8_K, exponents, x_at, padded, ws, 0, steps, acc);

  int pair[XB];      // (read again: registers are short in the walk)
#pragma unroll
  for (int x = 0; x < XB; ++x) pair[x] = pairs[min(p0 + (wm * XB + x) * 16 + lane % 16, count - 1)];
  if constexpr (GATED) {
    uint32_t* largest = reinterpret_cast<uint32_t*>(ring);      // [wave column][row]
    __syncthreads();      // every wave has read its last step
#pragma unroll
    for (int x = 0; x < XB; ++x) {
      const float wgt = in_weights ? in_weights[pair[x]] : 1.0f;
      uint32_t most = 0;
#pragma unroll
      for (int y = 0; y < HALF; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = tile_n * OUTS + (wn * HALF + y) * 16 + 4 * (lane / 16) + e;
          const float v = activated(acc[x][y][e] * wgt, acc[x][y + HALF][e] * wgt, gate);
          acc[x][y][e] = n < N ? v : 0.f;
          most = f8_larger(most, acc[x][y][e]);
        }
      most = f8_largest_of_row(most);
      if (lane < 16) largest[wn * ROWS + (wm * XB + x) * 16 + lane] = most;
    }
    __syncthreads();
    const int out_stretches = (N + F8_K - 1) / F8_K;
#pragma unroll
    for (int x = 0; x < XB; ++x) {
      const int r = (wm * XB + x) * 16 + lane % 16;
      uint32_t most = largest[r];
#pragma unroll
      for (int column = 1; column < WN; ++column) most = max(most, largest[column * ROWS + r]);
      const uint32_t exponent = f8_exponent(most);
      if (p0 + r >= count) continue;
      uint8_t* row = reinterpret_cast<uint8_t*>(out) + ((size_t)pair[x] * out_stretches + tile_n) * F8_K;
#pragma unroll
      for (int y = 0; y < HALF; ++y)
        *reinterpret_cast<uint32_t*>(row + (wn * HALF + y) * 16 + 4 * (lane / 16)) =
            f8_four(acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3], f8_scale(exponent));
      if (wn == 0 && lane < 16) out_exponents[((size_t)(tile_n / 4) * out_padded + pair[x]) * 4 + tile_n % 4] = (uint8_t)exponent;
    }
  } else {
    const bool fours = N % 4 == 0;
#pragma unroll
    for (int x = 0; x < XB; ++x) {
      if (p0 + (wm * XB + x) * 16 + lane % 16 >= count) continue;
      float* row = reinterpret_cast<float*>(out) + (size_t)pair[x] * N;
#pragma unroll
      for (int y = 0; y < HALF; ++y) {
        const int n = tile_n * OUTS + (wn * HALF + y) * 16 + 4 * (lane / 16);
        if (n >= N) continue;
        if (fours) {
          store_four(row + n, acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) row[n + e] = acc[x][y][e];
        }
      }
    }
  }
}

template <bool GATED, bool FULL, int XB>
__global__ __launch_bounds__(512, 2) void experts_ring_kernel(const uint8_t* __restrict__ a, const uint32_t* __restrict__ exponents, int padded, int in_div,
                                                              const int32_t* __restrict__ list, int capacity, const int32_t* __restrict__ counts, int E,
                                                              F8Weight w, void* __restrict__ out, uint8_t* __restrict__ out_exponents, int out_padded,
                                                              ExpertGate gate, const float* __restrict__ in_weights) {
  using Ring = ExpertsRing<GATED, FULL, XB>;
  constexpr int ROWS = Ring::ROWS, OUTS = Ring::OUTS;
  __shared__ __attribute__((aligned(16))) f8_u32x4_t ring[Ring::R * Ring::PIECES * 64];
  const int lane = threadIdx.x % 64, n_tiles = (w.rows + OUTS - 1) / OUTS;
  // Tiles of pairs of all experts: a wave adds up 64 experts at a time; every wave of the workgroup finds the same.  Workgroups go to the
  // eight XCDs in turn: every XCD takes a run of (expert, weight tile, tile of pairs) in this order.
  int total = 0;
  for (int e0 = 0; e0 < E; e0 += 64) total += e0 + lane < E ? (counts[e0 + lane] + ROWS - 1) / ROWS : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, BH_WAVE);
  total *= n_tiles;
  const int each = (total + 7) / 8, turn = blockIdx.x / 8, id = (blockIdx.x % 8) * each + turn;
  if (turn >= each || id >= total) return;      // the whole workgroup
  int expert = -1, before = 0, count = 0, at = 0;
  for (int e0 = 0; e0 < E && expert < 0; e0 += 64) {
    const int own = e0 + lane < E ? counts[e0 + lane] : 0, tiles = (own + ROWS - 1) / ROWS * n_tiles;
    int upto = tiles;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int lower = __shfl_up(upto, off, BH_WAVE);
      if (lane >= off) upto += lower;
    }
    const unsigned long long behind = __ballot(before + upto > id);
    if (behind) {
      const int l = __ffsll(behind) - 1;
      expert = e0 + l;
      count = __shfl(own, l, BH_WAVE);
      at = id - before - (__shfl(upto, l, BH_WAVE) - __shfl(tiles, l, BH_WAVE));
    } else {
      before += __shfl(upto, 63, BH_WAVE);
    }
  }
  expert = __builtin_amdgcn_readfirstlane(expert);
  count = __builtin_amdgcn_readfirstlane(count);
  at = __builtin_amdgcn_readfirstlane(at);
  const int row_tiles = (count + ROWS - 1) / ROWS, p0 = (at % row_tiles) * ROWS, tile_n = at / row_tiles;
  const int32_t* pairs = list + (size_t)expert * capacity;
  if (XB == 4 && count - p0 <= 64)
    experts_ring_tile<GATED, FULL, 2>(ring, a, exponents, padded, in_div, pairs, expert, count, p0, tile_n, w, out, out_exponents, out_padded, gate, in_weights);
  else
    experts_ring_tile<GATED, FULL, XB>(ring, a, exponents, padded, in_div, pairs, expert, count, p0, tile_n, w, out, out_exponents, out_padded, gate, in_weights);
}

// ---- the sum over a row's pairs --------------------------------------------------------------------------------
// VN: neighbouring outputs of a thread (4: a multiple of 4 outputs).
template <typename T, typename TC, int VN>
__global__ __launch_bounds__(256) void experts_sum_kernel(const float* __restrict__ y, const int32_t* __restrict__ chosen, const float* __restrict__ weights,
                                                          const T* __restrict__ through, TC* __restrict__ out, int E, int top, int D, int fresh) {
  const int row = blockIdx.x, d = VN * (blockIdx.y * blockDim.x + threadIdx.x);
  if (d >= D) return;
  float total[VN] = {};
#pragma unroll 4
  for (int j = 0; j < top; ++j) {
    const long pair = (long)row * top + j;
    const int e = chosen[pair];
    if (e < 0 || (e >= E && through == nullptr)) continue;
    const float f = weights ? weights[pair] : 1.0f;
    if constexpr (VN == 4) {
      const float4 share = e >= E ? load_four(through + (size_t)row * D + d) : load_four(y + pair * D + d);
      total[0] = fmaf(f, share.x, total[0]), total[1] = fmaf(f, share.y, total[1]), total[2] = fmaf(f, share.z, total[2]), total[3] = fmaf(f, share.w, total[3]);
    } else {
      total[0] = fmaf(f, e >= E ? to_f32(through[(size_t)row * D + d]) : y[pair * D + d], total[0]);
    }
  }
  TC* at = out + (size_t)row * D + d;
  if constexpr (VN == 4) {
    if (!fresh) {
      const float4 old = load_four(at);
      total[0] += old.x, total[1] += old.y, total[2] += old.z, total[3] += old.w;
    }
    store_four(at, total[0], total[1], total[2], total[3]);
  } else {
    *at = from_f32<TC>(fresh ? total[0] : to_f32(*at) + total[0]);
  }
}

}  // namespace

// Whether the pairs of a call go through `few`.
extern "C" int bh_experts_float8_few(int pairs, int E) { return pairs <= FEW_PAIRS && pairs <= 8 * E; }

// One of the two products of `few`: in [*][K] rows of `dtype`; out float32 [pairs][N]; gated: w holds gate and up of every expert.
extern "C" int bh_experts_float8_rows(const void* in, int dtype, int in_div, const int32_t* chosen, int pairs, int E, const void* w, const void* scales,
                                      float* out, int N, int K, int gated, float limit, float alpha, float shift, const float* in_weights, int full,
                                      hipStream_t stream) {
  BH_REQUIRE(pairs > 0 && pairs <= FEW_PAIRS && E > 0 && N > 0 && K > 0 && in_div > 0, "experts_float8: 1 to %d pairs of positive sizes, got %d", FEW_PAIRS, pairs);
  BH_REQUIRE((uintptr_t)w % 16 == 0, "experts_float8: the weights must be 16-byte aligned");
  const F8Weight weight = {(const uint8_t*)w, (const float*)scales, N, (K + F8_K - 1) / F8_K};
  BH_REQUIRE(E <= 65535, "experts_float8: up to 65,535 experts, got %d", E);
  BH_REQUIRE(full || !gated, "experts_float8: gate and up are summed in full");
  const ExpertGate gate = {limit, alpha, shift};
#define BH_F8_EXPERTS(T, GATED, FULL)                                                                                                              \
  do {                                                                                                                                             \
    if (f8_load_of(in, K) == F8_EVEN) launch_few<T, GATED, FULL, F8_EVEN>((const T*)in, in_div, chosen, pairs, E, weight, out, K, gate, in_weights, stream); \
    else launch_few<T, GATED, FULL, F8_VALUES>((const T*)in, in_div, chosen, pairs, E, weight, out, K, gate, in_weights, stream);                  \
  } while (0)
#define BH_F8_EXPERTS_OF(T)                                                                                \
  do {                                                                                                     \
    if (gated) BH_F8_EXPERTS(T, true, true);                                                               \
    else if (full) BH_F8_EXPERTS(T, false, true);                                                          \
    else BH_F8_EXPERTS(T, false, false);                                                                   \
  } while (0)
  if (dtype == BH_F32) BH_F8_EXPERTS_OF(float);
  else if (dtype == BH_BF16) BH_F8_EXPERTS_OF(bf16_t);
  else return bh_fail("experts_float8: unknown dtype %d", dtype);
#undef BH_F8_EXPERTS_OF
#undef BH_F8_EXPERTS
  return bh_check_launch("experts_float8_rows");
}

// Whether a call is one row's.
extern "C" int bh_experts_float8_one(int pairs, int top) { return pairs == top && top <= FEW_TOP; }

// Both products of one row and the sum: inner float32 [top][ff] is scratch.
extern "C" int bh_experts_float8_row(const void* x, int dtype, const int32_t* chosen, const float* weights, int weigh_input, const void* through, int E,
                                     const void* up, const void* up_scales, const void* down, const void* down_scales, float* inner, void* out, int c_dtype,
                                     int top, int K, int ff, int D, float limit, float alpha, float shift, int fresh, int full, hipStream_t stream) {
  BH_REQUIRE(top > 0 && top <= FEW_TOP && D > 0 && K > 0 && ff > 0 && E > 0, "experts_float8: a row of %d pairs, %d x %d x %d", top, K, ff, D);
  BH_REQUIRE(((uintptr_t)up | (uintptr_t)down) % 16 == 0, "experts_float8: the weights must be 16-byte aligned");
  BH_REQUIRE((dtype == BH_F32 || dtype == BH_BF16) && (c_dtype == BH_F32 || c_dtype == BH_BF16), "experts_float8: unknown dtype");
  BH_REQUIRE(!weigh_input || weights != nullptr, "experts_float8: inputs are weighed by weights");
  const F8Weight first = {(const uint8_t*)up, (const float*)up_scales, ff, (K + F8_K - 1) / F8_K};
  const F8Weight second = {(const uint8_t*)down, (const float*)down_scales, D, (ff + F8_K - 1) / F8_K};
  const ExpertGate gate = {limit, alpha, shift};
  const float* in_weights = weigh_input ? weights : nullptr;
  const float* out_weights = weigh_input ? nullptr : weights;
#define BH_F8_ONE_AS(T, LOAD) \
  experts_one_kernel<T, LOAD><<<dim3(first.blocks(), top), FEW_WAVES * 64, 0, stream>>>((const T*)x, chosen, E, first, inner, K, gate, in_weights)
#define BH_F8_ONE(T)                                                    \
  do {                                                                  \
    if (f8_load_of(x, K) == F8_EVEN) BH_F8_ONE_AS(T, F8_EVEN);          \
    else BH_F8_ONE_AS(T, F8_VALUES);                                    \
  } while (0)
  if (dtype == BH_F32) BH_F8_ONE(float);
  else BH_F8_ONE(bf16_t);
#undef BH_F8_ONE
#undef BH_F8_ONE_AS
#define BH_F8_SUM_AS(T, TC, FULL, LOAD) \
  experts_one_sum_kernel<T, TC, FULL, LOAD><<<(D + 7) / 8, ONE_WAVES * 64, 0, stream>>>(inner, chosen, out_weights, (const T*)through, E, second, (TC*)out, ff, top, fresh)
#define BH_F8_SUM(T, TC)                                                      \
  do {                                                                        \
    if (f8_load_of(inner, ff) == F8_EVEN) {                                   \
      if (full) BH_F8_SUM_AS(T, TC, true, F8_EVEN);                           \
      else BH_F8_SUM_AS(T, TC, false, F8_EVEN);                               \
    } else if (full) BH_F8_SUM_AS(T, TC, true, F8_VALUES);                    \
    else BH_F8_SUM_AS(T, TC, false, F8_VALUES);                               \
  } while (0)
  if (dtype == BH_F32) {
    if (c_dtype == BH_F32) BH_F8_SUM(float, float);
    else BH_F8_SUM(float, bf16_t);
  } else if (c_dtype == BH_F32) BH_F8_SUM(bf16_t, float);
  else BH_F8_SUM(bf16_t, bf16_t);
#undef BH_F8_SUM
#undef BH_F8_SUM_AS
  return bh_check_launch("experts_float8_row");
}

// One of the two products of `tiles`, from rows in 8 bits; lists [E][capacity] and counts [E] as experts_group makes them.  Gated: out is
// rows in 8 bits [pairs], row after row, with their exponents.
extern "C" int bh_experts_float8_tiles(const void* a, const void* exponents, int rows, int in_div, const int32_t* list, int capacity, const int32_t* counts,
                                       int pairs, int E, const void* w, const void* scales, void* out, void* out_exponents, int N, int K, int gated,
                                       float limit, float alpha, float shift, const float* in_weights, int full, hipStream_t stream) {
  BH_REQUIRE(rows > 0 && pairs > 0 && E > 0 && N > 0 && K > 0 && in_div > 0 && capacity > 0, "experts_float8: sizes must be positive");
  BH_REQUIRE(((uintptr_t)a | (uintptr_t)exponents | (uintptr_t)w | (uintptr_t)out) % 16 == 0, "experts_float8: rows and weights must be 16-byte aligned");
  BH_REQUIRE((long)(rows + 15) * ((K + 511) / 512 * 512) < (1L << 32), "experts_float8: %d rows of %d inputs do not lie within 4 GB", rows, K);
  BH_REQUIRE(!gated || out_exponents != nullptr, "experts_float8: rows in 8 bits have exponents");
  BH_REQUIRE(full || !gated, "experts_float8: gate and up are summed in full");
  const F8Weight weight = {(const uint8_t*)w, (const float*)scales, N, (K + F8_K - 1) / F8_K};
  const bool wide = pairs >= 48L * E;
  const int outs = gated ? 128 : 256, tile = wide ? 128 : 64;
  const long most = (long)((N + outs - 1) / outs) * (pairs / tile + (pairs < E ? pairs : E)) + 8;      // every expert's last tile may be a part of one
  BH_REQUIRE(most < (1L << 31), "experts_float8: %d pairs of %d outputs are too many", pairs, N);
  const ExpertGate gate = {limit, alpha, shift};
#define BH_F8_TILES(GATED, FULL, XB)                                                                                                            \
  experts_ring_kernel<GATED, FULL, XB><<<(unsigned)most, 512, 0, stream>>>((const uint8_t*)a, (const uint32_t*)exponents, (rows + 15) / 16 * 16, in_div, \
                                                                          list, capacity, counts, E, weight, out, (uint8_t*)out_exponents,      \
                                                                          (pairs + 15) / 16 * 16, gate, in_weights)
#define BH_F8_TILES_OF(GATED, FULL)          \
  do {                                       \
    if (wide) BH_F8_TILES(GATED, FULL, 4);   \
    else BH_F8_TILES(GATED, FULL, 2);        \
  } while (0)
  if (gated) BH_F8_TILES_OF(true, true);
  else if (full) BH_F8_TILES_OF(false, true);
  else BH_F8_TILES_OF(false, false);
#undef BH_F8_TILES_OF
#undef BH_F8_TILES
  return bh_check_launch("experts_float8_tiles");
}

extern "C" int bh_experts_float8_sum(const float* y, const int32_t* chosen, const float* weights, const void* through, int dtype, void* out, int c_dtype,
                                     int n_rows, int E, int top, int D, int fresh, hipStream_t stream) {
  BH_REQUIRE(n_rows > 0 && top > 0 && D > 0 && E > 0 && (D + 255) / 256 <= 65535, "experts_float8: %d rows of %d outputs", n_rows, D);
  BH_REQUIRE((dtype == BH_F32 || dtype == BH_BF16) && (c_dtype == BH_F32 || c_dtype == BH_BF16), "experts_float8: unknown dtype");
  const bool fours = D % 4 == 0 && ((uintptr_t)y | (uintptr_t)through | (uintptr_t)out) % 16 == 0;
  const dim3 grid(n_rows, (D / (fours ? 4 : 1) + 255) / 256);
#define BH_F8_SUM(T, TC)                                                                                                                         \
  do {                                                                                                                                           \
    if (fours) experts_sum_kernel<T, TC, 4><<<grid, 256, 0, stream>>>(y, chosen, weights, (const T*)through, (TC*)out, E, top, D, fresh);         \
    else experts_sum_kernel<T, TC, 1><<<grid, 256, 0, stream>>>(y, chosen, weights, (const T*)through, (TC*)out, E, top, D, fresh);               \
  } while (0)
  if (dtype == BH_F32) {
    if (c_dtype == BH_F32) BH_F8_SUM(float, float);
    else BH_F8_SUM(float, bf16_t);
  } else if (c_dtype == BH_F32) BH_F8_SUM(bf16_t, float);
  else BH_F8_SUM(bf16_t, bf16_t);
#undef BH_F8_SUM
  return bh_check_launch("experts_float8_sum");
}
