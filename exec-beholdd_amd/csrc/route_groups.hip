// The router of a mixture of experts whose rows use experts of a few groups only (HipKernels.route_in_groups).
//   score[e]  = 1 / (1 + exp(-z[e]))  or  exp(z[e] - max z) / sum exp(z - max z)          z: a row's E logits
//   by[e]     = score[e] + correction[e]                                                  what is chosen by
//   merit[g]  = the largest of by in group g, or the sum of its two largest; groups are runs of E / groups neighbours
//   chosen    = the `top` largest of by in the `keep` groups of largest merit, largest first; ties go to the lower index
//   weights   = score of the chosen, divided by their sum where asked for, times `factor`
// A row is a wave's.  Choices are whole numbers that a rounding would change, and scores of two experts differ by less than 32 bits tell
// apart in one row of 30,000 (256 experts): scores, merits and sums are in 64 bits, whose exponentials are a small part of the time.
// A score that is not a number counts as the lowest, so that the indices are always `top` different experts of open groups.
// Bound by the chain of `top` choices for few rows, by their instructions for many.  A choice finds the largest upper half of the scores' bits,
// ordered as whole numbers, in six steps between registers of neighbouring lanes; only where two lanes share it (one choice in thousands, or equal
// scores) the lower halves and the indices are compared.  Measured, us, in brackets with 64-bit scores, indices and weights handed between lanes
// through LDS at every step: 1 row of 128 3.8 (8.8), 1,234 of 160 7.0 (11.7), 8,192 of 256 15.0 (31.7), of which 7.6 are a launch and the scores,
// 3 the groups, 3.5 the choices but the first, 1.5 the weights' sum and division.
#include "common.h"

#define RG_MAX_TOP 32
#define RG_MAX_GROUPS 64
#define RG_WAVES 4

namespace {

struct Two {
  double first, second;
};
__device__ inline Two merged(Two a, Two b) {
  return {fmax(a.first, b.first), fmax(fmin(a.first, b.first), fmax(a.second, b.second))};
}

// The largest (or smallest) over the wave, for every lane.
template <typename JOIN>
__device__ inline uint32_t over_wave(uint32_t v, JOIN join) {
  v = join(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128 /* row_ror:8 */, 0xf, 0xf, true));
  v = join(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
  v = join(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
  v = join(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = join((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return join((uint32_t)b[0], (uint32_t)b[1]);
}
__device__ inline uint32_t wave_largest(uint32_t v) {
  return over_wave(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
// A number's bits in the order of the numbers; above 0, which stands for none.
__device__ inline unsigned long long ordered(double v) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  return bits >> 63 ? ~bits : bits | (1ull << 63);
}
// v with the lanes of a group of 16 turned by N.
template <int N>
__device__ inline double turned(double v) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bits, 0x120 + N /* row_ror */, 0xf, 0xf, true);
  const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(bits >> 32), 0x120 + N, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (unsigned long long)high << 32 | low);
}

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int off = BH_WAVE / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, BH_WAVE);
  return v;
}

// PER: experts a lane holds (lane, lane + 64, ...).  LDS: by of the wave's row, E doubles a wave.
template <int PER>
__global__ __launch_bounds__(RG_WAVES * 64) void route_groups_kernel(const float* __restrict__ logits, int stride, const float* __restrict__ correction,
                                                                    int32_t* __restrict__ chosen, float* __restrict__ weights, int n_rows, int E, int top,
                                                                    int groups, int keep, uint32_t per_each, int softmax, int top_two, int renorm, float factor) {
  extern __shared__ double by_of[];
  const int lane = threadIdx.x % BH_WAVE, wave = threadIdx.x / BH_WAVE, row = blockIdx.x * RG_WAVES + wave;
  if (row >= n_rows) return;      // nothing below meets other waves
  const float* z = logits + (size_t)row * stride;
  double* by_row = by_of + (size_t)wave * E;
  const double none = -__builtin_inf();
  double score[PER], by[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + i * BH_WAVE;
    score[i] = e < E ? (double)z[e] : none;
  }
  if (softmax) {
    double most = none, total = 0.;
#pragma unroll
    for (int i = 0; i < PER; ++i) most = fmax(most, score[i]);
#pragma unroll
    for (int off = BH_WAVE / 2; off > 0; off >>= 1) most = fmax(most, __shfl_xor(most, off, BH_WAVE));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      score[i] = lane + i * BH_WAVE < E ? exp(score[i] - most) : 0.;
      total += score[i];
    }
    total = wave_sum_f64(total);
#pragma unroll
    for (int i = 0; i < PER; ++i) score[i] /= total;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) score[i] = 1. / (1. + exp(-score[i]));
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + i * BH_WAVE;
    by[i] = e < E ? score[i] + (correction ? (double)correction[e] : 0.) : none;
    by[i] = by[i] == by[i] ? by[i] + 0. : none;      // (a negative zero becomes a positive one, whose bits it then shares)
  }
  unsigned taken = 0;      // bit i: this lane's expert lane + 64 i may not be chosen (any more)
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + i * BH_WAVE >= E) taken |= 1u << i;
  if (keep < groups) {
    const int each = E / groups;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + i * BH_WAVE < E) by_row[lane + i * BH_WAVE] = by[i];
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int room = 1;      // groups rounded up to a power of two: 64 / room lanes look through a group
    while (room < groups) room *= 2;
    const int lanes = BH_WAVE / room, group = lane / lanes;
    Two best = {none, none};
    if (group < groups)
      for (int i = lane % lanes; i < each; i += lanes) {
        const double v = by_row[group * each + i];
        best = {fmax(best.first, v), fmax(best.second, fmin(best.first, v))};
      }
    for (int off = lanes / 2; off > 0; off >>= 1) best = merged(best, Two{__shfl_xor(best.first, off, BH_WAVE), __shfl_xor(best.second, off, BH_WAVE)});
    double merit = top_two && each > 1 ? best.first + best.second : best.first;
    merit = merit == merit ? merit : none;      // (of two infinite ones)
    int better = 0;      // groups ahead of this lane's, each of a group's lanes comparing it with some
    for (int first = 0; first < groups; first += lanes) {
      const int g = first + lane % lanes;
      const double other = __shfl(merit, g * lanes % BH_WAVE, BH_WAVE);
      const unsigned long long ahead = __ballot(g < groups && (other > merit || (other == merit && g < group)));
      better += __popcll((ahead >> (group * lanes)) & (~0ull >> (BH_WAVE - lanes)));
    }
    const unsigned long long open = __ballot(group < groups && better < keep);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + i * BH_WAVE;
      if (e < E && !((open >> ((per_each ? (int)__umulhi((uint32_t)e, per_each) : e) * lanes)) & 1ull)) taken |= 1u << i;
    }
  }
  unsigned long long keys[PER];      // 0: not to be chosen (any more)
#pragma unroll
  for (int i = 0; i < PER; ++i) keys[i] = (taken >> i) & 1u ? 0 : ordered(by[i]);
  // Up to four experts a lane stand in order, largest first (neighbours change places, so equal ones stay in theirs), and a choice looks at the
  // first alone; more are looked through every time.
  constexpr bool SORTED = PER <= 4;
  int at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) at[i] = i;
  if constexpr (SORTED) {
#pragma unroll
    for (int last = PER - 1; last > 0; --last)
#pragma unroll
      for (int i = 0; i < last; ++i) {
        const bool change = keys[i + 1] > keys[i];
        const unsigned long long key = keys[i];
        const int index = at[i];
        keys[i] = change ? keys[i + 1] : key, at[i] = change ? at[i + 1] : index;
        keys[i + 1] = change ? key : keys[i + 1], at[i + 1] = change ? index : at[i + 1];
      }
  }
  int mine_index = 0;      // lane j keeps the j-th choice
  for (int j = 0; j < top; ++j) {
    unsigned long long best = keys[0];
    int best_i = at[0];
    if constexpr (!SORTED) {
#pragma unroll
      for (int i = 1; i < PER; ++i)
        if (keys[i] > best) {
          best = keys[i];
          best_i = i;
        }
    }
    const uint32_t high = (uint32_t)(best >> 32), most = wave_largest(high);
    unsigned long long having = __ballot(high == most);
    if (having & (having - 1)) {      // several lanes: the lower halves decide, then the index
      const uint32_t low = high == most ? (uint32_t)best : 0u, most_low = wave_largest(low);
      const uint32_t index = high == most && low == most_low ? (uint32_t)(lane + best_i * BH_WAVE) : 0xffffffffu;
      having = __ballot(index == over_wave(index, [](uint32_t a, uint32_t b) { return min(a, b); }) && high == most);
    }
    const int winner = __builtin_ctzll(having), which = __builtin_amdgcn_readlane(best_i, winner);
    if constexpr (SORTED) {
      if (lane == winner) {
#pragma unroll
        for (int i = 0; i + 1 < PER; ++i) keys[i] = keys[i + 1], at[i] = at[i + 1];
        keys[PER - 1] = 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (which == i && lane == winner) keys[i] = 0;
    }
    if (lane == j) mine_index = winner + which * BH_WAVE;
  }
  double mine = 0., sum = 0.;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const double theirs = __shfl(score[i], mine_index % BH_WAVE, BH_WAVE);
    if (mine_index / BH_WAVE == i) mine = theirs;
  }
  if (renorm) {      // (the first 32 lanes have choices)
    sum = lane < top ? mine : 0.;
    sum += turned<8>(sum);
    sum += turned<4>(sum);
    sum += turned<2>(sum);
    sum += turned<1>(sum);
    if (top > 16) sum += __shfl_xor(sum, 16, BH_WAVE);
  }
  if (lane < top) {
    if (renorm) mine = sum == 0. ? 0. : mine / sum;
    chosen[(size_t)row * top + lane] = mine_index;
    weights[(size_t)row * top + lane] = (float)(mine * (double)factor);
  }
}

}  // namespace

// logits [n_rows][stride]: a row's E logits are its first.
extern "C" int bh_route_in_groups(const float* logits, int stride, const float* correction, int32_t* chosen, float* weights, int n_rows, int E, int top,
                                  int groups, int keep, int softmax, int top_two, int renorm, float factor, hipStream_t stream) {
  BH_REQUIRE(n_rows > 0 && E > 0 && E <= 1024, "route_in_groups: 1 to 1024 experts, got %d", E);
  BH_REQUIRE(stride >= E, "route_in_groups: %d logits do not lie in a row of %d", E, stride);
  BH_REQUIRE(groups >= 1 && groups <= RG_MAX_GROUPS && E % groups == 0, "route_in_groups: %d experts do not make 1 to %d equal groups of which there are %d",
             E, RG_MAX_GROUPS, groups);
  BH_REQUIRE(keep >= 1 && keep <= groups, "route_in_groups: a row uses 1 to %d groups, got %d", groups, keep);
  BH_REQUIRE(top >= 1 && top <= RG_MAX_TOP && (long)top <= (long)keep * (E / groups), "route_in_groups: 1 to min(%d, %ld) experts a row, got %d",
             RG_MAX_TOP, (long)keep * (E / groups), top);
  const dim3 grid((n_rows + RG_WAVES - 1) / RG_WAVES);
  // e / each = the upper half of e * per_each for e < 1024: rounding 2^32 / each up adds less than 1024 / 2^32 to a quotient that is at least 1 / each
  // below the next whole number.  (Of one expert a group 2^32 does not fit: every expert is its group's.)
  const uint32_t per_each = E == groups ? 0u : (uint32_t)(((1ull << 32) + E / groups - 1) / (E / groups));
  const size_t lds = keep < groups ? (size_t)RG_WAVES * E * sizeof(double) : 0;
#define BH_ROUTE(PER)                                                                                                                         \
  route_groups_kernel<PER><<<grid, RG_WAVES * 64, lds, stream>>>(logits, stride, correction, chosen, weights, n_rows, E, top, groups, keep, per_each, \
                                                                softmax, top_two, renorm, factor)
  if (E <= BH_WAVE) BH_ROUTE(1);
  else if (E <= 2 * BH_WAVE) BH_ROUTE(2);
  else if (E <= 4 * BH_WAVE) BH_ROUTE(4);
  else BH_ROUTE(16);
#undef BH_ROUTE
  return bh_check_launch("route_in_groups");
}
