// Products of many rows with weights and activations in 8 bits: see gemm_float8_ring.hip.
#pragma once
#include "float8.h"

// The tile that a product runs on (an index of SHAPES in gemm_float8_ring.hip), in how many parts of K, and what that is estimated to take.
struct F8RingPlan {
  int tile, parts;
  double us;
};
// in_stretches: of the tiles whose gated outputs are a stretch of 128, with K whole.
F8RingPlan float8_ring_plan(int M, int N, int K, bool gated, bool full, bool in_stretches = false);
// a, exponents: rows in 8 bits, in blocks.  c: [M] rows of `ldc` elements; gated: w holds two matrices.  In more than one part the bare sums are
// left in `sums` [parts][M][N, gated 2 N] and `c` is not touched.
int float8_ring_launch(const F8RingPlan& plan, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, void* c, int c_dtype, float* sums, int accumulate,
                       int M, int ldc, int gated, int full, GateForm form, hipStream_t stream);
// A gated product on one of those, its outputs in 8 bits in blocks.  through_bf16: rounded to bfloat16 on their way there.
int float8_ring_launch_in_8(const F8RingPlan& plan, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, uint8_t* c, uint8_t* c_exponents, int through_bf16,
                            int M, int full, GateForm form, hipStream_t stream);
