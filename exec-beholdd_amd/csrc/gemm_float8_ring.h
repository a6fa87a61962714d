// Products of many rows with weights and activations in 8 bits: see gemm_float8_ring.hip.
#pragma once
#include "float8.h"

// The tile that a product of these sizes runs on (an index of SHAPES in gemm_float8_ring.hip), or -1: the tiles of gemm_float8.hip.
int float8_ring_tile(int M, int N, int K, bool gated, bool full);
// a, exponents: rows in 8 bits, in blocks.  c: [M] rows of `ldc` elements; gated: w holds two matrices.
int float8_ring_launch(int tile, const uint8_t* a, const uint32_t* exponents, const F8Weight& w, void* c, int c_dtype, int accumulate, int M, int ldc,
                       int gated, int full, GateForm form, hipStream_t stream);
