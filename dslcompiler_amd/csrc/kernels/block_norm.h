// block_norm.h -- launcher of the fused residual norm (block_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// Rows of N elements; ld*: row strides in elements (ldg 0: one gate row for
// all).  y, g, wpost and h_out may be null.
struct BlockNormArgs {
  const void *y, *h, *g, *wpost, *wpre;
  void *h_out, *out;
  int64_t ldy, ldh, ldg, ldho, ldo;
  int N;
  float scale, eps, offset;
};

// Largest N: 1024 threads of 4 chunks of 8 elements.
constexpr int64_t kBlockNormMaxN = 32768;

// M >= 1 (in as many launches as its threads need), 1 <= N <= kBlockNormMaxN; *_f32: fp32 instead of bf16 (y and
// the gate; the residual, in and out; the result; both weights).
hipError_t llk_launch_block_norm(const BlockNormArgs& a, int64_t M, bool y_f32, bool h_f32,
                                 bool o_f32, bool w_f32, hipStream_t s);
