// rotary.h -- rotary positions: arguments and launcher.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

struct RotarySide {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;  // strides in elements
  int heads;
};

struct RotaryArgs {
  RotarySide side[2];  // q and k; k may have no heads
  const int32_t* positions;  // [tokens]
  const uint64_t* turns;  // [pairs]: turns per position, in units of 2^-64
  float factor;
  int tokens, head_dim, pairs;
  int inverse;
};

// Tokens that one call takes: a dimension of a launch has fewer than 2^32 threads,
// 256 of them to a token at most.
constexpr int64_t kRotaryMaxTokens = ((int64_t)1 << 24) - 1;

hipError_t llk_launch_rotary(const RotaryArgs& a, bool f32, bool interleaved, hipStream_t s);
