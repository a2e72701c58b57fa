// q4.h -- weights in 4 bits with group scales: their layout and launchers.
//
//   W[k][n] = scale[k / group][n] * (code[k][n] - zero[k / group][n])
//
// Codes lie in units of 16 columns by 128 k (1 KiB), unit (tile, u) at (tile * U +
// u) KiB, U = ceil(K / 128), tile = n / 16.  A unit is 64 lane slots of 16 bytes:
// slot l, dword j holds the 8 codes of column l % 16, k = 32 j + 8 (l / 16) + t, so
// that a wave's 16-byte loads of a unit are four ready operands of a
// v_mfma_f32_16x16x32_bf16 but for the conversion.  In a dword, turned right by 4 i
// bits, codes t = 2 i and 2 i + 1 are at bits 3 to 6 and 19 to 22: there they are the
// upper mantissa bits of two bf16 between 1 and 2 (kCodeMask, kCodeOne), 1 + c / 16.
//
// Scales lie as [tile][group][16 columns] dwords: the scale as fp32 without its
// low 13 bits (bf16 and fp16 scales are exact in the 19 left), and there 16 + zero.
// Rows and columns that fill the last unit have code 0 and scale 0.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

constexpr int kQ4Columns = 16, kQ4Unit = 128, kQ4UnitBytes = 1024;

inline int64_t q4_tiles(int64_t n) { return (n + kQ4Columns - 1) / kQ4Columns; }
inline int64_t q4_units(int64_t k) { return (k + kQ4Unit - 1) / kQ4Unit; }
// Groups that are stored: those of whole units.
inline int64_t q4_groups(int64_t k, int group) { return q4_units(k) * (kQ4Unit / group); }

struct Q4Source {  // codes and scales as the caller has them
  const uint8_t* codes;  // [K][ld] 0..15
  const uint16_t* scales;  // [groups][ld_scales], bf16 or fp16
  const uint8_t* zeros;  // [groups][ld_zeros], or null: 8
  int64_t ld, ld_scales, ld_zeros;
  int K, N, group, f16;
};

struct Q4Side {
  const uint8_t* codes;
  const uint32_t* scales;
};

// The launch of a product.
struct Q4Plan {
  int rows;      // to a workgroup: 16 (the kernel for few rows), 32 or 64
  int tiles;     // column tiles to a workgroup (the kernel for few rows)
  int splits;    // of K, joined by a second kernel
  int stages;    // units of K to a split
  int64_t groups;  // workgroups of the main kernel
  size_t bytes;    // workspace
};

struct Q4Args {
  const uint16_t* x;
  int64_t ldx;
  Q4Side side[2];  // gate and up for the SwiGLU
  void* y;
  int64_t ldy;
  int M, N, K, group;
  int out;  // llk_dtype
  int accumulate;
  float* part;  // splits: [split][side][M][N] sums
  int splits, stages;
  int tiles;  // column tiles of the matrix
};

hipError_t llk_launch_q4_pack(const Q4Source& s, uint8_t* codes, uint32_t* scales, hipStream_t stream);
struct Q4QuantiseArgs {
  const uint16_t* w;  // bf16 [K][ld]
  int64_t ld, ld_codes, ld_scales, ld_zeros;
  uint8_t* codes;
  uint16_t* scales;
  uint8_t* zeros;  // null: symmetric
  int K, N, group, f16;
};
hipError_t llk_launch_q4_quantise(const Q4QuantiseArgs& a, hipStream_t stream);
Q4Plan llk_plan_q4(int64_t M, int64_t N, int64_t K, int sides);
hipError_t llk_launch_q4(const Q4Args& a, int sides, const Q4Plan& plan, hipStream_t stream);
hipError_t llk_launch_q4_tile(const Q4Args& a, int sides, int rows, hipStream_t stream);
hipError_t llk_launch_q4_join(const Q4Args& a, int sides, hipStream_t stream);

#ifdef __HIPCC__
#include "common.h"

namespace llk_gfx950 {

constexpr uint32_t kCodeMask = 0x00780078u, kCodeOne = 0x3f803f80u;

// kCodeOne in a vector register, which the compiler would not keep there by itself: with
// it v_and_or_b32 takes both constants, one of them a scalar.
__device__ __forceinline__ uint32_t q4_one() {
  uint32_t one;
  asm("v_mov_b32 %0, %1" : "=v"(one) : "s"(kCodeOne));
  return one;
}
// A dword's 8 codes as bf16 1 + c / 16.
__device__ __forceinline__ bf16x8 q4_decode8(uint32_t q, uint32_t one) {
  return __builtin_bit_cast(
      bf16x8, u32x4{(q & kCodeMask) | one, ((q >> 4) & kCodeMask) | one, ((q >> 8) & kCodeMask) | one,
                    (__builtin_amdgcn_alignbit(q, q, 12) & kCodeMask) | one});
}
__device__ __forceinline__ float q4_scale(uint32_t w) { return __uint_as_float(w & 0xffffe000u); }
// -(1 + z / 16)
__device__ __forceinline__ float q4_offset(uint32_t w) { return (float)(w & 0xffu) * -0.0625f; }

// Results from the sums of (code - zero) / 16: times 16, SiLU(g) u, added to what is
// there, rounded.
__device__ __forceinline__ void q4_store(const Q4Args& a, int sides, int m, int n, float v, float u) {
  const int64_t at = m * a.ldy + n;
  float r = sides == 2 ? swiglu_act(v * 16.0f, u * 16.0f) : v * 16.0f;
  if (a.out == kOutF32) {
    float* const y = static_cast<float*>(a.y) + at;
    *y = a.accumulate ? r + *y : r;
  } else {
    uint16_t* const y = static_cast<uint16_t*>(a.y) + at;
    if (a.accumulate)
      r += a.out == kOutBF16 ? bf16_bits_to_f32(*y) : (float)__builtin_bit_cast(_Float16, *y);
    *y = a.out == kOutBF16 ? f32_to_bf16_rne(r) : f32_to_f16_rne(r);
  }
}

}  // namespace llk_gfx950
#endif
