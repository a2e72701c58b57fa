// q4_pack.hip -- weights to 4 bits, and codes into the order of q4.h.  Both run
// once for a weight.
#include "common.h"
#include "q4.h"

namespace llk_gfx950 {
namespace {

__device__ __forceinline__ float widen(uint16_t h, bool f16) {
  return f16 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : bf16_bits_to_f32(h);
}

// Workgroup (x, y): the unit y of 4 tiles from 4 x on, through LDS.
__global__ void __launch_bounds__(256) q4_pack_kernel(Q4Source s, uint8_t* codes, uint32_t* scales,
                                                      int tiles, int units) {
  __shared__ uint8_t lds[kQ4Unit][64];
  const int n0 = blockIdx.x * 64, k0 = blockIdx.y * kQ4Unit;
  for (int i = threadIdx.x; i < kQ4Unit * 64; i += 256) {
    const int k = k0 + i / 64, n = n0 + i % 64;
    lds[i / 64][i % 64] = k < s.K && n < s.N ? s.codes[k * s.ld + n] & 15 : 0;
  }
  __syncthreads();
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int tile = blockIdx.x * 4 + wave;
  if (tile >= tiles) return;
  const int col = lane % 16, quarter = lane / 16;
  u32x4 out;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t d = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = lds[32 * j + 8 * quarter + 2 * i][wave * 16 + col];
      const uint32_t hi = lds[32 * j + 8 * quarter + 2 * i + 1][wave * 16 + col];
      const uint32_t at = lo << 3 | hi << 19;
      d |= i ? at << (4 * i) | at >> (32 - 4 * i) : at;
    }
    out[j] = d;
  }
  reinterpret_cast<u32x4*>(codes + ((int64_t)tile * units + blockIdx.y) * kQ4UnitBytes)[lane] = out;
  const int per = kQ4Unit / s.group, n = tile * kQ4Columns + col;
  if (quarter < per) {
    const int g = blockIdx.y * per + quarter;
    uint32_t w = 0;
    if (n < s.N && (int64_t)g * s.group < s.K) {
      const uint32_t z = s.zeros ? s.zeros[g * s.ld_zeros + n] & 15 : 8;
      w = (__float_as_uint(widen(s.scales[g * s.ld_scales + n], s.f16)) & 0xffffe000u) | (16 + z);
    }
    scales[((int64_t)tile * units * per + g) * kQ4Columns + col] = w;
  }
}

// A thread to a group of a column.  Symmetric: scale = largest magnitude / 7, codes
// around 8.  With zeros: scale = (largest - smallest) / 15 of the group's values and
// 0, the zero where 0 lies.  The scale is rounded to its type before the codes are
// made, so they are the nearest to what it stands for.
__global__ void __launch_bounds__(256) q4_quantise_kernel(Q4QuantiseArgs a) {
  const int n = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y;
  if (n >= a.N) return;
  const int k0 = g * a.group, k1 = min(a.K, k0 + a.group);
  float lo = 0.0f, hi = 0.0f;
  bool finite = true;
  for (int k = k0; k < k1; ++k) {
    const float w = bf16_bits_to_f32(a.w[k * a.ld + n]);
    finite &= fabsf(w) < __builtin_inff();
    lo = fminf(lo, w);
    hi = fmaxf(hi, w);
  }
  // hi - lo would overflow for the largest values
  float scale = a.zeros ? hi / 15.0f - lo / 15.0f : fmaxf(hi, -lo) / 7.0f;
  if (!finite) scale = __builtin_nanf("");
  const uint16_t bits = a.f16 ? f32_to_f16_rne(scale) : f32_to_bf16_rne(scale);
  scale = widen(bits, a.f16);
  a.scales[g * a.ld_scales + n] = bits;
  const bool some = scale > 0.0f && scale < __builtin_inff();
  float zero = 8.0f;
  if (a.zeros) {
    zero = some ? fminf(rintf(-lo / scale), 15.0f) : 0.0f;
    a.zeros[g * a.ld_zeros + n] = (uint8_t)zero;
  }
  for (int k = k0; k < k1; ++k) {
    const float w = bf16_bits_to_f32(a.w[k * a.ld + n]);
    const float c = some ? fminf(fmaxf(rintf(w / scale) + zero, 0.0f), 15.0f) : zero;
    a.codes[k * a.ld_codes + n] = (uint8_t)c;
  }
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_q4_pack(const Q4Source& src, uint8_t* codes, uint32_t* scales,
                              hipStream_t stream) {
  Q4Source s = src;
  int tiles = (int)q4_tiles(s.N), units = (int)q4_units(s.K);
  void* params[] = {&s, &codes, &scales, &tiles, &units};
  return hipLaunchKernel(reinterpret_cast<const void*>(&llk_gfx950::q4_pack_kernel),
                         dim3((tiles + 3) / 4, units), dim3(256), params, 0, stream);
}

hipError_t llk_launch_q4_quantise(const Q4QuantiseArgs& args, hipStream_t stream) {
  Q4QuantiseArgs a = args;
  void* params[] = {&a};
  return hipLaunchKernel(reinterpret_cast<const void*>(&llk_gfx950::q4_quantise_kernel),
                         dim3((a.N + 255) / 256, (a.K + a.group - 1) / a.group), dim3(256), params, 0,
                         stream);
}
