// q4_gemv.hip -- products of few rows with 4-bit weights (q4.h).
//
//   Y = X W,   W[k][n] = s (c - z)   with s and z of (k / group, n)
//
// A group's part of a sum is s (sum x (1 + c / 16) - (1 + z / 16) sum x) 16: the bf16
// 1 + c / 16 is a code put among mantissa bits (q4.h), exact, so a weight costs 7 / 8
// of an instruction and no rounding.  Both sums come from the matrix units
// (v_mfma_f32_16x16x32_bf16; the second with a column operand of ones, which leaves
// it in the lanes and registers of the first), in fp32, and are joined group by
// group, so that nothing larger than a group's sum is ever cancelled.
//
// The columns are the lanes of the result (one scale to a lane), the rows 4 i + l /
// 16 its register i, so up to 4 rows need one register of four.
//
// HBM bound: the waves of a workgroup take the units of a column tile in turn, and
// join their sums in LDS.
#include <algorithm>

#include "common.h"
#include "q4.h"

namespace llk_gfx950 {
namespace {

// A wave's operands of one unit.
template <int SIDES, int GROUP>
struct Unit {
  static constexpr int kGroups = kQ4Unit / GROUP;
  u32x4 codes[SIDES];
  uint32_t scales[SIDES][kGroups];
  u32x4 x[4];
};

// MR: registers of the result that hold rows (M <= 4 MR).
template <int SIDES, int GROUP, int MR>
__global__ void __launch_bounds__(1024) q4_gemv_kernel(Q4Args a) {
  extern __shared__ float sums[];  // [wave][side][row][16]
  using U = Unit<SIDES, GROUP>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int tile = blockIdx.x, rows = a.M;  // to 16
  const int units = (a.K + kQ4Unit - 1) / kQ4Unit;
  const int col = lane & 15, grp = lane >> 4;
  // the lane's row of X: operand row col is row 4 (col % 4) + col / 4
  const int row = (col & 3) * 4 + (col >> 2);
  const uint16_t* const x = a.x + (int64_t)row * a.ldx + grp * 8;

  auto load = [&](int u, U& o) {
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
      const int64_t at = (int64_t)tile * units + u;
      o.codes[s] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(a.side[s].codes + at * kQ4UnitBytes) + lane);
#pragma unroll
      for (int g = 0; g < U::kGroups; ++g)
        o.scales[s][g] = a.side[s].scales[(at * U::kGroups + g) * kQ4Columns + col];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o.x[j] = u32x4{0, 0, 0, 0};
    if (row < rows) {
      const int k = u * kQ4Unit + grp * 8;
      if ((u + 1) * kQ4Unit <= a.K) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o.x[j] = load16_any(x + u * kQ4Unit + 32 * j);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int left = a.K - (k + 32 * j);
          if (left >= 8) o.x[j] = load16_any(x + u * kQ4Unit + 32 * j);
          else if (left > 0) o.x[j] = load16_part(x + u * kQ4Unit + 32 * j, left);
        }
      }
    }
  };

  float acc[SIDES][MR];
#pragma unroll
  for (int s = 0; s < SIDES; ++s)
#pragma unroll
    for (int i = 0; i < MR; ++i) acc[s][i] = 0.0f;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{kCodeOne, kCodeOne, kCodeOne, kCodeOne});
  auto work = [&](const U& o) {
    constexpr int kSteps = 4 / U::kGroups;  // of 32 k, to a group
#pragma unroll
    for (int g = 0; g < U::kGroups; ++g) {
      f32x4 sx{0, 0, 0, 0}, part[SIDES];
#pragma unroll
      for (int s = 0; s < SIDES; ++s) part[s] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = g * kSteps; j < (g + 1) * kSteps; ++j) {
        const bf16x8 xs = __builtin_bit_cast(bf16x8, o.x[j]);
        sx = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xs, ones, sx, 0, 0, 0);
#pragma unroll
        for (int s = 0; s < SIDES; ++s)
          part[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xs, q4_decode8(o.codes[s][j]), part[s], 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < SIDES; ++s) {
        const uint32_t w = o.scales[s][g];
        const float scale = q4_scale(w), off = q4_offset(w);
#pragma unroll
        for (int i = 0; i < MR; ++i)
          acc[s][i] = __builtin_fmaf(scale, __builtin_fmaf(off, sx[i], part[s][i]), acc[s][i]);
      }
    }
  };
  if (wave < units) {
    U cur, next;
    load(wave, cur);
    for (int u = wave; u < units; u += waves) {
      if (u + waves < units) load(u + waves, next);
      work(cur);
      cur = next;
    }
  }

#pragma unroll
  for (int s = 0; s < SIDES; ++s)
#pragma unroll
    for (int i = 0; i < MR; ++i)
      sums[((wave * SIDES + s) * MR * 4 + 4 * i + grp) * 16 + col] = acc[s][i];
  __syncthreads();
  for (int t = threadIdx.x; t < rows * 16; t += blockDim.x) {
    const int m = t / 16, n = tile * kQ4Columns + t % 16;
    if (n >= a.N) continue;
    float v[SIDES];
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
      v[s] = 0.0f;
      for (int w = 0; w < waves; ++w) v[s] += sums[(w * SIDES + s) * MR * 64 + t];
    }
    q4_store(a, SIDES, m, n, v[0], v[SIDES - 1]);
  }
}

template <int SIDES, int GROUP>
hipError_t launch(const Q4Args& args, hipStream_t stream) {
  Q4Args a = args;
  void* params[] = {&a};
  const int units = (int)q4_units(a.K);
  const int waves = std::clamp(units, 1, 8);
  const int mr = std::min(4, (a.M + 3) / 4);
  const void* fn = mr == 1   ? reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, 1>)
                   : mr == 2 ? reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, 2>)
                   : mr == 3 ? reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, 3>)
                             : reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, 4>);
  return hipLaunchKernel(fn, dim3((unsigned)q4_tiles(a.N)), dim3(waves * 64), params,
                         (size_t)waves * SIDES * mr * 256, stream);
}
template <int SIDES>
hipError_t launch_group(const Q4Args& a, hipStream_t s) {
  return a.group == 32   ? launch<SIDES, 32>(a, s)
         : a.group == 64 ? launch<SIDES, 64>(a, s)
                         : launch<SIDES, 128>(a, s);
}

}  // namespace
}  // namespace llk_gfx950

// The kernel for 16 rows streams the weights once for them; the tile kernel shares
// them among 32 or 64.
Q4Plan llk_plan_q4(int64_t M, int64_t N, int64_t K, int sides) {
  Q4Plan p{16, 1, (int)q4_units(K), q4_tiles(N), 0};
  if (M <= 16) return p;
  p.rows = M <= 32 ? 32 : 64;
  const int64_t tiles = (M + p.rows - 1) / p.rows * ((N * sides + 255) / 256);
  const int64_t units = std::max<int64_t>(1, q4_units(K));
  // two workgroups to a CU, at least 4 units to each
  const int64_t s = std::clamp<int64_t>(512 / std::max<int64_t>(tiles, 1), 1, std::max<int64_t>(1, units / 4));
  p.stages = (int)((units + s - 1) / s);
  p.splits = (int)((units + p.stages - 1) / p.stages);
  p.groups = tiles * p.splits;
  p.bytes = p.splits > 1 ? (size_t)p.splits * sides * M * N * sizeof(float) : 0;
  return p;
}

hipError_t llk_launch_q4(const Q4Args& args, int sides, const Q4Plan& plan, hipStream_t stream) {
  using namespace llk_gfx950;
  Q4Args a = args;
  a.splits = plan.splits;
  a.stages = plan.stages;
  if (plan.rows > 16) return llk_launch_q4_tile(a, sides, plan.rows, stream);
  return sides == 2 ? launch_group<2>(a, stream) : launch_group<1>(a, stream);
}
