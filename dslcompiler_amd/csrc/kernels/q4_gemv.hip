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
// HBM bound.  A workgroup has a few column tiles and a range of K: its rows of X go
// to LDS once (read as operands from memory they are four times a unit's codes, and
// the vector memory path, not HBM, would be the limit), and its 8 waves take the
// range's units in turn, four of them on their way.  Their sums are joined in LDS, and
// those of a split K by a second kernel.  SwiGLU of 4096 x 14336, 1 row: 12.3 us, 5.0
// TB/s; 13824 x 5120, 5 rows: 11.4 us and 4.0 to join 6 splits (kernel times).
#include <algorithm>

#include "common.h"
#include "q4.h"

namespace llk_gfx950 {
namespace {

constexpr int kWaves = 8, kAhead = 4;

// MR: registers of the result that hold rows (M <= 4 MR).  C: column tiles.
template <int SIDES, int GROUP, int MR, int C>
__global__ void __launch_bounds__(kWaves * 64) q4_gemv_kernel(Q4Args a) {
  // X: [unit][row][16 chunks of 8 k], a chunk's place turned by the row, so that 16
  // rows' chunks meet all banks; then the waves' sums [wave][side][row][16]
  extern __shared__ __attribute__((aligned(16))) u32x4 lds[];
  constexpr int kGroups = kQ4Unit / GROUP, kTurns = kWaves / C;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = blockIdx.z * 16, rows = min(16, a.M - m0);
  const int units = (a.K + kQ4Unit - 1) / kQ4Unit;
  const int begin = blockIdx.y * a.stages, end = min(begin + a.stages, units);
  const int tile0 = blockIdx.x * C, turn = wave / C;
  // (past the last tile, the last again, not stored)
  const int64_t tile = (int64_t)min(tile0 + wave % C, a.tiles - 1) * units;

  // Codes and scales through buffers of the tile: units past its last read as zeros,
  // without a branch that would have every load waited for.
  struct Unit {
    u32x4 codes[SIDES];
    uint32_t scales[SIDES][kGroups];
  };
  __amdgpu_buffer_rsrc_t codes[SIDES], scales[SIDES];
#pragma unroll
  for (int s = 0; s < SIDES; ++s) {
    codes[s] = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.side[s].codes + tile * kQ4UnitBytes), 0, units * kQ4UnitBytes, kBufferWord3);
    scales[s] = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint32_t*>(a.side[s].scales + tile * kGroups * kQ4Columns), 0,
        units * kGroups * kQ4Columns * 4, kBufferWord3);
  }
  auto load = [&](int u, Unit& o) {
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
      // (2: not to stay in the caches; no other workgroup reads them)
      o.codes[s] = __builtin_amdgcn_raw_buffer_load_b128(codes[s], u * kQ4UnitBytes + lane * 16, 0, 2);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        o.scales[s][g] = __builtin_amdgcn_raw_buffer_load_b32(
            scales[s], ((u * kGroups + g) * kQ4Columns + col) * 4, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);  // in order, so that the oldest can be waited for
  };
  Unit ring[kAhead];
  const int first = begin + turn;
#pragma unroll
  for (int n = 0; n < kAhead; ++n) load(first + n * kTurns, ring[n]);

  for (int i = threadIdx.x; i < (end - begin) * rows * 16; i += kWaves * 64) {
    const int chunk = i & 15, m = (i >> 4) % rows, u = (i >> 4) / rows;
    const int k = (begin + u) * kQ4Unit + 8 * chunk, left = a.K - k;
    const uint16_t* const p = a.x + (int64_t)(m0 + m) * a.ldx + k;
    lds[(u * rows + m) * 16 + (chunk ^ m)] = left >= 8 ? load16_any(p) : load16_part(p, max(left, 0));
  }
  __syncthreads();

  // the lane's row of X: operand row col is row 4 (col % 4) + col / 4.  Rows past the
  // last are the last again: no other row sees them, and they are not stored.
  const int row = min((col & 3) * 4 + (col >> 2), rows - 1);
  float acc[SIDES][MR];
#pragma unroll
  for (int s = 0; s < SIDES; ++s)
#pragma unroll
    for (int i = 0; i < MR; ++i) acc[s][i] = 0.0f;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{kCodeOne, kCodeOne, kCodeOne, kCodeOne});
  const uint32_t code_one = q4_one();
  auto work = [&](int u, const Unit& o) {
    constexpr int kSteps = 4 / kGroups;  // of 32 k, to a group
    const u32x4* const xs = lds + ((u - begin) * rows + row) * 16;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      f32x4 sx{0, 0, 0, 0}, part[SIDES];
#pragma unroll
      for (int s = 0; s < SIDES; ++s) part[s] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = g * kSteps; j < (g + 1) * kSteps; ++j) {
        const bf16x8 x = __builtin_bit_cast(bf16x8, xs[(4 * j + grp) ^ row]);
        sx = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, ones, sx, 0, 0, 0);
#pragma unroll
        for (int s = 0; s < SIDES; ++s)
          part[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, q4_decode8(o.codes[s][j], code_one), part[s], 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < SIDES; ++s) {
        const float scale = q4_scale(o.scales[s][g]), off = q4_offset(o.scales[s][g]);
#pragma unroll
        for (int i = 0; i < MR; ++i)
          acc[s][i] = __builtin_fmaf(scale, __builtin_fmaf(off, sx[i], part[s][i]), acc[s][i]);
      }
    }
  };
  if (first < end) {
    for (int u = first;;) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        work(u, ring[n]);
        if ((u += kTurns) >= end) goto done;
        __builtin_amdgcn_sched_barrier(0);
        load(u + (kAhead - 1) * kTurns, ring[n]);
      }
    }
  }
done:
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int s = 0; s < SIDES; ++s)
#pragma unroll
    for (int i = 0; i < MR; ++i)
      sums[((wave * SIDES + s) * MR * 4 + 4 * i + grp) * 16 + col] = acc[s][i];
  __syncthreads();
  for (int t = threadIdx.x; t < rows * 16 * C; t += kWaves * 64) {
    const int c = t / 16 % C, m = t / (16 * C), n = (tile0 + c) * kQ4Columns + t % 16;
    if (n >= a.N) continue;
    float v[SIDES];
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
      v[s] = 0.0f;
#pragma unroll
      for (int w = 0; w < kTurns; ++w)
        v[s] += sums[(((w * C + c) * SIDES + s) * MR * 4 + m) * 16 + t % 16];
    }
    if (a.splits == 1) {
      q4_store(a, SIDES, m0 + m, n, v[0], v[SIDES - 1]);
    } else {  // (one group of rows)
#pragma unroll
      for (int s = 0; s < SIDES; ++s)
        a.part[(int64_t)((blockIdx.y * SIDES + s) * a.M + m) * a.N + n] = v[s];
    }
  }
}

template <int SIDES, int GROUP, int MR>
hipError_t launch(const Q4Args& args, const Q4Plan& plan, hipStream_t stream) {
  Q4Args a = args;
  void* params[] = {&a};
  const void* fn = plan.tiles == 1   ? reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, MR, 1>)
                   : plan.tiles == 2 ? reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, MR, 2>)
                                     : reinterpret_cast<const void*>(&q4_gemv_kernel<SIDES, GROUP, MR, 4>);
  const size_t lds =
      std::max((size_t)a.stages * std::min(a.M, 16) * 256, (size_t)kWaves * SIDES * MR * 256);
  // beyond 64 KiB, once per kernel and device
  static std::atomic<uint64_t> set[3];
  hipError_t e = hipSuccess;
  if (lds > 65536) e = ensure_dynamic_lds(fn, 163840, set[plan.tiles / 2]);
  if (e != hipSuccess) return e;
  e = hipLaunchKernel(fn, dim3((unsigned)((a.tiles + plan.tiles - 1) / plan.tiles), (unsigned)a.splits,
                           (unsigned)((a.M + 15) / 16)),
                      dim3(kWaves * 64), params, lds, stream);
  return e != hipSuccess || a.splits == 1 ? e : llk_launch_q4_join(a, SIDES, stream);
}
template <int SIDES, int GROUP>
hipError_t launch_rows(const Q4Args& a, const Q4Plan& p, hipStream_t s) {
  return a.M <= 4    ? launch<SIDES, GROUP, 1>(a, p, s)
         : a.M <= 8  ? launch<SIDES, GROUP, 2>(a, p, s)
         : a.M <= 12 ? launch<SIDES, GROUP, 3>(a, p, s)
                     : launch<SIDES, GROUP, 4>(a, p, s);
}
template <int SIDES>
hipError_t launch_group(const Q4Args& a, const Q4Plan& p, hipStream_t s) {
  return a.group == 32   ? launch_rows<SIDES, 32>(a, p, s)
         : a.group == 64 ? launch_rows<SIDES, 64>(a, p, s)
                         : launch_rows<SIDES, 128>(a, p, s);
}

}  // namespace
}  // namespace llk_gfx950

// The kernel for 16 rows streams the weights once for them; the tile kernel shares
// them among 32 or 64.  The figures are us a call in a replayed graph, the second
// kernel of a split K included, on weights that come from HBM, groups of 128 where
// nothing else is said.
Q4Plan llk_plan_q4(int64_t M, int64_t N, int64_t K, int sides) {
  const int64_t units = std::max<int64_t>(1, q4_units(K));
  Q4Plan p{};
  if (M == 0 || N == 0) return p;  // no launch
  int64_t s;  // splits of K
  const int64_t columns = q4_tiles(N);
  if (M <= 16 || K < 8) {  // (the tile kernel reads 8 elements of a row at once)
    // A workgroup's X takes 256 M bytes a unit of K.  Without a split of K a call is one
    // launch, about 3 us less than with the kernel that joins them; the columns are
    // then a launch's only parallelism, so that few tiles go to a workgroup.  1, 2 and
    // 4 tiles: 4096 x 4096, 1 row, 4.6, 5.6, 7.8; 4096 x 14336, 1 row, 9.1, 8.6, 8.8, 8
    // rows 14.8, 11.4, 10.8; SwiGLU of it, 1 row, 14.7, 13.9, 13.1, 8 rows 20.3, 15.5,
    // 15.0.  Near the limits the next choice may be a tenth faster: 4096 x 10240, 1 row,
    // 7.5, 8.3, 8.5; SwiGLU of 4096 x 11008, 1 row, 12.1, 13.2, 12.0.
    p.rows = 16;
    const bool two = sides == 2;
    const int64_t x = std::min<int64_t>(M, 16) * units, four = (columns + 3) / 4;
    if (x <= 256 || (x <= 640 && two && four >= 200)) {
      // (640 is all of a CU's LDS: SwiGLU of 5120 x 13824, 16 rows, 19.9, split by 2
      // 23.1, by 3 26.0)
      p.tiles = two && columns >= 800 ? 4 : columns >= (two ? 400 : 640) ? 2 : 1;
      s = 1;
    } else {
      // Two workgroups to a CU, 4 tiles each, at least 8 units.  13824 x 5120, 5 rows: 1
      // tile, 1 split 20.7, 2 tiles, 3 splits 14.6, 4 tiles, 6 splits 13.8; 16 rows, 3
      // splits with 1, 2 and 4 tiles 32.6, 23.1, 18.0, 4 tiles, 6 splits 16.8.  4096 x
      // 4096, 16 rows: 2 tiles, 2 splits 9.2, 4 and 4 8.3.
      p.tiles = 4;
      s = std::max((x + 319) / 320, std::min(480 / four, units / 8));
    }
  } else {
    // 64 rows read the codes half as often, 32 leave more workgroups that hide their
    // waits.  32 and 64: 4096 x 4096, 64 rows, 15.0, 18.6, 128 rows 20.7, 23.0; 13824 x
    // 5120, 128 rows, 36.0, 36.8, 255 rows 59.7, 56.1, 512 rows 145, 98; groups of 32,
    // 128 rows, 49.1, 50.6 (with 8 registers spilled), 255 rows 86, 82, groups of 64 41.1,
    // 40.0, 69, 62; SwiGLU of 4096 x 14336, 64 rows, 32.3, 33.6, 255 rows 87, 75.  Between
    // 129 and 192 rows it goes by how many workgroups there are: 129 rows, 4096 x 4096,
    // 21.8, 26.4; 13824 x 5120 40.2, 44.1; 5120 x 13824 57.7, 47.5.
    p.rows = M <= 128 ? 32 : 64;
    const int64_t tiles = (M + p.rows - 1) / p.rows * ((N * sides + 255) / 256);
    // Two workgroups to a CU, at least 4 units to each.  SwiGLU of 4096 x 14336, 32 rows:
    // 448 workgroups 21.7, 672 25.3, 896 27.0; 13824 x 5120, 17 rows, 440 17.6, 540 20.3,
    // 720 19.0.
    s = std::clamp<int64_t>(512 / std::max<int64_t>(tiles, 1), 1, std::max<int64_t>(1, units / 4));
  }
  p.stages = (int)((units + s - 1) / s);
  p.splits = (int)((units + p.stages - 1) / p.stages);
  p.groups = p.rows == 16 ? std::max((columns + p.tiles - 1) / p.tiles, (M + 15) / 16 * 256)
                          : (M + p.rows - 1) / p.rows * ((N * sides + 255) / 256) * p.splits;
  p.bytes = p.splits > 1 ? (size_t)p.splits * sides * M * N * sizeof(float) : 0;
  return p;
}

hipError_t llk_launch_q4(const Q4Args& args, int sides, const Q4Plan& plan, hipStream_t stream) {
  using namespace llk_gfx950;
  Q4Args a = args;
  a.splits = plan.splits;
  a.stages = plan.stages;
  a.tiles = (int)q4_tiles(a.N);
  if (plan.rows > 16) return llk_launch_q4_tile(a, sides, plan.rows, stream);
  return sides == 2 ? launch_group<2>(a, plan, stream) : launch_group<1>(a, plan, stream);
}
