// q4_tile.hip -- products of more than 16 rows with 4-bit weights (q4.h): the
// mathematics of q4_gemv.hip, 32 or 64 rows to a workgroup.
//
// Four waves share the rows, each with 64 columns of its own (32 of each side of a
// SwiGLU), whose codes it takes from memory straight into operands, a unit of 128 k
// ahead.  X goes through LDS in operand order, two buffers in turn, and with it the
// sums of each row over a group, which the threads that move X add up on the way.
//
// What bounds it from 64 rows on are the vector and the matrix instructions, which
// take turns: 13824 x 5120, 255 rows, 52 us (700 TFLOP/s; the kernel without the one
// that joins its splits, 9), vector 47% and matrix 36% of a SIMD's cycles; a column
// tile's sums and the next one's conversions between the products of one, in a given
// order, measured 8% more.  SwiGLU of 5120 x 13824, 17 rows, groups of 32, 26 us (and 5
// to join): the scales and zeros of 32 rows each 32 k; codes two units ahead measured 4%
// more.
#include <algorithm>

#include "common.h"
#include "q4.h"

namespace llk_gfx950 {
namespace {

constexpr int kWaves = 4, kTiles = 4;  // column tiles of a wave

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Sum of 8 bf16.
__device__ __forceinline__ float sum8(const u32x4& x) {
  const bf16x2 one = __builtin_bit_cast(bf16x2, kCodeOne);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t two = x[i];  // (a bit cast of the element itself would take the first)
    s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), one, s, false);
  }
  return s;
}
template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true));
}

template <int SIDES, int GROUP, int RT>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(2))) q4_tile_kernel(Q4Args a) {
  constexpr int kRows = 16 * RT, kGroups = kQ4Unit / GROUP, kSteps = 4 / kGroups;
  constexpr int kColumns = kWaves * kTiles * 16 / SIDES;  // of a side
  // X: [step of 32 k][row tile][lane] of 16 bytes, a lane's place within its 16 turned
  // by the chunk's number, so that the chunks of a row, which 16 threads write, meet
  // different banks
  __shared__ __attribute__((aligned(16))) u32x4 xs[2][4 * RT * 64];
  __shared__ __attribute__((aligned(16))) float sums[2][kGroups][kRows];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int tiles_m = (a.M + kRows - 1) / kRows, tiles_n = (a.N + kColumns - 1) / kColumns;
  const int id = xcd_remap(blockIdx.x, tiles_m * tiles_n * a.splits);
  const int m0 = id % tiles_m * kRows, n0 = id / tiles_m % tiles_n * kColumns;
  const int split = id / (tiles_m * tiles_n);
  const int units = (a.K + kQ4Unit - 1) / kQ4Unit;
  const int begin = split * a.stages, end = min(begin + a.stages, units);

  // The wave's column tiles; past N its last one's again (not stored).  Codes and
  // scales through buffers of the tiles: units past their last read as zeros, without
  // a branch that would have every load waited for.
  __amdgpu_buffer_rsrc_t codes[kTiles], scales[kTiles];
#pragma unroll
  for (int c = 0; c < kTiles; ++c) {
    const Q4Side& side = a.side[c / (kTiles / SIDES)];
    const int64_t tile =
        (int64_t)min(n0 / 16 + wave * (kTiles / SIDES) + c % (kTiles / SIDES), a.tiles - 1) * units;
    codes[c] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(side.codes + tile * kQ4UnitBytes),
                                                 0, units * kQ4UnitBytes, kBufferWord3);
    scales[c] = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint32_t*>(side.scales + tile * kGroups * kQ4Columns), 0,
        units * kGroups * kQ4Columns * 4, kBufferWord3);
  }
  struct Codes {
    u32x4 q[kTiles];
    uint32_t s[kTiles][kGroups];
  };
  auto load_codes = [&](int u, Codes& o) {
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
      o.q[c] = __builtin_amdgcn_raw_buffer_load_b128(codes[c], u * kQ4UnitBytes + lane * 16, 0, 0);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        o.s[c][g] = __builtin_amdgcn_raw_buffer_load_b32(
            scales[c], ((u * kGroups + g) * kQ4Columns + col) * 4, 0, 0);
    }
  };
  // X: thread t moves chunk t % 16 (8 k) of rows t / 16 + 16 i; rows past M are the
  // last one again.  A chunk past K is read where K ends, and put right as it is placed.
  const int chunk = t & 15, xrow = t >> 4;
  const uint16_t* xp[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) xp[i] = a.x + (int64_t)min(m0 + xrow + 16 * i, a.M - 1) * a.ldx;
  auto load_x = [&](int u, u32x4 (&x)[RT]) {  // (K >= 8)
    const int at = min(u * kQ4Unit + 8 * chunk, a.K - 8);
#pragma unroll
    for (int i = 0; i < RT; ++i) x[i] = load16_any(xp[i] + at);
  };
  auto end_x = [&](int u, u32x4 (&x)[RT]) {  // of the unit that K ends in
    const int past = u * kQ4Unit + 8 * chunk - (a.K - 8);  // elements
    if (past <= 0) return;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      u32x4 v = past >= 8 ? u32x4{0, 0, 0, 0} : x[i];
      if (past & 4) v = u32x4{v[2], v[3], 0, 0};
      if (past & 2) v = u32x4{v[1], v[2], v[3], 0};
      if (past & 1)
        v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
      x[i] = v;
    }
  };
  auto place_x = [&](int buf, const u32x4 (&x)[RT]) {
    const int step = chunk >> 2, quarter = chunk & 3;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      xs[buf][(step * RT + i) * 64 + quarter * 16 + (xrow ^ chunk)] = x[i];
      // over the 16 threads of the row, or 8 or 4 of them
      float s = sum8(x[i]);
      s = add_dpp<0xB1>(s);  // quad_perm: lane ^ 1
      s = add_dpp<0x4E>(s);  // lane ^ 2
      if constexpr (GROUP >= 64) s = add_dpp<0x141>(s);   // row_half_mirror
      if constexpr (GROUP >= 128) s = add_dpp<0x140>(s);  // row_mirror
      if (chunk % (GROUP / 8) == 0) sums[buf][chunk / (GROUP / 8)][xrow + 16 * i] = s;
    }
  };

  f32x4 acc[RT][kTiles];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < kTiles; ++c) acc[r][c] = f32x4{0, 0, 0, 0};
  const uint32_t code_one = q4_one();
  auto work = [&](int buf, const Codes& w) {
    bf16x8 x[2][RT];  // operands of a step, the next one's on their way
    auto read = [&](int j) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
        x[j & 1][r] =
            __builtin_bit_cast(bf16x8, xs[buf][(j * RT + r) * 64 + grp * 16 + (col ^ (4 * j + grp))]);
    };
    read(0);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      f32x4 part[RT][kTiles];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < kTiles; ++c) part[r][c] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = g * kSteps; j < (g + 1) * kSteps; ++j) {
        if (j < 3) read(j + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
          const bf16x8 q = q4_decode8(w.q[c][j], code_one);
#pragma unroll
          for (int r = 0; r < RT; ++r)
            part[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[j & 1][r], q, part[r][c], 0, 0, 0);
        }
      }
      f32x4 sx[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r)
        sx[r] = *reinterpret_cast<const f32x4*>(&sums[buf][g][16 * r + 4 * grp]);
#pragma unroll
      for (int c = 0; c < kTiles; ++c) {
        const float scale = q4_scale(w.s[c][g]), off = q4_offset(w.s[c][g]);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[r][c][i] =
                __builtin_fmaf(scale, __builtin_fmaf(off, sx[r][i], part[r][c][i]), acc[r][c][i]);
      }
    }
  };

  Codes even, odd;
  u32x4 x[RT];
  load_x(begin, x);
  __builtin_amdgcn_sched_barrier(0);  // loads in order, so that the oldest can be waited for
  load_codes(begin, even);
  // (two units to a turn: no loaded register is copied, which would wait for it)
  auto unit = [&](int u, int buf, const Codes& now, Codes& next) {
    if ((u + 1) * kQ4Unit > a.K) end_x(u, x);
    place_x(buf, x);  // its readers of two units ago are past the barrier of the last
    __syncthreads();
    load_x(u + 1, x);
    __builtin_amdgcn_sched_barrier(0);
    load_codes(u + 1, next);
    __builtin_amdgcn_sched_barrier(0);
    work(buf, now);
  };
  for (int u = begin;;) {
    unit(u, 0, even, odd);
    if (++u == end) break;
    unit(u, 1, odd, even);
    if (++u == end) break;
  }

  // lane: column col of each tile, rows 4 grp + i
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + 16 * r + 4 * grp + i;
      if (m >= a.M) continue;
#pragma unroll
      for (int c = 0; c < kTiles / SIDES; ++c) {
        const int n = n0 + (wave * (kTiles / SIDES) + c) * 16 + col;
        if (n >= a.N) continue;
        const float v = acc[r][c][i], w = acc[r][c + (SIDES - 1) * (kTiles / 2)][i];
        if (a.splits == 1) {
          q4_store(a, SIDES, m, n, v, w);
        } else {
          const int64_t plane = (int64_t)a.M * a.N, at = (int64_t)m * a.N + n;
          a.part[split * SIDES * plane + at] = v;
          if (SIDES == 2) a.part[(split * SIDES + 1) * plane + at] = w;
        }
      }
    }
}

// Joins the splits in their order.
template <int SIDES>
__global__ void __launch_bounds__(256) q4_join_kernel(Q4Args a) {
  const int64_t plane = (int64_t)a.M * a.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < plane; i += (int64_t)gridDim.x * 256) {
    float v[2] = {};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
      for (int k = 0; k < SIDES; ++k) v[k] += a.part[(s * SIDES + k) * plane + i];
    q4_store(a, SIDES, (int)(i / a.N), (int)(i % a.N), v[0], v[SIDES - 1]);
  }
}

template <int SIDES, int RT>
hipError_t launch(const Q4Args& args, hipStream_t stream) {
  Q4Args a = args;
  void* params[] = {&a};
  const void* fn = a.group == 32   ? reinterpret_cast<const void*>(&q4_tile_kernel<SIDES, 32, RT>)
                   : a.group == 64 ? reinterpret_cast<const void*>(&q4_tile_kernel<SIDES, 64, RT>)
                                   : reinterpret_cast<const void*>(&q4_tile_kernel<SIDES, 128, RT>);
  constexpr int kColumns = kWaves * kTiles * 16 / SIDES;
  const int64_t groups = (int64_t)((a.M + 16 * RT - 1) / (16 * RT)) * ((a.N + kColumns - 1) / kColumns) *
                         a.splits;
  const hipError_t e =
      hipLaunchKernel(fn, dim3((unsigned)groups), dim3(kWaves * 64), params, 0, stream);
  return e != hipSuccess || a.splits == 1 ? e : llk_launch_q4_join(a, SIDES, stream);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_q4_join(const Q4Args& args, int sides, hipStream_t stream) {
  using namespace llk_gfx950;
  Q4Args a = args;
  void* params[] = {&a};
  const int64_t all = ((int64_t)a.M * a.N + 255) / 256;
  return hipLaunchKernel(sides == 2 ? reinterpret_cast<const void*>(&q4_join_kernel<2>)
                                    : reinterpret_cast<const void*>(&q4_join_kernel<1>),
                         dim3((unsigned)std::min<int64_t>(all, 1 << 16)), dim3(256), params, 0, stream);
}

hipError_t llk_launch_q4_tile(const Q4Args& a, int sides, int rows, hipStream_t s) {
  using namespace llk_gfx950;
  if (sides == 2) return rows == 32 ? launch<2, 2>(a, s) : launch<2, 4>(a, s);
  return rows == 32 ? launch<1, 2>(a, s) : launch<1, 4>(a, s);
}
