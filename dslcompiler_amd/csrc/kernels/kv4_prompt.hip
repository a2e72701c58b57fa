// kv4_prompt.hip -- attention over the 4-bit cache for many rows (prompts and
// chunks of them): see kv4_attention.hip for the mathematics and the operands'
// order.
//
// A workgroup's 4 waves share 128 rows, 32 each, and step through the same
// keys, 64 at a time: every wave converts 16 keys and values from codes to bf16
// into LDS, where all four read them as operands.  Two buffers, so one barrier
// a step, and the codes of the step after next are on their way meanwhile.
#include "kv4_attention.h"

namespace llk_gfx950 {
namespace {

constexpr int kWaves = 4, kRT = 2, kRows = kKv4PromptRows, kTiles = 4;
constexpr int kStep = 16 * kTiles;
static_assert(kRows == kWaves * kRT * 16 && kStep == kv4_step(kRows), "row tile");

constexpr uint8_t kAbsent = 1, kNan = 2;
constexpr uint32_t kEveryTile = 0x01010101u;  // times a flag: that flag of every tile

template <int D>
struct PromptLds {
  uint8_t k[2][kStep * D * 2];  // [16-key tile][D / 32][64 lanes] of 16 bytes: A operands
  uint8_t v[2][kStep * D * 2];  // v_chunk
  // of each 16-key tile: lanes that hold part of a NaN block, and what a step
  // looks at first, kAbsent (its page does not exist) and kNan
  uint64_t nan[2][kTiles][TileCodes<D>::kScales];
  uint8_t flags[2][kTiles];
};

template <int D>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) kv4_prompt_kernel(Kv4AttentionArgs a) {
  constexpr int kD16 = D / 16, kJ = D / 32;
  __shared__ __attribute__((aligned(16))) PromptLds<D> lds;
  using Codes = TileCodes<D>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.y;
  const int head = blockIdx.x % a.cache.heads;
  // the last tiles, of the most keys, first; then the others from the first on,
  // so that the two workgroups a CU gets in one round have much and little to do
  const int nth = blockIdx.x / a.cache.heads;
  const int tile = 2 * nth < a.tiles ? a.tiles - 1 - nth : nth - (a.tiles + 1) / 2;
  RowTile rt;
  if (!row_tile<kRows>(a, tile, &rt)) return;
  const int used = used_splits(a, rt.steps);
  if (split >= used) return;
  const int begin = split * a.chunk;
  const int end = split == used - 1 ? rt.steps : begin + a.chunk;
  const int col = lane & 15, grp = lane >> 4;

  // Q: the lane's row of each of the wave's 16-row tiles
  const int wrow = wave * kRT * 16;
  bf16x8 q[kRT][kJ];
  int pos[kRT];
#pragma unroll
  for (int y = 0; y < kRT; ++y) {
    const int r = wrow + y * 16 + col;
    const int row = rt.row0 + (r < rt.rows ? r : 0);
    const int i = row / a.group, h = head * a.group + row % a.group;
    pos[y] = min(rt.first + i, rt.p_hi);
    const uint16_t* src = a.q + (int64_t)(rt.token0 + i) * a.q_token + (int64_t)h * a.q_head;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
      q[y][j] = __builtin_bit_cast(bf16x8, load16_any(src + Codes::element(j, lane)));
  }
  // positions of the wave's first and last row
  const int last = min(wrow + kRT * 16, rt.rows) - 1;
  const int w_lo = rt.first + (rt.row0 + wrow) / a.group;
  const int w_hi = last < wrow ? -1 : min(rt.first + (rt.row0 + last) / a.group, rt.p_hi);

  f32x4 o[kRT][kD16];
  float m[kRT], l[kRT];
#pragma unroll
  for (int y = 0; y < kRT; ++y) {
    m[y] = kNegInf, l[y] = 0.0f;
#pragma unroll
    for (int d = 0; d < kD16; ++d) o[y][d] = f32x4{0, 0, 0, 0};
  }

  const int page_mask = (1 << a.cache.page_shift) - 1;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;
  const int32_t* const table = a.batch.table + rt.s * a.batch.table_stride;
  auto key0 = [&](int step) { return (step < rt.sink ? step : step - rt.sink + rt.low) * kStep; };
  // the wave's 16 keys of a step
  auto fetch = [&](int step, Codes& c) {
    const int key = key0(step) + 16 * wave;
    int id = -1;
    if (key <= rt.p_hi) id = table[key >> a.cache.page_shift];
    c.present = id >= 0 && id < a.cache.pages;
    if (c.present)
      c.load(base + id * a.cache.page_stride + (int64_t)((key & page_mask) >> 4) * (17 * D), lane);
    else
      c.clear();
  };
  auto place = [&](int step, int buf, const Codes& c) {
    const bool past = key0(step) + 16 * wave + col > rt.p_hi;
    float ks[Codes::kScales], vs[Codes::kScales];
    uint64_t nan[Codes::kScales];
#pragma unroll
    for (int i = 0; i < Codes::kScales; ++i) {
      const uint32_t e = past ? 0u : c.vs[i];
      nan[i] = __ballot(e > 252u);
      vs[i] = __uint_as_float(e > 252u ? 0u : e << 23);
      ks[i] = __uint_as_float(c.ks[i] << 23);
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      *reinterpret_cast<bf16x8*>(lds.k[buf] + ((wave * kJ + j) * 64 + lane) * 16) =
          decode8(c.k[j], ks[Codes::scale_of(j)]);
      const int d = Codes::element(j, lane);
      *reinterpret_cast<bf16x8*>(lds.v[buf] + v_chunk<D>(wave, d >> 4, (d >> 3) & 1, col)) =
          decode8(c.v[j], vs[Codes::scale_of(j)]);
    }
    if (lane == 0) {
      uint64_t any = 0;
#pragma unroll
      for (int i = 0; i < Codes::kScales; ++i) any |= lds.nan[buf][wave][i] = nan[i];
      lds.flags[buf][wave] = (c.present ? 0 : kAbsent) | (any ? kNan : 0);
    }
  };

  Codes codes;
  if (begin < end) {
    fetch(begin, codes);
    place(begin, 0, codes);
    if (begin + 1 < end) fetch(begin + 1, codes);
  }
  __syncthreads();
  for (int step = begin; step < end; ++step) {
    const int buf = (step - begin) & 1;
    const int k0 = key0(step);
    // some row of the wave sees some key of the step
    const bool any = k0 <= w_hi &&
                     (!a.window || k0 + kStep - 1 > w_lo - a.window || k0 < a.sinks);
    if (any) {
      const uint32_t flags = __builtin_amdgcn_readfirstlane(
          *reinterpret_cast<const uint32_t*>(lds.flags[buf]));
      // every row sees every key
      const bool whole = k0 + kStep - 1 <= w_lo && !(flags & kAbsent * kEveryTile) &&
                         (!a.window || k0 > w_hi - a.window || k0 + kStep <= a.sinks);
      f32x4 st[kRT][kTiles];
      bf16x8 k[2][kJ];  // of this tile, and of the next, on its way
      auto read_k = [&](int x) {
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          k[x & 1][j] =
              *reinterpret_cast<const bf16x8*>(lds.k[buf] + ((x * kJ + j) * 64 + lane) * 16);
      };
      read_k(0);
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        if (x + 1 < kTiles) read_k(x + 1);
#pragma unroll
        for (int y = 0; y < kRT; ++y) st[y][x] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
          for (int y = 0; y < kRT; ++y)
            st[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[x & 1][j], q[y][j], st[y][x], 0, 0, 0);
      }
      bf16x8 p[kRT][kTiles / 2];
#pragma unroll
      for (int y = 0; y < kRT; ++y) {
        if (!whole) {
#pragma unroll
          for (int x = 0; x < kTiles; ++x) {
            const bool here = !(flags >> 8 * x & kAbsent);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              st[y][x][r] =
                  here && sees(a, pos[y], k0 + 16 * x + 4 * grp + r) ? st[y][x][r] : kNegInf;
          }
        }
        float top = m[y];
#pragma unroll
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, st[y][x][r]);
        if (__any(outgrown(a, top, m[y]))) {
          top = max_over_groups(top);
          const float alpha = rescale(a, top, m[y]);
          m[y] = top;
          l[y] *= alpha;
#pragma unroll
          for (int d = 0; d < kD16; ++d) o[y][d] *= alpha;
        }
        const float shift = m[y] == kNegInf ? 0.0f : m[y] * a.scale;
#pragma unroll
        for (int h = 0; h < kTiles / 2; ++h) {
          float e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            e[i] = __builtin_amdgcn_exp2f(
                __builtin_fmaf(st[y][2 * h + (i >> 2)][i & 3], a.scale, -shift));
            l[y] += e[i];
          }
          p[y][h] = __builtin_bit_cast(
              bf16x8, u32x4{f32x2_to_bf16x2_rne(e[0], e[1]), f32x2_to_bf16x2_rne(e[2], e[3]),
                            f32x2_to_bf16x2_rne(e[4], e[5]), f32x2_to_bf16x2_rne(e[6], e[7])});
        }
      }
      const int vkey = 4 * grp + (col >> 2), vhalf = (col >> 1) & 1;
#pragma unroll
      for (int h = 0; h < kTiles / 2; ++h)
#pragma unroll
        for (int d = 0; d < kD16; ++d) {
          v4i16 part[2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
            part[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_v4i16)(lds.v[buf] + v_chunk<D>(2 * h + x, d, vhalf, vkey) + (col & 1) * 8));
          const bf16x8 v = __builtin_bit_cast(
              bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int y = 0; y < kRT; ++y)
            o[y][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[y][h], o[y][d], 0, 0, 0);
        }
      if (flags & kNan * kEveryTile) {
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
          for (int c = 0; c < Codes::kScales; ++c)
#pragma unroll
            for (int y = 0; y < kRT; ++y)
              add_nan<D>(a, lds.nan[buf][x][c], c, k0 + 16 * x, pos[y], o[y]);
      }
    }
    if (step + 1 < end) {
      place(step + 1, buf ^ 1, codes);
      if (step + 2 < end) fetch(step + 2, codes);
    }
    __syncthreads();
  }

  float* const part = used > 1 ? part_of<D, kRows>(a, tile, head, split) : nullptr;
#pragma unroll
  for (int y = 0; y < kRT; ++y) {
    const int r = wrow + y * 16 + col;
    Joined sum(m[y]);
    sum.l = sum_over_groups(l[y]);
    if (r >= rt.rows) continue;
    if (part && grp == 0) part[kRows * D + r] = sum.m, part[kRows * (D + 1) + r] = sum.l;
#pragma unroll
    for (int d = 0; d < kD16; ++d) {
      if (part) {
        *reinterpret_cast<f32x4*>(part + r * D + d * 16 + 4 * grp) = o[y][d];
      } else {
        sum.o = o[y][d];
        sum.store(a, rt, head, r, d * 16 + 4 * grp);
      }
    }
  }
}

template <int D>
hipError_t prompt(const Kv4AttentionArgs& args, hipStream_t s) {
  Kv4AttentionArgs a = args;
  void* params[] = {&a};
  return hipLaunchKernel(reinterpret_cast<const void*>(&kv4_prompt_kernel<D>),
                         dim3((unsigned)(a.tiles * a.cache.heads), (unsigned)a.splits),
                         dim3(kWaves * 64), params, 0, s);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_prompt(const Kv4AttentionArgs& a, int D, hipStream_t s) {
  using namespace llk_gfx950;
  return D == 64 ? prompt<64>(a, s) : D == 128 ? prompt<128>(a, s) : prompt<256>(a, s);
}
