// kv4_prompt.hip -- attention over the 4-bit cache for many rows (prompts and
// chunks of them): the mathematics of kv4_attention.hip on 32 x 32 tiles
// (v_mfma_f32_32x32x16_bf16).
//
// Four waves share 128 rows, 32 each, and step through the same keys, 64 at a
// time: every wave converts 16 keys and values from codes to bf16 into LDS,
// where all four read them as operands, while the next step's codes are on their
// way.
//
// At D = 128 a step takes 1.4 us where a workgroup has its CU to itself and 2.1 us
// where two share it, which is what the registers leave room for: 1.05 us a step.
// With CUs kept full by equal tiles that is 940 TFLOP/s (2048 tokens of 32 heads
// over 6080 keys each: 218 us).  The tiles of a causal prompt are not equal: 2048
// tokens of 32 heads, 2 to 32 steps, take 53 us, 650 TFLOP/s of what causality
// leaves and no less than 16 heads do, since the longest tiles run most of their
// steps alone on their CU (6 us go by until a tile's first step is done); 8192
// tokens, whose tiles refill the CUs, 890.  Over the prompt of 2048 matrix units are
// busy 33% of the time, vector 38%, LDS 26%.  Two buffers in turn, 8 waves, 128 keys
// a step, wave priorities and other orders of the instructions measured no less.
#include <type_traits>

#include "kv4_attention.h"

namespace llk_gfx950 {
namespace {

constexpr int kRows = kKv4PromptRows, kTiles = 4;  // 16-key tiles of a step = waves of a group
constexpr int kStep = 16 * kTiles;
static_assert(kRows == kTiles * 32 && kStep == kv4_step(kRows), "row tile");

template <int D>
struct PromptLds {
  uint8_t k[kStep * D * 2];  // [32 keys][D / 16][64 lanes] of 16 bytes: A operands
  uint8_t v[kStep * D * 2];  // v_chunk
  // of each 16-key tile: lanes that hold part of a NaN block of V; bit 0 of
  // the flags: its page does not exist, bit 1: there is such a lane
  uint64_t nan[kTiles][TileCodes<D>::kScales];
  uint32_t flags[kTiles];
};

__device__ __forceinline__ float swap_max(float x) {  // over lane and lane ^ 32
  const auto r =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_sum(float x) {
  const auto r =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D>
__global__ void __launch_bounds__(kTiles * 64)
    __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) kv4_prompt_kernel(Kv4AttentionArgs a) {
  constexpr int kU = D / 16, kD32 = D / 32, kJ = D / 32;
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
  // a lane's row of S^T and O^T, and which 4 of every 8 keys (values) it holds;
  // its token and group of the codes
  const int lrow = lane & 31, half = lane >> 5, col = lane & 15;

  bf16x8 q[kU];
  int pos;
  {
    const int r = wave * 32 + lrow, row = rt.row0 + (r < rt.rows ? r : 0);
    const int token = row / a.group, qhead = head * a.group + row % a.group;
    pos = rt.first + token;
    const uint16_t* src =
        a.q + (int64_t)(rt.token0 + token) * a.q_token + (int64_t)qhead * a.q_head + half * 8;
#pragma unroll
    for (int u = 0; u < kU; ++u) q[u] = __builtin_bit_cast(bf16x8, load16_any(src + u * 16));
  }
  // positions of the wave's first and last row
  const int last = max(min(wave * 32 + 32, rt.rows) - 1, 0);
  const int w_lo = rt.first + (rt.row0 + min(wave * 32, last)) / a.group;
  const int w_hi = rt.first + (rt.row0 + last) / a.group;

  f32x16 o[kD32];
  float m = kNegInf, l = 0.0f;
#pragma unroll
  for (int d = 0; d < kD32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

  const int page_mask = (1 << a.cache.page_shift) - 1;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;
  const int32_t* const table = a.batch.table + rt.s * a.batch.table_stride;
  // first key of step `step`
  auto key0 = [&](int step) { return (step < rt.sink ? step : step - rt.sink + rt.low) * kStep; };
  // The wave converts 16 keys of a step, from the tile at k0 + 16 wave.  Its page
  // is asked for a step before its codes, by a vector load: a scalar one would
  // have every LDS wait of the step wait for it.  Where there is no page, the
  // codes are those of page 0, and no row sees them.
  auto page_of = [&](int k0) {
    const int key = k0 + 16 * wave;
    return key <= rt.p_hi ? __builtin_nontemporal_load(table + (key >> a.cache.page_shift)) : -1;
  };
  auto fetch = [&](int k0, int page, Codes& c) {
    const int id = __builtin_amdgcn_readfirstlane(page);
    c.present = id >= 0 && id < a.cache.pages;
    c.template load<false>(base + (c.present ? id : 0) * a.cache.page_stride +
                               (((k0 + 16 * wave) & page_mask) >> 4) * (17 * D),
                           lane);
  };
  // where the lane's first 8 values go
  const int kto = (((wave >> 1) * kU + (Codes::element(0, lane) >> 4)) * 64 +
                   (Codes::element(0, lane) >> 3 & 1) * 32 + (wave & 1) * 16 + col) * 16;
  uint64_t nan[Codes::kScales];
  auto place = [&](int k0, const Codes& c) {
    const bool past = !c.present || k0 + 16 * wave + col > rt.p_hi;
    float ks[Codes::kScales], vs[Codes::kScales];
#pragma unroll
    for (int i = 0; i < Codes::kScales; ++i) {
      const uint32_t e = past ? 0u : c.vs[i];
      nan[i] = __ballot(e > 252u);
      vs[i] = __uint_as_float(e > 252u ? 0u : e << 23);
      ks[i] = __uint_as_float(c.ks[i] << 23);
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int d = Codes::element(j, lane);
      *reinterpret_cast<bf16x8*>(lds.k + kto + (Codes::element(j, 0) >> 4) * 1024 + (j & 1) * 512) =
          decode8(c.k[j], ks[Codes::scale_of(j)]);
      *reinterpret_cast<bf16x8*>(lds.v + v_chunk<D>(wave, d >> 4, j & 1, col)) =
          decode8(c.v[j], vs[Codes::scale_of(j)]);
    }
  };
  // what the waves have to know of the tile placed last
  auto note = [&](bool present) {
    uint64_t any = 0;
#pragma unroll
    for (int i = 0; i < Codes::kScales; ++i) any |= nan[i];
    if (lane == 0) {
      lds.flags[wave] = (present ? 0 : 1) | (any ? 2 : 0);
#pragma unroll
      for (int i = 0; i < Codes::kScales; ++i) lds.nan[wave][i] = nan[i];
    }
  };

  // First keys of this step and the next two: the codes of the one and the page
  // of the other are on their way.
  Codes codes;
  int k0 = key0(begin), k1 = key0(begin + 1);
  fetch(k0, page_of(k0), codes);
  int page = page_of(k1);
  // Where the lane's operands lie in a buffer: K, and V's two halves (v_chunk's
  // swap apart, a constant step from one 32 values to the next).
  const int vkey = 4 * half + (col >> 2), vhalf = (col >> 1) & 1, vsub = (lane >> 4) & 1;
  const int kat = lane * 16;
  const int vat[2] = {v_chunk<D>(0, vsub, vhalf, vkey) + (col & 1) * 8,
                      v_chunk<D>(0, vsub, vhalf, vkey + 8) + (col & 1) * 8};
  // One step.
  auto work = [&] {
    const u32x4 tile_flags = *reinterpret_cast<const u32x4*>(lds.flags);
#pragma unroll
    for (int x = 0; x < 2; ++x) {  // 32 keys each
      f32x16 st;
#pragma unroll
      for (int e = 0; e < 16; ++e) st[e] = 0.0f;
#pragma unroll
      for (int u = 0; u < kU; ++u)
        st = mfma32(*reinterpret_cast<const bf16x8*>(lds.k + kat + (x * kU + u) * 1024), q[u], st);
      const int j0 = k0 + 32 * x;
      const uint32_t flags =
          __builtin_amdgcn_readfirstlane(tile_flags[2 * x] | tile_flags[2 * x + 1]);
      // every row sees every key
      const bool whole = j0 + 31 <= w_lo && !(flags & 1) &&
                         (!a.window || j0 > w_hi - a.window || j0 + 32 <= a.sinks);
      if (!whole) {
        auto mask = [&](auto first) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = j0 + 8 * (e >> 2) + 4 * half + (e & 3);
            st[e] = in_window(a, pos, j) || (first && j <= pos && j < a.sinks) ? st[e] : kNegInf;
          }
        };
        if (j0 < a.sinks) mask(std::true_type{});
        else mask(std::false_type{});
        if (flags & 1) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            st[e] = tile_flags[2 * x + (e >> 3)] & 1 ? kNegInf : st[e];
        }
      }
      // Keeps the scores in their registers: the compiler would take the tuple
      // apart here and copy its values on the way without a mask.
      asm("" : "+v"(st));
      float top = m;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, st[e]);
      if (__any(outgrown(a, top, m))) {
        top = swap_max(top);
        const float alpha = rescale(a, top, m);
        m = top;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < kD32; ++d) o[d] *= alpha;
      }
      const float shift = m == kNegInf ? 0.0f : m * a.scale;
      bf16x8 p[2];  // of 16 keys each
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t two[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e[2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
            e[n] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[g * 8 + 2 * i + n], a.scale, -shift));
          l += e[0];
          l += e[1];
          two[i] = f32x2_to_bf16x2_rne(e[0], e[1]);
        }
        p[g] = __builtin_bit_cast(bf16x8, u32x4{two[0], two[1], two[2], two[3]});
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int d = 0; d < kD32; ++d) {
          v4i16 part[2];
#pragma unroll
          for (int y = 0; y < 2; ++y)
            part[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_v4i16)(lds.v + vat[y] + ((2 * x + g) * kU + 2 * d) * 512));
          const bf16x8 v = __builtin_bit_cast(
              bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
          o[d] = mfma32(v, p[g], o[d]);
        }
    }
    if (__builtin_amdgcn_readfirstlane(tile_flags[0] | tile_flags[1] | tile_flags[2] |
                                       tile_flags[3]) & 2) {  // rare: see add_nan
      for (int g = 0; g < kTiles; ++g) {
        uint32_t seen = 0;
#pragma unroll 1
        for (int j = 0; j < 16; ++j) seen |= (uint32_t)sees(a, pos, k0 + 16 * g + j) << j;
#pragma unroll
        for (int d = 0; d < kD32; ++d) {
          // a lane holds values of one block (32 d on) in every register of o[d]
          const int c = D == 256 ? d >> 2 : 0;
          const uint64_t f = lds.nan[g][c];
          const uint32_t part = D == 64 ? (uint32_t)(f >> (32 * d)) | (uint32_t)(f >> (32 * d + 16))
                                        : (uint32_t)(f >> (16 * (d & 3)));
          if (part & seen & 0xffffu) o[d] += __builtin_nanf("");
        }
      }
    }
  };
  for (int step = begin; step < end; ++step) {
    __syncthreads();  // every wave is done with the step before
    place(k0, codes);
    note(codes.present);
    fetch(k1, page, codes);
    const int k2 = key0(step + 2);
    page = page_of(k2);
    __syncthreads();
    // some row of the wave sees some key of the step
    if (k0 <= w_hi && (!a.window || k0 + kStep - 1 > w_lo - a.window || k0 < a.sinks)) work();
    k0 = k1, k1 = k2;
  }

  l = swap_sum(l);
  const int r = wave * 32 + lrow;
  if (r >= rt.rows) return;
  const int token = (rt.row0 + r) / a.group;
  const int qhead = head * a.group + (rt.row0 + r) % a.group;
  // the lane's values: 32 d + 8 e + 4 half on
  if (used > 1) {
    float* const part = part_of<D, kRows>(a, tile, head, split);
    if (half == 0) part[kRows * D + r] = m, part[kRows * (D + 1) + r] = l;
#pragma unroll
    for (int d = 0; d < kD32; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(part + r * D + d * 32 + e * 8 + 4 * half) =
            f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
  } else {
    const float inv = 1.0f / l;
    if (half == 0) leave_stats(a, rt, head, rt.row0 + r, m, l);
    uint16_t* const dst = a.out + (int64_t)(rt.token0 + token) * a.out_token +
                          (int64_t)qhead * a.out_head + 4 * half;
#pragma unroll
    for (int d = 0; d < kD32; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        store8_any(dst + d * 32 + e * 8,
                   make_uint2(f32x2_to_bf16x2_rne(result(o[d][4 * e], l, inv),
                                                  result(o[d][4 * e + 1], l, inv)),
                              f32x2_to_bf16x2_rne(result(o[d][4 * e + 2], l, inv),
                                                  result(o[d][4 * e + 3], l, inv))));
  }
}

template <int D>
hipError_t prompt(const Kv4AttentionArgs& args, hipStream_t s) {
  Kv4AttentionArgs a = args;
  void* params[] = {&a};
  return hipLaunchKernel(reinterpret_cast<const void*>(&kv4_prompt_kernel<D>),
                         dim3((unsigned)(a.tiles * a.cache.heads), (unsigned)a.splits),
                         dim3(kTiles * 64), params, 0, s);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_prompt(const Kv4AttentionArgs& a, int D, hipStream_t s) {
  using namespace llk_gfx950;
  return D == 64 ? prompt<64>(a, s) : D == 128 ? prompt<128>(a, s) : prompt<256>(a, s);
}
