// kv4_attention.hip -- attention over the 4-bit paged cache (kv4.h).
//
//   out = softmax(scale q k^T, over the keys a query sees) v
//
// in one pass over the keys with a running maximum and sum.  The query heads
// of a key head and the sequence's new tokens together are the rows of a tile:
// row r is new token r / group, query head r % group.
//
// Keys and values come from the cache as codes; a key's 32-value block is one
// lane's 16 bytes, so K is converted in registers straight into the A operand
// of S^T = K Q^T (v_mfma_f32_16x16x32_bf16; any order of the D values serves as
// long as Q's is the same).  The lanes of S^T hold 4 keys of one query each,
// which is the B operand of O^T = V^T P^T once P is rounded to bf16, with the
// keys in the order the transposed LDS reads of V (ds_read_b64_tr_b16) give
// them: P never leaves its lane.  The codes' values are exact in bf16; P is
// rounded to it (by 2^-8 at most, as the result is) to run on the bf16 matrix
// instructions, while scores, maxima, sums and accumulators stay in fp32.
#include <algorithm>

#include "kv4_attention.h"

namespace llk_gfx950 {
namespace {

constexpr int kWaves = 4;  // of a workgroup, each over its own keys
constexpr int kStep = 32;  // keys to a step

// Waves to a SIMD that the registers are cut to: more have more bytes on their way
// until the registers no longer suffice.  D = 128, 16 rows: one token over 131072
// keys, 3 waves 34.8 us, 4 30.7.  Ragged sequences to 8192 keys (D = 256: 4096), 64
// with 16 rows, 32 with 32 rows, us: D = 64, 16 rows, 4 waves 52, 5 51.7, 6 49.5; 32
// rows, 3 waves 41, 5 88; D = 128, 16 rows, 3 to 5 waves 77; 32 rows, 1 wave 100, 2
// 65, 3 86; D = 256, 16 rows, 1 wave 113, 2 82, 3 112; 32 rows, 1 wave 113, 2 207.
template <int D, int RT>
constexpr int kMinWaves =
    D * RT <= 64 ? 5 : D * RT <= 128 ? (RT == 1 ? 4 : 3) : D * RT <= 256 ? 2 : 1;

// A workgroup's 4 waves share a row tile of 16 * RT rows and one split of its
// keys, each wave taking every fourth step of 32 keys with a running maximum
// of its own; at the end they are joined in LDS.
// Bound by HBM for 16 rows: 64 sequences of 4.2k keys on average (358 MB) take
// 68 us, 5.3 TB/s; one token over 131072 keys (143 MB) 28 us, 5.1 TB/s, and 4 to
// join the splits.  The codes of one row tile are read past the L2, since no
// other workgroup reads them.
// KEEP: the scores are stored too, for the call that adds the weights up.
template <int D, int RT, bool KEEP = false>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(kMinWaves<D, RT>))) kv4_attention_kernel(Kv4AttentionArgs a) {
  constexpr int R = 16 * RT, kD16 = D / 16, kJ = D / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves][kStep * D * 2];
  __shared__ float wave_m[kWaves][R], wave_l[kWaves][R];
  using Codes = TileCodes<D>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.y;
  const int head = blockIdx.x % a.cache.heads, tile = blockIdx.x / a.cache.heads;
  RowTile rt;
  if (!row_tile<R>(a, tile, &rt)) return;
  const int used = used_splits(a, rt.steps);
  if (split >= used) return;
  const int begin = split * a.chunk;
  const int end = split == used - 1 ? rt.steps : begin + a.chunk;
  const int col = lane & 15, grp = lane >> 4;

  // Q: the lane's row of each 16-row tile, in K's order of the D values
  bf16x8 q[RT][kJ];
  int pos[RT];  // the row's position (rows past the end repeat row 0 and are not stored)
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = x * 16 + col;
    const int row = rt.row0 + (r < rt.rows ? r : 0);
    const int i = row / a.group, h = head * a.group + row % a.group;
    pos[x] = rt.first + i;
    const uint16_t* src = a.q + (int64_t)(rt.token0 + i) * a.q_token + (int64_t)h * a.q_head;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
      q[x][j] = __builtin_bit_cast(bf16x8, load16_any(src + Codes::element(j, lane)));
  }

  f32x4 o[RT][kD16];
  float m[RT], l[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    m[x] = kNegInf, l[x] = 0.0f;
#pragma unroll
    for (int d = 0; d < kD16; ++d) o[x][d] = f32x4{0, 0, 0, 0};
  }

  const int page_mask = (1 << a.cache.page_shift) - 1;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;
  const int32_t* const table = a.batch.table + rt.s * a.batch.table_stride;
  auto key0 = [&](int step) { return (step < rt.sink ? step : step - rt.sink + rt.low) * kStep; };
  // A step's two pages are asked for a step before its codes, by vector loads
  // (scalar ones would have every LDS wait wait for them).  Where there is no
  // page, the codes are those of page 0, and no row sees them.
  int none;  // 0, not known to be uniform
  asm("v_mov_b32 %0, 0" : "=v"(none));
  struct Pages {
    int x[2];
  };
  auto pages_of = [&](int step) {
    Pages p;
    auto page = [&](int key) {
      return step < end && key <= rt.p_hi ? table[(key >> a.cache.page_shift) + none] : -1;
    };
    const int key = key0(step);
    p.x[0] = page(key);
    p.x[1] = page(key + 16);
    return p;
  };
  auto fetch = [&](int step, const Pages& p, Codes (&c)[2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int key = key0(step) + 16 * x, id = __builtin_amdgcn_readfirstlane(p.x[x]);
      c[x].present = id >= 0 && id < a.cache.pages;
      c[x].template load<RT == 1>(base + (c[x].present ? id : 0) * a.cache.page_stride +
                                      ((key & page_mask) >> 4) * (17 * D),
                                  lane);
    }
  };

  uint8_t* const vbuf = lds[wave];
  Codes next[2];
  Pages pages = pages_of(begin + wave);
  if (begin + wave < end) {
    fetch(begin + wave, pages, next);
    pages = pages_of(begin + wave + kWaves);
  }
  for (int step = begin + wave; step < end; step += kWaves) {
    Codes cur[2] = {next[0], next[1]};
    fetch(step + kWaves, pages, next);
    pages = pages_of(step + 2 * kWaves);
    const int k0 = key0(step);
    // every row sees every key of the step
    const bool whole = k0 + kStep - 1 <= rt.p_lo && cur[0].present && cur[1].present &&
                       (!a.window || k0 > rt.p_last - a.window || k0 + kStep <= a.sinks);
    // V to LDS.  A value of a key that some row does not see must not reach
    // that row even as 0 * NaN: positions past the tile's last read as finite
    // (a scale of 0), and NaN blocks go in as zeros and are added to the rows
    // that see them below.
    uint64_t nan[2][Codes::kScales];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const bool past = !cur[x].present || k0 + 16 * x + col > rt.p_hi;
      float vs[Codes::kScales];
#pragma unroll
      for (int c = 0; c < Codes::kScales; ++c) {
        const uint32_t e = past ? 0u : cur[x].vs[c];
        nan[x][c] = __ballot(e > 252u);
        vs[c] = __uint_as_float(e > 252u ? 0u : e << 23);
      }
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int d = Codes::element(j, lane);
        *reinterpret_cast<bf16x8*>(vbuf + v_chunk<D>(x, d >> 4, (d >> 3) & 1, col)) =
            decode8(cur[x].v[j], vs[Codes::scale_of(j)]);
      }
    }

    f32x4 st[RT][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int y = 0; y < RT; ++y) st[y][x] = f32x4{0, 0, 0, 0};
      float ks[Codes::kScales];
#pragma unroll
      for (int c = 0; c < Codes::kScales; ++c) ks[c] = __uint_as_float(cur[x].ks[c] << 23);
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const bf16x8 k = decode8(cur[x].k[j], ks[Codes::scale_of(j)]);
#pragma unroll
        for (int y = 0; y < RT; ++y)
          st[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[y][j], st[y][x], 0, 0, 0);
      }
    }

    if constexpr (KEEP) {
      if (col < a.group && k0 < a.kept_keys) {
        float* const to = a.kept + ((int64_t)blockIdx.x * a.group + col) * a.kept_keys + k0 + 4 * grp;
#pragma unroll
        for (int x = 0; x < 2; ++x) *reinterpret_cast<f32x4*>(to + 16 * x) = st[0][x];
      }
    }

    bf16x8 p[RT];
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = k0 + 16 * x + 4 * grp + r;
            st[y][x][r] = cur[x].present && sees(a, pos[y], j) ? st[y][x][r] : kNegInf;
          }
      }
      float top = m[y];
#pragma unroll
      for (int x = 0; x < 2; ++x)
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
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][i >> 2][i & 3], a.scale, -shift));
        l[y] += e[i];
      }
      p[y] = __builtin_bit_cast(
          bf16x8, u32x4{f32x2_to_bf16x2_rne(e[0], e[1]), f32x2_to_bf16x2_rne(e[2], e[3]),
                        f32x2_to_bf16x2_rne(e[4], e[5]), f32x2_to_bf16x2_rne(e[6], e[7])});
    }

    // Only this wave's own lanes wrote vbuf, and a wave's LDS operations run
    // in order; the fence keeps the compiler from moving the reads.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int vkey = 4 * grp + (col >> 2), vhalf = (col >> 1) & 1;
#pragma unroll
    for (int d = 0; d < kD16; ++d) {
      v4i16 part[2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        part[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_v4i16)(vbuf + v_chunk<D>(x, d, vhalf, vkey) + (col & 1) * 8));
      const bf16x8 v = __builtin_bit_cast(
          bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int y = 0; y < RT; ++y)
        o[y][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[y], o[y][d], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int c = 0; c < Codes::kScales; ++c) {
        if (nan[x][c] == 0) continue;
#pragma unroll
        for (int y = 0; y < RT; ++y) add_nan<D>(a, nan[x][c], c, k0 + 16 * x, pos[y], o[y]);
      }
  }

  // Join the waves: each leaves m, l and O; thread t then sums (row, d) pairs.
#pragma unroll
  for (int y = 0; y < RT; ++y) l[y] = sum_over_groups(l[y]);
  if (grp == 0) {
#pragma unroll
    for (int y = 0; y < RT; ++y)
      wave_m[wave][y * 16 + col] = m[y], wave_l[wave][y * 16 + col] = l[y];
  }
  float* const part = used > 1 ? part_of<D, R>(a, tile, head, split) : nullptr;
  // 16 rows at a time fit the waves' own V buffers (32 keys x 2 bytes = 16
  // rows x 4 bytes), as [16 rows][D / 4 chunks of 4, swapped by the row so that
  // 16 rows' writes meet all banks]
  constexpr int kChunks = D / 4;
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    f32x4* const mine = reinterpret_cast<f32x4*>(vbuf);
#pragma unroll
    for (int d = 0; d < kD16; ++d) mine[col * kChunks + ((d * 4 + grp) ^ col)] = o[y][d];
    __syncthreads();
    const int rows = min(16, rt.rows - y * 16);
    for (int i = threadIdx.x; i < rows * kChunks; i += kWaves * 64) {
      const int r = i / kChunks, ch = i % kChunks;
      Joined sum(wave_m[0][y * 16 + r]);
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum.m = fmaxf(sum.m, wave_m[w][y * 16 + r]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        sum.add(wave_m[w][y * 16 + r], wave_l[w][y * 16 + r],
                reinterpret_cast<const f32x4*>(lds[w])[r * kChunks + (ch ^ r)], a.scale);
      if (part) {
        reinterpret_cast<f32x4*>(part)[(y * 16 + r) * kChunks + ch] = sum.o;
        if (ch == 0) part[R * D + y * 16 + r] = sum.m, part[R * (D + 1) + y * 16 + r] = sum.l;
      } else {
        sum.store(a, rt, head, y * 16 + r, ch * 4);
      }
    }
    __syncthreads();
  }
}

// Up to so many splits a row is joined by one group of threads, more by a workgroup
// to a row.  The call by the one and the other, us: 32 rows, 4 splits 9.3 and 9.8, 8
// 10.2 both, 16 10.9 and 10.4, 64 17.4 and 13.0; 256 rows, 4 splits 10.4 and 10.6, 8
// 12.7 and 12.6, 12 14.0 and 13.7, 32 24.9 and 23.2; 2048 rows, 8 splits 16.5 and
// 18.7, 12 21.8 and 23.8, 16 26.9 and 27.4; 6400 rows, 8 splits 25 and 32.
constexpr int kJoinAlone = 8;

// Joins the splits of a row in their order.  A group of D / 4 threads takes 4 of
// the D elements each; with ALONE a group has a row to itself, otherwise a
// workgroup's groups share one row, each over every kGroups-th split.
template <int D, int R, bool ALONE>
__global__ void __launch_bounds__(256) kv4_join_kernel(Kv4AttentionArgs a) {
  constexpr int kPlane = R * (D + 2), kChunks = D / 4, kGroups = 256 / kChunks;
  const int head = blockIdx.x % a.cache.heads, tile = blockIdx.x / a.cache.heads;
  const int ch = threadIdx.x % kChunks, group = threadIdx.x / kChunks;
  const int r = ALONE ? blockIdx.y * kGroups + group : blockIdx.y;
  RowTile rt;
  if (!row_tile<R>(a, tile, &rt) || r >= rt.rows) return;
  const int used = used_splits(a, rt.steps);
  if (used <= 1) return;
  const float* const part = part_of<D, R>(a, tile, head, 0);
  Joined sum(kNegInf);
  auto add = [&](int s) {
    const float* p = part + s * kPlane;
    sum.add(p[R * D + r], p[R * (D + 1) + r],
            reinterpret_cast<const f32x4*>(p)[r * kChunks + ch], a.scale);
  };
  if constexpr (ALONE) {
#pragma unroll 4
    for (int s = 0; s < used; ++s) sum.m = fmaxf(sum.m, part[s * kPlane + R * D + r]);
#pragma unroll 4
    for (int s = 0; s < used; ++s) add(s);
  } else {
    __shared__ f32x4 other[kGroups][kChunks];
    __shared__ float other_l[kGroups];
    for (int s = threadIdx.x & 63; s < used; s += 64)
      sum.m = fmaxf(sum.m, part[s * kPlane + R * D + r]);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum.m = fmaxf(sum.m, __shfl_xor(sum.m, d));
#pragma unroll 4
    for (int s = group; s < used; s += kGroups) add(s);
    other[group][ch] = sum.o;
    if (ch == 0) other_l[group] = sum.l;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      sum.l += other_l[g];
      sum.o += other[g][ch];
    }
  }
  sum.store(a, rt, head, r, ch * 4);
}

template <int D, int R>
hipError_t join(const Kv4AttentionArgs& args, hipStream_t s) {
  Kv4AttentionArgs a = args;
  void* params[] = {&a};
  const int rows = a.batch.starts ? R : std::min(R, a.group);
  constexpr int kGroups = 1024 / D;
  const bool alone = a.splits <= kJoinAlone;
  return hipLaunchKernel(alone ? reinterpret_cast<const void*>(&kv4_join_kernel<D, R, true>)
                               : reinterpret_cast<const void*>(&kv4_join_kernel<D, R, false>),
                         dim3((unsigned)(a.tiles * a.cache.heads),
                              (unsigned)(alone ? (rows + kGroups - 1) / kGroups : rows)),
                         dim3(256), params, 0, s);
}

template <int D, int RT>
hipError_t attend(const Kv4AttentionArgs& args, hipStream_t s) {
  Kv4AttentionArgs a = args;
  void* params[] = {&a};
  const hipError_t e = hipLaunchKernel(
      RT == 1 && a.kept ? reinterpret_cast<const void*>(&kv4_attention_kernel<D, 1, true>)
                        : reinterpret_cast<const void*>(&kv4_attention_kernel<D, RT>),
      dim3((unsigned)(a.tiles * a.cache.heads), (unsigned)a.splits), dim3(kWaves * 64), params, 0, s);
  return e == hipSuccess && a.splits > 1 ? join<D, 16 * RT>(a, s) : e;
}

template <int D>
hipError_t attend_rows(const Kv4AttentionArgs& a, int rows, hipStream_t s) {
  if (rows == 16) return attend<D, 1>(a, s);
  if (rows == 32) return attend<D, 2>(a, s);
  const hipError_t e = llk_launch_kv4_prompt(a, D, s);
  return e == hipSuccess && a.splits > 1 ? join<D, kKv4PromptRows>(a, s) : e;
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_attention(const Kv4AttentionArgs& a, int D, int rows, hipStream_t s) {
  using namespace llk_gfx950;
  return D == 64    ? attend_rows<64>(a, rows, s)
         : D == 128 ? attend_rows<128>(a, rows, s)
                    : attend_rows<256>(a, rows, s);
}

size_t llk_kv4_attention_part_bytes(int64_t tiles, int heads, int splits, int rows, int D) {
  return splits > 1 ? (size_t)tiles * heads * splits * rows * (D + 2) * sizeof(float) : 0;
}
