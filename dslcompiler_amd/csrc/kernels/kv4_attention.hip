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
#include "common.h"
#include "kv4.h"

namespace llk_gfx950 {
namespace {

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16* lds_v4i16;

constexpr int kWaves = 4;  // of a workgroup, each over its own keys
constexpr float kNegInf = -__builtin_inff();

// A row tile: its sequence, the positions its rows ask from and the steps of
// kKv4Step keys it covers: `sink` steps from key 0, then those from `low`.
struct RowTile {
  int s, row0, rows;     // sequence; first row of the sequence; rows in it
  int first, token0;     // position and index of the sequence's first new token
  int p_lo, p_hi;        // positions of the tile's first and last query
  int sink, low, steps;  // steps over the first tokens; first other step; all steps
};

template <int R>
__device__ __forceinline__ bool row_tile(const Kv4AttentionArgs& a, int t, RowTile* o) {
  const Kv4Batch& b = a.batch;
  int first = 0, next = 0, tile0 = 0;
  if (!b.starts) {
    const int per = (a.group + R - 1) / R;
    o->s = t / per;
    first = o->s;
    next = first + 1;
    tile0 = o->s * per;
  } else {
    // sequence s has the tiles from floor(starts[s] * group / R) + s on
    auto from = [&](int s) { return (int64_t)b.starts[s] * a.group / R + s; };
    int lo = 0, hi = b.sequences - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (from(mid) <= t) lo = mid;
      else hi = mid - 1;
    }
    o->s = lo;
    first = b.starts[lo];
    next = b.starts[lo + 1];
    tile0 = (int)from(lo);
  }
  if (o->s >= b.sequences || t < tile0 || first < 0 || next > b.tokens) return false;
  const int64_t row0 = (int64_t)(t - tile0) * R, all = (int64_t)(next - first) * a.group;
  if (row0 >= all) return false;
  o->row0 = (int)row0;
  o->rows = (int)min((int64_t)R, all - row0);
  o->token0 = first;
  const int len = kv4_length(a.cache, b, o->s);
  // new tokens past the table's end see all it holds
  o->first = max(min(b.lens[o->s], kKv4MaxLength) - (next - first), -kKv4MaxLength);
  o->p_lo = o->first + o->row0 / a.group;
  o->p_hi = min(o->first + (o->row0 + o->rows - 1) / a.group, len - 1);
  o->sink = o->low = o->steps = 0;
  if (o->p_hi < 0) return true;
  const int end = o->p_hi / kKv4Step + 1;
  if (a.window) {
    o->low = max(0, o->p_lo - a.window + 1) / kKv4Step;
    o->sink = min((a.sinks + kKv4Step - 1) / kKv4Step, min(o->low, end));
  }
  o->low = min(o->low, end);
  o->steps = o->sink + end - o->low;
  return true;
}

// Splits that a tile's steps need (the last takes what the plan's `chunk`
// steps to a split leave over).
__device__ __forceinline__ int used_splits(const Kv4AttentionArgs& a, int steps) {
  return max(1, min(a.splits, (steps + a.chunk - 1) / a.chunk));
}

// Partial planes of (tile, key head, split): O [R][D], then m [R], l [R].
template <int D, int R>
__device__ __forceinline__ float* part_of(const Kv4AttentionArgs& a, int tile, int head, int split) {
  return a.part + (((int64_t)tile * a.cache.heads + head) * a.splits + split) * (R * (D + 2));
}

__device__ __forceinline__ float max_over_groups(float x) {
  // the four lanes of a query: lane, lane ^ 16, lane ^ 32, lane ^ 48
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 8 codes (a dword) as bf16: an MFMA operand's 16 bytes.
__device__ __forceinline__ bf16x8 decode8(uint32_t codes, float scale) {
  const u32x4 v{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
  return __builtin_bit_cast(bf16x8, v);
}

// One lane's share of a 16-token tile: D / 4 keys' codes and values' codes of
// token lane % 16 -- the contiguous D / 4 values from lane / 16 * D / 4 (D =
// 256: from 32 (lane / 16) and 128 + 32 (lane / 16)) -- and their scales.
template <int D>
struct TileCodes {
  static constexpr int kDwords = D / 32;             // of codes, 8 values each
  static constexpr int kScales = D == 256 ? 2 : 1;   // blocks the lane has part of
  uint32_t k[kDwords], v[kDwords];
  uint32_t ks[kScales], vs[kScales];  // scale bytes
  int present;                        // the tile's page exists

  __device__ __forceinline__ void load(const uint8_t* tile, int lane) {
    if constexpr (D == 64) {
      const int block = lane >> 5, half = (lane >> 4) & 1, tok = lane & 15;
      const int at = (block * 16 + tok) * 16 + half * 8;
      const uint2 a = *reinterpret_cast<const uint2*>(tile + at);
      const uint2 b = *reinterpret_cast<const uint2*>(tile + 8 * D + at);
      k[0] = a.x, k[1] = a.y, v[0] = b.x, v[1] = b.y;
      ks[0] = tile[16 * D + block * 16 + tok];
      vs[0] = tile[16 * D + D / 2 + block * 16 + tok];
    } else {
#pragma unroll
      for (int c = 0; c < kScales; ++c) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(tile + c * 1024 + lane * 16);
        const u32x4 b = *reinterpret_cast<const u32x4*>(tile + 8 * D + c * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[4 * c + i] = a[i], v[4 * c + i] = b[i];
        ks[c] = tile[16 * D + c * 64 + lane];
        vs[c] = tile[16 * D + D / 2 + c * 64 + lane];
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kDwords; ++i) k[i] = v[i] = 0;
#pragma unroll
    for (int i = 0; i < kScales; ++i) ks[i] = vs[i] = 0;
  }
  static __device__ __forceinline__ int scale_of(int dword) { return D == 256 ? dword / 4 : 0; }
  // First of the 8 values of dword j.
  static __device__ __forceinline__ int element(int j, int lane) {
    return D == 256 ? (j >> 2) * 128 + (lane >> 4) * 32 + (j & 3) * 8
                    : (lane >> 4) * (D / 4) + j * 8;
  }
};

// V of 32 keys in LDS, as bf16: [16-key tile][D / 16][half: 8 values][16 keys]
// of 16 bytes, the keys of the second half swapped by 8 so that the 32 lanes
// of a half wave, which read both halves of 8 keys, meet all 64 banks.
template <int D>
__device__ __forceinline__ int v_chunk(int x, int d16, int half, int key) {
  return ((x * (D / 16) + d16) * 2 + half) * 256 + (key ^ (half * 8)) * 16;
}

// Parts of a row's softmax (maximum m of the unscaled scores, sum l, 4 of the
// unnormalised outputs) joined into one; m is the largest of theirs.
struct Joined {
  float m, l = 0.0f;
  f32x4 o{0, 0, 0, 0};
  __device__ __forceinline__ explicit Joined(float top) : m(top) {}
  __device__ __forceinline__ void add(float pm, float pl, const f32x4& po, float scale) {
    const float f = __builtin_amdgcn_exp2f((pm - (m == kNegInf ? 0.0f : m)) * scale);
    l = __builtin_fmaf(f, pl, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(f, po[i], o[i]);
  }
  // Elements d..d + 3 of the tile's row r; zeros for a row that saw no key.
  __device__ __forceinline__ void store(const Kv4AttentionArgs& a, const RowTile& rt, int head,
                                        int r, int d) const {
    const int row = rt.row0 + r;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* dst = a.out + (int64_t)(rt.token0 + row / a.group) * a.out_token +
                    (int64_t)(head * a.group + row % a.group) * a.out_head + d;
    store8_any(dst, make_uint2(f32x2_to_bf16x2_rne(o[0] * inv, o[1] * inv),
                               f32x2_to_bf16x2_rne(o[2] * inv, o[3] * inv)));
  }
};

// A workgroup's 4 waves share a row tile of 16 * RT rows and one split of its
// keys, each wave taking every fourth step of 32 keys with a running maximum
// of its own; at the end they are joined in LDS.
template <int D, int RT>
__global__ void __launch_bounds__(kWaves * 64) kv4_attention_kernel(Kv4AttentionArgs a) {
  constexpr int R = 16 * RT, kD16 = D / 16, kJ = D / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves][kKv4Step * D * 2];
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
    pos[x] = min(rt.first + i, rt.p_hi);
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
  auto key0 = [&](int step) { return (step < rt.sink ? step : step - rt.sink + rt.low) * kKv4Step; };
  auto fetch = [&](int step, Codes (&c)[2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int key = key0(step) + 16 * x;
      int id = -1;
      if (key <= rt.p_hi) id = table[key >> a.cache.page_shift];
      c[x].present = id >= 0 && id < a.cache.pages;
      if (c[x].present)
        c[x].load(base + id * a.cache.page_stride + (int64_t)((key & page_mask) >> 4) * (17 * D),
                  lane);
      else
        c[x].clear();
    }
  };

  uint8_t* const vbuf = lds[wave];
  Codes next[2];
  if (begin + wave < end) fetch(begin + wave, next);
  for (int step = begin + wave; step < end; step += kWaves) {
    Codes cur[2] = {next[0], next[1]};
    if (step + kWaves < end) fetch(step + kWaves, next);
    const int k0 = key0(step);
    // every row sees every key of the step
    const bool whole = k0 + kKv4Step - 1 <= rt.p_lo && cur[0].present && cur[1].present &&
                       (!a.window || k0 > rt.p_hi - a.window || k0 + kKv4Step <= a.sinks);
    // V to LDS.  A value of a key that some row does not see must not reach
    // that row even as 0 * NaN: positions past the tile's last read as finite
    // (a scale of 0), and NaN blocks go in as zeros and are added to the rows
    // that see them below.
    uint64_t nan[2][Codes::kScales];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const bool past = k0 + 16 * x + col > rt.p_hi;
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

    bf16x8 p[RT];
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = k0 + 16 * x + 4 * grp + r;
            const bool seen = j <= pos[y] && cur[x].present &&
                              (!a.window || j > pos[y] - a.window || j < a.sinks);
            st[y][x][r] = seen ? st[y][x][r] : kNegInf;
          }
      }
      float top = m[y];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, st[y][x][r]);
      top = max_over_groups(top);
      if (__any(top > m[y])) {
        // of a row that has seen no key yet m is -inf, and l and o are 0
        const float alpha = __builtin_amdgcn_exp2f((m[y] - (top == kNegInf ? 0.0f : top)) * a.scale);
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
        for (int y = 0; y < RT; ++y) {
          uint32_t seen = 0;  // of the 16 keys, those the lane's row sees
          for (int i = 0; i < 16; ++i) {
            const int j = k0 + 16 * x + i;
            if (j <= pos[y] && (!a.window || j > pos[y] - a.window || j < a.sinks)) seen |= 1u << i;
          }
#pragma unroll
          for (int d = 0; d < kD16; ++d) {
            // lanes that hold part of the 16 values' block: those of one group
            const int e0 = d * 16;
            if (D == 256 && e0 / 128 != c) continue;
            const int g = D == 256 ? e0 % 128 / 32 : e0 / (D / 4);
            if ((uint32_t)(nan[x][c] >> (16 * g)) & seen & 0xffffu) o[y][d] += __builtin_nanf("");
          }
        }
      }
  }

  // Join the waves: each leaves m, l and O; thread t then sums (row, d) pairs.
#pragma unroll
  for (int y = 0; y < RT; ++y) l[y] = sum_over_groups(l[y]);
  if (grp == 0) {
#pragma unroll
    for (int y = 0; y < RT; ++y) wave_m[wave][y * 16 + col] = m[y], wave_l[wave][y * 16 + col] = l[y];
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

// Joins a tile's splits: a workgroup per (tile, key head), its threads over
// (row, pair of d).
template <int D, int R>
__global__ void __launch_bounds__(256) kv4_join_kernel(Kv4AttentionArgs a) {
  const int head = blockIdx.x % a.cache.heads, tile = blockIdx.x / a.cache.heads;
  RowTile rt;
  if (!row_tile<R>(a, tile, &rt)) return;
  const int used = used_splits(a, rt.steps);
  if (used <= 1) return;
  const float* const part = part_of<D, R>(a, tile, head, 0);
  constexpr int kPlane = R * (D + 2), kChunks = D / 4;
  for (int i = threadIdx.x; i < rt.rows * kChunks; i += 256) {
    const int r = i / kChunks, ch = i % kChunks;
    Joined sum(kNegInf);
    for (int s = 0; s < used; ++s) sum.m = fmaxf(sum.m, part[s * kPlane + R * D + r]);
    for (int s = 0; s < used; ++s) {
      const float* p = part + s * kPlane;
      sum.add(p[R * D + r], p[R * (D + 1) + r],
              reinterpret_cast<const f32x4*>(p)[r * kChunks + ch], a.scale);
    }
    sum.store(a, rt, head, r, ch * 4);
  }
}

template <int D, int RT>
hipError_t launch(const Kv4AttentionArgs& args, hipStream_t s) {
  Kv4AttentionArgs a = args;
  void* params[] = {&a};
  const unsigned x = (unsigned)(a.tiles * a.cache.heads);
  hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&kv4_attention_kernel<D, RT>),
                                 dim3(x, (unsigned)a.splits), dim3(kWaves * 64), params, 0, s);
  if (e == hipSuccess && a.splits > 1)
    e = hipLaunchKernel(reinterpret_cast<const void*>(&kv4_join_kernel<D, 16 * RT>), dim3(x),
                        dim3(256), params, 0, s);
  return e;
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_attention(const Kv4AttentionArgs& a, int D, int rows, hipStream_t s) {
  using namespace llk_gfx950;
  if (rows == 16)
    return D == 64 ? launch<64, 1>(a, s) : D == 128 ? launch<128, 1>(a, s) : launch<256, 1>(a, s);
  return D == 64 ? launch<64, 2>(a, s) : D == 128 ? launch<128, 2>(a, s) : launch<256, 2>(a, s);
}

size_t llk_kv4_attention_part_bytes(int64_t tiles, int heads, int splits, int rows, int D) {
  return splits > 1 ? (size_t)tiles * heads * splits * rows * (D + 2) * sizeof(float) : 0;
}
