// kv4_weigh.hip -- what weight an attention gave to every cached key, added up
// over its rows (new tokens and query heads of the key head):
//
//   w[j] = decay w[j] + sum over rows r that see j of exp2((s_rj - m_r) scale) / l_r
//
// with each row's reference m and sum l as the attention left them.  Every key has
// one wave that goes over all its rows, so nothing is added from two places and the
// sums come out the same every time.
//
// Single tokens (few rows): the attention stores its scores, 4 bytes for a row and key
// where the cache has 17/16 D, and they are read once more here.  Where it did not,
// or rows are many, the scores are computed again: a prompt has far more pairs of a
// row and a key than could be kept.
#include <algorithm>

#include "kv4_attention.h"

namespace llk_gfx950 {
namespace {

constexpr int kWaves = 4, kStep = 32;  // keys to a wave's step

// The sequence of a workgroup and its rows.
struct Weighed {
  int s, len, first, token0, rows;  // first: position of row 0's token
  __device__ __forceinline__ bool find(const Kv4AttentionArgs& a, int seq) {
    const Kv4Batch& b = a.batch;
    s = seq;
    const int from = b.starts ? b.starts[s] : s, next = b.starts ? b.starts[s + 1] : s + 1;
    if (from < 0 || next > b.tokens || next <= from) return false;
    len = kv4_length(a.cache, b, s);
    first = (int)max((int64_t)b.lens[s] - (next - from), -(int64_t)kKv4MaxLength);
    token0 = from;
    rows = (next - from) * a.group;
    return len > 0;
  }
};

// Sum over the 16 lanes of a group.
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// A row's reference and sum as what its weights are computed with.
struct RowWeight {
  float shift, inv;  // exp2(score a.scale - shift) inv
  // nothing of a row that saw nothing, or scores of -infinity only
  __device__ __forceinline__ RowWeight(const Kv4AttentionArgs& a, int64_t row, bool some) {
    const float2 ml = reinterpret_cast<const float2*>(a.stats)[row];
    some = some && ml.y != 0.0f;
    shift = some ? ml.x * a.scale : 0.0f;
    inv = some ? 1.0f / ml.y : 0.0f;
  }
  __device__ __forceinline__ float of(const Kv4AttentionArgs& a, float score) const {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(score, a.scale, -shift)) * inv;
  }
};
constexpr int kNowhere = -1 - kKv4MaxLength;  // the position of a row that sees no key

// Adds `mine` up in a slot.
__device__ __forceinline__ void add_weight(float* at, float decay, float mine) {
  *at = decay == 0.0f ? mine : __builtin_fmaf(decay, *at, mine);
}

// KEPT: of the first a.kept_keys keys the scores are there; of later ones they are
// computed as for calls that kept none.
template <int D, bool KEPT>
__global__ void __launch_bounds__(kWaves * 64)
    kv4_weigh_kernel(Kv4AttentionArgs a, Kv4Marks marks, float decay, int steps) {
  constexpr int kJ = D / 32;
  using Codes = TileCodes<D>;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % a.cache.heads;
  Weighed w;
  if (!w.find(a, blockIdx.x / a.cache.heads)) return;
  const int size = 1 << a.cache.page_shift;
  const int32_t* const table = a.batch.table + w.s * a.batch.table_stride;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;

  if constexpr (KEPT) {
    // 4 keys to a lane; the rows are the query heads of the sequence's token
    const int end = min(w.len, a.kept_keys);
    for (int k0 = (blockIdx.y * kWaves + wave) * 256; k0 < end; k0 += gridDim.y * kWaves * 256) {
      const int key = k0 + 4 * lane;
      if (key >= end) break;
      const int id = table[key >> a.cache.page_shift];
      const float* from = a.kept + (int64_t)blockIdx.x * a.group * a.kept_keys + key;
      f32x4 sum{0, 0, 0, 0};
#pragma unroll 4
      for (int g = 0; g < a.group; ++g) {
        const RowWeight row(a, (int64_t)w.token0 * (a.cache.heads * a.group) + head * a.group + g, true);
        const f32x4 st = *reinterpret_cast<const f32x4*>(from + (int64_t)g * a.kept_keys);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += sees(a, w.first, key + i) ? row.of(a, st[i]) : 0.0f;
      }
      if (id < 0 || id >= a.cache.pages) continue;
      float* const at = marks.weights + id * marks.weights_page + (int64_t)head * size + (key & (size - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + i < w.len) add_weight(at + i, decay, sum[i]);
    }
  }
  const int all = (w.len + kStep - 1) / kStep;
  const int64_t stride = (int64_t)gridDim.y * kWaves * steps;
  int64_t begin = (int64_t)(blockIdx.y * kWaves + wave) * steps + (KEPT ? a.kept_keys / kStep : 0);
  if (begin >= all) return;

  // the lane's row of the 16 from row0 on: Q in K's order, and its statistics
  bf16x8 q[kJ];
  int pos;
  float shift, inv;
  auto rows_from = [&](int row0) {
    const int row = row0 + col < w.rows ? row0 + col : row0;
    const int i = row / a.group, h = head * a.group + row % a.group;
    const uint16_t* const src = a.q + (int64_t)(w.token0 + i) * a.q_token + (int64_t)h * a.q_head;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
      q[j] = __builtin_bit_cast(bf16x8, load16_any(src + Codes::element(j, lane)));
    const bool some = row0 + col < w.rows;
    const RowWeight r(a, (int64_t)(w.token0 + i) * (a.cache.heads * a.group) + h, some);
    shift = r.shift;
    inv = r.inv;
    pos = some ? w.first + i : kNowhere;
  };
  const bool one = w.rows <= 16;
  if (one) rows_from(0);
  for (int64_t step = begin; step < all;) {
    const int k0 = (int)step * kStep;
    Codes c[2];
    int page[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int key = k0 + 16 * x;
      page[x] = key < w.len ? table[key >> a.cache.page_shift] : -1;
      c[x].present = page[x] >= 0 && page[x] < a.cache.pages;
      c[x].template load<false>(base + (c[x].present ? page[x] : 0) * a.cache.page_stride +
                                    ((key & (size - 1)) >> 4) * (17 * D),
                                lane);
    }
    float sum[2][4] = {};
    // rows before the first token that is not before the step's first key see none
    const int from =
        one ? 0 : (int)min((int64_t)max(0, k0 - w.first) * a.group / 16 * 16, (int64_t)w.rows);
    for (int row0 = from; row0 < w.rows; row0 += 16) {
      if (!one) {
        if (a.window && k0 + kStep - 1 <= w.first + row0 / a.group - a.window && k0 >= a.sinks) break;
        rows_from(row0);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        f32x4 st{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          st = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              decode8(c[x].k[j], __uint_as_float(c[x].ks[Codes::scale_of(j)] << 23)), q[j], st, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], a.scale, -shift)) * inv;
          sum[x][r] += sees(a, pos, k0 + 16 * x + 4 * grp + r) ? e : 0.0f;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[x][r] = sum16(sum[x][r]);
      const int key = k0 + 16 * x + 4 * grp + col;  // of lane col < 4
      const float mine = col == 0 ? sum[x][0] : col == 1 ? sum[x][1] : col == 2 ? sum[x][2] : sum[x][3];
      if (col < 4 && key < w.len && c[x].present) {
        add_weight(marks.weights + page[x] * marks.weights_page + (int64_t)head * size +
                       (key & (size - 1)),
                   decay, mine);
      }
    }
    if (++step == begin + steps) step = begin += stride;
  }
}

// Many rows: a wave has 32 keys, in registers as operands, and meets all rows that
// see them, 64 at a time in LDS, which the workgroup's four waves (128 keys) share.
// S^T = K Q^T on v_mfma_f32_32x32x16_bf16, any order of the D values: of a key's, the
// lane's half of the wave has the first or second half.
constexpr int kKeys = 32, kQueries = 64;

template <int D>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(2))) kv4_weigh_rows_kernel(Kv4AttentionArgs a, Kv4Marks marks,
                                                                  float decay, int tiles) {
  constexpr int kU = D / 16, kBlocks = D / 64, kChunks = D / 8;
  // Q: [32 rows][step u][half][row] of 16 bytes, a row's place turned by the chunk's
  // number, so that the chunks of a row meet different banks when they are written
  __shared__ __attribute__((aligned(16))) u32x4 qs[2][kQueries / 32 * kU * 64];
  __shared__ float2 weight[2][kQueries];  // shift, inv
  __shared__ int position[2][kQueries];
  const int t = threadIdx.x, lane = t & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // The first tiles of keys, seen by the most rows, first, then the others from the
  // last on, so that the two workgroups a CU gets in a round have much and little to do.
  const int groups = a.batch.sequences * a.cache.heads;
  const int nth = blockIdx.x / groups, head = blockIdx.x % groups % a.cache.heads;
  const int tile = 2 * nth < tiles ? nth : tiles - 1 - (nth - (tiles + 1) / 2);
  Weighed w;
  if (!w.find(a, blockIdx.x % groups / a.cache.heads)) return;
  const int size = 1 << a.cache.page_shift;
  const int32_t* const table = a.batch.table + w.s * a.batch.table_stride;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;
  const int heads = a.cache.heads * a.group;

  for (int64_t first_key = (int64_t)tile * (kWaves * kKeys); first_key < w.len;
       first_key += (int64_t)tiles * (kWaves * kKeys)) {
    const int k0 = (int)first_key + wave * kKeys;  // the wave's keys
    // the lane's key, its page, and its blocks
    const int key = k0 + col, id = key < w.len ? table[key >> a.cache.page_shift] : -1;
    const bool present = id >= 0 && id < a.cache.pages;
    bf16x8 k[kU];
    {
      const uint8_t* const at = base + (present ? id : 0) * a.cache.page_stride +
                                ((key & (size - 1)) >> 4) * (17 * D);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int block = half * kBlocks + b;
        const u32x4 c = *reinterpret_cast<const u32x4*>(at + (block * 16 + (key & 15)) * 16);
        const float scale = __uint_as_float((uint32_t)at[16 * D + block * 16 + (key & 15)] << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[4 * b + i] = decode8(c[i], scale);
      }
    }
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.0f;

    // rows of the first token that is not before the first key of the workgroup, to
    // the last that its window reaches
    const int64_t from = (int64_t)max(0, (int)first_key - w.first) * a.group;
    int64_t to = w.rows;
    if (a.window && first_key >= a.sinks)
      to = min(to, max((int64_t)0, first_key + kWaves * kKeys - 1 + a.window - w.first) * a.group);
    u32x4 x[kQueries * kChunks / 256];
    float2 ml;
    int at = 0;
    auto row_at = [&](int64_t r) { return r < w.rows ? (int)r : w.rows - 1; };
    auto load = [&](int64_t row0) {
#pragma unroll
      for (int i = 0; i < kQueries * kChunks / 256; ++i) {
        const int n = i * 256 + t, row = row_at(row0 + n / kChunks);
        const uint16_t* const src = a.q + (int64_t)(w.token0 + row / a.group) * a.q_token +
                                    (int64_t)(head * a.group + row % a.group) * a.q_head;
        x[i] = load16_any(src + n % kChunks * 8);
      }
      if (t < kQueries) {
        const int row = row_at(row0 + t);
        const bool some = row0 + t < w.rows;
        const RowWeight r(a, (int64_t)(w.token0 + row / a.group) * heads + head * a.group + row % a.group,
                          some);
        ml = make_float2(r.shift, r.inv);
        at = some ? w.first + row / a.group : kNowhere;
      }
    };
    auto place = [&](int buf) {
#pragma unroll
      for (int i = 0; i < kQueries * kChunks / 256; ++i) {
        const int n = i * 256 + t, q = n / kChunks, c = n % kChunks;  // chunk c: half c / kU, step c % kU
        qs[buf][((q / 32 * kU + c % kU) * 2 + c / kU) * 32 + ((q ^ c) & 31)] = x[i];
      }
      if (t < kQueries) weight[buf][t] = ml, position[buf][t] = at;
    };
    __syncthreads();  // the last reads of the tile of keys before
    if (from < to) load(from);
    int buf = 0;
    for (int64_t row0 = from; row0 < to; row0 += kQueries, buf ^= 1) {
      place(buf);  // its readers of two rounds ago are past the barrier of the last
      __syncthreads();
      if (row0 + kQueries < to) load(row0 + kQueries);
      // every row sees every key of the wave
      const int p_lo = w.first + (int)(row0 / a.group);
      const int p_hi = w.first + (int)(min(row0 + kQueries, (int64_t)w.rows) - 1) / a.group;
      const bool whole = row0 + kQueries <= w.rows && k0 + kKeys - 1 <= p_lo &&
                         (!a.window || k0 > p_hi - a.window || k0 + kKeys <= a.sinks);
      if (k0 > p_hi) continue;  // none does
#pragma unroll
      for (int h = 0; h < kQueries / 32; ++h) {
        f32x16 st;
#pragma unroll
        for (int i = 0; i < 16; ++i) st[i] = 0.0f;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int c = half * kU + u;
          st = mfma32(k[u],
                      __builtin_bit_cast(bf16x8, qs[buf][((h * kU + u) * 2 + half) * 32 + ((col ^ c) & 31)]),
                      st);
        }
        const float2 r = weight[buf][32 * h + col];
        if (whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sum[i] = __builtin_fmaf(
                __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], a.scale, -r.x)), r.y, sum[i]);
        } else {
          const int pos = position[buf][32 * h + col];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], a.scale, -r.x)) * r.y;
            sum[i] += sees(a, pos, k0 + 8 * (i >> 2) + 4 * half + (i & 3)) ? e : 0.0f;
          }
        }
      }
    }
    // over the 32 lanes of a half wave; lane n stores the sum of its half's key n
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = sum16(sum[i]);
      s += __shfl_xor(s, 16);
      mine = col == i ? s : mine;
    }
    const int own = k0 + 8 * (col >> 2) + 4 * half + (col & 3);  // of lanes col < 16
    const int page = __shfl(present ? id : -1, own - k0 & 31);
    if (col < 16 && own < w.len && page >= 0)
      add_weight(marks.weights + page * marks.weights_page + (int64_t)head * size + (own & (size - 1)),
                 decay, mine);
  }
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_weigh(const Kv4AttentionArgs& args, const Kv4Marks& m, float decay, int D,
                                int64_t max_len, hipStream_t s) {
  using namespace llk_gfx950;
  Kv4AttentionArgs a = args;
  Kv4Marks marks = m;
  int64_t len = std::min<int64_t>((int64_t)a.batch.table_pages << a.cache.page_shift, kKv4MaxLength);
  if (max_len > 0) len = std::min(len, max_len);
  len = std::max<int64_t>(len, 1);
  const int64_t groups = (int64_t)a.batch.sequences * a.cache.heads;
  if (!a.kept && (int64_t)a.batch.tokens * a.group > 16 * (int64_t)a.batch.sequences) {
    // (fewer workgroups go round for the rest)
    int tiles = (int)std::min<int64_t>((len + kWaves * kKeys - 1) / (kWaves * kKeys),
                                       kKv4MaxWorkgroups / groups);
    void* params[] = {&a, &marks, &decay, &tiles};
    const void* fn = D == 64    ? reinterpret_cast<const void*>(&kv4_weigh_rows_kernel<64>)
                     : D == 128 ? reinterpret_cast<const void*>(&kv4_weigh_rows_kernel<128>)
                                : reinterpret_cast<const void*>(&kv4_weigh_rows_kernel<256>);
    return hipLaunchKernel(fn, dim3((unsigned)(groups * tiles)), dim3(kWaves * 64), params, 0, s);
  }
  const int64_t all = (len + kStep - 1) / kStep;  // steps of a sequence, at most
  // about 8192 waves; with kept scores 256 keys to a wave
  int steps = a.kept ? 8 : (int)std::max<int64_t>(1, all * groups / 8192);
  void* params[] = {&a, &marks, &decay, &steps};
  const void* fn =
      a.kept ? (D == 64    ? reinterpret_cast<const void*>(&kv4_weigh_kernel<64, true>)
                : D == 128 ? reinterpret_cast<const void*>(&kv4_weigh_kernel<128, true>)
                           : reinterpret_cast<const void*>(&kv4_weigh_kernel<256, true>))
             : (D == 64    ? reinterpret_cast<const void*>(&kv4_weigh_kernel<64, false>)
                : D == 128 ? reinterpret_cast<const void*>(&kv4_weigh_kernel<128, false>)
                           : reinterpret_cast<const void*>(&kv4_weigh_kernel<256, false>));
  const int64_t per = (int64_t)steps * kWaves;
  return hipLaunchKernel(fn, dim3((unsigned)groups, (unsigned)std::min<int64_t>((all + per - 1) / per, 65535)),
                         dim3(kWaves * 64), params, 0, s);
}
