// kv4_weigh.hip -- what weight an attention gave to every cached key, added up
// over its rows (new tokens and query heads of the key head):
//
//   w[j] = decay w[j] + sum over rows r that see j of exp2((s_rj - m_r) scale) / l_r
//
// with each row's reference m and sum l as the attention left them.  Every key has
// one wave that goes over all its rows, so nothing is added from two places and the
// sums come out the same every time.
//
// Single tokens without `starts`, to 16 query heads of a key head: the attention
// stores its scores, 4 bytes for a row and key where the cache has 17/16 D, and they are
// read once more here (also those of keys outside a window, which are not used).  Where
// it did not, the scores are computed again: a prompt has far more pairs of a row and a
// key than could be kept, and the buffer goes by sequence, of which a batch with
// `starts` may have some with more tokens than one.  64 ragged sequences to 8192 keys, 32 query heads on 8: the
// attention 84 us with its scores stored (68 without) and 15 here (kernel times).  A call
// in a replayed graph, 4337 keys on average: 66 without weights, 95 with, 126 by
// `starts`; with a window of 256 10, 24 and 65.
#include <algorithm>
#include <type_traits>

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
  __device__ __forceinline__ RowWeight(const Kv4AttentionArgs& a, int64_t row, bool some)
      : RowWeight(a, reinterpret_cast<const float2*>(a.stats)[row], some) {}
  __device__ __forceinline__ RowWeight(const Kv4AttentionArgs& a, float2 ml, bool some) {
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

// Many rows: four waves share 128 keys, 32 of each, in registers as operands, four
// more have the same keys, and the rows that see them go through LDS, 64 at a time,
// half of them for either four.  S^T = K Q^T on v_mfma_f32_32x32x16_bf16, any order of
// the D values: of a key's, the lane's half of the wave has the first or second half.
//
// A prompt of 2048 tokens, 32 heads, takes 41 us (400 TFLOP/s of what causality
// leaves).  No unit is near its limit: vector instructions take 39% of a SIMD's
// cycles, products 20%, LDS 22% of a CU's, without bank conflicts; taking out the
// products or the exponentials changed nothing, keeping the rows in LDS a tenth.  At D =
// 128 it has 193 registers, so eight waves to a CU, all in step by a barrier a round, and
// they wait for 36% of their time.  A round's scores carried over to the next round's
// products gained nothing; 64 keys to a wave need more registers than there are (61 us).
constexpr int kRowWaves = 8, kRowThreads = kRowWaves * 64, kRowKeys = 128;

template <int D>
__global__ void __launch_bounds__(kRowThreads)
    __attribute__((amdgpu_waves_per_eu(2))) kv4_weigh_rows_kernel(Kv4AttentionArgs a, Kv4Marks marks,
                                                                  float decay, int tiles) {
  constexpr int kU = D / 16, kBlocks = D / 64, kChunks = D / 8;
  constexpr int kKeyWaves = kRowKeys / 32, kParts = kRowWaves / kKeyWaves;
  constexpr int kQueries = 32 * kParts;  // rows to a round
  // Q: [32 rows][step u][half][row] of 16 bytes, a row's place turned by the chunk's
  // number, so that the chunks of a row meet different banks when they are written
  __shared__ __attribute__((aligned(16))) u32x4 qs[2][kParts * kU * 64];
  __shared__ float2 weight[2][kQueries];  // shift, inv
  __shared__ int position[2][kQueries];
  __shared__ float others[kParts][kRowKeys];  // the parts' sums
  const int t = threadIdx.x, lane = t & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6) % kKeyWaves;
  const int part = __builtin_amdgcn_readfirstlane(t >> 6) / kKeyWaves;  // which 32 rows
  // the first tiles of keys, seen by the most rows, first
  const int groups = a.batch.sequences * a.cache.heads;
  const int tile = blockIdx.x / groups, head = blockIdx.x % groups % a.cache.heads;
  Weighed w;
  if (!w.find(a, blockIdx.x % groups / a.cache.heads)) return;
  const int size = 1 << a.cache.page_shift;
  const int32_t* const table = a.batch.table + w.s * a.batch.table_stride;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;
  const int heads = a.cache.heads * a.group;

  for (int64_t first_key = (int64_t)tile * kRowKeys; first_key < w.len;
       first_key += (int64_t)tiles * kRowKeys) {
    const int k0 = (int)first_key + wave * 32;  // the wave's keys
    bf16x8 k[kU];
    {
      // the lane's key, its page (0 without one; its sum is not stored), its blocks
      const int key = k0 + col, id = key < w.len ? table[key >> a.cache.page_shift] : 0;
      const uint8_t* const at = base + (id >= 0 && id < a.cache.pages ? id : 0) * a.cache.page_stride +
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
    const int64_t seen_from = (int64_t)max(0, (int)first_key - w.first) * a.group;
    int64_t seen_to = w.rows;
    if (a.window && first_key >= a.sinks)
      seen_to = min(seen_to, max((int64_t)0, first_key + kRowKeys - 1 + a.window - w.first) * a.group);
    const int from = (int)min(seen_from, seen_to), to = (int)seen_to;
    // The thread's chunks are of kLoads rows, kRowThreads / kChunks apart, and one row's
    // statistics.  Their addresses go from round to round by a constant, and by
    // another where a row's query head passes the last (never, if a round's rows are a
    // multiple of their number).
    constexpr int kLoads = kQueries * kChunks / kRowThreads;
    static_assert(kLoads * kRowThreads == kQueries * kChunks && kQueries <= kRowThreads, "rounds");
    u32x4 x[kLoads];
    float2 ml;
    int at = 0;
    const int tokens = kQueries / a.group, rest = kQueries % a.group;
    const int last = w.rows - 1;
    const uint16_t* const q =
        a.q + w.token0 * a.q_token + (int64_t)head * a.group * a.q_head + t % kChunks * 8;
    const float2* const stats =
        reinterpret_cast<const float2*>(a.stats) + (int64_t)w.token0 * heads + head * a.group;
    auto q_at = [&](int row) { return q + row / a.group * a.q_token + row % a.group * a.q_head; };
    const int64_t q_step = tokens * a.q_token + rest * a.q_head, q_wrap = a.q_token - a.group * a.q_head;
    const uint16_t* src[kLoads];
    int q_head[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = from + (i * kRowThreads + t) / kChunks;
      src[i] = q_at(row);
      q_head[i] = row % a.group;
    }
    const int own_row = from + t % kQueries;
    int token = own_row / a.group, own_head = own_row % a.group;
    auto load = [&](int row0) {
      if (row0 >= to) return;
      const bool whole = row0 + kQueries <= w.rows;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint16_t* p = src[i];
        if (!whole && row0 + (i * kRowThreads + t) / kChunks > last) p = q_at(last);
        x[i] = load16_any(p);
        src[i] += q_step;
        if (rest) {
          q_head[i] += rest;
          if (q_head[i] >= a.group) q_head[i] -= a.group, src[i] += q_wrap;
        }
      }
      if (t < kQueries) {
        const bool some = row0 + t <= last;
        ml = stats[some ? (int64_t)token * heads + own_head : 0];
        at = some ? w.first + token : kNowhere;
        token += tokens;
        own_head += rest;
        if (own_head >= a.group) own_head -= a.group, ++token;
      }
    };
    auto place = [&](int buf) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        // row n, chunk c: half c / kU, step c % kU
        const int n = (i * kRowThreads + t) / kChunks, c = t % kChunks;
        qs[buf][((n / 32 * kU + c % kU) * 2 + c / kU) * 32 + ((n ^ c) & 31)] = x[i];
      }
      if (t < kQueries) {  // (only here, so that the load before is not waited for at once)
        const RowWeight r(a, ml, at != kNowhere);
        weight[buf][t] = make_float2(r.shift, r.inv);
        position[buf][t] = at;
      }
    };
    int p_lo = w.first + from / a.group, lo_head = from % a.group;  // of a round's first row
    auto round = [&](int row0, auto which) {
      constexpr int buf = decltype(which)::value;
      place(buf);  // its readers of two rounds ago are past the barrier of the last
      __syncthreads();
      load(row0 + kQueries);
      const int p_hi = p_lo + (lo_head + kQueries - 1) / a.group;  // (rows past the last: more)
      const int p_first = row0 + kQueries <= w.rows ? p_lo : kNowhere;
      p_lo += tokens;
      lo_head += rest;
      if (lo_head >= a.group) lo_head -= a.group, ++p_lo;
      // (all operands are asked for before the first product: left to itself the
      // compiler reads each where it is used and waits for it)
      bf16x8 o[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        o[u] = __builtin_bit_cast(
            bf16x8, qs[buf][((part * kU + u) * 2 + half) * 32 + ((col ^ (half * kU + u)) & 31)]);
      const float2 r = weight[buf][32 * part + col];
      const int pos = position[buf][32 * part + col];
      __builtin_amdgcn_sched_barrier(0);
      f32x16 st;
#pragma unroll
      for (int i = 0; i < 16; ++i) st[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < kU; ++u) st = mfma32(k[u], o[u], st);
      // every row sees every key
      if (k0 + 31 <= p_first && (!a.window || k0 > p_hi - a.window || k0 + 32 <= a.sinks)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sum[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(st[i], a.scale, -r.x)), r.y,
                                  sum[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], a.scale, -r.x)) * r.y;
          sum[i] += sees(a, pos, k0 + 8 * (i >> 2) + 4 * half + (i & 3)) ? e : 0.0f;
        }
      }
    };
    __syncthreads();  // the last reads of the tile of keys before
    load(from);
    for (int row0 = from; row0 < to; row0 += 2 * kQueries) {
      round(row0, std::integral_constant<int, 0>{});
      if (row0 + kQueries < to) round(row0 + kQueries, std::integral_constant<int, 1>{});
    }

    // over the 32 lanes of a half wave, then the parts; lane n has its half's key n
    float own_sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = sum16(sum[i]);
      s += __shfl_xor(s, 16);
      own_sum = col == i ? s : own_sum;
    }
    if (col < 16) others[part][wave * 32 + 8 * (col >> 2) + 4 * half + (col & 3)] = own_sum;
    __syncthreads();
    if (t < kRowKeys) {
      const int64_t key = first_key + t;
      float all = 0.0f;
#pragma unroll
      for (int n = 0; n < kParts; ++n) all += others[n][t];
      const int id = key < w.len ? table[key >> a.cache.page_shift] : -1;
      if (id >= 0 && id < a.cache.pages)
        add_weight(marks.weights + id * marks.weights_page + (int64_t)head * size + (key & (size - 1)),
                   decay, all);
    }
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
    int tiles = (int)std::min<int64_t>((len + kRowKeys - 1) / kRowKeys, kKv4MaxWorkgroups / 2 / groups);
    void* params[] = {&a, &marks, &decay, &tiles};
    const void* fn = D == 64    ? reinterpret_cast<const void*>(&kv4_weigh_rows_kernel<64>)
                     : D == 128 ? reinterpret_cast<const void*>(&kv4_weigh_rows_kernel<128>)
                                : reinterpret_cast<const void*>(&kv4_weigh_rows_kernel<256>);
    return hipLaunchKernel(fn, dim3((unsigned)(groups * tiles)), dim3(kRowThreads), params, 0, s);
  }
  const int64_t all = (len + kStep - 1) / kStep;  // steps of a sequence, at most
  // about 8192 waves; with kept scores 256 keys to a wave
  int steps = a.kept ? 8 : (int)std::clamp<int64_t>(all * groups / 8192, 1, all);
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
