// kv4_weigh.hip -- what weight an attention gave to every cached key, added up
// over its rows (new tokens and query heads of the key head):
//
//   w[j] = decay w[j] + sum over rows r that see j of exp2((s_rj - m_r) scale) / l_r
//
// with each row's reference m and sum l as the attention left them.  The scores are
// computed once more: of a row's keys only the sums survive a pass over them, and to
// keep them would take 4 bytes a pair.  A wave has keys of its own, which it goes
// over all rows for, so nothing is added from two places and the sums come out the
// same every time.
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

template <int D>
__global__ void __launch_bounds__(kWaves * 64)
    kv4_weigh_kernel(Kv4AttentionArgs a, Kv4Marks marks, float decay, int steps) {
  constexpr int kJ = D / 32;
  using Codes = TileCodes<D>;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % a.cache.heads;
  Weighed w;
  if (!w.find(a, blockIdx.x / a.cache.heads)) return;
  const int all = (w.len + kStep - 1) / kStep;
  const int64_t stride = (int64_t)gridDim.y * kWaves * steps;
  int64_t begin = (int64_t)(blockIdx.y * kWaves + wave) * steps;
  if (begin >= all) return;
  const int size = 1 << a.cache.page_shift;
  const int32_t* const table = a.batch.table + w.s * a.batch.table_stride;
  const uint8_t* const base = a.cache.data + head * a.cache.head_bytes;

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
    const float2 ml = reinterpret_cast<const float2*>(
        a.stats)[(int64_t)(w.token0 + i) * (a.cache.heads * a.group) + h];
    // a row that saw nothing, or scores of -infinity only, gives nothing; nor does
    // one past the last
    const bool some = row0 + col < w.rows && ml.y != 0.0f;
    shift = some ? ml.x * a.scale : 0.0f;
    inv = some ? 1.0f / ml.y : 0.0f;
    pos = some ? w.first + i : -1 - (int)kKv4MaxLength;  // of no key's reach
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
        float* const at = marks.weights + page[x] * marks.weights_page + (int64_t)head * size +
                          (key & (size - 1));
        *at = decay == 0.0f ? mine : __builtin_fmaf(decay, *at, mine);
      }
    }
    if (++step == begin + steps) step = begin += stride;
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
  const int64_t all = std::max<int64_t>(1, (len + kStep - 1) / kStep);  // steps of a sequence, at most
  const int64_t groups = (int64_t)a.batch.sequences * a.cache.heads;
  // about 8192 waves
  int steps = (int)std::max<int64_t>(1, all * groups / 8192);
  void* params[] = {&a, &marks, &decay, &steps};
  const void* fn = D == 64    ? reinterpret_cast<const void*>(&kv4_weigh_kernel<64>)
                   : D == 128 ? reinterpret_cast<const void*>(&kv4_weigh_kernel<128>)
                              : reinterpret_cast<const void*>(&kv4_weigh_kernel<256>);
  const int64_t per = (int64_t)steps * kWaves;
  return hipLaunchKernel(fn, dim3((unsigned)groups, (unsigned)std::min<int64_t>((all + per - 1) / per, 65535)),
                         dim3(kWaves * 64), params, 0, s);
}
