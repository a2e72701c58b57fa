// kv4_evict.hip -- which slots of the cache stay, by the weight that attention gave
// them, and the cache moved together.
//
// Plan: a workgroup to a sequence's head.  The slots' order is that of a 32-bit key:
// the weight's bits, turned so that they order like numbers, under the largest key
// for the protected ones.  The `keep`-th largest key is found digit by digit (8 bits,
// counts in LDS), and of those equal to it the lowest slots stay.  Slots below `keep`
// that stay are not moved: the holes among them take, in order, those from `keep` on
// that stay.  So few bytes move however long the cache is, and none is read after it
// was written: sources lie from `keep` on, targets below.
//
// Move: a wave to 64 slots below `keep`; 16 codes' bytes and their scale to a lane.
#include <algorithm>

#include "common.h"
#include "kv4.h"

namespace llk_gfx950 {
namespace {

constexpr int kThreads = 1024, kPlanWaves = kThreads / 64;

struct Slots {  // of a sequence's head
  const Kv4EvictPlan& p;
  const int32_t* table;
  int head, last;
  __device__ __forceinline__ bool at(int j, int64_t* page, int* off) const {
    const int id = table[j >> p.page_shift];
    *page = id;
    *off = (head << p.page_shift) + (j & ((1 << p.page_shift) - 1));
    return id >= 0 && id < p.pages;
  }
  __device__ __forceinline__ uint32_t key(int j) const {
    int64_t page;
    int off;
    if (!at(j, &page, &off)) return 0;
    if (p.marks.positions) {
      const int pos = p.marks.positions[page * p.marks.positions_page + off];
      if ((int64_t)pos > (int64_t)last - p.recent || pos < p.first) return 0xffffffffu;
    }
    const float w = p.marks.weights[page * p.marks.weights_page + off];
    if (w != w) return 1;
    const uint32_t u = __float_as_uint(w + 0.0f);  // -0 as 0
    return u >> 31 ? ~u : u | 0x80000000u;
  }
};

// Sum over the workgroup, and of the threads before this one.
__device__ __forceinline__ int scan(int x, int* before, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int mine = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(mine, d);
    if (lane >= d) mine += o;
  }
  if (lane == 63) part[wave] = mine;
  __syncthreads();
  int all = 0, base = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    base += w < wave ? part[w] : 0;
    all += part[w];
  }
  __syncthreads();
  *before = base + mine - x;
  return all;
}

__global__ void __launch_bounds__(kThreads) kv4_evict_plan_kernel(Kv4EvictPlan p) {
  __shared__ int counts[256], part[kPlanWaves];
  __shared__ int shared_last, shared_digit, shared_above;
  const int s = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int64_t cap = min((int64_t)p.batch.table_pages << p.page_shift, (int64_t)kKv4MaxLength);
  const int n = (int)max((int64_t)0, min((int64_t)p.batch.lens[s], cap));
  int32_t* const source = p.source + ((int64_t)s * p.heads + head) * p.keep;
  if (head == 0 && threadIdx.x == 0) p.lens[s] = min(p.batch.lens[s], p.keep);
  for (int j = threadIdx.x + (n > p.keep ? p.keep : 0); j < p.keep; j += kThreads) source[j] = j;
  if (n <= p.keep) return;
  Slots slots{p, p.batch.table + s * p.batch.table_stride, head, 0};

  if (p.marks.positions) {  // the newest position
    if (threadIdx.x == 0) shared_last = INT32_MIN;
    __syncthreads();
    int last = INT32_MIN;
    for (int j = threadIdx.x; j < n; j += kThreads) {
      int64_t page;
      int off;
      if (slots.at(j, &page, &off))
        last = max(last, p.marks.positions[page * p.marks.positions_page + off]);
    }
    atomicMax(&shared_last, last);
    __syncthreads();
    slots.last = shared_last;
  }

  // the keep-th largest key, and how many of those equal to it stay
  uint32_t key = 0;
  int left = p.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) counts[threadIdx.x] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += kThreads) {
      const uint32_t k = slots.key(j);
      if (shift == 24 || (k ^ key) >> (shift + 8) == 0) atomicAdd(&counts[k >> shift & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + counts[d] < left) above += counts[d--];
      shared_digit = d;
      shared_above = above;
    }
    __syncthreads();
    key |= (uint32_t)shared_digit << shift;
    left -= shared_above;
    __syncthreads();
  }

  // Those from keep on that stay, in order, to the front of source; `equal` of the
  // slots equal to the key lie before a round of slots.
  int equal = 0, extras = 0;
  auto stays = [&](int j, int bound) {
    const uint32_t k = j < bound ? slots.key(j) : 0;
    int before;
    const int same = j < bound && k == key;
    const int all = scan(same, &before, part);
    const bool stay = j < bound && (k > key || (same && equal + before < left));
    equal += all;
    return stay;
  };
  for (int j0 = 0; j0 < p.keep; j0 += kThreads) stays(j0 + threadIdx.x, p.keep);
  const int below = equal;
  for (int j0 = p.keep; j0 < n; j0 += kThreads) {
    const bool stay = stays(j0 + threadIdx.x, n);
    int before;
    const int all = scan(stay, &before, part);
    if (stay) source[extras + before] = j0 + threadIdx.x;
    extras += all;
  }
  __syncthreads();
  // From the last slots below keep to the first: hole i, at or after slot i, takes
  // source[i], which no slot after the round has any use for.
  int holes = extras;  // in this round and before it
  equal = below;
  for (int j0 = (p.keep - 1) / kThreads * kThreads; j0 >= 0; j0 -= kThreads) {
    const int j = j0 + threadIdx.x;
    const uint32_t k = j < p.keep ? slots.key(j) : 0;
    const int same = j < p.keep && k == key;
    int before, nth;
    equal -= scan(same, &before, part);
    const bool hole = j < p.keep && !(k > key || (same && equal + before < left));
    holes -= scan(hole, &nth, part);
    const int from = hole ? source[holes + nth] : j;
    __syncthreads();
    if (j < p.keep) source[j] = from;
    __syncthreads();
  }
}

constexpr int kMoveWaves = 4;

template <int D>
__global__ void __launch_bounds__(kMoveWaves * 64)
    kv4_evict_kernel(Kv4Cache c, Kv4Batch b, Kv4Marks marks, const int32_t* source, int keep,
                     int32_t* lens) {
  __shared__ int2 moves[kMoveWaves][64];
  constexpr int kBlocks = D / 16;  // of a token's key and value
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = blockIdx.x / c.heads, head = blockIdx.x % c.heads;
  const int64_t cap = min((int64_t)b.table_pages << c.page_shift, (int64_t)kKv4MaxLength);
  const int32_t* const table = b.table + s * b.table_stride;
  const int32_t* const from = source + ((int64_t)s * c.heads + head) * keep;
  const int size = 1 << c.page_shift;
  if (lens && head == 0 && blockIdx.y == 0 && threadIdx.x == 0) lens[s] = min(lens[s], keep);
  for (int j0 = (blockIdx.y * kMoveWaves + wave) * 64; j0 < keep; j0 += gridDim.y * kMoveWaves * 64) {
    const int j = j0 + lane, src = j < keep ? from[j] : j;
    // (a source below keep could be a target itself: never one of a plan's)
    const bool moved = src != j && src >= keep && src < cap && j < cap;
    const uint64_t mask = __ballot(moved);
    if (moved) moves[wave][__popcll(mask & ((1ull << lane) - 1))] = make_int2(j, src);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int all = __popcll(mask) * kBlocks;
    for (int i = lane; i < all; i += 64) {
      const int2 m = moves[wave][i / kBlocks];
      const int part = i % kBlocks / (kBlocks / 2), block = i % (kBlocks / 2);
      const int to = table[m.x >> c.page_shift], of = table[m.y >> c.page_shift];
      if (to < 0 || to >= c.pages || of < 0 || of >= c.pages) continue;
      auto at = [&](int page, int slot) {
        return c.data + page * c.page_stride + head * c.head_bytes +
               (int64_t)((slot & (size - 1)) >> 4) * (17 * D);
      };
      uint8_t* const dst = at(to, m.x);
      const uint8_t* const org = at(of, m.y);
      const int code = part * 8 * D + block * 256, scale = 16 * D + part * (D / 2) + block * 16;
      *reinterpret_cast<u32x4*>(dst + code + (m.x & 15) * 16) =
          *reinterpret_cast<const u32x4*>(org + code + (m.y & 15) * 16);
      dst[scale + (m.x & 15)] = org[scale + (m.y & 15)];
      if (i % kBlocks == 0) {
        const int64_t dm = (int64_t)head * size + (m.x & (size - 1));
        const int64_t om = (int64_t)head * size + (m.y & (size - 1));
        if (marks.weights)
          marks.weights[to * marks.weights_page + dm] = marks.weights[of * marks.weights_page + om];
        if (marks.positions)
          marks.positions[to * marks.positions_page + dm] =
              marks.positions[of * marks.positions_page + om];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_evict_plan(const Kv4EvictPlan& plan, int64_t, hipStream_t s) {
  Kv4EvictPlan p = plan;
  void* params[] = {&p};
  return hipLaunchKernel(reinterpret_cast<const void*>(&llk_gfx950::kv4_evict_plan_kernel),
                         dim3((unsigned)(p.batch.sequences * p.heads)), dim3(llk_gfx950::kThreads),
                         params, 0, s);
}

hipError_t llk_launch_kv4_evict(const Kv4Cache& cache, const Kv4Batch& batch, const Kv4Marks& m,
                                const int32_t* source, int keep, int32_t* lens, int D,
                                hipStream_t s) {
  using namespace llk_gfx950;
  Kv4Cache c = cache;
  Kv4Batch b = batch;
  Kv4Marks marks = m;
  void* params[] = {&c, &b, &marks, &source, &keep, &lens};
  const void* fn = D == 64    ? reinterpret_cast<const void*>(&kv4_evict_kernel<64>)
                   : D == 128 ? reinterpret_cast<const void*>(&kv4_evict_kernel<128>)
                              : reinterpret_cast<const void*>(&kv4_evict_kernel<256>);
  const int blocks = std::min((keep + kMoveWaves * 64 - 1) / (kMoveWaves * 64), 65535);
  return hipLaunchKernel(fn, dim3((unsigned)(b.sequences * c.heads), (unsigned)blocks),
                         dim3(kMoveWaves * 64), params, 0, s);
}
