// kv4_evict.hip -- which slots of the cache stay, by the weight that attention gave
// them, and the cache moved together.
//
// Plan: a workgroup to a sequence's head.  The slots' order is that of a 32-bit key:
// the weight's bits, turned so that they order like numbers, under the largest key
// for the protected ones.  The `keep`-th largest key is found from its upper bits
// down, and of those equal to it the lowest slots stay.  Slots below `keep`
// that stay are not moved: the holes among them take, in order, those from `keep` on
// that stay.  So few bytes move however long the cache is, and none is read after it
// was written: sources lie from `keep` on, targets below.
//
// What bounds it is the chain of its passes: one sequence's 8 heads 10 us, 512 heads of
// up to 8192 slots 28 us (36 with two bits of the key a pass, counted by ballots).
//
// Move: a lane to a slot below `keep`, with all of its token's blocks on their way at
// once.  HBM: a token's 16 bytes of every 256 and its scales' single bytes are parts of
// lines that are moved whole.  512 heads 64 us; with loads that stay in the caches 90,
// with the blocks of a token on neighbouring lanes 101.
#include <algorithm>

#include "common.h"
#include "kv4.h"

namespace llk_gfx950 {
namespace {

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
template <int WAVES>
__device__ __forceinline__ int scan_threads(int x, int* before, int* part) {
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
#pragma unroll 1
  for (int w = 0; w < WAVES; ++w) {
    base += w < wave ? part[w] : 0;
    all += part[w];
  }
  __syncthreads();
  *before = base + mine - x;
  return all;
}

// Any length: the keys are read from memory at every pass.
template <int THREADS>
__device__ __forceinline__ void plan_long(const Kv4EvictPlan& p, int s, int head, int n,
                                          int32_t* source) {
  __shared__ int counts[256], part[THREADS / 64];
  __shared__ int shared_last, shared_digit, shared_above;
  Slots slots{p, p.batch.table + s * p.batch.table_stride, head, 0};

  if (p.marks.positions) {  // the newest position
    if (threadIdx.x == 0) shared_last = INT32_MIN;
    __syncthreads();
    int last = INT32_MIN;
    for (int j = threadIdx.x; j < n; j += THREADS) {
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
    for (int i = threadIdx.x; i < 256; i += THREADS) counts[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += THREADS) {
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
    const int all = scan_threads<THREADS / 64>(same, &before, part);
    const bool stay = j < bound && (k > key || (same && equal + before < left));
    equal += all;
    return stay;
  };
  for (int j0 = 0; j0 < p.keep; j0 += THREADS) stays(j0 + threadIdx.x, p.keep);
  const int below = equal;
  for (int j0 = p.keep; j0 < n; j0 += THREADS) {
    const bool stay = stays(j0 + threadIdx.x, n);
    int before;
    const int all = scan_threads<THREADS / 64>(stay, &before, part);
    if (stay) source[extras + before] = j0 + threadIdx.x;
    extras += all;
  }
  __syncthreads();
  // From the last slots below keep to the first: hole i, at or after slot i, takes
  // source[i], which no slot after the round has any use for.
  int holes = extras;  // in this round and before it
  equal = below;
  for (int j0 = (p.keep - 1) / THREADS * THREADS; j0 >= 0; j0 -= THREADS) {
    const int j = j0 + threadIdx.x;
    const uint32_t k = j < p.keep ? slots.key(j) : 0;
    const int same = j < p.keep && k == key;
    int before, nth;
    equal -= scan_threads<THREADS / 64>(same, &before, part);
    const bool hole = j < p.keep && !(k > key || (same && equal + before < left));
    holes -= scan_threads<THREADS / 64>(hole, &nth, part);
    const int from = hole ? source[holes + nth] : j;
    __syncthreads();
    if (j < p.keep) source[j] = from;
    __syncthreads();
  }
}

// Sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ uint32_t row_sum(uint32_t x) {
  x += __builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true);  // row_ror:8
  x += __builtin_amdgcn_mov_dpp(x, 0x124, 0xf, 0xf, true);
  x += __builtin_amdgcn_mov_dpp(x, 0x122, 0xf, 0xf, true);
  x += __builtin_amdgcn_mov_dpp(x, 0x121, 0xf, 0xf, true);
  return x;
}

// Sums over the lanes up to this one, in DPP steps.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// Up to PER * THREADS slots: the keys stay in registers, slot THREADS i + t in thread
// t's i-th.  The keep-th largest is found by its upper 11 bits, then the next 11 and
// the last 10, each time by counting the keys that agree so far in LDS (a weight's
// sign, exponent and two bits of its mantissa spread over enough counters that lanes
// seldom meet).  GUARD: some positions are protected.
template <int PER, int THREADS, bool GUARD>
__device__ __forceinline__ void plan_short(const Kv4EvictPlan& p, int s, int head, int n,
                                           int32_t* source) {
  constexpr int kWaves = THREADS / 64, kParts = PER * kWaves;
  static_assert(kWaves <= 16 && PER * THREADS <= 16384, "counts and slots of 16 bits");
  constexpr int kBins = 2048, kOwn = kBins / THREADS;  // counters, and of a thread
  __shared__ int bins[kBins];
  __shared__ int totals[16];  // of the waves
  __shared__ int found[3];
  __shared__ uint32_t part[kParts];
  __shared__ uint16_t extra[PER * THREADS / 2];
  __shared__ int newest;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int32_t* const table = p.batch.table + s * p.batch.table_stride;
  // (slots past n read slot n - 1's, absent ones page 0's marks: all loads are in
  // flight at once)
  const int inner = (1 << p.page_shift) - 1;
  int page[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) page[i] = table[min(i * THREADS + t, n - 1) >> p.page_shift];
  float w[PER];
  int pos[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool here = page[i] >= 0 && page[i] < p.pages;
    const int64_t id = here ? page[i] : 0;
    const int off = (head << p.page_shift) + (min(i * THREADS + t, n - 1) & inner);
    w[i] = p.marks.weights[id * p.marks.weights_page + off];
    if constexpr (GUARD) pos[i] = p.marks.positions[id * p.marks.positions_page + off];
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) bins[i * THREADS + t] = 0;
  if (t < 16) totals[t] = 0;
  int last = INT32_MIN;
  if constexpr (GUARD) {
    if (t == 0) newest = INT32_MIN;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      last = max(last, page[i] >= 0 && page[i] < p.pages ? pos[i] : INT32_MIN);
    atomicMax(&newest, last);
    __syncthreads();
    last = __builtin_amdgcn_readfirstlane(newest);
  }
  // positions from here on are protected
  const int64_t cut = (int64_t)last - p.recent + 1;
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t u = __float_as_uint(w[i] + 0.0f);  // -0 as 0
    key[i] = u >> 31 ? ~u : u | 0x80000000u;
    if (w[i] != w[i]) key[i] = 1;
    if constexpr (GUARD) {
      if (pos[i] >= cut || pos[i] < p.first) key[i] = 0xffffffffu;
    }
    if (page[i] < 0 || page[i] >= p.pages || i * THREADS + t >= n) key[i] = 0;
  }
  __syncthreads();

  // `least`: the bits seen so far of the keep-th largest key, and zeros.  `reach`
  // keys are not below it; `left` of those that agree with it are to stay.  Slots
  // past n have the key 0, as absent ones, and the last places.
  uint32_t least = 0;
  int reach = 0, left = p.keep;
#pragma unroll
  for (int shift = 21, width = 11; shift >= 0; width = shift == 10 ? 10 : 11, shift -= width) {
    const uint32_t mask = (1u << width) - 1;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (shift == 21 || (key[i] ^ least) >> (shift + width) == 0)
        atomicAdd(&bins[mask - (key[i] >> shift & mask)], 1);
    __syncthreads();
    int mine[kOwn], all = 0;  // counters from the largest digit on
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      mine[i] = bins[t * kOwn + i];
      bins[t * kOwn + i] = 0;
      all += mine[i];
    }
    const int up_to = wave_scan(all);
    if (lane == 63) totals[wave] = up_to;
    __syncthreads();
    int base = (lane & 15) < wave ? totals[lane & 15] : 0;
    base = (int)row_sum((uint32_t)base);
    int before = base + up_to - all;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (before < left && left <= before + mine[i]) {
        found[0] = (int)mask - (t * kOwn + i);
        found[1] = before;
        found[2] = mine[i];
      }
      before += mine[i];
    }
    __syncthreads();
    least |= (uint32_t)__builtin_amdgcn_readfirstlane(found[0]) << shift;
    const int above = __builtin_amdgcn_readfirstlane(found[1]);
    const int same = __builtin_amdgcn_readfirstlane(found[2]);
    reach = p.keep - left + above + same;
    left -= above;
    if (reach == p.keep) break;  // all that agree stay
  }

  // part to the sums before each entry
  auto scan = [&] {
    __syncthreads();
    if (wave == 0) {
      uint32_t base = 0;
#pragma unroll
      for (int i = 0; i < kParts; i += 64) {
        const int v = i + lane < kParts ? (int)part[i + lane] : 0, up_to = wave_scan(v);
        if (i + lane < kParts) part[i + lane] = base + up_to - v;
        base += __builtin_amdgcn_readlane(up_to, 63);
      }
    }
    __syncthreads();
  };
  auto before = [&](uint64_t mask) {  // lanes of it before this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
  };
  uint32_t stays = 0;  // bit i: the thread's i-th slot
#pragma unroll
  for (int i = 0; i < PER; ++i) stays |= (uint32_t)(key[i] >= least) << i;
  if (reach != p.keep) {
    // All bits are seen, and more keys are equal to the keep-th largest than stay:
    // the lowest slots of them, `left`.
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t same = (uint32_t)__popcll(__ballot(key[i] == least));
      if (lane == 0) part[i * kWaves + wave] = same;
    }
    scan();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int nth = (int)(part[i * kWaves + wave] + before(__ballot(key[i] == least)));
      if (key[i] == least && nth >= left) stays &= ~(1u << i);
    }
    __syncthreads();
  }
  // holes below keep in the lower half of a count, those from keep on that stay in
  // the upper
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool low = i * THREADS + t < p.keep, stay = stays >> i & 1;
    const uint32_t holes = (uint32_t)__popcll(__ballot(low && !stay));
    const uint32_t more = (uint32_t)__popcll(__ballot(!low && stay));
    if (lane == 0) part[i * kWaves + wave] = holes | more << 16;
  }
  scan();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool more = i * THREADS + t >= p.keep && (stays >> i & 1);
    const uint32_t nth = (part[i * kWaves + wave] >> 16) + before(__ballot(more));
    if (more) extra[nth] = (uint16_t)(i * THREADS + t);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * THREADS + t;
    const bool hole = j < p.keep && !(stays >> i & 1);
    const uint32_t nth = (part[i * kWaves + wave] & 0xffffu) + before(__ballot(hole));
    if (j < p.keep) source[j] = hole ? extra[nth] : j;
  }
}

template <int PER, int THREADS, bool GUARD>
__global__ void __launch_bounds__(THREADS)
    __attribute__((amdgpu_waves_per_eu(PER <= 8 ? 8 : 4))) kv4_evict_plan_kernel(Kv4EvictPlan p) {
  const int s = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int64_t cap = min((int64_t)p.batch.table_pages << p.page_shift, (int64_t)kKv4MaxLength);
  const int n = (int)max((int64_t)0, min((int64_t)p.batch.lens[s], cap));
  int32_t* const source = p.source + ((int64_t)s * p.heads + head) * p.keep;
  if (head == 0 && threadIdx.x == 0) p.lens[s] = min(p.batch.lens[s], p.keep);
  if (n <= p.keep) {
    for (int j = threadIdx.x; j < p.keep; j += THREADS) source[j] = j;
    return;
  }
  if (n <= PER * THREADS) plan_short<PER, THREADS, GUARD>(p, s, head, n, source);
  else plan_long<THREADS>(p, s, head, n, source);
}

template <int PER, int THREADS>
hipError_t plan(const Kv4EvictPlan& args, hipStream_t s) {
  Kv4EvictPlan p = args;
  void* params[] = {&p};
  return hipLaunchKernel(
      p.marks.positions ? reinterpret_cast<const void*>(&kv4_evict_plan_kernel<PER, THREADS, true>)
                        : reinterpret_cast<const void*>(&kv4_evict_plan_kernel<PER, THREADS, false>),
      dim3((unsigned)(p.batch.sequences * p.heads)), dim3(THREADS), params, 0, s);
}

constexpr int kMoveWaves = 4;

template <int D>
__global__ void __launch_bounds__(kMoveWaves * 64)
    kv4_evict_kernel(Kv4Cache c, Kv4Batch b, Kv4Marks marks, const int32_t* source, int keep,
                     int32_t* lens) {
  constexpr int kBlocks = D / 16;  // of a token's key and value
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = blockIdx.x / c.heads, head = blockIdx.x % c.heads;
  const int64_t cap = min((int64_t)b.table_pages << c.page_shift, (int64_t)kKv4MaxLength);
  const int32_t* const table = b.table + s * b.table_stride;
  const int32_t* const from = source + ((int64_t)s * c.heads + head) * keep;
  const int size = 1 << c.page_shift;
  if (lens && head == 0 && blockIdx.y == 0 && threadIdx.x == 0) lens[s] = min(lens[s], keep);
  for (int j = (blockIdx.y * kMoveWaves + wave) * 64 + lane; j < keep; j += gridDim.y * kMoveWaves * 64) {
    const int src = from[j];
    // (a source below keep could be a target itself: never one of a plan's)
    if (src == j || src < keep || src >= cap || j >= cap) continue;
    const int to = table[j >> c.page_shift], of = table[src >> c.page_shift];
    if (to < 0 || to >= c.pages || of < 0 || of >= c.pages) continue;
    const int x = j & (size - 1), y = src & (size - 1);
    uint8_t* const dst = c.data + to * c.page_stride + head * c.head_bytes + (int64_t)(x >> 4) * (17 * D);
    const uint8_t* const org =
        c.data + of * c.page_stride + head * c.head_bytes + (int64_t)(y >> 4) * (17 * D);
    const int64_t dm = (int64_t)head * size + x, om = (int64_t)head * size + y;
    u32x4 codes[kBlocks];
    uint8_t scales[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      codes[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(org + i * 256 + (y & 15) * 16));
      scales[i] = org[16 * D + i * 16 + (y & 15)];
    }
    float w = 0.0f;
    int pos = 0;
    if (marks.weights) w = marks.weights[of * marks.weights_page + om];
    if (marks.positions) pos = marks.positions[of * marks.positions_page + om];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      *reinterpret_cast<u32x4*>(dst + i * 256 + (x & 15) * 16) = codes[i];
      dst[16 * D + i * 16 + (x & 15)] = scales[i];
    }
    if (marks.weights) marks.weights[to * marks.weights_page + dm] = w;
    if (marks.positions) marks.positions[to * marks.positions_page + dm] = pos;
  }
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_evict_plan(const Kv4EvictPlan& p, int64_t max_len, hipStream_t s) {
  using namespace llk_gfx950;
  int64_t len = (int64_t)p.batch.table_pages << p.page_shift;
  if (max_len > 0) len = std::min(len, max_len);
  // Slots in registers: 2, 8 or 16 to a thread; a longer sequence reads its marks at
  // every pass.  Measured, us, of 64 sequences of 8 heads: 2000 slots 12.5, 27.3 and
  // 53.7; 8000 slots 117 (at every pass), 20.1 and 47.6.
  return len <= 2048 ? plan<2, 1024>(p, s) : len <= 8192 ? plan<8, 1024>(p, s) : plan<16, 1024>(p, s);
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
