// block_norm.hip -- what stands between two blocks of a decoder layer, in one
// pass over the residual stream: the norm after a block, its gate and residual
// scale, the residual sum, and the norm before the next block.
//
//   u  = y * rsqrt(mean(y^2) + eps) * (w_post + offset)     (or y itself)
//   h' = h + scale * g * u                                  (g: gate, or 1)
//   n  = h' * rsqrt(mean(h'^2) + eps) * (w_pre + offset)
//
// HBM bound: y, h and g are read once and h', n written once, since a row stays
// in registers between the two sums (a workgroup per row, CH chunks of 8
// elements per thread; with 4 chunks, above 16384 columns, part of it spills unless
// y and the weights are bf16: 4097 rows of fp32 with a gate, 16384 columns 268 us,
// 5.0 TB/s, 32768 columns 688 us, 3.9; of bf16 127 us, 5.3, and 290 us, 4.6).  All arithmetic and both sums are in fp32; h' is
// rounded to the residual's type only where it is stored, so n is the norm of
// the unrounded sum.
#include "block_norm.h"

#include <algorithm>

#include "common.h"

namespace llk_gfx950 {
namespace {

// 8 consecutive elements as fp32: one (bf16) or two (fp32) 16-byte loads at
// any alignment; `n` (1..8) of them at a row's end.
template <bool F32>
struct Chunk;
template <>
struct Chunk<false> {
  u32x4 raw;
  __device__ __forceinline__ void load(const void* p, int64_t at, int n) {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    raw = n >= 8 ? load16_any(q) : load16_part(q, n);
  }
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? raw[i >> 1] & 0xffff0000u : raw[i >> 1] << 16);
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, int n, const float (&v)[8]) {
    uint16_t* q = static_cast<uint16_t*>(p) + at;
    const u32x4 r{f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]),
                  f32x2_to_bf16x2_rne(v[4], v[5]), f32x2_to_bf16x2_rne(v[6], v[7])};
    if (n >= 8) {
      store16_any(q, r);
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < n) q[i] = (uint16_t)(i & 1 ? r[i >> 1] >> 16 : r[i >> 1]);
    }
  }
};
template <>
struct Chunk<true> {
  u32x4 raw[2];
  __device__ __forceinline__ void load(const void* p, int64_t at, int n) {
    const uint32_t* q = static_cast<const uint32_t*>(p) + at;
    if (n >= 8) {
      raw[0] = load16_any(q);
      raw[1] = load16_any(q + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i >> 2][i & 3] = i < n ? q[i] : 0u;
    }
  }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(raw[i >> 2][i & 3]); }
  static __device__ __forceinline__ void store(void* p, int64_t at, int n, const float (&v)[8]) {
    float* q = static_cast<float*>(p) + at;
    if (n >= 8) {
      store16_any(q, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
      store16_any(q + 4, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < n) q[i] = v[i];
    }
  }
};

// Sum over the workgroup (a multiple of 64 threads, at most 1024), the same
// value in every thread.  Each call of a kernel gets a `part` of its own, so
// one barrier is enough.
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
  for (int w = 0; w < waves; ++w) s += part[w];
  return s;
}

// One row per workgroup, its elements in registers: thread t holds chunks t,
// t + blockDim, ... (at most CH).
template <int CH, bool YF, bool RF, bool OF, bool WF>
__global__ void __launch_bounds__(1024) block_norm_kernel(BlockNormArgs a) {
  __shared__ float part[2][16];
  const int64_t m = blockIdx.x;
  const int N = a.N, chunks = (N + 7) >> 3;
  const int64_t yo = m * a.ldy, ho = m * a.ldh, go = m * a.ldg;
  Chunk<YF> y[CH], g[CH];
  Chunk<RF> h[CH];
  Chunk<WF> wpost[CH], wpre[CH];
  int c[CH], n[CH];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    c[k] = threadIdx.x + k * blockDim.x;
    n[k] = c[k] < chunks ? min(8, N - 8 * c[k]) : 0;
  }
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (n[k] == 0) continue;
    h[k].load(a.h, ho + 8 * c[k], n[k]);
    if (a.y) y[k].load(a.y, yo + 8 * c[k], n[k]);
    if (a.g) g[k].load(a.g, go + 8 * c[k], n[k]);
  }
  // the weights too before the first sum, not each after its own
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (n[k] == 0) continue;
    if (a.wpost) wpost[k].load(a.wpost, 8 * c[k], n[k]);
    wpre[k].load(a.wpre, 8 * c[k], n[k]);
  }
  float r = 1.0f;
  if (a.wpost) {
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (n[k])
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(y[k].get(i), y[k].get(i), ss);
    r = 1.0f / sqrtf(block_sum(ss, part[0]) / (float)N + a.eps);
  }
  float v[CH][8];
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (n[k] == 0) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = h[k].get(i);
      if (a.y) {
        float u = y[k].get(i);
        if (a.wpost) u = u * r * (wpost[k].get(i) + a.offset);
        if (a.g) u *= g[k].get(i);
        x = __builtin_fmaf(a.scale, u, x);
      }
      // past a row's end the loads gave zeros, whose sum is zero too
      v[k][i] = x;
      ss = __builtin_fmaf(x, x, ss);
    }
    if (a.h_out) Chunk<RF>::store(a.h_out, m * a.ldho + 8 * c[k], n[k], v[k]);
  }
  r = 1.0f / sqrtf(block_sum(ss, part[1]) / (float)N + a.eps);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (n[k] == 0) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] = v[k][i] * r * (wpre[k].get(i) + a.offset);
    Chunk<OF>::store(a.out, m * a.ldo + 8 * c[k], n[k], v[k]);
  }
}

template <int CH, bool YF, bool RF, bool OF>
const void* pick_w(bool wf) {
  return wf ? reinterpret_cast<const void*>(&block_norm_kernel<CH, YF, RF, OF, true>)
            : reinterpret_cast<const void*>(&block_norm_kernel<CH, YF, RF, OF, false>);
}
template <int CH, bool YF, bool RF>
const void* pick_o(bool of, bool wf) {
  return of ? pick_w<CH, YF, RF, true>(wf) : pick_w<CH, YF, RF, false>(wf);
}
template <int CH>
const void* pick(bool yf, bool rf, bool of, bool wf) {
  if (yf) return rf ? pick_o<CH, true, true>(of, wf) : pick_o<CH, true, false>(of, wf);
  return rf ? pick_o<CH, false, true>(of, wf) : pick_o<CH, false, false>(of, wf);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_block_norm(const BlockNormArgs& a, int64_t M, bool y_f32, bool h_f32,
                                 bool o_f32, bool w_f32, hipStream_t s) {
  using namespace llk_gfx950;
  const int chunks = (a.N + 7) / 8;
  // Chunks to a thread: one where few rows leave CUs idle, two where there are
  // enough; more only where 1024 threads are too few.  Bf16 rows of 5120 with a gate,
  // one and two chunks, us: 17 rows 6.3 and 6.7, 256 6.8 and 7.2, 512 10.0 both, 640
  // 12.2 and 11.2, 1024 15.0 and 13.6, 4097 50 and 41.  (fp32 rows of 4096 without
  // one do better with one chunk at any number: 1024 rows 13.3 and 13.8, 4097 41 and
  // 45.)
  int ch = M <= 512 ? 1 : 2;
  while (chunks > ch * 1024) ch *= 2;
  const int threads = ((chunks + ch - 1) / ch + 63) / 64 * 64;
  const void* fn = ch == 1   ? pick<1>(y_f32, h_f32, o_f32, w_f32)
                   : ch == 2 ? pick<2>(y_f32, h_f32, o_f32, w_f32)
                             : pick<4>(y_f32, h_f32, o_f32, w_f32);
  BlockNormArgs args = a;
  void* params[] = {&args};
  // a dimension of a launch takes fewer than 2^32 threads; with more it runs some
  // of them only, and says nothing
  const int64_t most = ((int64_t)1 << 31) / threads;
  auto advance = [&](const void*& p, int64_t ld, bool f32) {
    if (p) p = static_cast<const uint8_t*>(p) + most * ld * (f32 ? 4 : 2);
  };
  for (int64_t left = M;; left -= most) {
    const hipError_t e =
        hipLaunchKernel(fn, dim3((unsigned)std::min(left, most)), dim3(threads), params, 0, s);
    if (e != hipSuccess || left <= most) return e;
    advance(args.y, a.ldy, y_f32);
    advance(args.g, a.ldg, y_f32);
    advance(args.h, a.ldh, h_f32);
    if (args.h_out) args.h_out = static_cast<uint8_t*>(args.h_out) + most * a.ldho * (h_f32 ? 4 : 2);
    args.out = static_cast<uint8_t*>(args.out) + most * a.ldo * (o_f32 ? 4 : 2);
  }
}
