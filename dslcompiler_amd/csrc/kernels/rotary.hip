// rotary.hip -- rotary positions of queries and keys, in one launch.
//
// Pair i of a head at position p is turned by p f_i.  f_i is held as turns in
// units of 2^-64, so p times it modulo 2^64 is the exact fraction of a turn however
// far p lies (fp32 would lose an angle of 2^20 by 0.06); its upper 32 bits, as a
// signed number, give the angle to 2^-32 of a turn, and fp32 keeps 24 bits of it.
//
// HBM bound.  The cosines and sines of a workgroup's tokens are computed once,
// into LDS, and serve all heads of q and k.  16384 tokens of 32 + 8 heads of 128, bf16:
// 57.8 us, 5.8 TB/s of reads and writes (partly from the last-level cache).  That is with
// pairs in eights; other numbers of pairs go one at a time, and what is copied one
// value at a time: 4096 tokens of 40 heads of 96, 12 pairs 35.5 us, 48 pairs 16.1; of 80,
// 10 pairs 30.5, 16 pairs 18.4, 40 pairs 13.5.
#include <algorithm>

#include "common.h"
#include "rotary.h"

namespace llk_gfx950 {
namespace {

// 8 consecutive elements, as fp32.
template <bool F32>
struct Eight {
  float v[8];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    if constexpr (F32) {
      const float* q = static_cast<const float*>(p) + at;
      const f32x4 a = __builtin_bit_cast(f32x4, load16_any(q));
      const f32x4 b = __builtin_bit_cast(f32x4, load16_any(q + 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
      const u32x4 r = load16_any(static_cast<const uint16_t*>(p) + at);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t at) const {
    if constexpr (F32) {
      float* q = static_cast<float*>(p) + at;
      store16_any(q, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
      store16_any(q + 4, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
    } else {
      store16_any(static_cast<uint16_t*>(p) + at,
                  u32x4{f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]),
                        f32x2_to_bf16x2_rne(v[4], v[5]), f32x2_to_bf16x2_rne(v[6], v[7])});
    }
  }
};
template <bool F32>
__device__ __forceinline__ float load1(const void* p, int64_t at) {
  return F32 ? static_cast<const float*>(p)[at]
             : bf16_bits_to_f32(static_cast<const uint16_t*>(p)[at]);
}
template <bool F32>
__device__ __forceinline__ void store1(void* p, int64_t at, float v) {
  if constexpr (F32) static_cast<float*>(p)[at] = v;
  else static_cast<uint16_t*>(p)[at] = f32_to_bf16_rne(v);
}

__device__ __forceinline__ void turn(float& x, float& y, float2 cs) {
  const float a = x, b = y;
  x = __builtin_fmaf(a, cs.x, -(b * cs.y));
  y = __builtin_fmaf(b, cs.x, a * cs.y);
}

// A workgroup takes `per` tokens, of all heads; a thread's items are 16 values of a
// head (WIDE: both halves of 8 pairs, or 8 pairs side by side) or one pair.
template <bool F32, bool SIDE_BY_SIDE, bool WIDE>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a, int per) {
  extern __shared__ float2 turns[];  // [per][pairs]: cosine, sine
  const int t0 = blockIdx.x * per, tokens = min(per, a.tokens - t0);
  for (int i = threadIdx.x; i < tokens * a.pairs; i += 256) {
    const int64_t p = a.positions[t0 + i / a.pairs];
    const uint64_t angle = (uint64_t)p * a.turns[i % a.pairs];
    // half turns, from -1 to 1
    const float half = (float)(int32_t)(angle >> 32) * 0x1p-31f;
    float s, c;
    sincospif(half, &s, &c);
    turns[i] = make_float2(c * a.factor, (a.inverse ? -s : s) * a.factor);
  }
  __syncthreads();
  constexpr int kPairs = WIDE ? 8 : 1;
  const int items = a.pairs / kPairs;  // of a head
  const int rest = a.head_dim - 2 * a.pairs;  // values that are only copied
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const RotarySide& x = a.side[side];
    const int all = tokens * x.heads * items;
    for (int i = threadIdx.x; i < all; i += 256) {
      const int item = i % items, head = i / items % x.heads, t = i / items / x.heads;
      const int64_t from = (int64_t)(t0 + t) * x.in_token + (int64_t)head * x.in_head;
      const int64_t to = (int64_t)(t0 + t) * x.out_token + (int64_t)head * x.out_head;
      const float2* const cs = turns + t * a.pairs + item * kPairs;
      const int first = SIDE_BY_SIDE ? 2 * kPairs * item : kPairs * item;
      const int second = SIDE_BY_SIDE ? first + kPairs : first + a.pairs;
      if constexpr (WIDE) {
        Eight<F32> u, w;
        u.load(x.in, from + first);
        w.load(x.in, from + second);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          if constexpr (SIDE_BY_SIDE) {
            Eight<F32>& e = n < 4 ? u : w;
            turn(e.v[n % 4 * 2], e.v[n % 4 * 2 + 1], cs[n]);
          } else {
            turn(u.v[n], w.v[n], cs[n]);
          }
        }
        u.store(x.out, to + first);
        w.store(x.out, to + second);
      } else {
        float u = load1<F32>(x.in, from + first), w = load1<F32>(x.in, from + second);
        turn(u, w, cs[0]);
        store1<F32>(x.out, to + first, u);
        store1<F32>(x.out, to + second, w);
      }
    }
    if (rest == 0 || (x.in == x.out && x.in_token == x.out_token && x.in_head == x.out_head)) continue;
    // what is not turned: 8 values or one at a time
    const int wide = WIDE && rest % 8 == 0 ? 8 : 1, parts = rest / wide;
    for (int i = threadIdx.x; i < tokens * x.heads * parts; i += 256) {
      const int part = i % parts, head = i / parts % x.heads, t = i / parts / x.heads;
      const int at = 2 * a.pairs + part * wide;
      const int64_t from = (int64_t)(t0 + t) * x.in_token + (int64_t)head * x.in_head + at;
      const int64_t to = (int64_t)(t0 + t) * x.out_token + (int64_t)head * x.out_head + at;
      if (wide == 8) {
        if constexpr (F32) {
          const u32x4 lo = load16_any(static_cast<const float*>(x.in) + from);
          const u32x4 hi = load16_any(static_cast<const float*>(x.in) + from + 4);
          store16_any(static_cast<float*>(x.out) + to, lo);
          store16_any(static_cast<float*>(x.out) + to + 4, hi);
        } else {
          store16_any(static_cast<uint16_t*>(x.out) + to,
                      load16_any(static_cast<const uint16_t*>(x.in) + from));
        }
      } else if constexpr (F32) {
        static_cast<uint32_t*>(x.out)[to] = static_cast<const uint32_t*>(x.in)[from];
      } else {
        static_cast<uint16_t*>(x.out)[to] = static_cast<const uint16_t*>(x.in)[from];
      }
    }
  }
}

template <bool F32, bool SIDE_BY_SIDE>
hipError_t launch(const RotaryArgs& args, hipStream_t s) {
  RotaryArgs a = args;
  const bool wide = a.pairs % 8 == 0;
  const int items = (a.side[0].heads + a.side[1].heads) * (wide ? a.pairs / 8 : a.pairs);
  // An item to a thread, not more than 256 cosines, and two workgroups to a CU.
  // Measured, us, 1, 2, 4 and 8 tokens to a workgroup: 16384 tokens, 40 heads of 128,
  // 57.8, 59.0, 60.9, 60.6; 9 heads of 64 15.8, 10.4, 8.5, 7.5; 64 tokens, 40 heads of
  // 128, 3.0, 3.4, 4.1.
  int per = std::max(1, std::min(std::min(256 / a.pairs, 256 / items), a.tokens / 512));
  void* params[] = {&a, &per};
  return hipLaunchKernel(wide ? reinterpret_cast<const void*>(&rotary_kernel<F32, SIDE_BY_SIDE, true>)
                              : reinterpret_cast<const void*>(&rotary_kernel<F32, SIDE_BY_SIDE, false>),
                         dim3((a.tokens + per - 1) / per), dim3(256), params,
                         (size_t)per * a.pairs * sizeof(float2), s);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_rotary(const RotaryArgs& a, bool f32, bool interleaved, hipStream_t s) {
  using namespace llk_gfx950;
  if (f32) return interleaved ? launch<true, true>(a, s) : launch<true, false>(a, s);
  return interleaved ? launch<false, true>(a, s) : launch<false, false>(a, s);
}
