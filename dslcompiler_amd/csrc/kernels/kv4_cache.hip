// kv4_cache.hip -- quantises keys and values as they are written to the 4-bit
// paged cache (kv4.h), and reads them back.
//
// Write: a block of 32 values with largest magnitude a gets the smallest power
// of two X with a <= 7 X as its scale (held to 2^-126 .. 2^125): the codes'
// largest step lies between 4 and 6, and a value of up to 7 X, rounded to 6 X,
// is no further off than one in the middle of that step, while the next larger
// X would double every step.  Each value is then the nearest code (ties to
// even).  A block with an infinity or a NaN is stored as NaN.
//
// HBM bound.  A wave takes one block of 16 tokens: 4 lanes to a token, 8 values
// (16 bytes of bf16, 4 of codes) to a lane, which exchange their largest
// magnitudes in registers.  Consecutive tokens' codes are contiguous, so the
// codes of a wave are one run of 256 bytes and the values 16 runs of 64.  The
// tokens' places are looked up once for all blocks that the wave goes through.
// (With a workgroup to a token, its lanes over the values: 43530 tokens of 8
// heads of 128 written in 119 us and read in 110, here in 59 and 52, 3.8 and 4.3
// TB/s; a prompt of 2048 tokens of 32 heads 15 and 19, here 11.5 and 10.9.)
#include <algorithm>

#include "common.h"
#include "kv4.h"

namespace llk_gfx950 {
namespace {

// x of the lane that differs in bit 0 (bit 1) of the lane number.
template <int CTRL>
__device__ __forceinline__ uint32_t quad_perm(uint32_t x) {
  return __builtin_amdgcn_mov_dpp(x, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E;

// A block of 16 tokens: number c of heads * 2 * D / 32.
template <int D>
struct Block {
  int head, part, block;  // part: 0 key, 1 value
  __device__ __forceinline__ explicit Block(int c) {
    constexpr int kBlocks = D / 32;
    block = c % kBlocks;
    part = c / kBlocks % 2;
    head = c / kBlocks / 2;
  }
  __device__ __forceinline__ int code_at(int tok) const {
    return part * 8 * D + (block * 16 + tok) * 16;
  }
  __device__ __forceinline__ int scale_at(int tok) const {
    return 16 * D + part * (D / 2) + block * 16 + tok;
  }
  __device__ __forceinline__ uint16_t* row(const Kv4Rows& r, int64_t t) const {
    return (part ? r.v + t * r.v_token + head * r.v_head : r.k + t * r.k_token + head * r.k_head) +
           block * 32;
  }
};

// Byte BYTE's two codes as bf16.
template <int BYTE>
__device__ __forceinline__ uint32_t decode2(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
}

// The blocks of a wave: every 4 gridDim.y-th of all, kAhead of them on their way
// at once.
constexpr int kWaves = 4, kAhead = 4;
struct Walk {
  int c, step;
  __device__ __forceinline__ Walk()
      : c(blockIdx.y * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
        step(gridDim.y * kWaves) {}
};

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Byte BYTE of `codes` replaced by the codes of two bf16 values.
template <int BYTE>
__device__ __forceinline__ uint32_t encode2(uint32_t codes, uint32_t two, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2_t, two), scale,
                                                   BYTE);
}

// MARKS: the tokens' marks too.
template <int D, bool MARKS>
__global__ void __launch_bounds__(kWaves * 64)
    kv4_write_kernel(Kv4Cache c, Kv4Batch b, Kv4Rows r, Kv4Marks marks, const int32_t* at) {
  const int lane = threadIdx.x & 63, quarter = lane & 3, t = blockIdx.x * 16 + (lane >> 2);
  uint8_t* tile = nullptr;
  int tok = 0;
  if (t >= b.tokens || !kv4_place(c, b, t, 17 * D, &tile, &tok)) return;
  const int blocks = c.heads * (D / 16);
  if constexpr (MARKS) {
    // a thread to a head of the token
    int own, page = 0, slot = 0;
    kv4_slot(c, b, t, &own, &page, &slot);
    const int pos = at ? at[t] : own, size = 1 << c.page_shift;
    for (int h = (blockIdx.y * kWaves + (threadIdx.x >> 6)) * 4 + quarter; h < c.heads;
         h += gridDim.y * kWaves * 4) {
      if (marks.weights) marks.weights[page * marks.weights_page + (int64_t)h * size + slot] = 0.0f;
      if (marks.positions) marks.positions[page * marks.positions_page + (int64_t)h * size + slot] = pos;
    }
  }
  for (Walk w; w.c < blocks; w.c += kAhead * w.step) {
    u32x4 x[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
      if (w.c + n * w.step < blocks)
        x[n] = load16_any(Block<D>(w.c + n * w.step).row(r, t) + quarter * 8);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (w.c + n * w.step >= blocks) break;
      const Block<D> k(w.c + n * w.step);
      // largest magnitude as bf16 bits, which order like the magnitudes: finite
      // ones, infinity, NaN
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top = max_u32(top, max_u32(x[n][i] & 0x7fffu, (x[n][i] >> 16) & 0x7fffu));
      top = max_u32(top, quad_perm<kXor1>(top));
      top = max_u32(top, quad_perm<kXor2>(top));
      // exponent of a, plus one where its mantissa is beyond 1.75, minus 2
      int e = (int)((top + 0x1fu) >> 7) - 2;
      e = min(max(e, 1), 252);
      const float scale = __uint_as_float((uint32_t)e << 23);
      uint32_t codes = 0;
      codes = encode2<0>(codes, x[n][0], scale);
      codes = encode2<1>(codes, x[n][1], scale);
      codes = encode2<2>(codes, x[n][2], scale);
      codes = encode2<3>(codes, x[n][3], scale);
      const bool finite = top < 0x7f80u;
      uint8_t* const dst = tile + k.head * c.head_bytes;
      *reinterpret_cast<uint32_t*>(dst + k.code_at(tok) + quarter * 4) = finite ? codes : 0u;
      if (quarter == 0) dst[k.scale_at(tok)] = (uint8_t)(finite ? e : 255);
    }
  }
}

// 16 bytes to any 2-byte aligned address, PAST the L2 for more than it keeps.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
template <bool PAST>
__device__ __forceinline__ void store16(void* p, const u32x4& v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, static_cast<u32x4_any*>(p));
  else store16_any(p, v);
}

template <int D, bool PAST>
__global__ void __launch_bounds__(kWaves * 64) kv4_read_kernel(Kv4Cache c, Kv4Batch b, Kv4Rows r) {
  const int lane = threadIdx.x & 63, quarter = lane & 3, t = blockIdx.x * 16 + (lane >> 2);
  if (t >= b.tokens) return;
  uint8_t* tile = c.data;
  int tok = 0;
  const bool held = kv4_place(c, b, t, 17 * D, &tile, &tok);
  const int blocks = c.heads * (D / 16);
  for (Walk w; w.c < blocks; w.c += kAhead * w.step) {
    uint32_t codes[kAhead], e[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (w.c + n * w.step >= blocks) break;
      const Block<D> k(w.c + n * w.step);
      const uint8_t* const src = tile + k.head * c.head_bytes;  // page 0's without a place
      codes[n] = *reinterpret_cast<const uint32_t*>(src + k.code_at(tok) + quarter * 4);
      e[n] = src[k.scale_at(tok)];
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (w.c + n * w.step >= blocks) break;
      const uint32_t some = held ? codes[n] : 0u;
      const float scale = __uint_as_float((held ? e[n] : 0u) << 23);
      store16<PAST>(
          Block<D>(w.c + n * w.step).row(r, t) + quarter * 8,
          u32x4{decode2<0>(some, scale), decode2<1>(some, scale), decode2<2>(some, scale),
                decode2<3>(some, scale)});
    }
  }
}

// 16 tokens to a workgroup, and enough workgroups along the blocks for 2048 in
// all, at least one block to a wave.
template <class K>
hipError_t launch_rows(K kernel, const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, int D,
                       hipStream_t s, const Kv4Marks* marks = nullptr, const int32_t* at = nullptr) {
  const unsigned groups = (unsigned)((b.tokens + 15) / 16);
  const unsigned most = (unsigned)(c.heads * (D / 16) + kWaves - 1) / kWaves;
  const unsigned y = std::min(std::max((2048 + groups - 1) / groups, 1u), std::min(most, 65535u));
  Kv4Cache ca = c;
  Kv4Batch ba = b;
  Kv4Rows ra = r;
  Kv4Marks ma = marks ? *marks : Kv4Marks{};
  void* params[] = {&ca, &ba, &ra, &ma, &at};  // (the read takes the first three)
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(groups, y), dim3(kWaves * 64),
                         params, 0, s);
}

template <int D>
hipError_t write(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, const Kv4Marks* marks,
                 const int32_t* at, hipStream_t s) {
  return launch_rows(marks ? &kv4_write_kernel<D, true> : &kv4_write_kernel<D, false>, c, b, r, D, s,
                     marks, at);
}
// From 64 MiB of keys and values on they are written past the L2.  8 heads of 128,
// through the L2 and past it, us, into memory other than the last call's: 50 MB 14.2
// and 16.6, 67 MB 24 and 21, 101 MB 38 and 29, 134 MB 57 and 39, 178 MB 76 and 52, 268
// MB 113 and 78.  (Into the same memory again and again, as a replayed graph does, the
// caches hold it for longer: 67 MB 17.5 and 21, 134 MB 30 and 39, 147 MB 47 and 44.)
template <int D>
hipError_t read(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, hipStream_t s) {
  const bool past = (int64_t)b.tokens * c.heads * D * 4 >= (int64_t)64 << 20;
  return past ? launch_rows(&kv4_read_kernel<D, true>, c, b, r, D, s)
              : launch_rows(&kv4_read_kernel<D, false>, c, b, r, D, s);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_write(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, int D,
                                hipStream_t s, const Kv4Marks* marks, const int32_t* at) {
  using namespace llk_gfx950;
  return D == 64    ? write<64>(c, b, r, marks, at, s)
         : D == 128 ? write<128>(c, b, r, marks, at, s)
                    : write<256>(c, b, r, marks, at, s);
}

hipError_t llk_launch_kv4_read(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, int D,
                               hipStream_t s) {
  using namespace llk_gfx950;
  return D == 64 ? read<64>(c, b, r, s) : D == 128 ? read<128>(c, b, r, s) : read<256>(c, b, r, s);
}
