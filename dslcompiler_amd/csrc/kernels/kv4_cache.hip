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
// HBM bound: 16 bytes of bf16 per thread (8 values; 4 threads to a block, which
// exchange their largest magnitudes in registers), 4 bytes of codes.
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

// A thread's 8 values: number u of a token's 2 * heads * D / 8.
template <int D>
struct Unit {
  int head, part, block, quarter;
  __device__ __forceinline__ explicit Unit(int u) {
    constexpr int kPer = D / 8;
    quarter = u % 4;
    block = u % kPer / 4;
    part = u / kPer % 2;  // 0 key, 1 value
    head = u / kPer / 2;
  }
  __device__ __forceinline__ int element() const { return block * 32 + quarter * 8; }
  __device__ __forceinline__ int code_at(int tok) const {
    return part * 8 * D + (block * 16 + tok) * 16 + quarter * 4;
  }
  __device__ __forceinline__ int scale_at(int tok) const {
    return 16 * D + part * (D / 2) + block * 16 + tok;
  }
};

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Byte BYTE of `codes` replaced by the codes of two bf16 values.
template <int BYTE>
__device__ __forceinline__ uint32_t encode2(uint32_t codes, uint32_t two, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2_t, two), scale,
                                                   BYTE);
}

template <int D>
__global__ void __launch_bounds__(256) kv4_write_kernel(Kv4Cache c, Kv4Batch b, Kv4Rows r) {
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= b.tokens) return;
  uint8_t* tile;
  int tok;
  if (!kv4_place(c, b, t, 17 * D, &tile, &tok)) return;
  const int units = c.heads * (D / 4);
  for (int i = threadIdx.x; i < units; i += blockDim.x) {
    const Unit<D> u(i);
    const uint16_t* src = u.part ? r.v + t * r.v_token + u.head * r.v_head
                                 : r.k + t * r.k_token + u.head * r.k_head;
    const u32x4 x = load16_any(src + u.element());
    // largest magnitude as bf16 bits, which order like the magnitudes: finite
    // ones, infinity, NaN
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      top = max_u32(top, max_u32(x[k] & 0x7fffu, (x[k] >> 16) & 0x7fffu));
    top = max_u32(top, quad_perm<kXor1>(top));
    top = max_u32(top, quad_perm<kXor2>(top));
    // exponent of a, plus one where its mantissa is beyond 1.75, minus 2
    int e = (int)((top + 0x1fu) >> 7) - 2;
    e = min(max(e, 1), 252);
    uint32_t codes = 0;
    if (top >= 0x7f80u) {
      e = 255;
    } else {
      const float scale = __uint_as_float((uint32_t)e << 23);
      codes = encode2<0>(codes, x[0], scale);
      codes = encode2<1>(codes, x[1], scale);
      codes = encode2<2>(codes, x[2], scale);
      codes = encode2<3>(codes, x[3], scale);
    }
    uint8_t* dst = tile + u.head * c.head_bytes;
    *reinterpret_cast<uint32_t*>(dst + u.code_at(tok)) = codes;
    if (u.quarter == 0) dst[u.scale_at(tok)] = (uint8_t)e;
  }
}

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Cache c, Kv4Batch b, Kv4Rows r) {
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= b.tokens) return;
  uint8_t* tile = nullptr;
  int tok = 0;
  const bool held = kv4_place(c, b, t, 17 * D, &tile, &tok);
  const int units = c.heads * (D / 4);
  for (int i = threadIdx.x; i < units; i += blockDim.x) {
    const Unit<D> u(i);
    u32x4 x{0, 0, 0, 0};
    if (held) {
      const uint8_t* src = tile + u.head * c.head_bytes;
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + u.code_at(tok));
      const float scale = __uint_as_float((uint32_t)src[u.scale_at(tok)] << 23);
      x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
      x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
      x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
      x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    }
    uint16_t* dst = u.part ? r.v + t * r.v_token + u.head * r.v_head
                           : r.k + t * r.k_token + u.head * r.k_head;
    store16_any(dst + u.element(), x);
  }
}

// A token's units across a workgroup, several tokens to one where they are few.
template <class K>
hipError_t launch_rows(K kernel, const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, int D,
                       hipStream_t s) {
  const int units = c.heads * (D / 4);
  const unsigned x = units < 256 ? units : 256, y = 256 / x;
  Kv4Cache ca = c;
  Kv4Batch ba = b;
  Kv4Rows ra = r;
  void* params[] = {&ca, &ba, &ra};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel),
                         dim3((unsigned)((b.tokens + y - 1) / y)), dim3(x, y), params, 0, s);
}

}  // namespace
}  // namespace llk_gfx950

hipError_t llk_launch_kv4_write(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, int D,
                                hipStream_t s) {
  using namespace llk_gfx950;
  return D == 64    ? launch_rows(&kv4_write_kernel<64>, c, b, r, D, s)
         : D == 128 ? launch_rows(&kv4_write_kernel<128>, c, b, r, D, s)
                    : launch_rows(&kv4_write_kernel<256>, c, b, r, D, s);
}

hipError_t llk_launch_kv4_read(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& r, int D,
                               hipStream_t s) {
  using namespace llk_gfx950;
  return D == 64    ? launch_rows(&kv4_read_kernel<64>, c, b, r, D, s)
         : D == 128 ? launch_rows(&kv4_read_kernel<128>, c, b, r, D, s)
                    : launch_rows(&kv4_read_kernel<256>, c, b, r, D, s);
}
