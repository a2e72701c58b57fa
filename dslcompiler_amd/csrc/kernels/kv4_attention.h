// kv4_attention.h -- device side of the attention over the 4-bit cache that its
// kernels share: row tiles and the keys they cover, the codes' conversion, V's
// place in LDS, partial results.
#pragma once

#include "common.h"
#include "kv4.h"

namespace llk_gfx950 {

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16* lds_v4i16;

constexpr float kNegInf = -__builtin_inff();

// A row tile: its sequence, the positions its rows ask from and the steps of
// kv4_step(R) keys it covers: `sink` steps from key 0, then those from `low`.
struct RowTile {
  int s, row0, rows;     // sequence; first row of the sequence; rows in it
  int first, token0;     // position and index of the sequence's first new token
  int p_lo, p_last;      // positions of the tile's first and last query
  int p_hi;              // the last of them that the sequence holds: no later key is read
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
  // A new token past what the table holds keeps its position, of which causality
  // and the window go; the keys there are absent.  (len, if lens is beyond the
  // table, is whole pages, so no 16 keys that are read lie partly past it.)
  o->first = (int)max((int64_t)b.lens[o->s] - (next - first), -(int64_t)kKv4MaxLength);
  o->p_lo = o->first + o->row0 / a.group;
  o->p_last = o->first + (o->row0 + o->rows - 1) / a.group;
  o->p_hi = min(o->p_last, len - 1);
  o->sink = o->low = o->steps = 0;
  if (o->p_hi < 0) return true;
  constexpr int kStep = kv4_step(R);
  const int end = o->p_hi / kStep + 1;
  if (a.window) {
    o->low = max(0, o->p_lo - a.window + 1) / kStep;
    o->sink = min((a.sinks + kStep - 1) / kStep, min(o->low, end));
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

// The reference m of a row's exponentials is its largest score so far, but
// follows it only once it has grown by a factor of 2^8 of the weights: until then
// they are at most 2^8, at no loss (the sums are fp32 and bf16 keeps its 8 bits),
// and the accumulators need no rescaling, which 16 rows' maxima would ask for
// at nearly every step.  top: the largest of the lane's scores and m.
__device__ __forceinline__ bool outgrown(const Kv4AttentionArgs& a, float top, float m) {
  return (top - m) * a.scale > 8.0f;  // m -inf: once there is a score
}
// What l and the accumulators are multiplied by when m becomes top.  Of a row
// without a score yet m is -inf, and they are 0.
__device__ __forceinline__ float rescale(const Kv4AttentionArgs& a, float top, float m) {
  return __builtin_amdgcn_exp2f((m - (top == kNegInf ? 0.0f : top)) * a.scale);
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

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool ONCE, class T>
__device__ __forceinline__ T read(const uint8_t* p) {
  const T* q = reinterpret_cast<const T*>(p);
  if constexpr (ONCE) return __builtin_nontemporal_load(q);
  else return *q;
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

  // ONCE: no other workgroup reads the tile, so it need not stay in L2.
  template <bool ONCE>
  __device__ __forceinline__ void load(const uint8_t* tile, int lane) {
    if constexpr (D == 64) {
      const int block = lane >> 5, half = (lane >> 4) & 1, tok = lane & 15;
      const int at = (block * 16 + tok) * 16 + half * 8;
      const u32x2 a = read<ONCE, u32x2>(tile + at), b = read<ONCE, u32x2>(tile + 8 * D + at);
#pragma unroll
      for (int i = 0; i < 2; ++i) k[i] = a[i], v[i] = b[i];
      ks[0] = tile[16 * D + block * 16 + tok];
      vs[0] = tile[16 * D + D / 2 + block * 16 + tok];
    } else {
#pragma unroll
      for (int c = 0; c < kScales; ++c) {
        const u32x4 a = read<ONCE, u32x4>(tile + c * 1024 + lane * 16);
        const u32x4 b = read<ONCE, u32x4>(tile + 8 * D + c * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[4 * c + i] = a[i], v[4 * c + i] = b[i];
        ks[c] = tile[16 * D + c * 64 + lane];
        vs[c] = tile[16 * D + D / 2 + c * 64 + lane];
      }
    }
  }
  static __device__ __forceinline__ int scale_of(int dword) { return D == 256 ? dword / 4 : 0; }
  // First of the 8 values of dword j.
  static __device__ __forceinline__ int element(int j, int lane) {
    return D == 256 ? (j >> 2) * 128 + (lane >> 4) * 32 + (j & 3) * 8
                    : (lane >> 4) * (D / 4) + j * 8;
  }
};

// V of 16-key tiles in LDS, as bf16: [16-key tile][D / 16][half: 8 values][16
// keys] of 16 bytes, the keys of the second half swapped by 8 and those of every
// other 16 values by 4, so that the 32 lanes of a half wave, which read both
// halves of 8 keys' 16 values or of 4 keys' 32, meet all 64 banks.
template <int D>
__device__ __forceinline__ int v_chunk(int x, int d16, int half, int key) {
  return ((x * (D / 16) + d16) * 2 + half) * 256 + (key ^ (half * 8) ^ ((d16 & 1) * 4)) * 16;
}

// Whether the query at position pos sees key j (of a page that exists): among
// the last a.span keys up to its own (all, without a window: pos - j, unsigned,
// is at least 2^31 for a later key), or as one of the first.
__device__ __forceinline__ bool in_window(const Kv4AttentionArgs& a, int pos, int j) {
  return (uint32_t)(pos - j) < a.span;
}
__device__ __forceinline__ bool sees(const Kv4AttentionArgs& a, int pos, int j) {
  return in_window(a, pos, j) || (j <= pos && j < a.sinks);
}

// Values of NaN blocks go into the products as zeros (0 * NaN would reach the
// rows that do not see them); here they are added to the lane's row, at
// position pos, if it sees them.  flags: the lanes of the 16-key tile from key0
// on that hold part of such a block (scale c of TileCodes); o: the row's
// accumulators.  Rare, so not unrolled over the keys.
template <int D>
__device__ void add_nan(const Kv4AttentionArgs& a, uint64_t flags, int c, int key0, int pos,
                        f32x4 (&o)[D / 16]) {
  uint32_t seen = 0;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) seen |= (uint32_t)sees(a, pos, key0 + i) << i;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    // the lanes that hold these 16 values: those of group g
    if (D == 256 && d / 8 != c) continue;
    const int g = D == 256 ? d % 8 / 2 : d * 16 / (D / 4);
    if ((uint32_t)(flags >> (16 * g)) & seen & 0xffffu) o[d] += __builtin_nanf("");
  }
}

// An output of a row whose weights' sum is l (inv: 1 / l).  l is 0 if the row saw
// no key, or only scores of -infinity: then zero, whatever o holds (add_nan's NaN).
__device__ __forceinline__ float result(float o, float l, float inv) {
  return l == 0.0f ? 0.0f : o * inv;
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
  // Elements d..d + 3 of the tile's row r.
  __device__ __forceinline__ void store(const Kv4AttentionArgs& a, const RowTile& rt, int head,
                                        int r, int d) const {
    const int row = rt.row0 + r;
    const float inv = 1.0f / l;
    uint16_t* dst = a.out + (int64_t)(rt.token0 + row / a.group) * a.out_token +
                    (int64_t)(head * a.group + row % a.group) * a.out_head + d;
    store8_any(dst, make_uint2(f32x2_to_bf16x2_rne(result(o[0], l, inv), result(o[1], l, inv)),
                               f32x2_to_bf16x2_rne(result(o[2], l, inv), result(o[3], l, inv))));
  }
};

}  // namespace llk_gfx950
