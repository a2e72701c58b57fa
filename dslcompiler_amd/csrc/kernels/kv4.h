// kv4.h -- the 4-bit paged cache of keys and values: its layout, the device
// side of its addressing, and its launchers.
//
// A token's key (value) of one head, D values, is cut into blocks of 32.  A
// block is a scale byte E standing for 2^(E - 127) and 32 four-bit codes: a
// sign over an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6 -- the element and scale
// types of the OCP Microscaling (MX) FP4 format, which gfx950 converts in
// hardware (two values per instruction, the scale included).  Byte i of a
// block's 16 holds value 2i in its low half and 2i + 1 in its high half.
// E = 255 stands for a block of NaN; 1 <= E <= 252 otherwise, so every other
// value is a finite bf16, exactly.
//
// 16 consecutive tokens of a page and head are one tile of 17 D bytes:
//
//   key codes [D/32][16 tokens][16 bytes], value codes likewise,
//   key scales [D/32][16 tokens], value scales likewise
//
// in which a tile's D/32 x 16 blocks are the lanes of a wave in the order of a
// v_mfma_f32_16x16x32_bf16 A operand (lane = block * 16 + token): one 1 KiB
// wave load (D = 128) is a ready operand but for the conversion, and a tile's
// keys, values and scales are one contiguous run of memory.
// The cache is [pages][heads][page_size / 16 tiles].
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// The cache's memory.  Every page holds heads * head_bytes bytes.
struct Kv4Cache {
  uint8_t* data;
  int64_t page_stride;  // bytes
  int64_t head_bytes;   // page_size * 17 D / 16
  int pages, heads, page_shift;  // page_size = 1 << page_shift
};

// The call's sequences.  starts null: one new token each.
struct Kv4Batch {
  const int32_t *table, *lens, *starts;
  int64_t table_stride;
  int table_pages;  // pages named per sequence
  int sequences, tokens;
};

// What is kept of every slot beside the cache, [pages][heads][page_size] each (either
// may be null): the attention weight it got, and its token's position.
struct Kv4Marks {
  float* weights;
  int32_t* positions;
  int64_t weights_page, positions_page;  // page strides in elements
};

struct Kv4AttentionArgs {
  Kv4Cache cache;
  Kv4Batch batch;
  const uint16_t* q;
  uint16_t* out;
  int64_t q_token, q_head, out_token, out_head;  // strides in elements
  float* part;        // split partials: see kv4_attention.hip
  int group;          // query heads to a key head
  int window, sinks;  // window 0: none
  uint32_t span;      // the window, or 2^31
  int tiles;          // row tiles (of all sequences)
  int splits, chunk;  // splits of a sequence's key steps, steps to a split
  float scale;        // of q.k, times log2(e)
  float* stats;       // null, or [tokens][q heads][2]: a row's reference score and sum
  // null, or the scores of single tokens' rows of 16 at most: [sequence][key head][row]
  // [kept_keys], of the first kept_keys keys (a multiple of 256)
  float* kept;
  int kept_keys;
};

// A dimension of a launch takes fewer than 2^32 threads (with more it runs some of
// them only): workgroups of 256, and tokens at 16 to a workgroup of the write and
// the read.
constexpr int64_t kKv4MaxWorkgroups = ((int64_t)1 << 24) - 1;
constexpr int64_t kKv4MaxMoved = kKv4MaxWorkgroups * 16;

// k, v (out for read): element strides of tokens and heads.
struct Kv4Rows {
  uint16_t *k, *v;
  int64_t k_token, k_head, v_token, v_head;
};
// marks: of the tokens that are written, weight 0 and position at[token] (null: the
// slot's number).
hipError_t llk_launch_kv4_write(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& rows, int D,
                                hipStream_t s, const Kv4Marks* marks = nullptr,
                                const int32_t* at = nullptr);
hipError_t llk_launch_kv4_read(const Kv4Cache& c, const Kv4Batch& b, const Kv4Rows& rows, int D,
                               hipStream_t s);

// Attention: `rows` is the row tile (query heads of a key head times tokens):
// 16 or 32, whose keys a workgroup's waves divide, or kKv4PromptRows, which
// they divide instead.
constexpr int kKv4PromptRows = 128;
hipError_t llk_launch_kv4_prompt(const Kv4AttentionArgs& a, int D, hipStream_t s);
hipError_t llk_launch_kv4_attention(const Kv4AttentionArgs& a, int D, int rows, hipStream_t s);
size_t llk_kv4_attention_part_bytes(int64_t tiles, int heads, int splits, int rows, int D);

// After an attention that left its rows' statistics, and their scores where it kept
// them: adds every key's weights up.
hipError_t llk_launch_kv4_weigh(const Kv4AttentionArgs& a, const Kv4Marks& marks, float decay, int D,
                                int64_t max_len, hipStream_t s);

// Which slots of a sequence's heads stay, and where they come from.
struct Kv4EvictPlan {
  Kv4Marks marks;
  Kv4Batch batch;
  int pages, heads, page_shift;  // of the marks
  int keep, recent, first;
  int32_t* lens;    // [sequences]
  int32_t* source;  // [sequences][heads][keep]
};
hipError_t llk_launch_kv4_evict_plan(const Kv4EvictPlan& p, int64_t max_len, hipStream_t s);
hipError_t llk_launch_kv4_evict(const Kv4Cache& c, const Kv4Batch& b, const Kv4Marks& marks,
                                const int32_t* source, int keep, int32_t* lens, int D,
                                hipStream_t s);
// Longest sequence (and window); positions and their sums fit 32 bits.
constexpr int kKv4MaxLength = 1 << 30;
// Keys that one step of a tile of `rows` rows covers.
constexpr int kv4_step(int rows) { return rows == kKv4PromptRows ? 64 : 32; }

#ifdef __HIPCC__
namespace llk_gfx950 {

// Positions a sequence holds: what its length says, within the table.
__device__ __forceinline__ int kv4_length(const Kv4Cache& c, const Kv4Batch& b, int s) {
  const int64_t cap = min((int64_t)b.table_pages << c.page_shift, (int64_t)kKv4MaxLength);
  return (int)max((int64_t)0, min((int64_t)b.lens[s], cap));
}

// The page of a position, or -1 where the table names none that exists.
__device__ __forceinline__ int kv4_page(const Kv4Cache& c, const Kv4Batch& b, int s, int pos) {
  const int id = b.table[s * b.table_stride + (pos >> c.page_shift)];
  return id >= 0 && id < c.pages ? id : -1;
}

// The sequence of new token t: the last one that starts at or before it.
__device__ __forceinline__ int kv4_sequence(const Kv4Batch& b, int t) {
  if (!b.starts) return t;
  int lo = 0, hi = b.sequences - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.starts[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Where new token t of the call lies: its position, page and slot in the page;
// false if it has no place (outside every sequence, before position 0, past the
// table, on a page that does not exist).
__device__ __forceinline__ bool kv4_slot(const Kv4Cache& c, const Kv4Batch& b, int t, int* pos,
                                         int* page, int* slot) {
  const int s = kv4_sequence(b, t);
  if (s >= b.sequences) return false;
  const int first = b.starts ? b.starts[s] : s, next = b.starts ? b.starts[s + 1] : s + 1;
  if (t < first || t >= next) return false;
  const int64_t p = (int64_t)b.lens[s] - (next - t);
  if (p < 0 || p >= kKv4MaxLength || p >= (int64_t)b.table_pages << c.page_shift) return false;
  *pos = (int)p;
  *page = kv4_page(c, b, s, (int)p);
  *slot = (int)p & ((1 << c.page_shift) - 1);
  return *page >= 0;
}

// The same as its 16-token tile (of head 0) and its number in it.
__device__ __forceinline__ bool kv4_place(const Kv4Cache& c, const Kv4Batch& b, int t,
                                          int tile_bytes, uint8_t** tile, int* tok) {
  int pos, page, slot;
  if (!kv4_slot(c, b, t, &pos, &page, &slot)) return false;
  *tile = c.data + page * c.page_stride + (int64_t)(slot >> 4) * tile_bytes;
  *tok = slot & 15;
  return true;
}

}  // namespace llk_gfx950
#endif
