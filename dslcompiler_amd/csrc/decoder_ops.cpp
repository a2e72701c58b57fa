// decoder_ops.cpp -- C entry points of the operators around the MLP in a
// decoder block (include/llk/llk_abi.h): the fused residual norm, the 4-bit paged cache
// with the attention that reads it, the weights that it gave, and eviction by them.
// Kernels: kernels/block_norm.hip, kernels/kv4_cache.hip, kernels/kv4_attention.hip,
// kernels/kv4_prompt.hip, kernels/kv4_weigh.hip, kernels/kv4_evict.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "abi_support.h"
#include "kernels/block_norm.h"
#include "kernels/kv4.h"
#include "llk/llk_abi.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return llk::setError(code, buf);
}
int fail_hip(hipError_t e, const char* what) {
  return fail(LLK_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
hipStream_t stream_of(const llk_kernel_context* ctx) {
  return ctx ? static_cast<hipStream_t>(ctx->stream) : nullptr;
}

// --- block norm ------------------------------------------------------------

bool norm_type(int t) { return t == LLK_BF16 || t == LLK_FP32; }
size_t type_size(int t) { return t == LLK_FP32 ? 4 : 2; }

// A [M, N] operand of the block norm; one_row: M rows of it may be one row
// (stride0 0).
int check_rows(const llk_tensor2d* t, const char* name, int64_t M, int64_t N, int type,
               bool one_row) {
  if (t->dim0 != M || t->dim1 != N)
    return fail(LLK_ERR_SHAPE, "%s shape (%lld, %lld) != (%lld, %lld)", name, (long long)t->dim0,
                (long long)t->dim1, (long long)M, (long long)N);
  if (!norm_type(type)) return fail(LLK_ERR_DTYPE, "%s type %d unsupported (bf16 or f32)", name, type);
  if (M == 0) return LLK_OK;
  if (!t->data) return fail(LLK_ERR_INVALID_ARGUMENT, "%s.data is NULL", name);
  if (t->stride1 != 1 && N > 1)
    return fail(LLK_ERR_LAYOUT, "%s.stride1 is %lld; only unit inner stride is supported", name,
                (long long)t->stride1);
  if (M > 1 && t->stride0 < N && !(one_row && t->stride0 == 0))
    return fail(LLK_ERR_LAYOUT, "%s.stride0 (%lld) < dim1 (%lld)", name, (long long)t->stride0,
                (long long)N);
  if (reinterpret_cast<uintptr_t>(t->data) % type_size(type))
    return fail(LLK_ERR_LAYOUT, "%s.data is not aligned to its elements", name);
  return LLK_OK;
}

// --- 4-bit cache -----------------------------------------------------------

bool page_size_ok(int64_t p) { return p >= 16 && p <= 4096 && (p & (p - 1)) == 0; }
bool head_dim_ok(int64_t d) { return d == 64 || d == 128 || d == 256; }

constexpr int64_t kMaxTokens = (int64_t)1 << 30;

int check_cache(const llk_kv4_cache* c, Kv4Cache* out) {
  if (!c) return fail(LLK_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (!head_dim_ok(c->head_dim))
    return fail(LLK_ERR_SHAPE, "cache head_dim %lld unsupported (64, 128 or 256)",
                (long long)c->head_dim);
  if (!page_size_ok(c->page_size))
    return fail(LLK_ERR_SHAPE, "cache page_size %lld unsupported (a power of two, 16 to 4096)",
                (long long)c->page_size);
  if (c->pages < 1 || c->pages > 0x7fffffff || c->heads < 1 || c->heads > 65535)
    return fail(LLK_ERR_SHAPE, "cache of %lld pages and %lld heads unsupported",
                (long long)c->pages, (long long)c->heads);
  if (!c->data) return fail(LLK_ERR_INVALID_ARGUMENT, "cache.data is NULL");
  const int64_t head_bytes = llk_kv4_head_bytes(c->page_size, c->head_dim);
  if (reinterpret_cast<uintptr_t>(c->data) % 16 || c->page_stride % 16)
    return fail(LLK_ERR_LAYOUT, "cache data and page_stride must be multiples of 16 bytes");
  if (c->pages > 1 && c->page_stride < c->heads * head_bytes)
    return fail(LLK_ERR_LAYOUT, "cache.page_stride (%lld) < %lld heads of %lld bytes",
                (long long)c->page_stride, (long long)c->heads, (long long)head_bytes);
  out->data = static_cast<uint8_t*>(c->data);
  out->page_stride = c->page_stride;
  out->head_bytes = head_bytes;
  out->pages = (int)c->pages;
  out->heads = (int)c->heads;
  out->page_shift = __builtin_ctzll((unsigned long long)c->page_size);
  return LLK_OK;
}

int check_batch(const llk_kv4_batch* b, Kv4Batch* out) {
  if (!b) return fail(LLK_ERR_INVALID_ARGUMENT, "batch is NULL");
  if (b->sequences < 0 || b->sequences > kMaxTokens || b->tokens < 0 || b->tokens > kMaxTokens)
    return fail(LLK_ERR_SHAPE, "batch of %lld sequences and %lld tokens unsupported",
                (long long)b->sequences, (long long)b->tokens);
  if (!b->starts && b->tokens != b->sequences)
    return fail(LLK_ERR_SHAPE, "without starts there is one token per sequence: %lld != %lld",
                (long long)b->tokens, (long long)b->sequences);
  if (b->table_pages < 0 || b->table_pages > 0x7fffffff)
    return fail(LLK_ERR_SHAPE, "table of %lld pages unsupported", (long long)b->table_pages);
  if (b->sequences > 0 && (!b->lens || (b->table_pages > 0 && !b->table)))
    return fail(LLK_ERR_INVALID_ARGUMENT, "batch.table or batch.lens is NULL");
  if (b->sequences > 1 && b->table_stride < 0)
    return fail(LLK_ERR_LAYOUT, "batch.table_stride (%lld) < 0", (long long)b->table_stride);
  out->table = b->table;
  out->lens = b->lens;
  out->starts = b->starts;
  out->table_stride = b->table_stride;
  out->table_pages = (int)b->table_pages;
  out->sequences = (int)b->sequences;
  out->tokens = (int)b->tokens;
  return LLK_OK;
}

// bf16 [tokens, heads, head_dim] rows.  result: no two elements may share
// memory.
int check_rows3(const llk_tensor3d* t, const char* name, int64_t tokens, int64_t heads, int64_t D,
                bool result) {
  if (!t) return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", name);
  if (t->dim0 != tokens || t->dim1 != heads || t->dim2 != D)
    return fail(LLK_ERR_SHAPE, "%s shape (%lld, %lld, %lld) != (%lld, %lld, %lld)", name,
                (long long)t->dim0, (long long)t->dim1, (long long)t->dim2, (long long)tokens,
                (long long)heads, (long long)D);
  if (tokens == 0 || heads == 0) return LLK_OK;
  if (!t->data) return fail(LLK_ERR_INVALID_ARGUMENT, "%s.data is NULL", name);
  if (reinterpret_cast<uintptr_t>(t->data) % 2)
    return fail(LLK_ERR_LAYOUT, "%s.data is not aligned to its elements", name);
  if (t->stride2 != 1)
    return fail(LLK_ERR_LAYOUT, "%s.stride2 is %lld; only unit inner stride is supported", name,
                (long long)t->stride2);
  const int64_t s0 = tokens > 1 ? t->stride0 : INT64_MAX, s1 = heads > 1 ? t->stride1 : INT64_MAX;
  if (s0 < 0 || s1 < 0) return fail(LLK_ERR_LAYOUT, "%s has a negative stride", name);
  if (result) {
    const int64_t inner = std::min(s0, s1), outer = std::max(s0, s1);
    const int64_t n = s0 < s1 ? tokens : heads;  // of the inner one
    if ((inner != INT64_MAX && inner < D) ||
        (outer != INT64_MAX && outer / std::max<int64_t>(inner, 1) < n - 1) ||
        (outer != INT64_MAX && outer < inner * (n - 1) + D))
      return fail(LLK_ERR_LAYOUT, "%s has rows that overlap (strides %lld, %lld)", name,
                  (long long)t->stride0, (long long)t->stride1);
  }
  return LLK_OK;
}

uint16_t* bf16_of(const llk_tensor3d* t) { return static_cast<uint16_t*>(t->data); }

// Checks shared by write and read; *empty: nothing to do.
int check_move(const llk_tensor3d* k, const llk_tensor3d* v, const llk_kv4_cache* cache,
               const llk_kv4_batch* batch, bool result, Kv4Cache* c, Kv4Batch* b, Kv4Rows* r,
               bool* empty) {
  int rc;
  if ((rc = check_cache(cache, c)) || (rc = check_batch(batch, b))) return rc;
  if ((rc = check_rows3(k, "k", b->tokens, c->heads, cache->head_dim, result)) ||
      (rc = check_rows3(v, "v", b->tokens, c->heads, cache->head_dim, result)))
    return rc;
  if (b->tokens > kKv4MaxMoved)
    return fail(LLK_ERR_SHAPE, "%d tokens are too many for one call (%lld)", b->tokens,
                (long long)kKv4MaxMoved);
  *r = Kv4Rows{bf16_of(k), bf16_of(v), k->stride0, k->stride1, v->stride0, v->stride1};
  // (a read without sequences gives zeros)
  *empty = b->tokens == 0 || (b->sequences == 0 && !result);
  int dev;
  return *empty ? LLK_OK : llk::current_gfx950(&dev);
}

// Marks of a cache's slots.  need: 1 the weights, 2 the positions.
int check_marks(const llk_kv4_marks* m, int64_t pages, int64_t heads, int64_t page_size, int need,
                Kv4Marks* out) {
  if (!m) return fail(LLK_ERR_INVALID_ARGUMENT, "marks is NULL");
  if (((need & 1) && !m->weights) || ((need & 2) && !m->positions))
    return fail(LLK_ERR_INVALID_ARGUMENT, "marks.%s is NULL",
                (need & 1) && !m->weights ? "weights" : "positions");
  if (reinterpret_cast<uintptr_t>(m->weights) % 4 || reinterpret_cast<uintptr_t>(m->positions) % 4)
    return fail(LLK_ERR_LAYOUT, "marks are not aligned to their elements");
  const int64_t least = heads * page_size;
  if (pages > 1 && ((m->weights && m->weights_stride < least) ||
                    (m->positions && m->positions_stride < least)))
    return fail(LLK_ERR_LAYOUT, "a page stride of the marks (%lld, %lld) < %lld heads of %lld slots",
                (long long)m->weights_stride, (long long)m->positions_stride, (long long)heads,
                (long long)page_size);
  *out = Kv4Marks{m->weights, m->positions, m->weights_stride, m->positions_stride};
  return LLK_OK;
}

struct AttentionPlan {
  int rows;  // row tile
  int64_t tiles;
  int splits, chunk;
  size_t bytes;
};

// The launch of one attention call, from what the host knows: not the
// sequences' lengths, which are device memory, but the longest (max_len, or
// what the table holds).
AttentionPlan plan_attention(const Kv4Batch& b, int page_shift, int heads, int group, int D,
                             int window, int sinks, int64_t max_len) {
  AttentionPlan p{};
  const int64_t rows_each = b.starts ? ((int64_t)b.tokens * group + b.sequences - 1) / b.sequences
                                     : group;
  // Tiles of 16 and 32 rows read the keys once more per tile and split them over
  // the chip; one of 128 rows converts each key once for 4 waves, and pays when
  // it is full.  Measured, D = 128, context 8000, us: 16 rows a sequence, 16
  // sequences: 37 by 16 rows, 48 by 32; 24 on average: 52 by 32, 121 by 128; 96:
  // 117 and 166; 128, one sequence: 28.6 and 26.6; 256, 16 sequences: 187 both
  // (context 1000: 93 and 33).
  p.rows = rows_each <= 16 ? 16 : rows_each <= 96 ? 32 : kKv4PromptRows;
  p.tiles = b.starts ? (int64_t)b.tokens * group / p.rows + b.sequences
                     : (int64_t)b.sequences * ((group + p.rows - 1) / p.rows);
  int64_t len = std::min<int64_t>((int64_t)b.table_pages << page_shift, kKv4MaxLength);
  if (max_len > 0) len = std::min(len, max_len);
  const int64_t step = kv4_step(p.rows);
  int64_t steps = (len + step - 1) / step;
  if (window > 0)
    steps = std::min<int64_t>(steps, (sinks + step - 1) / step +
                                         (window + p.rows / group + step - 1) / step + 2);
  const int64_t groups = p.tiles * heads;
  // Splits of the keys: enough workgroups for the chip, none of a few steps only,
  // since a second kernel joins them.  Measured, D = 128, us.
  int64_t s;
  if (p.rows == kKv4PromptRows) {
    // About 512 workgroups, two to a CU: 64 groups at 8000 keys 60, by 256 85, by
    // 1024 74; 256 groups of 4000 keys, 2 splits 91, 4 99.  Steps a split: 64
    // groups at 1000 keys by 4 21, by 8 24, one split 30; 136 groups 31, 29 and
    // 31; 256 groups, by 8 38, one split 32.
    s = std::min<int64_t>(std::max<int64_t>(1, 512 / groups),
                          steps / std::clamp<int64_t>(groups / 16, 4, 16));
  } else {
    // About 2048 workgroups: 512 groups at 8000 keys, 4 splits 78, 8 79, 15 86.
    // At most 64: 8 groups at 30000 (16 rows) 20.8, 105 splits 24.9.  Steps a
    // split: 64 groups at 2000, 7 splits 13.2, 3 14.2; 512 groups at 500, one
    // split 12.2, two 17.1.
    s = std::min<int64_t>(std::min<int64_t>(64, (2048 + groups - 1) / groups),
                          steps / (groups >= 256 ? 16 : 8));
  }
  s = std::max<int64_t>(s, 1);
  p.chunk = (int)std::max<int64_t>(1, (steps + s - 1) / s);
  p.splits = (int)std::max<int64_t>(1, (steps + p.chunk - 1) / p.chunk);
  p.bytes = llk_kv4_attention_part_bytes(p.tiles, heads, p.splits, p.rows, D);
  return p;
}

// Checks and plans an attention call; *empty: nothing to do.
int check_attention(const llk_tensor3d* q, const llk_kv4_cache* cache, const llk_kv4_batch* batch,
                    const llk_attention_params* params, Kv4AttentionArgs* a, AttentionPlan* plan,
                    bool* empty) {
  int rc;
  if ((rc = check_cache(cache, &a->cache)) || (rc = check_batch(batch, &a->batch))) return rc;
  if (!q || !params)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", q ? "params" : "q");
  const int64_t heads = cache->heads;
  if (q->dim1 < 1 || q->dim1 % heads != 0 || q->dim1 / heads > 4096)
    return fail(LLK_ERR_SHAPE, "q heads (%lld) are not a multiple (to 4096) of the cache's %lld",
                (long long)q->dim1, (long long)heads);
  if ((rc = check_rows3(q, "q", batch->tokens, q->dim1, cache->head_dim, false))) return rc;
  if (!(params->scale > 0.0f) || !std::isfinite(params->scale))
    return fail(LLK_ERR_INVALID_ARGUMENT, "scale %g is not positive and finite", params->scale);
  if (params->window < 0 || params->sinks < 0 || batch->max_len < 0)
    return fail(LLK_ERR_INVALID_ARGUMENT, "window, sinks and max_len must not be negative");
  a->q = static_cast<const uint16_t*>(q->data);
  a->q_token = q->stride0;
  a->q_head = q->stride1;
  a->group = (int)(q->dim1 / heads);
  a->window = (int)std::min<int64_t>(params->window, kKv4MaxLength);
  a->span = a->window ? (uint32_t)a->window : 1u << 31;
  a->sinks = a->window ? (int)std::min<int64_t>(params->sinks, kKv4MaxLength) : 0;
  a->scale = (float)((double)params->scale * 1.4426950408889634);  // log2(e)
  *empty = batch->tokens == 0 || batch->sequences == 0;
  if (*empty) return LLK_OK;
  if (batch->tokens * a->group > kMaxTokens)
    return fail(LLK_ERR_SHAPE, "%lld tokens of %d query heads to a key head are too many",
                (long long)batch->tokens, a->group);
  *plan = plan_attention(a->batch, a->cache.page_shift, a->cache.heads, a->group,
                         (int)cache->head_dim, a->window, a->sinks, batch->max_len);
  if (plan->tiles * heads > kKv4MaxWorkgroups)
    return fail(LLK_ERR_SHAPE, "%lld row tiles of %lld heads are too many for one call (%lld)",
                (long long)plan->tiles, (long long)heads, (long long)kKv4MaxWorkgroups);
  a->tiles = (int)plan->tiles;
  a->splits = plan->splits;
  a->chunk = plan->chunk;
  return LLK_OK;
}

// The workspace of an attention that adds its weights up: the splits' parts, the rows'
// statistics, and the scores of single tokens' rows.
// (Bytes of scores: beyond it they are computed again, as with `starts`: 64 sequences to
// 8192 keys, 32 query heads on 8, 126 us a call in a replayed graph for 95.)
constexpr int64_t kMaxKept = (int64_t)512 << 20;
struct WeighPlan {
  size_t stats, kept, bytes;  // where they begin; all
  int kept_keys;              // of a sequence, or 0: none are kept
};
WeighPlan plan_weigh(const AttentionPlan& p, const Kv4AttentionArgs& a, const llk_tensor3d* q,
                     int64_t max_len) {
  WeighPlan w{};
  w.stats = (p.bytes + 255) / 256 * 256;
  w.kept = w.stats + ((size_t)(q->dim0 * q->dim1) * 2 * sizeof(float) + 255) / 256 * 256;
  w.bytes = w.kept;
  if (!a.batch.starts && p.rows == 16 && a.group <= 16) {
    int64_t len = std::min<int64_t>((int64_t)a.batch.table_pages << a.cache.page_shift, kKv4MaxLength);
    if (max_len > 0) len = std::min(len, max_len);
    const int64_t keys = (len + 255) / 256 * 256;
    const double bytes = (double)(q->dim0 * q->dim1) * (double)keys * sizeof(float);
    // (4 group bytes for a key and head, of which the cache has 17/16 head_dim)
    if (keys > 0 && bytes <= (double)kMaxKept) {
      w.kept_keys = (int)keys;
      w.bytes += (size_t)bytes;
    }
  }
  return w;
}

// The sequences' heads are workgroups of up to 1024 threads along one dimension.
int check_heads(const Kv4Batch& b, int64_t heads) {
  constexpr int64_t kMost = ((int64_t)1 << 22) - 1;
  return b.sequences * heads <= kMost
             ? LLK_OK
             : fail(LLK_ERR_SHAPE, "%d sequences of %lld heads are too many for one call (%lld)",
                    b.sequences, (long long)heads, (long long)kMost);
}

int attend(const llk_tensor3d* q, const llk_kv4_cache* cache, const llk_kv4_batch* batch,
           const llk_attention_params* params, const llk_kv4_marks* marks, float decay,
           llk_tensor3d* out, llk_kernel_context* ctx) {
  Kv4AttentionArgs a{};
  AttentionPlan p{};
  Kv4Marks m{};
  bool empty = false;
  int rc = check_attention(q, cache, batch, params, &a, &p, &empty);
  if (rc || (rc = check_rows3(out, "out", batch->tokens, q->dim1, cache->head_dim, true))) return rc;
  if (marks) {
    if ((rc = check_marks(marks, cache->pages, cache->heads, cache->page_size, 1, &m)) ||
        (rc = check_heads(a.batch, cache->heads)))
      return rc;
    if (!(decay >= 0.0f) || !std::isfinite(decay))
      return fail(LLK_ERR_INVALID_ARGUMENT, "decay %g is negative or not finite", decay);
  }
  if (empty) return LLK_OK;
  // (the scores that are not kept are computed from q once more)
  if (marks && out->data == q->data)
    return fail(LLK_ERR_INVALID_ARGUMENT, "with weights out must not be q");
  a.out = bf16_of(out);
  a.out_token = out->stride0;
  a.out_head = out->stride1;
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  llk::CallWorkspace ws;
  const WeighPlan weigh = marks ? plan_weigh(p, a, q, batch->max_len) : WeighPlan{};
  if ((rc = ws.begin(dev, marks ? weigh.bytes : p.bytes, ctx))) return rc;
  a.part = static_cast<float*>(ws.ptr());
  if (marks) {
    a.stats = reinterpret_cast<float*>(static_cast<uint8_t*>(ws.ptr()) + weigh.stats);
    a.kept_keys = weigh.kept_keys;
    if (a.kept_keys) a.kept = reinterpret_cast<float*>(static_cast<uint8_t*>(ws.ptr()) + weigh.kept);
  }
  hipError_t e = llk_launch_kv4_attention(a, (int)cache->head_dim, p.rows, stream_of(ctx));
  if (marks && e == hipSuccess)
    e = llk_launch_kv4_weigh(a, m, decay, (int)cache->head_dim, batch->max_len, stream_of(ctx));
  ws.end();
  return e == hipSuccess ? LLK_OK : fail_hip(e, "cache attention kernel");
}

}  // namespace

extern "C" {

int llk_block_norm(const llk_tensor2d* y, const llk_tensor2d* residual, llk_tensor2d* residual_out,
                   llk_tensor2d* out, const llk_block_norm_params* p, llk_kernel_context* ctx) {
  if (!residual || !out || !p)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL",
                !residual ? "residual" : !out ? "out" : "params");
  const int64_t M = residual->dim0, N = residual->dim1;
  if (M < 0 || N < 1 || N > kBlockNormMaxN)
    return fail(LLK_ERR_SHAPE, "residual of (%lld, %lld) unsupported (1 to %lld columns)",
                (long long)M, (long long)N, (long long)kBlockNormMaxN);
  int rc;
  if ((rc = check_rows(residual, "residual", M, N, p->residual_dtype, false)) ||
      (rc = check_rows(out, "out", M, N, p->out_dtype, false)))
    return rc;
  BlockNormArgs a{};
  if (y) {
    if ((rc = check_rows(y, "y", M, N, p->y_dtype, false))) return rc;
    if (!residual_out)
      return fail(LLK_ERR_INVALID_ARGUMENT, "residual_out is NULL (it receives the sum with y)");
  } else if (p->post_weight || p->gate.data) {
    return fail(LLK_ERR_INVALID_ARGUMENT, "post_weight and gate apply to y, which is NULL");
  }
  if (residual_out && (rc = check_rows(residual_out, "residual_out", M, N, p->residual_dtype, false)))
    return rc;
  if (p->gate.data && (rc = check_rows(&p->gate, "gate", M, N, p->y_dtype, true))) return rc;
  if (!p->pre_weight) return fail(LLK_ERR_INVALID_ARGUMENT, "pre_weight is NULL");
  if (!norm_type(p->weight_dtype))
    return fail(LLK_ERR_DTYPE, "weight type %d unsupported (bf16 or f32)", p->weight_dtype);
  for (const void* w : {p->pre_weight, p->post_weight})
    if (reinterpret_cast<uintptr_t>(w) % type_size(p->weight_dtype))
      return fail(LLK_ERR_LAYOUT, "a weight is not aligned to its elements");
  if (!(p->eps >= 0.0f)) return fail(LLK_ERR_INVALID_ARGUMENT, "eps %g is negative", p->eps);
  if (M == 0) return LLK_OK;
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  a.h = residual->data;
  a.ldh = residual->stride0;
  a.out = out->data;
  a.ldo = out->stride0;
  a.wpre = p->pre_weight;
  if (y) {
    a.y = y->data;
    a.ldy = y->stride0;
    a.wpost = p->post_weight;
    if (p->gate.data) {
      a.g = p->gate.data;
      a.ldg = p->gate.stride0;
    }
  }
  if (residual_out) {
    a.h_out = residual_out->data;
    a.ldho = residual_out->stride0;
  }
  a.N = (int)N;
  a.scale = p->residual_scale;
  a.eps = p->eps;
  a.offset = p->weight_offset;
  const hipError_t e =
      llk_launch_block_norm(a, M, p->y_dtype == LLK_FP32, p->residual_dtype == LLK_FP32,
                            p->out_dtype == LLK_FP32, p->weight_dtype == LLK_FP32, stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "block norm kernel");
}

int64_t llk_kv4_head_bytes(int64_t page_size, int64_t head_dim) {
  return page_size_ok(page_size) && head_dim_ok(head_dim) ? page_size / 16 * 17 * head_dim : 0;
}

int llk_kv4_write(const llk_tensor3d* k, const llk_tensor3d* v, const llk_kv4_cache* cache,
                  const llk_kv4_batch* batch, llk_kernel_context* ctx) {
  Kv4Cache c;
  Kv4Batch b;
  Kv4Rows r;
  bool empty = false;
  const int rc = check_move(k, v, cache, batch, false, &c, &b, &r, &empty);
  if (rc || empty) return rc;
  const hipError_t e = llk_launch_kv4_write(c, b, r, (int)cache->head_dim, stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "cache write kernel");
}

int llk_kv4_read(const llk_kv4_cache* cache, const llk_kv4_batch* batch, llk_tensor3d* k,
                 llk_tensor3d* v, llk_kernel_context* ctx) {
  Kv4Cache c;
  Kv4Batch b;
  Kv4Rows r;
  bool empty = false;
  const int rc = check_move(k, v, cache, batch, true, &c, &b, &r, &empty);
  if (rc || empty) return rc;
  const hipError_t e = llk_launch_kv4_read(c, b, r, (int)cache->head_dim, stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "cache read kernel");
}

int llk_kv4_attention_describe(const llk_tensor3d* q, const llk_kv4_cache* cache,
                               const llk_kv4_batch* batch, const llk_attention_params* params,
                               llk_attention_plan* out) {
  if (!out) return fail(LLK_ERR_INVALID_ARGUMENT, "plan is NULL");
  Kv4AttentionArgs a{};
  AttentionPlan p{};
  bool empty = false;
  const int rc = check_attention(q, cache, batch, params, &a, &p, &empty);
  if (rc) return rc;
  *out = llk_attention_plan{};
  if (empty) return LLK_OK;
  out->rows = p.rows;
  out->splits = p.splits;
  out->workgroups = p.tiles * a.cache.heads * p.splits;
  out->launches = p.splits > 1 ? 2 : 1;
  out->workspace_bytes = p.bytes;
  return LLK_OK;
}

int llk_kv4_attention(const llk_tensor3d* q, const llk_kv4_cache* cache,
                      const llk_kv4_batch* batch, const llk_attention_params* params,
                      llk_tensor3d* out, llk_kernel_context* ctx) {
  return attend(q, cache, batch, params, nullptr, 0.0f, out, ctx);
}

int llk_kv4_write_marked(const llk_tensor3d* k, const llk_tensor3d* v, const llk_kv4_cache* cache,
                         const llk_kv4_batch* batch, const llk_kv4_marks* marks, const int32_t* at,
                         llk_kernel_context* ctx) {
  Kv4Cache c;
  Kv4Batch b;
  Kv4Rows r;
  Kv4Marks m;
  bool empty = false;
  int rc = check_cache(cache, &c);
  if (rc || (rc = check_marks(marks, cache->pages, cache->heads, cache->page_size, 0, &m)) ||
      (rc = check_move(k, v, cache, batch, false, &c, &b, &r, &empty)))
    return rc;
  if (empty) return LLK_OK;
  const hipError_t e =
      llk_launch_kv4_write(c, b, r, (int)cache->head_dim, stream_of(ctx), &m, at);
  return e == hipSuccess ? LLK_OK : fail_hip(e, "cache write kernel");
}

int llk_kv4_attention_weigh(const llk_tensor3d* q, const llk_kv4_cache* cache,
                            const llk_kv4_batch* batch, const llk_attention_params* params,
                            const llk_kv4_marks* marks, float decay, llk_tensor3d* out,
                            llk_kernel_context* ctx) {
  if (!marks) return fail(LLK_ERR_INVALID_ARGUMENT, "marks is NULL");
  return attend(q, cache, batch, params, marks, decay, out, ctx);
}

int llk_kv4_attention_weigh_describe(const llk_tensor3d* q, const llk_kv4_cache* cache,
                                     const llk_kv4_batch* batch, const llk_attention_params* params,
                                     llk_attention_plan* out) {
  const int rc = llk_kv4_attention_describe(q, cache, batch, params, out);
  if (rc || out->launches == 0) return rc;
  Kv4AttentionArgs a{};
  AttentionPlan p{};
  bool empty = false;
  check_attention(q, cache, batch, params, &a, &p, &empty);
  out->launches += 1;
  out->workspace_bytes = plan_weigh(p, a, q, batch->max_len).bytes;
  return LLK_OK;
}

int llk_kv4_evict_plan(const llk_kv4_marks* marks, int64_t pages, int64_t heads, int64_t page_size,
                       const llk_kv4_batch* batch, const llk_kv4_evict_params* params,
                       int32_t* lens, int32_t* source, llk_kernel_context* ctx) {
  Kv4EvictPlan p{};
  int rc;
  if ((rc = check_batch(batch, &p.batch))) return rc;
  if (!page_size_ok(page_size))
    return fail(LLK_ERR_SHAPE, "page_size %lld unsupported (a power of two, 16 to 4096)",
                (long long)page_size);
  if (pages < 1 || pages > 0x7fffffff || heads < 1 || heads > 65535)
    return fail(LLK_ERR_SHAPE, "marks of %lld pages and %lld heads unsupported", (long long)pages,
                (long long)heads);
  if (!params) return fail(LLK_ERR_INVALID_ARGUMENT, "params is NULL");
  if (params->keep < 1 || params->keep > kKv4MaxLength)
    return fail(LLK_ERR_SHAPE, "keep %lld unsupported (1 to %d)", (long long)params->keep,
                kKv4MaxLength);
  if (params->recent < 0 || params->first < 0 || params->recent > params->keep ||
      params->first > params->keep - params->recent)
    return fail(LLK_ERR_INVALID_ARGUMENT, "recent %lld and first %lld are negative or beyond keep %lld",
                (long long)params->recent, (long long)params->first, (long long)params->keep);
  const bool guarded = params->recent > 0 || params->first > 0;
  if ((rc = check_marks(marks, pages, heads, page_size, guarded ? 3 : 1, &p.marks)) ||
      (rc = check_heads(p.batch, heads)))
    return rc;
  if (batch->sequences == 0) return LLK_OK;
  if (!lens || !source)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", lens ? "source" : "lens");
  // every head's workgroup reads the old lengths, all of them while some are written
  const uintptr_t at = reinterpret_cast<uintptr_t>(lens), old = reinterpret_cast<uintptr_t>(batch->lens);
  const uintptr_t bytes = (uintptr_t)batch->sequences * sizeof(int32_t);
  if (at < old + bytes && old < at + bytes)
    return fail(LLK_ERR_INVALID_ARGUMENT, "the new lengths must not replace batch.lens, or a part of it");
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  if (!guarded) p.marks.positions = nullptr;
  p.pages = (int)pages;
  p.heads = (int)heads;
  p.page_shift = __builtin_ctzll((unsigned long long)page_size);
  p.keep = (int)params->keep;
  p.recent = (int)params->recent;
  p.first = (int)params->first;
  p.lens = lens;
  p.source = source;
  const hipError_t e = llk_launch_kv4_evict_plan(p, batch->max_len, stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "eviction plan kernel");
}

int llk_kv4_evict(const llk_kv4_cache* cache, const llk_kv4_batch* batch, const int32_t* source,
                  int64_t keep, const llk_kv4_marks* marks, int32_t* lens, llk_kernel_context* ctx) {
  Kv4Cache c;
  Kv4Batch b;
  Kv4Marks m{};
  int rc;
  if ((rc = check_cache(cache, &c))) return rc;
  if (!batch) return fail(LLK_ERR_INVALID_ARGUMENT, "batch is NULL");
  if (batch->sequences > 0 && !source) return fail(LLK_ERR_INVALID_ARGUMENT, "source is NULL");
  llk_kv4_batch used = *batch;  // its table and sequences
  used.lens = source;           // (not read)
  used.starts = nullptr;
  used.tokens = used.sequences;
  if ((rc = check_batch(&used, &b))) return rc;
  if (keep < 1 || keep > kKv4MaxLength)
    return fail(LLK_ERR_SHAPE, "keep %lld unsupported (1 to %d)", (long long)keep, kKv4MaxLength);
  if (marks && (rc = check_marks(marks, cache->pages, cache->heads, cache->page_size, 0, &m))) return rc;
  if ((rc = check_heads(b, cache->heads))) return rc;
  if (b.sequences == 0) return LLK_OK;
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  const hipError_t e = llk_launch_kv4_evict(c, b, m, source, (int)keep, lens, (int)cache->head_dim,
                                            stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "eviction kernel");
}

}  // extern "C"
