// q4_ops.cpp -- C entry points of the weights in 4 bits (include/llk/llk_abi.h).
// Kernels: kernels/q4_pack.hip, kernels/q4_gemv.hip (few rows; the plan of both),
// kernels/q4_tile.hip.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "abi_support.h"
#include "kernels/q4.h"
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

bool group_ok(int64_t g) { return g == 32 || g == 64 || g == 128; }
// The packing kernels have a unit of K in a dimension of their grid (to 65535), and
// indexes of 32 bits.
constexpr int64_t kMaxK = (int64_t)65535 * 32, kMaxN = (int64_t)1 << 26;

int check_sizes(int64_t K, int64_t N, int64_t group) {
  if (!group_ok(group))
    return fail(LLK_ERR_SHAPE, "group of %lld unsupported (32, 64 or 128)", (long long)group);
  if (K < 0 || N < 0 || K > kMaxK || N > kMaxN)
    return fail(LLK_ERR_SHAPE, "4-bit weights of (%lld, %lld) unsupported", (long long)K,
                (long long)N);
  return LLK_OK;
}

// A [rows, cols] operand with unit inner stride of elements of `size` bytes.
int check_matrix(const llk_tensor2d* t, const char* name, int64_t rows, int64_t cols, size_t size) {
  if (!t) return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", name);
  if (t->dim0 != rows || t->dim1 != cols)
    return fail(LLK_ERR_SHAPE, "%s shape (%lld, %lld) != (%lld, %lld)", name, (long long)t->dim0,
                (long long)t->dim1, (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return LLK_OK;
  if (!t->data) return fail(LLK_ERR_INVALID_ARGUMENT, "%s.data is NULL", name);
  if (t->stride1 != 1 && cols > 1)
    return fail(LLK_ERR_LAYOUT, "%s.stride1 is %lld; only unit inner stride is supported", name,
                (long long)t->stride1);
  if (rows > 1 && t->stride0 < cols)
    return fail(LLK_ERR_LAYOUT, "%s.stride0 (%lld) < dim1 (%lld)", name, (long long)t->stride0,
                (long long)cols);
  if (reinterpret_cast<uintptr_t>(t->data) % size)
    return fail(LLK_ERR_LAYOUT, "%s.data is not aligned to its elements", name);
  return LLK_OK;
}

int check_scale_type(int type) {
  return type == LLK_BF16 || type == LLK_FP16
             ? LLK_OK
             : fail(LLK_ERR_DTYPE, "scale type %d unsupported (bf16 or fp16)", type);
}

int check_packed(const llk_q4_weights* w, const char* name) {
  if (!w) return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", name);
  int rc = check_sizes(w->K, w->N, w->group);
  if (rc) return rc;
  if (w->K == 0 || w->N == 0) return LLK_OK;
  if (!w->codes || !w->scales)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s.codes or %s.scales is NULL", name, name);
  if (reinterpret_cast<uintptr_t>(w->codes) % 16 || reinterpret_cast<uintptr_t>(w->scales) % 16)
    return fail(LLK_ERR_LAYOUT, "%s.codes and %s.scales must be 16-byte aligned", name, name);
  return LLK_OK;
}

constexpr int64_t kMaxRows = (int64_t)1 << 24;
// A dimension of a launch takes fewer than 2^32 threads: workgroups of 256.
constexpr int64_t kMaxGroups = ((int64_t)1 << 24) - 1;

int product(const llk_tensor2d* x, const llk_q4_weights* const (&w)[2], int sides, llk_tensor2d* y,
            int y_dtype, bool accumulate, llk_kernel_context* ctx) {
  const char* const names[2] = {sides == 2 ? "wg" : "w", "wu"};
  int rc;
  for (int s = 0; s < sides; ++s)
    if ((rc = check_packed(w[s], names[s]))) return rc;
  const int64_t K = w[0]->K, N = w[0]->N;
  if (sides == 2 && (w[1]->K != K || w[1]->N != N || w[1]->group != w[0]->group))
    return fail(LLK_ERR_SHAPE, "wg (%lld, %lld, groups of %lld) and wu (%lld, %lld, groups of %lld) differ",
                (long long)K, (long long)N, (long long)w[0]->group, (long long)w[1]->K,
                (long long)w[1]->N, (long long)w[1]->group);
  if (!x || !y) return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", x ? "y" : "x");
  const int64_t M = x->dim0;
  if (M < 0 || M > kMaxRows) return fail(LLK_ERR_SHAPE, "x of %lld rows unsupported", (long long)M);
  if ((rc = check_matrix(x, "x", M, K, 2))) return rc;
  if (y_dtype != LLK_BF16 && y_dtype != LLK_FP32 && (sides == 2 || y_dtype != LLK_FP16))
    return fail(LLK_ERR_DTYPE, "y type %d unsupported", y_dtype);
  if ((rc = check_matrix(y, "y", M, N, y_dtype == LLK_FP32 ? 4 : 2))) return rc;
  if (M == 0 || N == 0) return LLK_OK;
  Q4Args a{};
  a.x = static_cast<const uint16_t*>(x->data);
  a.ldx = x->stride0;
  for (int s = 0; s < sides; ++s)
    a.side[s] = Q4Side{static_cast<const uint8_t*>(w[s]->codes),
                       static_cast<const uint32_t*>(w[s]->scales)};
  a.y = y->data;
  a.ldy = y->stride0;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.group = (int)w[0]->group;
  a.out = y_dtype;
  a.accumulate = accumulate;
  const Q4Plan plan = llk_plan_q4(M, N, K, sides);
  if (plan.groups > kMaxGroups)
    return fail(LLK_ERR_SHAPE, "%lld rows of %lld columns are too many for one call", (long long)M,
                (long long)N);
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  llk::CallWorkspace ws;
  if ((rc = ws.begin(dev, plan.bytes, ctx))) return rc;
  a.part = static_cast<float*>(ws.ptr());
  const hipError_t e = llk_launch_q4(a, sides, plan, stream_of(ctx));
  ws.end();
  return e == hipSuccess ? LLK_OK : fail_hip(e, "4-bit product kernel");
}

}  // namespace

extern "C" {

size_t llk_q4_code_bytes(int64_t K, int64_t N) {
  return K < 0 || N < 0 || K > kMaxK || N > kMaxN
             ? 0
             : (size_t)(q4_tiles(N) * q4_units(K)) * kQ4UnitBytes;
}

size_t llk_q4_scale_bytes(int64_t K, int64_t N, int64_t group) {
  return K < 0 || N < 0 || K > kMaxK || N > kMaxN || !group_ok(group)
             ? 0
             : (size_t)(q4_tiles(N) * q4_groups(K, (int)group)) * kQ4Columns * 4;
}

size_t llk_q4_scratch_size(int64_t M, int64_t N, int64_t K, int sides) {
  return M < 0 || N < 0 || K < 0 || M > kMaxRows || K > kMaxK || N > kMaxN || sides < 1 || sides > 2
             ? 0
             : llk_plan_q4(M, N, K, sides).bytes;
}

int llk_q4_quantise(const llk_tensor2d* w, int64_t group, llk_tensor2d* codes, llk_tensor2d* scales,
                    int scale_dtype, llk_tensor2d* zeros, llk_kernel_context* ctx) {
  if (!w) return fail(LLK_ERR_INVALID_ARGUMENT, "w is NULL");
  const int64_t K = w->dim0, N = w->dim1;
  int rc;
  if ((rc = check_sizes(K, N, group)) || (rc = check_scale_type(scale_dtype))) return rc;
  const int64_t groups = (K + group - 1) / group;
  if ((rc = check_matrix(w, "w", K, N, 2)) || (rc = check_matrix(codes, "codes", K, N, 1)) ||
      (rc = check_matrix(scales, "scales", groups, N, 2)) ||
      (zeros && (rc = check_matrix(zeros, "zeros", groups, N, 1))))
    return rc;
  if (K == 0 || N == 0) return LLK_OK;
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  Q4QuantiseArgs a{};
  a.w = static_cast<const uint16_t*>(w->data);
  a.ld = w->stride0;
  a.codes = static_cast<uint8_t*>(codes->data);
  a.ld_codes = codes->stride0;
  a.scales = static_cast<uint16_t*>(scales->data);
  a.ld_scales = scales->stride0;
  if (zeros) {
    a.zeros = static_cast<uint8_t*>(zeros->data);
    a.ld_zeros = zeros->stride0;
  }
  a.K = (int)K;
  a.N = (int)N;
  a.group = (int)group;
  a.f16 = scale_dtype == LLK_FP16;
  const hipError_t e = llk_launch_q4_quantise(a, stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "4-bit quantise kernel");
}

int llk_q4_pack(const llk_tensor2d* codes, const llk_tensor2d* scales, int scale_dtype,
                const llk_tensor2d* zeros, const llk_q4_weights* out, llk_kernel_context* ctx) {
  int rc;
  if ((rc = check_packed(out, "out")) || (rc = check_scale_type(scale_dtype))) return rc;
  const int64_t K = out->K, N = out->N, groups = (K + out->group - 1) / out->group;
  if ((rc = check_matrix(codes, "codes", K, N, 1)) ||
      (rc = check_matrix(scales, "scales", groups, N, 2)) ||
      (zeros && (rc = check_matrix(zeros, "zeros", groups, N, 1))))
    return rc;
  if (K == 0 || N == 0) return LLK_OK;
  int dev;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  Q4Source s{};
  s.codes = static_cast<const uint8_t*>(codes->data);
  s.ld = codes->stride0;
  s.scales = static_cast<const uint16_t*>(scales->data);
  s.ld_scales = scales->stride0;
  if (zeros) {
    s.zeros = static_cast<const uint8_t*>(zeros->data);
    s.ld_zeros = zeros->stride0;
  }
  s.K = (int)K;
  s.N = (int)N;
  s.group = (int)out->group;
  s.f16 = scale_dtype == LLK_FP16;
  const hipError_t e = llk_launch_q4_pack(s, static_cast<uint8_t*>(out->codes),
                                          static_cast<uint32_t*>(out->scales), stream_of(ctx));
  return e == hipSuccess ? LLK_OK : fail_hip(e, "4-bit pack kernel");
}

int llk_q4_gemm(const llk_tensor2d* x, const llk_q4_weights* w, llk_tensor2d* y, int y_dtype,
                int accumulate, llk_kernel_context* ctx) {
  return product(x, {w, nullptr}, 1, y, y_dtype, accumulate != 0, ctx);
}

int llk_q4_swiglu(const llk_tensor2d* x, const llk_q4_weights* wg, const llk_q4_weights* wu,
                  llk_tensor2d* y, int y_dtype, llk_kernel_context* ctx) {
  return product(x, {wg, wu}, 2, y, y_dtype, false, ctx);
}

}  // extern "C"
