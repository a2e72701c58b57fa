// rotary_ops.cpp -- C entry points of the rotary positions (include/llk/llk_abi.h).
// Kernel: kernels/rotary.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "abi_support.h"
#include "kernels/rotary.h"
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

constexpr double kPi = 3.14159265358979323846;
constexpr int64_t kMaxHeadDim = 1024, kMaxHeads = 4096;

bool positive(double v) { return v > 0.0 && std::isfinite(v); }

// bf16 or fp32 [tokens, heads, head_dim] rows.  result: no two elements may share
// memory.
int check_rows(const llk_tensor3d* t, const char* name, int64_t tokens, int64_t heads, int64_t D,
               size_t size, bool result) {
  if (!t) return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", name);
  if (t->dim0 != tokens || t->dim1 != heads || t->dim2 != D)
    return fail(LLK_ERR_SHAPE, "%s shape (%lld, %lld, %lld) != (%lld, %lld, %lld)", name,
                (long long)t->dim0, (long long)t->dim1, (long long)t->dim2, (long long)tokens,
                (long long)heads, (long long)D);
  if (tokens == 0 || heads == 0) return LLK_OK;
  if (!t->data) return fail(LLK_ERR_INVALID_ARGUMENT, "%s.data is NULL", name);
  if (reinterpret_cast<uintptr_t>(t->data) % size)
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

}  // namespace

extern "C" {

int llk_rotary_frequencies(const llk_rotary_params* p, double* frequencies, double* attention_factor) {
  if (!p || !frequencies || !attention_factor)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL",
                !p ? "params" : !frequencies ? "frequencies" : "attention_factor");
  const int64_t rot = p->rotary_dim;
  if (rot < 2 || rot > kMaxHeadDim || rot % 2)
    return fail(LLK_ERR_SHAPE, "rotary_dim %lld unsupported (even, 2 to %lld)", (long long)rot,
                (long long)kMaxHeadDim);
  if (!(p->base > 1.0) || !std::isfinite(p->base))
    return fail(LLK_ERR_INVALID_ARGUMENT, "base %g is not finite and above 1", p->base);
  if (p->scaling < LLK_ROTARY_PLAIN || p->scaling > LLK_ROTARY_BANDS)
    return fail(LLK_ERR_INVALID_ARGUMENT, "scaling %d unknown", p->scaling);
  const bool scaled = p->scaling != LLK_ROTARY_PLAIN;
  const bool by_turns = p->scaling == LLK_ROTARY_YARN || p->scaling == LLK_ROTARY_BANDS;
  const double s = p->factor;
  if (scaled && !positive(s)) return fail(LLK_ERR_INVALID_ARGUMENT, "factor %g is not positive", s);
  if (by_turns && !positive(p->trained))
    return fail(LLK_ERR_INVALID_ARGUMENT, "trained length %g is not positive", p->trained);
  if (by_turns && !(positive(p->slow) && p->fast > p->slow && std::isfinite(p->fast)))
    return fail(LLK_ERR_INVALID_ARGUMENT, "turns from %g to %g do not rise", p->slow, p->fast);
  if (p->scaling == LLK_ROTARY_BASE && rot == 2)
    return fail(LLK_ERR_SHAPE, "a scaled base needs a rotary_dim above 2");
  const double base =
      p->scaling == LLK_ROTARY_BASE ? p->base * std::pow(s, (double)rot / (double)(rot - 2)) : p->base;
  if (!(base > 1.0) || !std::isfinite(base))
    return fail(LLK_ERR_INVALID_ARGUMENT, "scaled base %g is not finite and above 1", base);
  // the pair that turns so often over the trained length
  auto pair = [&](double turns) {
    return (double)rot * std::log(p->trained / (2.0 * kPi * turns)) / (2.0 * std::log(base));
  };
  double low = 0, high = 0;
  if (p->scaling == LLK_ROTARY_YARN) {
    low = std::max(std::floor(pair(p->fast)), 0.0);
    high = std::min(std::ceil(pair(p->slow)), (double)(rot - 1));
  }
  for (int64_t i = 0; i < rot / 2; ++i) {
    double f = std::pow(base, -2.0 * (double)i / (double)rot);
    if (p->scaling == LLK_ROTARY_LINEAR) f /= s;
    if (p->scaling == LLK_ROTARY_YARN) {
      const double r =
          std::min(std::max(((double)i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      f = r * f / s + (1.0 - r) * f;
    }
    if (p->scaling == LLK_ROTARY_BANDS) {
      const double turns = p->trained * f / (2.0 * kPi);
      const double r = std::min(std::max((turns - p->slow) / (p->fast - p->slow), 0.0), 1.0);
      f = (1.0 - r) * f / s + r * f;
    }
    frequencies[i] = f;
  }
  *attention_factor = p->scaling == LLK_ROTARY_YARN && s > 1.0 ? 0.1 * std::log(s) + 1.0 : 1.0;
  return LLK_OK;
}

int llk_rotary_turns(const double* frequencies, int64_t pairs, uint64_t* turns) {
  if (!frequencies || !turns)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", frequencies ? "turns" : "frequencies");
  if (pairs < 1 || pairs > kMaxHeadDim / 2)
    return fail(LLK_ERR_SHAPE, "%lld pairs unsupported (1 to %lld)", (long long)pairs,
                (long long)kMaxHeadDim / 2);
  for (int64_t i = 0; i < pairs; ++i) {
    if (!std::isfinite(frequencies[i]))
      return fail(LLK_ERR_INVALID_ARGUMENT, "frequency %lld is not finite", (long long)i);
    // (long double has the 64 bits that the fraction of a turn is kept to)
    constexpr long double kTwoPi = 6.283185307179586476925286766559L;
    const long double x = (long double)frequencies[i] / kTwoPi;
    const long double t = rintl((x - floorl(x)) * 0x1p64L);
    turns[i] = t >= 0x1p64L ? 0 : (uint64_t)t;
  }
  return LLK_OK;
}

int llk_rotary(const llk_tensor3d* q, const llk_tensor3d* k, const int32_t* positions,
               const uint64_t* turns, int64_t pairs, float factor, int dtype, int flags,
               llk_tensor3d* q_out, llk_tensor3d* k_out, llk_kernel_context* ctx) {
  if (!q) return fail(LLK_ERR_INVALID_ARGUMENT, "q is NULL");
  if (!k != !k_out) return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", k ? "k_out" : "k");
  if (dtype != LLK_BF16 && dtype != LLK_FP32)
    return fail(LLK_ERR_DTYPE, "type %d unsupported (bf16 or f32)", dtype);
  if (flags & ~(LLK_ROTARY_INTERLEAVED | LLK_ROTARY_INVERSE))
    return fail(LLK_ERR_INVALID_ARGUMENT, "flags %d unknown", flags);
  const int64_t T = q->dim0, D = q->dim2;
  if (T < 0 || T > kRotaryMaxTokens)
    return fail(LLK_ERR_SHAPE, "%lld tokens unsupported (to %lld)", (long long)T,
                (long long)kRotaryMaxTokens);
  if (D < 2 || D > kMaxHeadDim || pairs < 1 || 2 * pairs > D)
    return fail(LLK_ERR_SHAPE, "%lld pairs of heads of %lld unsupported (heads to %lld)",
                (long long)pairs, (long long)D, (long long)kMaxHeadDim);
  if (!std::isfinite(factor)) return fail(LLK_ERR_INVALID_ARGUMENT, "factor %g is not finite", factor);
  const size_t size = dtype == LLK_FP32 ? 4 : 2;
  RotaryArgs a{};
  const llk_tensor3d* const in[2] = {q, k};
  const llk_tensor3d* const out[2] = {q_out, k_out};
  const char* const names[4] = {"q", "k", "q_out", "k_out"};
  int64_t heads = 0;
  for (int s = 0; s < (k ? 2 : 1); ++s) {
    const int64_t H = in[s]->dim1;
    if (H < 0 || H > kMaxHeads)
      return fail(LLK_ERR_SHAPE, "%lld heads unsupported (to %lld)", (long long)H, (long long)kMaxHeads);
    int rc;
    if ((rc = check_rows(in[s], names[s], T, H, D, size, false)) ||
        (rc = check_rows(out[s], names[2 + s], T, H, D, size, true)))
      return rc;
    a.side[s] = RotarySide{in[s]->data, out[s]->data, in[s]->stride0, in[s]->stride1,
                           out[s]->stride0, out[s]->stride1, (int)H};
    heads += H;
  }
  if (T == 0 || heads == 0) return LLK_OK;
  if (!positions || !turns)
    return fail(LLK_ERR_INVALID_ARGUMENT, "%s is NULL", positions ? "turns" : "positions");
  int dev, rc;
  if ((rc = llk::current_gfx950(&dev))) return rc;
  a.positions = positions;
  a.turns = turns;
  a.factor = factor;
  a.tokens = (int)T;
  a.head_dim = (int)D;
  a.pairs = (int)pairs;
  a.inverse = (flags & LLK_ROTARY_INVERSE) != 0;
  const hipError_t e =
      llk_launch_rotary(a, dtype == LLK_FP32, (flags & LLK_ROTARY_INTERLEAVED) != 0,
                        ctx ? static_cast<hipStream_t>(ctx->stream) : nullptr);
  return e == hipSuccess ? LLK_OK
                         : fail(LLK_ERR_HIP, "rotary kernel: %s", hipGetErrorString(e));
}

}  // extern "C"
