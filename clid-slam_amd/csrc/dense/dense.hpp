// What the dense operators (layer, cross entropy of a class head, label of each row) share: element types, activations, the
// running softmax statistics, argument checks.
//
// Softmax statistics.  A row's statistics over a set of columns are (m, r): the largest z and r = sum over the OTHER columns of
// exp(z - m).  log sum exp = m + log1p(r), so the log-probability of the largest column is -log1p(r) and the loss of a target t
// is (m - z_t) + log1p(r): a confident row keeps its relative accuracy where m + log(1 + r) would round it away.  Two sets
// join as: the larger m wins, r = r_win + (1 + r_lose) exp(m_lose - m_win).  A set of -inf alone has m = -inf, r = 0; one that holds a NaN or
// +inf has r = NaN.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/clid_dense.h"
#include "../../../include/clid_native.h"

extern "C" void clid_set_error(const char* fmt, ...);

namespace clid_dense {

using bf16 = __hip_bfloat16;
using f16 = __half;

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(f16 v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T down(float v);
template <> __device__ __forceinline__ float down<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 down<bf16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ f16 down<f16>(float v) { return __float2half(v); }

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// ---- activations: act(z) and dy act'(z), in fp32 ------------------------------------------------------------------------
// Phi(z) by the Chebyshev fit of erfc(x) = t exp(-x^2 + p(t)), t = 2 / (2 + x), of Press et al., Numerical Recipes, 6.2 (relative
// error 1.2e-7 for x >= 0): one exp, one reciprocal and nine FMAs without a branch, where the library's erf takes two branches.
__device__ __forceinline__ float normal_cdf(float z) {
  const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.f));
  float p = 0.17087277f;
  p = fmaf(p, t, -0.82215223f);
  p = fmaf(p, t, 1.48851587f);
  p = fmaf(p, t, -1.13520398f);
  p = fmaf(p, t, 0.27886807f);
  p = fmaf(p, t, -0.18628806f);
  p = fmaf(p, t, 0.09678418f);
  p = fmaf(p, t, 0.37409196f);
  p = fmaf(p, t, 1.00002368f);
  p = fmaf(p, t, -1.26551223f);
  const float half = 0.5f * t * __builtin_amdgcn_exp2f(fmaf(-x, x, p) * 1.4426950408889634f);
  return z < 0.f ? half : 1.f - half;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case CLID_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case CLID_ACT_LEAKY_RELU: return z > 0.f ? z : 0.01f * z;
    case CLID_ACT_GELU: return z * normal_cdf(z);
    case CLID_ACT_SILU: return z * sigmoid(z);
    default: return z;
  }
}
// dy act'(z).  relu selects, as torch's does: a unit whose z <= 0 hands back 0 whatever it was sent (0 times an overflowed dy would be NaN), and a
// NaN z hands dy on.
__device__ __forceinline__ float act_grad(float dy, float z, int act) {
  switch (act) {
    case CLID_ACT_RELU: return z <= 0.f ? 0.f : dy;
    case CLID_ACT_LEAKY_RELU: return z > 0.f ? dy : 0.01f * dy;
    case CLID_ACT_GELU: return dy * fmaf(z * 0.3989422804014327f, __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f), normal_cdf(z));
    case CLID_ACT_SILU: {
      const float p = sigmoid(z);
      return dy * (p * (1.f + z * (1.f - p)));
    }
    default: return dy;
  }
}

// z as the backward pass gets it (clid_linear_args.z_out): fp32, or fp16 for both 16-bit types (a slope is wrong by the rounding of z times
// its own slope, 2^-12 |z| in fp16, 2^-9 |z| in bf16; beyond 65504 every slope is constant).  Rounding must not turn a slope of 1 into one of
// 0 (a tiny z becoming 0) nor a finite z into an infinity (z p (1 - p) of silu is inf * 0 there).
template <typename T> struct KeptZ { using Z = f16; };
template <> struct KeptZ<float> { using Z = float; };
template <typename Z> __device__ __forceinline__ Z keep_z(float z);
template <> __device__ __forceinline__ float keep_z<float>(float z) { return z; }
template <> __device__ __forceinline__ f16 keep_z<f16>(float z) {
  f16 h = down<f16>(z);
  const float b = up(h);
  if (b == 0.f && z != 0.f) h = down<f16>(copysignf(5.9604645e-8f, z));               // 2^-24, the smallest fp16
  if (fabsf(b) > 65504.f && fabsf(z) <= 3.4028235e38f) h = down<f16>(copysignf(65504.f, z));
  return h;
}

// ---- softmax statistics ---------------------------------------------------------------------------------------------------
struct Stat {
  float m, r;
  int at;  // the lowest column that holds m (labels only)
};
// does (m, at) come before (n, bt)?  A NaN counts as largest, then the larger value, then the lower column.
__device__ __forceinline__ bool ahead(float m, int at, float n, int bt) {
  const bool mn = m != m, nn = n != n;
  if (mn || nn) return mn && (!nn || at < bt);
  return m > n || (m == n && at < bt);
}
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  const bool first = ahead(a.m, a.at, b.m, b.at);
  const Stat w = first ? a : b, l = first ? b : a;
  return {w.m, w.r + (l.m == neg_inf() ? l.r : (1.f + l.r) * expf(l.m - w.m)), w.at};
}

// ---- host: argument checks ----------------------------------------------------------------------------------------------
inline bool sizes_ok(int64_t rows, int32_t k, int32_t n) {
  return rows >= 0 && rows < (int64_t(1) << 31) && k >= 1 && n >= 1 && k < (1 << 20) && n < (1 << 20) &&
         rows * (k > n ? k : n) <= (int64_t(1) << 40) && int64_t(k) * n <= (int64_t(1) << 40);
}
inline int64_t up256(int64_t v) { return (v + 255) & ~int64_t(255); }

}  // namespace clid_dense

#define DENSE_CHECK_LAUNCH(what)                                              \
  do {                                                                        \
    hipError_t e__ = hipGetLastError();                                       \
    if (e__ != hipSuccess) {                                                  \
      clid_set_error("%s: HIP error: %s", what, hipGetErrorString(e__));      \
      return CLID_E_HIP;                                                      \
    }                                                                         \
  } while (0)
