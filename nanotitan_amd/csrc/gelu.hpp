// GELU, erf form: gelu(x) = x Phi(x) and gelu'(x) = Phi(x) + x phi(x), with Phi
// the standard normal CDF, Phi(x) = erfc(-x/sqrt2)/2, and phi(x) =
// exp(-x^2/2)/sqrt(2 pi). One for the 16-bit grouped GEMMs' epilogues and, in
// each type, for the kernels beside them, so that an expert's hidden values do not
// depend on the path. (The register-staged and generic GEMMs, which take 16-bit
// widths that are no multiple of 8, form 1 + erf: gemm_common.hpp.)
#pragma once

#include "common.hpp"

namespace nt {

// For 16-bit outputs. erfc(z), z >= 0, is the Chebyshev fit of Press et al.,
// Numerical Recipes ("erfcc": t = 1/(1 + z/2), erfc(z) = t exp(-z^2 + P(t)),
// fractional error below 1.2e-7 everywhere), evaluated with the hardware exp2
// and reciprocal: far below the half-ulp of bf16 / fp16, in the tail too (where
// a fit of erf with an absolute bound was off by 5e-4 at -4 and 1e-2 at -8), and
// about half the instructions of the library erff.
__device__ __forceinline__ float erfc_nonneg(float z, float& ez2) {
  constexpr float kLog2e = 1.4426950408889634f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.5f, z, 1.0f));
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
  ez2 = __builtin_amdgcn_exp2f(-z * z * kLog2e);           // exp(-z^2)
  return t * ez2 * __builtin_amdgcn_exp2f(p * kLog2e);
}
__device__ __forceinline__ float norm_cdf(float x, float& ez2) {
  const float c = 0.5f * erfc_nonneg(fabsf(x) * 0.70710678118654752f, ez2);
  return x >= 0.f ? 1.0f - c : c;
}

// Phi(x) and exp(-x^2/2) for values of type T. float32 takes the library's erf
// and exp, as the float32 GEMMs' epilogue does (the fit: 8.5e-8 against 3.7e-8
// of relative error on normal inputs).
template <typename T>
__device__ __forceinline__ float gelu_cdf(float x, float& bell) {
  return norm_cdf(x, bell);
}
template <>
__device__ __forceinline__ float gelu_cdf<float>(float x, float& bell) {
  bell = expf(-0.5f * x * x);
  return 0.5f * (1.f + erff(x * 0.70710678118654752f));
}

}  // namespace nt
