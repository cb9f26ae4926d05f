// silu(g) = g / (1 + e^-g) and its derivative beside other factors, for any g.
#pragma once
#include "mvpa_common.cuh"
#include "tc_ptx.cuh"

namespace mvpa {
namespace {

// For results in 16 bits.  With a = e^(-|g| / 4) (which leaves the normal numbers below |g| = 349, where the product with any
// factor rounds to zero) the factor s = 1 / (1 + e^-g) of a negative g is a^4 / (1 + a^4), taken into a product in four parts, so that
// nothing underflows that the result does not.  Relative errors of a^4: |g| 2^-23.7 from the rounding of a's argument (2^-18 near 50, 2^-15.3
// at the end), and an ulp or two of a, four times over, 2^-20; the result's own rounding to bf16 is one of up to 2^-8.
struct Sigmoid {
  float part, r;  // e^(-|g| / 4) where g < 0, else 1;  1 / (1 + e^-|g|)
  float other;    // 1 - s
  __device__ __forceinline__ explicit Sigmoid(float g) {
    const float a = ptx::ex2(fabsf(g) * (-0.25f * kLog2e)), a2 = a * a, e = a2 * a2;
    r = __fdividef(1.f, 1.f + e);
    part = g < 0.f ? a : 1.f;
    other = g < 0.f ? r : e * r;
  }
  // a b s: each product on the way is at most the larger of |a| and |b| or the result, so none overflows before it.
  __device__ __forceinline__ float times(float a, float b) const { return (a * part * part * r) * (b * part * part); }
  // a b s (1 + g (1 - s)).  The last two factors are one number between -0.1 and 1.1, which goes into `a` before `b` does, as half of it.
  __device__ __forceinline__ float times_slope(float a, float b, float g) const {
    return (a * part * part * (r * fmaf(g, 0.5f * other, 0.5f))) * (b * part * part) * 2.f;
  }
};

// silu(g) u, for results in 32 bits: the library's exponential, and the same parts where e^-|g| would leave the normal numbers.
__device__ __forceinline__ float silu_mul_f32(float g, float u) {
  if (fabsf(g) < 80.f || g > 0.f) return g / (1.f + expf(-g)) * u;
  const float a = expf(0.25f * g);
  return (g * a * a) * (u * a * a);
}

}  // namespace
}  // namespace mvpa
