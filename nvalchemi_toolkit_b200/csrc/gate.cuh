// SPDX-License-Identifier: Apache-2.0
// Activations of the gated feed-forward block and their derivatives:
//   silu: g s, s = 1 / (1 + e^-g);  act' = s (1 + g (1 - s))
//   gelu: g Phi(g);                 act' = Phi(g) + g phi(g)
#pragma once
#include <cuda_runtime.h>

namespace nva {

enum Act : int { kSilu = 0, kGelu = 1 };

// 2^x and 1 / x by the special function unit, one instruction each (subnormal results become 0; 2 and 1 ulp): the epilogues
// of the 16-bit products are bound by what they issue.
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// act(g) and act'(g).  EXACT, for float32 results: a few 2^-24 of the value at every g (silu 5, gelu 8 with its tail; the
// derivatives of the sum of their terms' magnitudes), without branches, so that a thread's values run side by side.  Else with
// the fast functions, 3e-6 of the value, which is little beside half a step of 16 bits.  Infinities give NaN or infinity.
template <bool EXACT, int ACT>
__device__ __forceinline__ void activate(float g, float& a, float& da) {
  if constexpr (ACT == kSilu && !EXACT) {
    const float e = fast_exp2(-kLog2e * g), s = fast_rcp(1.f + e);
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == kSilu) {  // by e^-|g|, which cannot overflow; s and 1 - s both keep their digits
    const float e = expf(-fabsf(g)), q = __fdividef(1.f, 1.f + e), eq = e * q, s = g < 0.f ? eq : q, r = g < 0.f ? q : eq;
    a = g * s;
    da = s * (1.f + g * r);
  } else {
    // Phi(-|g|) = e^(-g^2 / 2) t P(t) with t = 1 / (1 + |g| / sqrt(8)): P is a polynomial fitted to the least relative error
    // (reweighted least squares on 4000 points) over |g| <= 16, where the exponential has long left the fp32 range; 4.4e-8 with
    // nine coefficients, 1.8e-6 with seven.  Relative, because act(g) of a negative g is all tail.  Its exponential is the
    // derivative's as well.
    float e, q;
    if constexpr (EXACT) {
      constexpr float c[9] = {0.141042367f, 0.14120248f, 0.121443897f, 0.101771072f, -0.0143238446f, 0.140501097f, -0.244882271f,
                              0.142906472f, -0.0296612736f};
      const float z = fminf(fabsf(g), 16.f), h = z * z, low = fmaf(z, z, -h), t = __fdividef(1.f, fmaf(0.35355339059327376f, z, 1.f));
      e = expf(-0.5f * h);
      e = fmaf(-0.5f * low, e, e);  // what rounding the square left
      float p = c[8];
#pragma unroll
      for (int i = 7; i >= 0; --i) p = fmaf(p, t, c[i]);
      q = e * t * p;
    } else {
      const float t = fast_rcp(1.f + 0.35355339059327376f * fabsf(g));
      e = fast_exp2(-0.5f * kLog2e * g * g);
      q = e * t * (0.141146347f + t * (0.139064237f + t * (0.139263988f + t * (0.0229727123f + t * (0.18885614f +
          t * (-0.174219206f + t * 0.0429148637f))))));
    }
    const float cdf = g < 0.f ? q : 1.f - q;
    a = g * cdf;
    da = cdf + g * 0.39894228040143268f * e;
  }
}

}  // namespace nva
