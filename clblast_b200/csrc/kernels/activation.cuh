// Activation functions of the fused products and their derivatives, evaluated in fp32 (fp64 nowhere).
//
//   relu       z for z > 0, else 0 (a NaN stays a NaN)                  slope: 1 for z > 0, else 0
//   gelu       z P(z), P the normal distribution function               slope: P(z) + z p(z), p its density
//   gelu_tanh  z s(2u), u = sqrt(2/pi) (z + 0.044715 z^3)               slope: s + 2 z s (1 - s) u'
//              (0.5 (1 + tanh u) = s(2u), s the logistic function)
//   silu       z s(z)                                                   slope: s (1 + z (1 - s))
//
// P(z) is taken as erfc(-z / sqrt 2) / 2, which keeps its relative precision where 1 + erf cancels (z << 0). Arguments
// that only scale a vanishing factor are clamped, so that an infinite z gives the limit instead of inf * 0.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200 {

enum Act : int { kActIdentity = 161, kActRelu = 162, kActGelu = 163, kActGeluTanh = 164, kActSilu = 165 };

// FAST: for results in 16 bits. The hardware's base-2 exponential and reciprocal, a relative error of 2^-20 + |x| 2^-22 in
// all, where 2^x is the exponential taken: its argument comes rounded (x = -z^2 / 2 log2 e for gelu: 2^-20 near zero, 2^-18
// at z = 3, 2^-15 where the value leaves the range at z = -13). Half a step of half precision is 2^-11, of its numbers below
// 2^-14 more, and z P(z) is below that from z = -4 on. Without FAST the full-precision functions, for results in single
// precision. A gelu in the epilogue of 8192 x 8192 x 512 costs 195 us more than the identity with erfcf.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2E = 1.4426950408889634f;

// s(x) = 1 / (1 + exp(-x)) and, for slopes, 1 - s(x) = exp(-x) s(x), which the subtraction would leave with an absolute
// error of s's last place. The argument is -x log2(e) for FAST, else -x. An exponential beyond the range makes s zero;
// the other factor is held finite there, so that their product is zero too (a NaN passes through s).
template <bool FAST>
__device__ __forceinline__ float logistic(float minus_x, float* complement = nullptr) {
  const float e = FAST ? exp2_fast(minus_x) : expf(minus_x);
  const float s = FAST ? rcp_fast(1.f + e) : 1.f / (1.f + e);
  if (complement) *complement = fminf(e, 3.0e38f) * s;
  return s;
}

// P(z), the normal distribution function, and exp(-z^2 / 2). With t = 1 / (1 + q |z|) the tail P(-|z|) is
// exp(-z^2 / 2) t c(t); c is a polynomial of degree six fitted here to the smallest relative error over |z| < 13.4 (6.4e-7;
// beyond, the exponential has left the range), so that a vanishing P keeps the relative precision of its exponential.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z, float* bell = nullptr) {
  if (FAST) {
    const float e = exp2_fast(z * z * (-0.5f * kLog2E));
    const float t = rcp_fast(fmaf(0.26516504294495533f, fabsf(z), 1.f));
    float c = -0.06754792165618550f;
    c = fmaf(c, t, 0.19396880130252385f);
    c = fmaf(c, t, -0.06479847023409181f);
    c = fmaf(c, t, 0.14153061996590430f);
    c = fmaf(c, t, 0.08333235214270828f);
    c = fmaf(c, t, 0.10784457380456717f);
    c = fmaf(c, t, 0.10566972585255615f);
    const float tail = e * (t * c);
    if (bell) *bell = e;
    return z < 0.f ? tail : 1.f - tail;
  }
  if (bell) *bell = expf(-0.5f * z * z);
  return 0.5f * erfcf(z * -0.70710678118654752f);
}

// -2u, times log2(e) for FAST
template <bool FAST>
__device__ __forceinline__ float gelu_tanh_arg(float z) {
  constexpr float k = -1.5957691216057308f * (FAST ? kLog2E : 1.f);  // 2 sqrt(2/pi)
  return z * fmaf(k * 0.044715f, z * z, k);
}
template <bool FAST>
__device__ __forceinline__ float silu_arg(float z) { return FAST ? -kLog2E * z : -z; }

template <bool FAST, int ACT>
__device__ __forceinline__ float act_value(float z) {
  switch (ACT) {
    case kActRelu: return z < 0.f ? 0.f : z;
    case kActGelu: return fmaxf(z, -60.f) * normal_cdf<FAST>(z);
    case kActGeluTanh: return fmaxf(z, -60.f) * logistic<FAST>(gelu_tanh_arg<FAST>(z));
    case kActSilu: return fmaxf(z, -200.f) * logistic<FAST>(silu_arg<FAST>(z));
    default: return z;
  }
}

template <bool FAST, int ACT>
__device__ __forceinline__ float act_slope(float z) {
  switch (ACT) {
    case kActRelu: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case kActGelu: {
      float e;
      const float cdf = normal_cdf<FAST>(z, &e);
      const float zc = fminf(fmaxf(z, -60.f), 60.f);
      return fmaf(zc * 0.3989422804014327f, e, cdf);
    }
    case kActGeluTanh: {
      float rest;
      const float s = logistic<FAST>(gelu_tanh_arg<FAST>(z), &rest);
      const float zc = fminf(fmaxf(z, -60.f), 60.f);
      constexpr float k2 = 1.5957691216057308f;
      return fmaf(zc * fmaf(k2 * 3.f * 0.044715f, zc * zc, k2), s * rest, s);
    }
    case kActSilu: {
      float rest;
      const float s = logistic<FAST>(silu_arg<FAST>(z), &rest);
      return fmaf(fminf(fmaxf(z, -200.f), 200.f) * rest, s, s);
    }
    default: return 1.f;
  }
}

// Calls f with the activation as a compile-time constant. The choice is made once per block of values: taken per value
// it keeps the compiler from interleaving the values' chains (8192 x 8192 x 512 with relu: 299 us against 110 without).
template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case kActRelu: f(ActTag<kActRelu>()); break;
    case kActGelu: f(ActTag<kActGelu>()); break;
    case kActGeluTanh: f(ActTag<kActGeluTanh>()); break;
    case kActSilu: f(ActTag<kActSilu>()); break;
    default: f(ActTag<kActIdentity>());
  }
}

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }

}  // namespace b200
