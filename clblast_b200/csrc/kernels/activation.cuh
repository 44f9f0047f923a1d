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

// s(x) = 1 / (1 + exp(-x)) and, for slopes, 1 - s(x) = exp(-x) s(x), which the subtraction would leave with an absolute
// error of s's last place. FAST: the hardware exponential and reciprocal, a relative error of about 2^-21, far below the
// 2^-11 of a half result; without it the full-precision functions, for results in single precision. x is held above
// -80, so that the exponential stays finite (a NaN passes).
template <bool FAST>
__device__ __forceinline__ float logistic(float x, float* complement = nullptr) {
  const float xc = x < -80.f ? -80.f : x;
  const float e = FAST ? __expf(-xc) : expf(-xc);
  const float s = FAST ? __fdividef(1.f, 1.f + e) : 1.f / (1.f + e);
  if (complement) *complement = e * s;
  return s;
}

template <bool FAST>
__device__ __forceinline__ float gelu_tanh_arg(float z) {  // 2u
  constexpr float k2 = 1.5957691216057308f;  // 2 sqrt(2/pi)
  return k2 * z * (1.f + 0.044715f * z * z);
}

template <bool FAST>
__device__ __forceinline__ float act_value(int act, float z) {
  switch (act) {
    case kActRelu: return z < 0.f ? 0.f : z;
    case kActGelu: return fmaxf(z, -60.f) * (0.5f * erfcf(z * -0.70710678118654752f));
    case kActGeluTanh: return fmaxf(z, -60.f) * logistic<FAST>(gelu_tanh_arg<FAST>(z));
    case kActSilu: return fmaxf(z, -80.f) * logistic<FAST>(z);
    default: return z;
  }
}

template <bool FAST>
__device__ __forceinline__ float act_slope(int act, float z) {
  const float zc = fminf(fmaxf(z, -60.f), 60.f);
  switch (act) {
    case kActRelu: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case kActGelu: {
      const float e = FAST ? __expf(-0.5f * zc * zc) : expf(-0.5f * zc * zc);
      return 0.5f * erfcf(z * -0.70710678118654752f) + zc * (0.3989422804014327f * e);
    }
    case kActGeluTanh: {
      float rest;
      const float s = logistic<FAST>(gelu_tanh_arg<FAST>(z), &rest);
      constexpr float k2 = 1.5957691216057308f;
      return s + zc * s * rest * k2 * (1.f + 3.f * 0.044715f * zc * zc);
    }
    case kActSilu: {
      float rest;
      const float s = logistic<FAST>(z, &rest);
      return s * (1.f + fminf(fmaxf(z, -80.f), 200.f) * rest);
    }
    default: return 1.f;
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
