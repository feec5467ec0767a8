// Activations of the mixed-precision linear-layer routines and their derivatives, in FP32.
//
//   relu       z < 0 ? 0 : z                           (a NaN stays a NaN)
//   gelu       z * Phi(z), Phi the normal distribution function
//   gelu_tanh  z * sigma(2u), u = sqrt(2/pi) (z + 0.044715 z^3); equal to z/2 (1 + tanh u)
//   silu       z * sigma(z), sigma(z) = 1 / (1 + exp(-z))
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/paralia_c.h"

namespace paralia {

// max and min that hand a NaN on.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x and 1/x of the special-function unit, two units in the last place or so; results below
// 2^-126 are 0. The plain intrinsics wrap them in code for subnormal numbers, which nothing here
// needs and which the epilogue of a product pays for 32768 times a tile.
__device__ __forceinline__ float exp2_f32(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_f32(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float GELU_C = 0.7978845608028654f;    // sqrt(2/pi)
constexpr float GELU_A = 0.044715f;
constexpr float INV_SQRT_2PI = 0.3989422804014327f;

// 1 / (1 + 2^y); 0 from y = 128 on.
__device__ __forceinline__ float sigmoid_exp2(float y) { return rcp_f32(1.0f + exp2_f32(y)); }

// Phi(-x) = erfc(x / sqrt(2)) / 2 for x >= 0, by the Chebyshev fit of erfc with a relative error below
// 1.2e-7 everywhere (Press et al., Numerical Recipes, "erfcc"): erfc(w) = t exp(-w^2 + P(t)),
// t = 1 / (1 + w/2). The factors log2(e) of the exponent and 1/2 of the result are in the constants.
__device__ __forceinline__ float normal_tail(float x) {
  constexpr float L = LOG2E;
  const float t = rcp_f32(fmaf(0.35355339059327373f, x, 1.0f));
  float p = 0.17087277f * L;
  p = fmaf(p, t, -0.82215223f * L);
  p = fmaf(p, t, 1.48851587f * L);
  p = fmaf(p, t, -1.13520398f * L);
  p = fmaf(p, t, 0.27886807f * L);
  p = fmaf(p, t, -0.18628806f * L);
  p = fmaf(p, t, 0.09678418f * L);
  p = fmaf(p, t, 0.37409196f * L);
  p = fmaf(p, t, 1.00002368f * L);
  p = fmaf(p, t, -1.26551223f * L - 1.0f);
  const float w = 0.8493218002880191f * x;    // sqrt(log2(e) / 2): w^2 is the exponent to base 2
  return t * exp2_f32(fmaf(-w, w, p));
}

// The sigmoid, or the tail probability, is 0 from where it falls below 2^-126. z is clamped to the left of
// that place, where it is 0 already: act(-inf) is then 0 and not inf * 0. What a finite z loses is below
// |z| * 2^-126 at the place itself, 1e-36 at most (BF16 has numbers down to there, so nothing nearer
// will do as a clamp: silu(-85) is -1e-35). A NaN stays a NaN throughout.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == PARALIA_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (ACT == PARALIA_ACT_GELU) {
    const float c = max_nan(z, -30.0f), h = normal_tail(fabsf(c));
    return c * (c > 0.0f ? 1.0f - h : h);
  }
  if (ACT == PARALIA_ACT_GELU_TANH) {
    constexpr float K1 = -2.0f * GELU_C * LOG2E, K2 = K1 * GELU_A;
    const float c = max_nan(z, -10.2f);   // the exponent is 132 there
    return c * sigmoid_exp2(c * fmaf(K2, c * c, K1));
  }
  if (ACT == PARALIA_ACT_SILU) {
    const float c = max_nan(z, -90.0f);   // the exponent is 129 there
    return c * sigmoid_exp2(-LOG2E * c);
  }
  return z;
}

// act'(z), clamped on both sides for the same reason: act'(+-inf) is 1 or 0.
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == PARALIA_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == PARALIA_ACT_GELU) {
    const float c = min_nan(max_nan(z, -30.0f), 30.0f);
    const float h = normal_tail(fabsf(c)), w = 0.8493218002880191f * c;
    return fmaf(c * INV_SQRT_2PI, exp2_f32(-w * w), c > 0.0f ? 1.0f - h : h);
  }
  if (ACT == PARALIA_ACT_GELU_TANH) {
    constexpr float K1 = -2.0f * GELU_C * LOG2E, K2 = K1 * GELU_A;
    const float c = min_nan(max_nan(z, -10.2f), 10.2f), q = c * c;
    const float g = sigmoid_exp2(c * fmaf(K2, q, K1));
    return fmaf(c * fmaf(6.0f * GELU_C * GELU_A, q, 2.0f * GELU_C), g * (1.0f - g), g);
  }
  if (ACT == PARALIA_ACT_SILU) {
    const float c = min_nan(max_nan(z, -90.0f), 90.0f);
    const float g = sigmoid_exp2(-LOG2E * c);
    return fmaf(c * g, 1.0f - g, g);
  }
  return 1.0f;
}

// Run `f` with the activation, or with the activation and the element type, as compile-time
// constants: f(IntC<ACT>()), f(IntC<ACT>(), IntC<BF16>()).
template <int V>
struct IntC {
  static constexpr int value = V;
};
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case PARALIA_ACT_RELU: f(IntC<PARALIA_ACT_RELU>()); break;
    case PARALIA_ACT_GELU: f(IntC<PARALIA_ACT_GELU>()); break;
    case PARALIA_ACT_GELU_TANH: f(IntC<PARALIA_ACT_GELU_TANH>()); break;
    case PARALIA_ACT_SILU: f(IntC<PARALIA_ACT_SILU>()); break;
    default: f(IntC<PARALIA_ACT_NONE>()); break;
  }
}

template <typename F>
__device__ __forceinline__ void with_act_type(int act, bool bf16, F f) {
  if (bf16) with_act(act, [&](auto a) { f(a, IntC<1>()); });
  else with_act(act, [&](auto a) { f(a, IntC<0>()); });
}

// One 16-bit element to and from FP32; `bf` tells BF16 from FP16.
__device__ __forceinline__ float load16(const void* p, int64_t i, bool bf) {
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return bf ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ void store16(void* p, int64_t i, float v, bool bf) {
  static_cast<uint16_t*>(p)[i] =
      bf ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
// Two packed 16-bit elements (the lower half first) to and from FP32.
__device__ __forceinline__ float2 unpack16(uint32_t v, bool bf) {
  if (bf) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf) {
  uint32_t r;
  if (bf) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    r = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    r = *reinterpret_cast<const uint32_t*>(&h);
  }
  return r;
}

}  // namespace paralia
