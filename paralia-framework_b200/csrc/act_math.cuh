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

// 1 / (1 + exp(-x)) for x >= -80: below that the caller clamps, since exp(-x) leaves the range
// of the fast division.
__device__ __forceinline__ float sigmoid_f32(float x) {
  return __fdividef(1.0f, 1.0f + __expf(-x));
}

constexpr float GELU_C = 0.7978845608028654f;    // sqrt(2/pi)
constexpr float GELU_A = 0.044715f;
constexpr float INV_SQRT2 = 0.7071067811865476f;
constexpr float INV_SQRT_2PI = 0.3989422804014327f;

// The three smooth activations vanish to the left faster than any 16-bit type resolves, so z
// is clamped there: act(-inf) is then 0 and not inf * 0. A NaN stays a NaN throughout.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == PARALIA_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (ACT == PARALIA_ACT_GELU) {
    const float c = max_nan(z, -30.0f);
    return 0.5f * c * erfcf(-c * INV_SQRT2);
  }
  if (ACT == PARALIA_ACT_GELU_TANH) {
    const float c = max_nan(z, -9.0f);    // 2u = -66 there
    return c * sigmoid_f32(2.0f * GELU_C * c * fmaf(GELU_A * c, c, 1.0f));
  }
  if (ACT == PARALIA_ACT_SILU) {
    const float c = max_nan(z, -80.0f);
    return c * sigmoid_f32(c);
  }
  return z;
}

// act'(z), clamped on both sides for the same reason: act'(+-inf) is 1 or 0.
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == PARALIA_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == PARALIA_ACT_GELU) {
    const float c = min_nan(max_nan(z, -30.0f), 30.0f);
    return fmaf(c * INV_SQRT_2PI, __expf(-0.5f * c * c), 0.5f * erfcf(-c * INV_SQRT2));
  }
  if (ACT == PARALIA_ACT_GELU_TANH) {
    const float c = min_nan(max_nan(z, -9.0f), 9.0f);
    const float q = GELU_A * c * c;
    const float g = sigmoid_f32(2.0f * GELU_C * c * (1.0f + q));
    return fmaf(2.0f * GELU_C * c * (1.0f + 3.0f * q), g * (1.0f - g), g);
  }
  if (ACT == PARALIA_ACT_SILU) {
    const float c = min_nan(max_nan(z, -80.0f), 80.0f);
    const float g = sigmoid_f32(c);
    return fmaf(c * g, 1.0f - g, g);
  }
  return 1.0f;
}

// Run `f` with the activation as a compile-time constant: f(std::integral_constant<int, ACT>).
template <int V>
struct ActC {
  static constexpr int value = V;
};
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case PARALIA_ACT_RELU: f(ActC<PARALIA_ACT_RELU>()); break;
    case PARALIA_ACT_GELU: f(ActC<PARALIA_ACT_GELU>()); break;
    case PARALIA_ACT_GELU_TANH: f(ActC<PARALIA_ACT_GELU_TANH>()); break;
    case PARALIA_ACT_SILU: f(ActC<PARALIA_ACT_SILU>()); break;
    default: f(ActC<PARALIA_ACT_NONE>()); break;
  }
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
