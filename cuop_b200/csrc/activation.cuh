// Activations of the feed-forward layers and their derivatives, in fp32.
#pragma once

#include "common.cuh"

namespace cuopx {

// s(z) = 1 / (1 + exp(-z)).  exp(-z) = inf gives 0, the limit.
__device__ __forceinline__ float sigmoid_f(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// s'(z) = e / (1 + e)^2 with e = exp(-|z|): no cancellation in 1 - s(z), no overflow.
__device__ __forceinline__ float sigmoid_slope_f(float z) {
  const float e = __expf(-fabsf(z));
  const float r = __fdividef(1.f, 1.f + e);
  return e * r * r;
}

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluTanhTwoC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluTanhA = 0.044715f;

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == CUOPX_ACT_RELU) return z > 0.f ? z : 0.f;
  // Phi(z) = erfc(-z / sqrt 2) / 2 keeps its relative accuracy in the lower tail.
  if constexpr (ACT == CUOPX_ACT_GELU) return z * (0.5f * erfcf(-kSqrtHalf * z));
  if constexpr (ACT == CUOPX_ACT_GELU_TANH) return z * sigmoid_f(kGeluTanhTwoC * (z + kGeluTanhA * z * z * z));
  if constexpr (ACT == CUOPX_ACT_SILU) return z * sigmoid_f(z);
  if constexpr (ACT == CUOPX_ACT_SIGMOID) return sigmoid_f(z);
  return z;
}

// Value and derivative at z.
template <int ACT>
__device__ __forceinline__ float act_slope(float z, float& value) {
  if constexpr (ACT == CUOPX_ACT_RELU) {
    value = z > 0.f ? z : 0.f;
    return z > 0.f ? 1.f : 0.f;
  }
  if constexpr (ACT == CUOPX_ACT_GELU) {
    const float phi = 0.5f * erfcf(-kSqrtHalf * z);
    value = z * phi;
    const float d = kInvSqrt2Pi * __expf(-0.5f * z * z);
    return d > 0.f ? fmaf(z, d, phi) : phi;  // z infinite or its square beyond the range: z d -> 0
  }
  if constexpr (ACT == CUOPX_ACT_GELU_TANH) {
    const float u = kGeluTanhTwoC * (z + kGeluTanhA * z * z * z);
    const float s = sigmoid_f(u), d = sigmoid_slope_f(u);
    value = z * s;
    return d > 0.f ? fmaf(z * d, kGeluTanhTwoC * (1.f + 3.f * kGeluTanhA * z * z), s) : s;
  }
  if constexpr (ACT == CUOPX_ACT_SILU) {
    const float s = sigmoid_f(z), d = sigmoid_slope_f(z);
    value = z * s;
    return d > 0.f ? fmaf(z, d, s) : s;
  }
  if constexpr (ACT == CUOPX_ACT_SIGMOID) {
    value = sigmoid_f(z);
    return sigmoid_slope_f(z);
  }
  value = z;
  return 1.f;
}

// Calls f with std::integral_constant<int, ACT>: one uniform branch around a
// loop over elements instead of one per element.
template <typename F>
__host__ __device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case CUOPX_ACT_RELU: f(std::integral_constant<int, CUOPX_ACT_RELU>{}); break;
    case CUOPX_ACT_GELU: f(std::integral_constant<int, CUOPX_ACT_GELU>{}); break;
    case CUOPX_ACT_GELU_TANH: f(std::integral_constant<int, CUOPX_ACT_GELU_TANH>{}); break;
    case CUOPX_ACT_SILU: f(std::integral_constant<int, CUOPX_ACT_SILU>{}); break;
    case CUOPX_ACT_SIGMOID: f(std::integral_constant<int, CUOPX_ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, CUOPX_ACT_NONE>{}); break;
  }
}

}  // namespace cuopx
