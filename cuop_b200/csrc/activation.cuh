// Activations of the feed-forward layers and their derivatives, in fp32.
#pragma once

#include "common.cuh"

namespace cuopx {

constexpr float kGeluTanhTwoC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluTanhA = 0.044715f;

// 2^x and 1 / x to about one unit in the last place (PTX approx forms; 2^x
// overflows to infinity, and 1 / infinity is 0).
__device__ __forceinline__ float2 exp2_2(float2 x) {
  float2 r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(x.y));
  return r;
}
__device__ __forceinline__ float2 rcp_2(float2 x) {
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(x.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(x.y));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Everything below works on pairs: the packed forms halve the instructions
// that surround the two exponentials and divisions.

// s(z) = 1 / (1 + exp(-z)); exp(-z) = inf gives 0, the limit.
__device__ __forceinline__ float2 sigmoid_2(float2 z, float2& e) {
  e = exp2_2(mul2(z, both(-kLog2e)));
  return rcp_2(add2(e, both(1.f)));
}

// s'(z) = s (1 - s) with 1 - s = e s, e = exp(-z): no cancellation.  e s is
// taken to be 1 at most, and where e = inf and s = 0 (the minimum of NaN and 1
// is 1), so that s = 0 gives s' = 0; s = NaN gives NaN.
__device__ __forceinline__ float2 sigmoid_slope_2(float2 e, float2 s) {
  const float2 r = mul2(e, s);
  return mul2(make_float2(fminf(r.x, 1.f), fminf(r.y, 1.f)), s);
}

// The normal density phi(z) and distribution function Phi(z): for x >= 0
//   Phi(-x) = phi(x) M(x),  M(x) = t (c0 + c1 t + ... + c6 t^6),  t = 1 / (1 + p x),
// and Phi(x) = 1 - Phi(-x).  The form is that of Hastings (1955); p and the
// coefficients are fitted here to Mills' ratio M = sqrt(pi / 2) erfcx(x / sqrt 2)
// by Remez exchange for the least relative error over 0 <= x <= 14: 6.3e-7, and
// 9.6e-7 with its evaluation in fp32, 1/250 of an fp16 rounding.  So Phi keeps
// its relative accuracy in the lower tail, where a fit for absolute error with
// five terms is 3 % off at -12; the two terms more cost 7 us of 120 in the dZ
// pass of 4096 x 28672 and nothing measurable in forward passes.  One
// exponential and one division give both phi and Phi.  phi is 0 where
// exp(-z^2 / 2) leaves fp32's normal range (|z| > 13.2).
__device__ __forceinline__ float2 normal_2(float2 z, float2& density) {
  const float2 t = rcp_2(fma2(both(0.265f), make_float2(fabsf(z.x), fabsf(z.y)), both(1.f)));
  density = mul2(both(0.39894228040143268f), exp2_2(mul2(mul2(z, z), both(-0.5f * kLog2e))));
  float2 q = fma2(both(-0.16991689880208605f), t, both(0.489477059912886f));
  q = fma2(q, t, both(-0.1663471276747126f));
  q = fma2(q, t, both(0.35717779071072653f));
  q = fma2(q, t, both(0.20791627927404013f));
  q = fma2(q, t, both(0.27030672238464215f));
  q = fma2(q, t, both(0.2646995312161768f));
  q = mul2(mul2(q, t), density);
  return make_float2(z.x >= 0.f ? 1.f - q.x : q.x, z.y >= 0.f ? 1.f - q.y : q.y);
}

// 2 sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float2 gelu_tanh_arg_2(float2 z) {
  return mul2(z, fma2(both(kGeluTanhTwoC * kGeluTanhA), mul2(z, z), both(kGeluTanhTwoC)));
}

template <int ACT>
__device__ __forceinline__ float2 act_value2(float2 z) {
  float2 e;
  if constexpr (ACT == CUOPX_ACT_RELU) return make_float2(z.x > 0.f ? z.x : 0.f, z.y > 0.f ? z.y : 0.f);
  if constexpr (ACT == CUOPX_ACT_GELU) return mul2(z, normal_2(z, e));
  if constexpr (ACT == CUOPX_ACT_GELU_TANH) return mul2(z, sigmoid_2(gelu_tanh_arg_2(z), e));
  if constexpr (ACT == CUOPX_ACT_SILU) return mul2(z, sigmoid_2(z, e));
  if constexpr (ACT == CUOPX_ACT_SIGMOID) return sigmoid_2(z, e);
  return z;
}

// a b + c where a's factor d of the product has not vanished, c where it has:
// z may be infinite there, or its powers beyond the range, and z d -> 0.
__device__ __forceinline__ float2 vanishing_fma2(float2 d, float2 a, float2 b, float2 c) {
  const float2 v = fma2(a, b, c);
  return make_float2(d.x > 0.f ? v.x : c.x, d.y > 0.f ? v.y : c.y);
}

// Value and derivative at z.  The derivative of an infinite z is its limit; the
// value needs a finite z (-inf * 0 is NaN).
template <int ACT>
__device__ __forceinline__ float2 act_slope2(float2 z, float2& value) {
  float2 e;
  if constexpr (ACT == CUOPX_ACT_RELU) {
    value = act_value2<ACT>(z);
    return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
  }
  if constexpr (ACT == CUOPX_ACT_GELU) {
    const float2 phi = normal_2(z, e);
    value = mul2(z, phi);
    return vanishing_fma2(e, z, e, phi);
  }
  if constexpr (ACT == CUOPX_ACT_GELU_TANH) {
    const float2 s = sigmoid_2(gelu_tanh_arg_2(z), e);
    const float2 d = sigmoid_slope_2(e, s);
    value = mul2(z, s);
    return vanishing_fma2(d, mul2(z, d), fma2(both(3.f * kGeluTanhTwoC * kGeluTanhA), mul2(z, z), both(kGeluTanhTwoC)), s);
  }
  if constexpr (ACT == CUOPX_ACT_SILU) {
    const float2 s = sigmoid_2(z, e);
    const float2 d = sigmoid_slope_2(e, s);
    value = mul2(z, s);
    return vanishing_fma2(d, z, d, s);
  }
  if constexpr (ACT == CUOPX_ACT_SIGMOID) {
    value = sigmoid_2(z, e);
    return sigmoid_slope_2(e, value);
  }
  value = z;
  return both(1.f);
}

// The value at one element.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  return act_value2<ACT>(both(z)).x;
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
