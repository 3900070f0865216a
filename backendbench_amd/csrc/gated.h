// The activations of the gated projection and their derivatives.
#pragma once
#include "../../include/mi355_train.h"
#include "common.h"

namespace mi355 {

__device__ __forceinline__ float gate_exp(float v) { return expf(v); }
__device__ __forceinline__ double gate_exp(double v) { return exp(v); }
__device__ __forceinline__ float gate_erfc(float v) { return erfcf(v); }
__device__ __forceinline__ double gate_erfc(double v) { return erfc(v); }

// 1 / (1 + exp(-v)) from exp(-|v|): no overflow, and full relative accuracy on the negative side.
template <typename A> __device__ __forceinline__ A gate_sigmoid(A v) {
  const A e = gate_exp(v < A(0) ? v : -v);
  return (v < A(0) ? e : A(1)) / (A(1) + e);
}
// act(g) = g * q(g) for all three: q = sigmoid(g), Phi(g), or (1 + tanh z) / 2 = sigmoid(2 z).
// Phi comes from erfc, which keeps its relative accuracy in the negative tail.
template <int ACT, typename A> __device__ __forceinline__ A gate_q(A g) {
  if constexpr (ACT == MI355_SILU) return gate_sigmoid(g);
  if constexpr (ACT == MI355_GELU) return A(0.5) * gate_erfc(g * A(-0.70710678118654752440));
  return gate_sigmoid(A(1.59576912160573071176) * (g + A(0.044715) * g * g * g));  // 2 sqrt(2 / pi) (g + 0.044715 g^3)
}
// act'(g) given q = gate_q(g).
template <int ACT, typename A> __device__ __forceinline__ A gate_grad(A g, A q) {
  if constexpr (ACT == MI355_SILU) return q * (A(1) + g * (A(1) - q));
  if constexpr (ACT == MI355_GELU) return q + g * gate_exp(A(-0.5) * g * g) * A(0.39894228040143267794);
  const A d = q * (A(1) - q);  // 0 far out, where g * g may already be infinite
  return d == A(0) ? q : q + g * d * A(1.59576912160573071176) * (A(1) + A(3 * 0.044715) * g * g);
}

}  // namespace mi355
