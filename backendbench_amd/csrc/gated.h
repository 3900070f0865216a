// The activations of the gated projection and their derivatives.
#pragma once
#include <type_traits>

#include "../../include/mi355_train.h"
#include "elementwise.h"  // VecN

namespace mi355 {

__device__ __forceinline__ float gate_exp(float v) { return expf(v); }
__device__ __forceinline__ double gate_exp(double v) { return exp(v); }
__device__ __forceinline__ float gate_erfc(float v) { return erfcf(v); }
__device__ __forceinline__ double gate_erfc(double v) { return erfc(v); }
__device__ __forceinline__ float gate_div(float a, float b) { return a / b; }
__device__ __forceinline__ double gate_div(double a, double b) { return a / b; }

// float arithmetic whose result is rounded to 16 bits: the hardware's exp2 and reciprocal (1 ulp each; the exponential's
// argument is rounded once more, |v| 2^-24 of relative error) instead of the library's exact-rounding sequences.
struct GateHalf {
  float v;
  __device__ __forceinline__ GateHalf(float f) : v(f) {}
  __device__ __forceinline__ operator float() const { return v; }
};
__device__ __forceinline__ float gate_exp(GateHalf a) { return __builtin_amdgcn_exp2f(a.v * 1.44269504088896340736f); }
// erfc(v) = t P(t) exp(-v^2), t = 1 / (1 + 0.46 v), for v >= 0: P of degree 7 fitted here to erfc(v) exp(v^2) / t over all of
// t in (0, 1] for the smallest relative error, 6.8e-7, so the far tail keeps its digits; erfc(-v) = 2 - erfc(v).
__device__ __forceinline__ float gate_erfc(GateHalf a) {
  const float v = __builtin_fabsf(a.v), t = __builtin_amdgcn_rcpf(1.f + 0.46f * v);
  float p = 0.0677143769f;
  p = __builtin_fmaf(p, t, -0.226629397f);
  p = __builtin_fmaf(p, t, 0.169191163f);
  p = __builtin_fmaf(p, t, 0.0526105011f);
  p = __builtin_fmaf(p, t, 0.186847832f);
  p = __builtin_fmaf(p, t, 0.231181876f);
  p = __builtin_fmaf(p, t, 0.259557266f);
  p = __builtin_fmaf(p, t, 0.259527059f);
  const float e = p * t * __builtin_amdgcn_exp2f(v * v * -1.44269504088896340736f);
  return a.v < 0.f ? 2.f - e : e;
}
__device__ __forceinline__ float gate_div(GateHalf a, float b) { return a.v * __builtin_amdgcn_rcpf(b); }

// 1 / (1 + exp(-v)) from exp(-|v|): no overflow, and full relative accuracy on the negative side.
template <typename A, typename F> __device__ __forceinline__ F gate_sigmoid(F v) {
  const F e = gate_exp(A(v < F(0) ? v : -v));
  return gate_div(A(v < F(0) ? e : F(1)), F(1) + e);
}
// act(g) = g * q(g) for all three: q = sigmoid(g), Phi(g), or (1 + tanh z) / 2 = sigmoid(2 z).
// Phi comes from erfc, which keeps its relative accuracy in the negative tail.
template <int ACT, typename A, typename F> __device__ __forceinline__ F gate_q(F g) {
  if constexpr (ACT == MI355_SILU) return gate_sigmoid<A>(g);
  if constexpr (ACT == MI355_GELU) return F(0.5) * gate_erfc(A(g * F(-0.70710678118654752440)));
  return gate_sigmoid<A>(F(1.59576912160573071176) * (g + F(0.044715) * g * g * g));  // 2 sqrt(2 / pi) (g + 0.044715 g^3)
}
// act'(g) given q = gate_q(g).
template <int ACT, typename A, typename F> __device__ __forceinline__ F gate_grad(F g, F q) {
  if constexpr (ACT == MI355_SILU) return q * (F(1) + g * (F(1) - q));
  if constexpr (ACT == MI355_GELU) return q + g * gate_exp(A(F(-0.5) * g * g)) * F(0.39894228040143267794);
  const F d = q * (F(1) - q);  // 0 far out, where g * g may already be infinite
  return d == F(0) ? q : q + g * d * F(1.59576912160573071176) * (F(1) + F(3 * 0.044715) * g * g);
}
// The arithmetic for results of type T.
template <typename T> using GateMath = std::conditional_t<sizeof(T) == 2, GateHalf, typename OpMath<T>::type>;

// 16 bytes at an address that is only a multiple of an element's size.
template <int B> struct AnyVec;
template <> struct AnyVec<2> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct AnyVec<4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct AnyVec<8> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(8))); };
// 16 bytes without their first `count` elements: the rest moves to the front, zeros follow.  The end of a row is read as the
// 16 bytes that end with it, without a branch per element, and moved into place when it is needed.
template <typename T> __device__ __forceinline__ u32x4 drop_front(u32x4 v, int count) {
  const int bytes = count * (int)sizeof(T);
  if (bytes & 8) v = u32x4{v[2], v[3], 0u, 0u};
  if (bytes & 4) v = u32x4{v[1], v[2], v[3], 0u};
  if constexpr (sizeof(T) == 2) {
    if (bytes & 2) v = u32x4{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
  }
  return bytes >= 16 ? u32x4{0u, 0u, 0u, 0u} : v;
}

// The V = 16 / sizeof(T) elements of a row of n from the c-th on, zeros behind its end.  Rows of at least V: in two steps, so that
// all loads of a thread are on their way before the first is moved; shorter rows element by element.
template <typename T, int V = 16 / sizeof(T)> __device__ __forceinline__ u32x4 load_within(const T* row, int64_t c, int64_t n) {
  return __builtin_nontemporal_load(reinterpret_cast<const typename AnyVec<sizeof(T)>::type*>(row + (c + V <= n ? c : n - V)));
}
template <typename T, int V = 16 / sizeof(T)> __device__ __forceinline__ u32x4 placed(u32x4 v, int64_t c, int64_t n) {
  const int64_t over = c + V - n;
  return drop_front<T>(v, over <= 0 ? 0 : over < V ? (int)over : V);
}
template <typename T, int V = 16 / sizeof(T)> __device__ __forceinline__ VecN<T, V> load_short(const T* row, int64_t c, int64_t n) {
  VecN<T, V> v{};
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (c + j < n) v.v[j] = row[c + j];
  return v;
}

// 8 or 16 bytes at such an address.
template <int BYTES, int ALIGN> struct AnyPart { typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN))); };
template <typename T, int V> __device__ __forceinline__ void store_any(T* p, const VecN<T, V>& v) {
  using Part = typename AnyPart<sizeof(T) * V, sizeof(T)>::type;
  *reinterpret_cast<Part*>(p) = __builtin_bit_cast(Part, v);
}

// body(ACT) with an integral constant.
template <typename Body> static int dispatch_act(int act, const char* name, Body body) {
  switch (act) {
    case MI355_SILU: body(std::integral_constant<int, MI355_SILU>()); return MI355_OK;
    case MI355_GELU: body(std::integral_constant<int, MI355_GELU>()); return MI355_OK;
    case MI355_GELU_TANH: body(std::integral_constant<int, MI355_GELU_TANH>()); return MI355_OK;
    default: return set_error(MI355_ERR_INVALID, "%s: unknown activation %d", name, act);
  }
}

// One gated projection: x [M][K], weight [2F][K] (gate rows, then up rows), both K-contiguous; h [M][F]; pre [M][2F] or null.
struct GatedArgs {
  const void* x;
  const void* w;
  void* h;
  void* pre;
  int64_t x_rs, w_rs, M, F, K;
  int act, dtype;
};
// gated_x16.hip
bool gated_x16_takes(const GatedArgs& a);
int launch_gated_x16(const GatedArgs& a, hipStream_t st);
// gemm.hip: 128 rows by 64 features per workgroup; K % 64 == 0, 16-byte aligned rows
int launch_gated_small2(const GatedArgs& a, hipStream_t st);
// gated_rows.hip: few rows, 16-byte aligned ones of whole 16-byte units faster
bool gated_rows_aligned(const GatedArgs& a);
bool gated_rows_takes(const GatedArgs& a);
int launch_gated_rows(const GatedArgs& a, hipStream_t st);
// gated_dots.hip: a handful of rows of any float type, at any address
bool gated_dots_takes(const GatedArgs& a);
int launch_gated_dots(const GatedArgs& a, hipStream_t st);


// Its backward pass: dh [M][F], pre [M][2F], dx [M][K] and dw [2F][K] dense, dx or dw null when not wanted.
struct GatedBackwardArgs {
  const void *dh, *x, *w, *pre;
  void *dx, *dw;
  int64_t x_rs, w_rs, M, F, K;
  int act, dtype;
};
// gated_backward_rows.hip: few rows of any type, strides and alignment
bool gated_backward_rows_takes(int64_t M, int64_t K);
int64_t gated_backward_rows_workspace(int64_t M, int64_t F, int64_t K, int dtype);
int launch_gated_backward_rows(const GatedBackwardArgs& a, void* workspace, hipStream_t st);

}  // namespace mi355
