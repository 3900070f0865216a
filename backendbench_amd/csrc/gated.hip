// The gated projection of a feed-forward block, h = act(x Wg^T) * (x Wu^T), W = [Wg; Wu] of 2F rows: which kernel takes a
// call, and the activation as a kernel of its own behind a product (fp32, fp64, and layouts no single kernel takes).
#include <string.h>

#include "gated.h"
#include "elementwise.h"

namespace mi355 {

// Columns f .. f + V - 1 of one row per work item.  P: type of pre as read.
template <typename T, typename P, int ACT, int V, bool SAVE>
__global__ __launch_bounds__(256) void gated_act_kernel(const P* __restrict__ pre, T* __restrict__ h, T* __restrict__ pre_out,
                                                       int64_t items, int64_t per_row, int64_t F) {
  using A = typename OpMath<T>::type;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t m = items < (int64_t(1) << 32) ? (uint32_t)i / (uint32_t)per_row : i / per_row;
    const int64_t f = (i - m * per_row) * V;
    const VecN<P, V> g = ld_nt<P, V>(pre + m * 2 * F + f), u = ld_nt<P, V>(pre + m * 2 * F + F + f);
    VecN<T, V> r, sg, su;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const A ga = static_cast<A>(g.v[j]), ua = static_cast<A>(u.v[j]);
      r.v[j] = static_cast<T>(ga * gate_q<ACT, GateMath<T>>(ga) * ua);
      if constexpr (SAVE) {
        sg.v[j] = static_cast<T>(ga);
        su.v[j] = static_cast<T>(ua);
      }
    }
    st<T, V>(h + m * F + f, r);
    if constexpr (SAVE) {
      st<T, V>(pre_out + m * 2 * F + f, sg);
      st<T, V>(pre_out + m * 2 * F + F + f, su);
    }
  }
}

template <typename T, typename P>
static int run_gated_act(const void* pre, void* h, void* pre_out, int64_t M, int64_t F, int act, hipStream_t st) {
  constexpr int V = 16 / sizeof(P);  // whole 16-byte reads
  const bool vec = F % V == 0 && aligned16(pre) && aligned16(h) && aligned16(pre_out);
  const int rc = dispatch_act(act, "mi355_gated_act", [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    auto go = [&](auto v, auto save) {
      constexpr int VV = decltype(v)::value;
      const int64_t items = M * (F / VV);
      hipLaunchKernelGGL((gated_act_kernel<T, P, ACT, VV, decltype(save)::value>), dim3((unsigned)grid_for(items, 256, 1 << 20)), dim3(256), 0, st,
                         static_cast<const P*>(pre), static_cast<T*>(h), static_cast<T*>(pre_out), items, F / VV, F);
    };
    using std::integral_constant;
    if (pre_out != nullptr) vec ? go(integral_constant<int, V>(), std::true_type()) : go(integral_constant<int, 1>(), std::true_type());
    else vec ? go(integral_constant<int, V>(), std::false_type()) : go(integral_constant<int, 1>(), std::false_type());
  });
  return rc != MI355_OK ? rc : check_launch("mi355_gated_act");
}

}  // namespace mi355

using namespace mi355;

extern "C" int mi355_gated_act(const void* pre, int pre_dtype, void* h, void* pre_out, int dtype, int64_t M, int64_t F, int act,
                               void* stream) {
  MI355_REQUIRE(M >= 0 && F >= 0, "mi355_gated_act: negative extent");
  MI355_REQUIRE(act >= MI355_SILU && act <= MI355_GELU_TANH, "mi355_gated_act: unknown activation %d", act);
  if (M == 0 || F == 0) return MI355_OK;
  MI355_REQUIRE(pre != nullptr && h != nullptr, "mi355_gated_act: NULL data pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (pre_dtype == MI355_F32 && dtype == MI355_F16) return run_gated_act<f16_t, float>(pre, h, pre_out, M, F, act, st);
  if (pre_dtype == MI355_F32 && dtype == MI355_BF16) return run_gated_act<bf16_t, float>(pre, h, pre_out, M, F, act, st);
  if (pre_dtype != dtype)
    return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_act: no kernel for %s from %s", dtype_name(dtype), dtype_name(pre_dtype));
  MI355_DISPATCH_FLOAT(dtype, "mi355_gated_act", return run_gated_act<T, T>(pre, h, pre_out, M, F, act, st));
}

extern "C" int mi355_gated_linear(const void* x, int64_t x_rs, const void* weight, int64_t w_rs, void* h, void* pre, int64_t M, int64_t F,
                                  int64_t K, int act, int dtype, void* stream) {
  MI355_REQUIRE(M >= 0 && F >= 0 && K >= 0, "mi355_gated_linear: negative extent");
  MI355_REQUIRE(act >= MI355_SILU && act <= MI355_GELU_TANH, "mi355_gated_linear: unknown activation %d", act);
  if (M == 0 || F == 0) return MI355_OK;
  MI355_REQUIRE(x != nullptr && weight != nullptr && h != nullptr, "mi355_gated_linear: NULL data pointer");
  MI355_REQUIRE(x_rs >= K && w_rs >= K, "mi355_gated_linear: rows overlap (strides %lld, %lld for K = %lld)", (long long)x_rs,
                (long long)w_rs, (long long)K);
  const GatedArgs a{x, weight, h, pre, x_rs, w_rs, M, F, K, act, dtype};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if ((dtype == MI355_BF16 || dtype == MI355_F16) && M < (1 << 30) && F < (1 << 29) && K > 0 && K < (1 << 30)) {
    const bool rows16 = a.x_rs % 8 == 0 && a.w_rs % 8 == 0 && aligned16(x) && aligned16(weight);
    const bool few = M <= kGatedRows, t128 = rows16 && K % 64 == 0, t256 = rows16 && gated_x16_takes(a);
    const char* form = knobs().gated_form;  // a test and measurement knob: one form, where it applies
    if (form[0] != 0) {
      if (few && (strcmp(form, "rows") == 0 || strcmp(form, "direct") == 0)) return launch_gated_rows(a, st);
      if (t128 && strcmp(form, "tile128") == 0) return launch_gated_small2(a, st);
      if (t256 && strcmp(form, "tile256") == 0) return launch_gated_x16(a, st);
    }
    // Measured ([M, 4096] x 2 * 11008 and [M, 2048] x 2 * 5504, us): rows against 128-row tiles 46.7 / 48.7 and 17.7 / 19 at 32
    // rows, 60 / 48 and 23 / 19.4 at 48, 69 / 49.5 and 26.4 / 19.8 at 64; 128- against 256-row tiles 55 / 77 and 22 / 41 with 172
    // and 86 of the former, 22.7 / 42 with 172, 78 / 79.5 and 42 / 43.5 with 344, 122 / 89 and 64 / 48 with 688.
    const int64_t tiles = ((M + 127) / 128) * ((F + 63) / 64);  // of 128 rows by 64 features
    if (few && (M <= 32 || !t128)) return launch_gated_rows(a, st);
    if (t128 && tiles <= (t256 ? kNumCU : 2 * kNumCU)) return launch_gated_small2(a, st);
    if (t256) return launch_gated_x16(a, st);
  }
  return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_linear: no single kernel for M=%lld F=%lld K=%lld %s", (long long)M, (long long)F,
                   (long long)K, dtype_name(dtype));
}
