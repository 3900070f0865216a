// The gated projection of a feed-forward block, h = act(x Wg^T) * (x Wu^T), W = [Wg; Wu] of 2F rows: which kernel takes a
// call, and the activation as a kernel of its own behind a product (more than a few rows of fp32 and fp64).
#include <string.h>

#include "gated.h"
#include "elementwise.h"

namespace mi355 {

// Columns f .. f + V - 1 of one row per work item.
template <typename T, int ACT, int V>
__global__ __launch_bounds__(256) void gated_act_kernel(const T* __restrict__ pre, T* __restrict__ h, int64_t items, int64_t per_row, int64_t F) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t m = items < (int64_t(1) << 32) ? (uint32_t)i / (uint32_t)per_row : i / per_row;
    const int64_t f = (i - m * per_row) * V;
    const VecN<T, V> g = ld<T, V>(pre + m * 2 * F + f), u = ld<T, V>(pre + m * 2 * F + F + f);
    VecN<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = g.v[j] * gate_q<ACT, T>(g.v[j]) * u.v[j];
    st<T, V>(h + m * F + f, r);
  }
}

// dst [R][ld] = src [R][C] (rows rs apart, any alignment), columns C .. ld - 1 zeros; one 16-byte piece of dst per work item.
template <typename B>
__global__ __launch_bounds__(256) void pad_rows_kernel(const B* __restrict__ src, int64_t rs, int64_t C, B* __restrict__ dst, int64_t pieces,
                                                      int64_t items) {
  constexpr int V = 16 / sizeof(B);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t r = items < (int64_t(1) << 32) ? (uint32_t)i / (uint32_t)pieces : i / pieces;
    const int64_t c = (i - r * pieces) * V;
    const B* row = src + r * rs;
    st<B, V>(dst + i * V, C < V ? load_short(row, c, C) : __builtin_bit_cast(VecN<B, V>, placed<B>(load_within(row, c, C), c, C)));
  }
}

template <typename T>
static int run_gated_act(const void* pre, void* h, int64_t M, int64_t F, int act, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = F % V == 0 && aligned16(pre) && aligned16(h);
  const int rc = dispatch_act(act, "mi355_gated_act", [&](auto a) {
    auto go = [&](auto v) {
      constexpr int VV = decltype(v)::value;
      const int64_t items = M * (F / VV);
      hipLaunchKernelGGL((gated_act_kernel<T, decltype(a)::value, VV>), dim3((unsigned)grid_for(items, 256, 1 << 20)), dim3(256), 0, st,
                         static_cast<const T*>(pre), static_cast<T*>(h), items, F / VV, F);
    };
    vec ? go(std::integral_constant<int, V>()) : go(std::integral_constant<int, 1>());
  });
  return rc != MI355_OK ? rc : check_launch("mi355_gated_act");
}

}  // namespace mi355

using namespace mi355;

extern "C" int mi355_gated_act(const void* pre, void* h, int dtype, int64_t M, int64_t F, int act, void* stream) {
  MI355_REQUIRE(M >= 0 && F >= 0, "mi355_gated_act: negative extent");
  MI355_REQUIRE(act >= MI355_SILU && act <= MI355_GELU_TANH, "mi355_gated_act: unknown activation %d", act);
  if (M == 0 || F == 0) return MI355_OK;
  MI355_REQUIRE(pre != nullptr && h != nullptr, "mi355_gated_act: NULL data pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MI355_F32) return run_gated_act<float>(pre, h, M, F, act, st);
  if (dtype == MI355_F64) return run_gated_act<double>(pre, h, M, F, act, st);
  return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_act: unsupported dtype %s", dtype_name(dtype));
}

extern "C" int mi355_pad_rows(const void* src, int64_t src_rs, int64_t R, int64_t C, void* dst, int64_t ld, int element_size, void* stream) {
  MI355_REQUIRE(R >= 0 && C >= 0 && ld >= C && src_rs >= C, "mi355_pad_rows: bad extents");
  MI355_REQUIRE((element_size == 2 || element_size == 4) && ld * element_size % 16 == 0, "mi355_pad_rows: rows of %lld elements of %d bytes",
                (long long)ld, element_size);
  if (R == 0 || ld == 0) return MI355_OK;
  MI355_REQUIRE((src != nullptr || C == 0) && dst != nullptr && aligned16(dst), "mi355_pad_rows: NULL or misaligned pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t pieces = ld * element_size / 16, items = R * pieces;
  const dim3 grid((unsigned)grid_for(items, 256, 1 << 20));
  if (element_size == 2) hipLaunchKernelGGL((pad_rows_kernel<uint16_t>), grid, dim3(256), 0, st, static_cast<const uint16_t*>(src), src_rs, C, static_cast<uint16_t*>(dst), pieces, items);
  else hipLaunchKernelGGL((pad_rows_kernel<uint32_t>), grid, dim3(256), 0, st, static_cast<const uint32_t*>(src), src_rs, C, static_cast<uint32_t*>(dst), pieces, items);
  return check_launch("mi355_pad_rows");
}

extern "C" int mi355_gated_linear(const void* x, int64_t x_rs, const void* weight, int64_t w_rs, void* h, void* pre, int64_t M, int64_t F,
                                  int64_t K, int act, int dtype, void* stream) {
  MI355_REQUIRE(M >= 0 && F >= 0 && K >= 0, "mi355_gated_linear: negative extent");
  MI355_REQUIRE(act >= MI355_SILU && act <= MI355_GELU_TANH, "mi355_gated_linear: unknown activation %d", act);
  if (M == 0 || F == 0) return MI355_OK;
  MI355_REQUIRE(x != nullptr && weight != nullptr && h != nullptr, "mi355_gated_linear: NULL data pointer");
  if (M == 1) x_rs = K;  // (nothing is read at that distance)
  MI355_REQUIRE(x_rs >= K && w_rs >= K, "mi355_gated_linear: rows overlap (strides %lld, %lld for K = %lld)", (long long)x_rs,
                (long long)w_rs, (long long)K);
  const GatedArgs a{x, weight, h, pre, x_rs, w_rs, M, F, K, act, dtype};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const char* form = knobs().gated_form;  // a test and measurement knob: one form, where it applies
  const bool dots = gated_dots_takes(a);
  if (dots && strcmp(form, "dots") == 0) return launch_gated_dots(a, st);
  if ((dtype == MI355_BF16 || dtype == MI355_F16) && M < (1 << 30) && F < (1 << 29) && K > 0 && K < (1 << 30)) {
    const int64_t tiles = ((M + 127) / 128) * ((F + 63) / 64);  // of 128 rows by 64 features
    const bool rows16 = a.x_rs % 8 == 0 && a.w_rs % 8 == 0 && aligned16(x) && aligned16(weight);
    const bool few = gated_rows_takes(a), t128 = rows16 && K % 64 == 0 && tiles < (1 << 23), t256 = rows16 && gated_x16_takes(a);
    if (few && strcmp(form, "rows") == 0) return launch_gated_rows(a, st);
    if (t128 && strcmp(form, "tile128") == 0) return launch_gated_small2(a, st);
    if (t256 && strcmp(form, "tile256") == 0) return launch_gated_x16(a, st);
    // Measured, us (graphs, inputs that no cache holds).  Rows against 128-row tiles up to 32 rows: 40 / 48, 16 / 19 and 16 / 47 at
    // [32, 4096] x 2 * 11008, [32, 2048] x 2 * 5504 and [32, 8192] x 2 * 1376.  Beyond, the rows' kernel takes one round of the CUs
    // per 4096 features and the tiles a time that grows with K, however few they are.  64 rows (33: the rows' side 3 - 14 % less):
    //      F   K = 512      1024         2048         2560         4096         8192
    //   4096   6.2 /  7.8    8.3 / 10.5  13.3 / 19.6  15.9 / 28.0  21.5 / 33.8  36.3 / 65.6
    //   4160  10.2 /  7.9   13.3 / 10.5  19.3 / 19.8  23.9 / 27.2  32.5 / 34.3  55.7 / 66.8
    //   5504  10.5 /  7.9   13.7 / 12.2  20.8 / 20.7  25.4 / 29.0  33.2 / 36.7  61.9 / 70.1
    //   8192  10.9 /  8.2   15.3 / 16.6  24.5 / 26.3  28.9 / 31.7  39.1 / 45.1  68.0 / 83.7
    //   8256  14.8 /  8.2   19.7 / 16.8  29.8 / 26.5  37.2 / 31.2  50.5 / 45.8  88.7 / 88.2
    //  11008  15.6 /  9.2   20.9 / 19.6  32.4 / 30.9  39.9 / 35.4  51.4 / 52.1  98.2 / 97.8
    // 128- against 256-row tiles 55 / 79 and 22 / 42 with 172 and 86 of the former, 23 / 43 with 172, 86 / 87 and 42 / 45 with
    // 344, 122 / 90 and 65 / 50 with 688.
    const bool rows_win = M <= 32 || tiles <= kNumCU / 4 || (tiles <= kNumCU / 2 && K > 2048);
    if (dots && !gated_rows_aligned(a)) return launch_gated_dots(a, st);
    if (few && (rows_win || !t128)) return launch_gated_rows(a, st);
    if (t128 && tiles <= (t256 ? kNumCU : 2 * kNumCU)) return launch_gated_small2(a, st);
    if (t256) return launch_gated_x16(a, st);
    if (t128 && K % 128 == 0) return launch_gated_small2(a, st);  // (K % 128 == 64 with many tiles: padded rows are faster)
  }
  if (dots && strcmp(form, "rows") != 0) return launch_gated_dots(a, st);
  if (dtype == MI355_F32 && gated_rows_takes(a)) return launch_gated_rows(a, st);
  return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_linear: no single kernel for M=%lld F=%lld K=%lld %s", (long long)M, (long long)F,
                   (long long)K, dtype_name(dtype));
}
