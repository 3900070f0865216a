// The gated projection, backward (up to 16 rows: gated_backward_rows.hip): with gate = pre[:, :F], up = pre[:, F:],
//   dpre = [dh up act'(gate) | dh act(gate)],   dx = dpre W,   dW = dpre^T x.
//
// One elementwise kernel leaves dpre and its transpose, both in the products' types and paddings, and this library's
// products do the rest.  dpre^T is written out (another 2 M F elements) because the product kernels run 25 % faster on a
// K-contiguous left operand than on a transposed one: [22016, 4096] x [4096, 4096] takes 585 us from dpre as it is and 473
// from its transpose, which costs 28 us to write.  dpre is rounded to the inputs' type: it is the operand of two matrix
// products, whose matrix instructions take that type; everything before it is fp32 and the products accumulate in fp32.  A second
// operand for what the rounding leaves out would double both products, 1.0 of the 1.1 ms at [4096, 4096] x 2 * 11008; without it the
// error against 64 bits is 0.0023 of the result's norm in bf16, 0.0017 of it from rounding the result alone.  In f16 the rounding
// bounds the range too: beyond 65504 dpre becomes infinite (a loss scale's overflow), in its row of dx and its row of dW alone.
#include "gated.h"
#include "elementwise.h"

namespace mi355 {

constexpr int kGbTile = 64;

// The first `count` elements of v.
template <typename T, int V> __device__ __forceinline__ void gb_store(T* p, int64_t count, const VecN<T, V>& v) {
  if (count >= V) {
    *reinterpret_cast<typename AnyVec<sizeof(T)>::type*>(p) = __builtin_bit_cast(u32x4, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < count) p[j] = v.v[j];
  }
}

// Tiles of TM rows by 64 features, 256 threads: 64 rows, so that the transpose goes out in whole 128-byte lines (6.2 TB/s at
// [4096, 2 * 11008] bf16, 102 us), or 16 where tiles of 64 would leave most CUs idle ([197, 2 * 1001] fp32: 64 tiles 15 us,
// 256 tiles 6.5).  ROW: dpre [M][ld] (columns 2F .. ld - 1 become zeros); COL: its transpose dpre_t [2F][ld_t] (columns M ..
// ld_t - 1 become zeros), through LDS.  Vector accesses at any alignment.
template <typename T, int ACT, bool ROW, bool COL, int TM>
__global__ __launch_bounds__(256) void gated_dpre_kernel(const T* __restrict__ dh, const T* __restrict__ pre, T* __restrict__ dpre, int64_t ld,
                                                        T* __restrict__ dpre_t, int64_t ld_t, int64_t M, int64_t F, int tiles_f) {
  using A = typename OpMath<T>::type;
  constexpr int V = 16 / sizeof(T);
  constexpr int VECS = TM * kGbTile / V, PER = (VECS + 255) / 256;  // vectors of the tile, and per thread
  constexpr int LD = TM + 4 / sizeof(T);            // one bank further per feature
  __shared__ T turned[COL ? 2 : 1][COL ? kGbTile : 1][COL ? LD : 1];
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_f) * TM, f0 = (int64_t)(blockIdx.x % tiles_f) * kGbTile;
  VecN<T, V> gv[PER], uv[PER], dv[PER];
  auto column = [&](int i) { return f0 + (threadIdx.x + 256 * i) * V % kGbTile; };
  auto row = [&](int i) {  // (tiles of 16 rows: of threads past them too; rows past M read the last, their dh becomes zero)
    const int64_t m = m0 + (threadIdx.x + 256 * i) * V / kGbTile;
    return m < M ? m : M - 1;
  };
  if (F >= V) {
    u32x4 g[PER], u[PER], d[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      g[i] = load_within(pre + row(i) * 2 * F, column(i), F);
      u[i] = load_within(pre + row(i) * 2 * F + F, column(i), F);
      d[i] = load_within(dh + row(i) * F, column(i), F);
    }
    const bool whole = f0 + kGbTile <= F && m0 + TM <= M;  // of the block
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t c = m0 + (int64_t)(threadIdx.x + 256 * i) * V / kGbTile < M ? column(i) : F;  // (F: zeros)
      gv[i] = __builtin_bit_cast(VecN<T, V>, whole ? g[i] : placed<T>(g[i], c, F));
      uv[i] = __builtin_bit_cast(VecN<T, V>, whole ? u[i] : placed<T>(u[i], c, F));
      dv[i] = __builtin_bit_cast(VecN<T, V>, whole ? d[i] : placed<T>(d[i], c, F));
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t c = m0 + (int64_t)(threadIdx.x + 256 * i) * V / kGbTile < M ? column(i) : F;
      gv[i] = load_short(pre + row(i) * 2 * F, c, F);
      uv[i] = load_short(pre + row(i) * 2 * F + F, c, F);
      dv[i] = load_short(dh + row(i) * F, c, F);
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = (threadIdx.x + 256 * i) * V;
    const int64_t m = m0 + e / kGbTile, f = f0 + e % kGbTile;
    if (e >= TM * kGbTile) break;
    VecN<T, V> dg, du;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const A g = static_cast<A>(gv[i].v[j]), u = static_cast<A>(uv[i].v[j]), d = static_cast<A>(dv[i].v[j]);
      const A q = gate_q<ACT, GateMath<T>>(g);
      dg.v[j] = static_cast<T>(d * u * gate_grad<ACT, GateMath<T>>(g, q));
      du.v[j] = static_cast<T>(d * (g * q));
      if constexpr (COL) {  // (rows past M hold zeros: dv is zero there)
        turned[0][e % kGbTile + j][e / kGbTile] = dg.v[j];
        turned[1][e % kGbTile + j][e / kGbTile] = du.v[j];
      }
    }
    if constexpr (ROW) {
      const int64_t there = m < M ? F - f : 0;
      gb_store(dpre + m * ld + f, there, dg);
      gb_store(dpre + m * ld + F + f, there, du);
    }
  }
  if constexpr (ROW) {
    if (f0 + kGbTile >= F && ld > 2 * F) {
      for (int e = threadIdx.x; e < TM * (int)(ld - 2 * F); e += 256) {
        const int64_t m = m0 + e / (int)(ld - 2 * F);
        if (m < M) dpre[m * ld + 2 * F + e % (int)(ld - 2 * F)] = static_cast<T>(0.f);
      }
    }
  }
  if constexpr (COL) {
    __syncthreads();
    constexpr int W = 16 / sizeof(T);  // ld_t is a multiple of it
#pragma unroll
    for (int i = 0; i < 2 * TM * kGbTile / W / 256; ++i) {
      const int e = (threadIdx.x + 256 * i) * W;
      const int which = e / (TM * kGbTile), fl = e / TM % kGbTile, ml = e % TM;
      if (f0 + fl >= F || m0 + ml >= ld_t) continue;
      VecN<T, W> v;
#pragma unroll
      for (int j = 0; j < W; ++j) v.v[j] = turned[which][fl][ml + j];
      st<T, W>(dpre_t + ((int64_t)which * F + f0 + fl) * ld_t + m0 + ml, v);
    }
  }
}

// dst [C][ld] = src [R][C]^T (rows rs apart), columns R .. ld - 1 zeros.  Elements are moved as bits.
template <typename B>
__global__ __launch_bounds__(256) void turn_pad_kernel(const B* __restrict__ src, int64_t rs, B* __restrict__ dst, int64_t ld, int64_t R, int64_t C,
                                                      int tiles_c) {
  constexpr int LD = kGbTile + 4 / sizeof(B);
  __shared__ B tile[kGbTile][LD];
  const int64_t r0 = (int64_t)(blockIdx.x / tiles_c) * kGbTile, c0 = (int64_t)(blockIdx.x % tiles_c) * kGbTile;
  constexpr int V = 16 / sizeof(B), PER = kGbTile * kGbTile / V / 256;
  VecN<B, V> v[PER];
  auto row = [&](int i) {  // (rows past R become zeros)
    const int64_t r = r0 + (threadIdx.x + 256 * i) * V / kGbTile;
    return src + (r < R ? r : R - 1) * rs;
  };
  auto column = [&](int i) { return r0 + (threadIdx.x + 256 * i) * V / kGbTile < R ? c0 + (threadIdx.x + 256 * i) * V % kGbTile : C; };
  if (C >= V) {
    u32x4 raw[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) raw[i] = load_within(row(i), column(i), C);
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = __builtin_bit_cast(VecN<B, V>, placed<B>(raw[i], column(i), C));
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = load_short(row(i), column(i), C);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = (threadIdx.x + 256 * i) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) tile[e % kGbTile + j][e / kGbTile] = v[i].v[j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = (threadIdx.x + 256 * i) * V;
    const int64_t c = c0 + e / kGbTile, r = r0 + e % kGbTile;
    VecN<B, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = tile[e / kGbTile][e % kGbTile + j];
    if (c < C && r < ld) st<B, V>(dst + c * ld + r, o);  // ld is a multiple of 64
  }
}

static int64_t round_up(int64_t v, int64_t unit) { return (v + unit - 1) / unit * unit; }

// How the two products take their operands, and where the intermediate ones lie in the workspace.
struct GatedBackwardPlan {
  bool turn_w, turn_x;  // a transposed, zero-padded copy of the weight / of x stands in for it
  int64_t ld, ld_t;     // row lengths of dpre and dpre^T, = the products' K
  int64_t dpre, dpre_t, wt, xt, scratch, bytes;  // offsets
};
static GatedBackwardPlan plan_gated_backward(int64_t M, int64_t F, int64_t K, int dtype, bool want_dx, bool want_dw, bool w_rows16, bool x_rows16) {
  GatedBackwardPlan p{};
  const int es = dtype_size(dtype);
  const bool any = dtype == MI355_F64;  // the fp64 product takes any strides: dpre alone, no copies
  const int64_t V = 16 / es;
  // The row-major right operand as it is: aligned rows of whole vectors, and a product's K that its kernels take - from 256
  // rows on a multiple of 64, whose kernels pay for a copy of the weight; where something is padded anyway then to 128,
  // which lets the fastest, 256x256-tile kernel in.
  const bool many = es == 2 && M >= 256;
  p.turn_w = !any && !(w_rows16 && K % V == 0 && 2 * F % (many ? 64 : es == 2 ? 8 : 16) == 0);
  p.turn_x = !any && !(x_rows16 && K % V == 0 && M % 64 == 0);
  p.ld = p.turn_w ? round_up(2 * F, many ? 128 : 64) : 2 * F;
  p.ld_t = p.turn_x ? round_up(M, many ? 128 : 64) : M;
  int64_t at = 0;
  auto take = [&](bool wanted, int64_t bytes) {
    const int64_t here = at;
    if (wanted) at = round_up(at + bytes, 256);
    return here;
  };
  p.dpre = take(want_dx || (any && want_dw), M * p.ld * es);
  p.dpre_t = take(want_dw && !any, 2 * F * p.ld_t * es);
  p.wt = take(want_dx && p.turn_w, K * p.ld * es);
  p.xt = take(want_dw && p.turn_x, K * p.ld_t * es);
  const int64_t s1 = want_dx ? mi355_gemm_workspace_bytes(M, K, p.ld, dtype) : 0;
  const int64_t s2 = want_dw ? mi355_gemm_workspace_bytes(2 * F, K, any ? M : p.ld_t, dtype) : 0;
  p.scratch = take(true, s1 > s2 ? s1 : s2);  // the two products run one after the other
  p.bytes = at;
  return p;
}

template <typename T>
static int run_dpre(const void* dhv, const void* prev, void* dpre, int64_t ld, void* dpre_t, int64_t ld_t, int64_t M, int64_t F, int act, hipStream_t st) {
  const T *dh = static_cast<const T*>(dhv), *pre = static_cast<const T*>(prev);
  // (the transpose is padded past the last row's tile when its rows are padded to more than one)
  const int64_t rows = dpre_t != nullptr ? ld_t : M, tiles_f = (F + kGbTile - 1) / kGbTile;
  const bool small = tiles_f * ((rows + kGbTile - 1) / kGbTile) < kNumCU;
  const int64_t tiles_m = small ? (rows + 15) / 16 : (rows + kGbTile - 1) / kGbTile;
  MI355_REQUIRE(tiles_f * tiles_m < (int64_t(1) << 24), "mi355_gated_linear_backward: M=%lld F=%lld is too large", (long long)M, (long long)F);
  auto launch = [&](auto a, auto row, auto col, auto tm) {
    hipLaunchKernelGGL((gated_dpre_kernel<T, decltype(a)::value, decltype(row)::value, decltype(col)::value, decltype(tm)::value>),
                       dim3((unsigned)(tiles_f * tiles_m)), dim3(256), 0, st, dh, pre, static_cast<T*>(dpre), ld, static_cast<T*>(dpre_t), ld_t, M, F,
                       (int)tiles_f);
  };
  auto go = [&](auto a, auto row, auto col) {
    small ? launch(a, row, col, std::integral_constant<int, 16>()) : launch(a, row, col, std::integral_constant<int, kGbTile>());
  };
  using std::false_type;
  using std::true_type;
  return dispatch_act(act, "mi355_gated_linear_backward", [&](auto a) {
    if constexpr (std::is_same<T, double>::value) {
      go(a, true_type(), false_type());  // (no transpose: the fp64 product takes any strides)
    } else {
      if (dpre != nullptr && dpre_t != nullptr) go(a, true_type(), true_type());
      else if (dpre != nullptr) go(a, true_type(), false_type());
      else go(a, false_type(), true_type());
    }
  });
}

static int run_turn_pad(const void* src, int64_t rs, void* dst, int64_t ld, int64_t R, int64_t C, int es, hipStream_t st) {
  const int64_t tiles_c = (C + kGbTile - 1) / kGbTile, tiles_r = round_up(ld, kGbTile) / kGbTile;
  MI355_REQUIRE(tiles_c * tiles_r < (int64_t(1) << 24), "mi355_gated_linear_backward: an operand of %lld x %lld is too large", (long long)R, (long long)C);
  const dim3 grid((unsigned)(tiles_c * tiles_r));
  if (es == 2) hipLaunchKernelGGL((turn_pad_kernel<uint16_t>), grid, dim3(256), 0, st, static_cast<const uint16_t*>(src), rs, static_cast<uint16_t*>(dst), ld, R, C, (int)tiles_c);
  else hipLaunchKernelGGL((turn_pad_kernel<uint32_t>), grid, dim3(256), 0, st, static_cast<const uint32_t*>(src), rs, static_cast<uint32_t*>(dst), ld, R, C, (int)tiles_c);
  return check_launch("mi355_gated_linear_backward");
}

static bool rows16(const void* p, int64_t rs, int es) { return aligned16(p) && rs * es % 16 == 0; }

}  // namespace mi355

using namespace mi355;

extern "C" int64_t mi355_gated_linear_backward_workspace_bytes(int64_t M, int64_t F, int64_t K, int dtype) {
  if (M <= 0 || F <= 0 || K <= 0 || dtype_size(dtype) < 2) return 0;
  if (gated_backward_rows_takes(M, K)) return gated_backward_rows_workspace(M, F, K, dtype);
  int64_t most = 0;
  for (int aligned = 0; aligned < 4; ++aligned)
    for (int wanted = 1; wanted < 4; ++wanted) {
      const int64_t b = plan_gated_backward(M, F, K, dtype, wanted & 1, wanted & 2, aligned & 1, aligned & 2).bytes;
      most = b > most ? b : most;
    }
  return most;
}

extern "C" int mi355_gated_linear_backward(const void* dh, const void* x, int64_t x_rs, const void* weight, int64_t w_rs, const void* pre,
                                           void* dx, void* dweight, int64_t M, int64_t F, int64_t K, int act, int dtype,
                                           void* workspace, int64_t workspace_bytes, void* stream) {
  MI355_REQUIRE(M >= 0 && F >= 0 && K >= 0, "mi355_gated_linear_backward: negative extent");
  MI355_REQUIRE(act >= MI355_SILU && act <= MI355_GELU_TANH, "mi355_gated_linear_backward: unknown activation %d", act);
  if (dtype != MI355_F32 && dtype != MI355_F16 && dtype != MI355_BF16 && dtype != MI355_F64)
    return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_linear_backward: unsupported dtype %s", dtype_name(dtype));
  if (dx == nullptr && dweight == nullptr) return MI355_OK;
  MI355_REQUIRE(M > 0 && F > 0 && K > 0, "mi355_gated_linear_backward: an empty extent: the gradients are zeros or empty, which this call does not write");
  MI355_REQUIRE(M < (1 << 30) && F < (1 << 29) && K < (1 << 30), "mi355_gated_linear_backward: extents too large");
  MI355_REQUIRE(dh != nullptr && x != nullptr && weight != nullptr && pre != nullptr, "mi355_gated_linear_backward: NULL data pointer");
  if (M == 1) x_rs = K;  // (nothing is read at that distance)
  MI355_REQUIRE(x_rs >= K && w_rs >= K, "mi355_gated_linear_backward: rows overlap (strides %lld, %lld for K = %lld)", (long long)x_rs,
                (long long)w_rs, (long long)K);
  if (gated_backward_rows_takes(M, K)) {
    const int64_t need = gated_backward_rows_workspace(M, F, K, dtype);
    MI355_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned16(workspace),
                  "mi355_gated_linear_backward: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    return launch_gated_backward_rows(GatedBackwardArgs{dh, x, weight, pre, dx, dweight, x_rs, w_rs, M, F, K, act, dtype}, workspace,
                                      static_cast<hipStream_t>(stream));
  }
  const int es = dtype_size(dtype);
  const bool any = dtype == MI355_F64;
  const GatedBackwardPlan p = plan_gated_backward(M, F, K, dtype, dx != nullptr, dweight != nullptr, rows16(weight, w_rs, es), rows16(x, x_rs, es));
  MI355_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes && aligned16(workspace),
                "mi355_gated_linear_backward: needs a 16-byte aligned workspace of %lld bytes", (long long)p.bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  void* dpre = dx != nullptr || any ? ws + p.dpre : nullptr;
  void* dpre_t = dweight != nullptr && !any ? ws + p.dpre_t : nullptr;
  void* scratch = ws + p.scratch;
  const int64_t scratch_bytes = p.bytes - p.scratch;
  int rc = MI355_ERR_UNSUPPORTED;
  switch (dtype) {
    case MI355_F32: rc = run_dpre<float>(dh, pre, dpre, p.ld, dpre_t, p.ld_t, M, F, act, st); break;
    case MI355_F16: rc = run_dpre<f16_t>(dh, pre, dpre, p.ld, dpre_t, p.ld_t, M, F, act, st); break;
    case MI355_BF16: rc = run_dpre<bf16_t>(dh, pre, dpre, p.ld, dpre_t, p.ld_t, M, F, act, st); break;
    default: rc = run_dpre<double>(dh, pre, dpre, p.ld, dpre_t, p.ld_t, M, F, act, st); break;
  }
  if (rc == MI355_OK) rc = check_launch("mi355_gated_linear_backward");
  if (rc == MI355_OK && dx != nullptr) {
    if (p.turn_w) {
      rc = run_turn_pad(weight, w_rs, ws + p.wt, p.ld, 2 * F, K, es, st);
      if (rc == MI355_OK)
        rc = mi355_gemm(dpre, p.ld, 1, ws + p.wt, 1, p.ld, nullptr, 0, 0, dx, M, K, p.ld, 1.0, 0.0, dtype, scratch, scratch_bytes, stream);
    } else {
      rc = mi355_gemm(dpre, p.ld, 1, weight, w_rs, 1, nullptr, 0, 0, dx, M, K, 2 * F, 1.0, 0.0, dtype, scratch, scratch_bytes, stream);
    }
  }
  if (rc == MI355_OK && dweight != nullptr) {
    if (any) {
      rc = mi355_gemm(dpre, 1, p.ld, x, x_rs, 1, nullptr, 0, 0, dweight, 2 * F, K, M, 1.0, 0.0, dtype, scratch, scratch_bytes, stream);
    } else if (p.turn_x) {
      rc = run_turn_pad(x, x_rs, ws + p.xt, p.ld_t, M, K, es, st);
      if (rc == MI355_OK)
        rc = mi355_gemm(dpre_t, p.ld_t, 1, ws + p.xt, 1, p.ld_t, nullptr, 0, 0, dweight, 2 * F, K, p.ld_t, 1.0, 0.0, dtype, scratch, scratch_bytes, stream);
    } else {
      rc = mi355_gemm(dpre_t, p.ld_t, 1, x, x_rs, 1, nullptr, 0, 0, dweight, 2 * F, K, M, 1.0, 0.0, dtype, scratch, scratch_bytes, stream);
    }
  }
  return rc;
}
