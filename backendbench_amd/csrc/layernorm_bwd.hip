// Layer norm, backward, over M dense rows of N: with xhat = (x - mean) rstd and g = dy w,
//   dx = rstd (g - mean_N(g) - xhat mean_N(g xhat)),   dw = sum_M dy xhat,   db = sum_M dy.
//
//   general  any type, length and alignment, two passes over x and dy: a block per row leaves the row's two means,
//            then every thread walks one column down a group of rows, writing dx and carrying that column's dw and
//            db in registers;
//   finish   adds the partial dw and db of the row groups in a fixed order (no atomics: the same call gives the
//            same bits).
#include "../../include/mi355_train.h"
#include "rowtile.h"

namespace mi355 {

constexpr int kLbBlock = 256;
constexpr int kLbMaxGroups = 256;  // row groups that leave a partial dw / db each

// sums[row] = {mean_N(g), mean_N(g xhat)}.
template <typename T, typename Wt, typename S>
__global__ __launch_bounds__(kLbBlock) void lb_row_means_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                               const S* __restrict__ mean, const S* __restrict__ rstd,
                                                               const Wt* __restrict__ w, S* __restrict__ sums, int64_t M, int64_t N) {
  __shared__ S red[2][kLbBlock / kWave];
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const S mu = mean[row], rs = rstd[row];
    S a = 0, b = 0;
    for (int64_t c = threadIdx.x; c < N; c += kLbBlock) {
      S g = static_cast<S>(dy[row * N + c]);
      if (w) g *= static_cast<S>(w[c]);
      a += g;
      b += g * ((static_cast<S>(x[row * N + c]) - mu) * rs);
    }
    __syncthreads();  // the previous row's sums have been read
    a = block_allreduce(a, SumOp(), red[0], S(0));
    b = block_allreduce(b, SumOp(), red[1], S(0));
    if (threadIdx.x == 0) {
      sums[2 * row] = a / static_cast<S>(N);
      sums[2 * row + 1] = b / static_cast<S>(N);
    }
  }
}

// One column per thread, blockIdx.y = row group; partial[group][0 / 1][N] = the group's dw / db.
template <typename T, typename Wt, typename S>
__global__ __launch_bounds__(kLbBlock) void lb_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                             const S* __restrict__ mean, const S* __restrict__ rstd,
                                                             const Wt* __restrict__ w, const S* __restrict__ sums, T* __restrict__ dx,
                                                             S* __restrict__ partial, int64_t M, int64_t N, int64_t rows_per_group) {
  const int64_t c = (int64_t)blockIdx.x * kLbBlock + threadIdx.x;
  if (c >= N) return;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_group, r1 = r0 + rows_per_group < M ? r0 + rows_per_group : M;
  const S gamma = w ? static_cast<S>(w[c]) : S(1);
  S dw = 0, db = 0;
  for (int64_t r = r0; r < r1; ++r) {
    const S rs = rstd[r];
    const S d = static_cast<S>(dy[r * N + c]);
    const S xhat = (static_cast<S>(x[r * N + c]) - mean[r]) * rs;
    dw += d * xhat;
    db += d;
    if (dx) dx[r * N + c] = static_cast<T>(rs * (d * gamma - sums[2 * r] - xhat * sums[2 * r + 1]));
  }
  if (partial) {
    partial[(int64_t)blockIdx.y * 2 * N + c] = dw;
    partial[(int64_t)blockIdx.y * 2 * N + N + c] = db;
  }
}

// dw and db: the groups' partials, summed by 4 x 64 threads (64 columns, every fourth group each).
template <typename Wt, typename S>
__global__ __launch_bounds__(kLbBlock) void lb_finish_kernel(const S* __restrict__ partial, Wt* __restrict__ dw, Wt* __restrict__ db,
                                                            int64_t N, int groups) {
  __shared__ S part[4][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;  // of the 2N columns [dw | db]
  const int q = threadIdx.x / 64;
  S s = 0;
  if (c < 2 * N)
    for (int g = q; g < groups; g += 4) s += partial[(int64_t)g * 2 * N + c];
  part[q][threadIdx.x % 64] = s;
  __syncthreads();
  if (q != 0 || c >= 2 * N) return;
  s = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
  Wt* out = c < N ? dw : db;
  if (out) out[c < N ? c : c - N] = static_cast<Wt>(s);
}

struct LbPlan {
  int64_t groups, rows_per_group;
};
// Row groups of the column pass: enough blocks for four per CU, at least 64 (no thread then adds more than a 64th of a
// column), at most one per row.
static LbPlan lb_plan(int64_t M, int64_t N) {
  const int64_t cols = (N + kLbBlock - 1) / kLbBlock;
  int64_t g = (4 * kNumCU + cols - 1) / cols;
  if (g > kLbMaxGroups) g = kLbMaxGroups;
  if (g < 64) g = 64;
  if (g > M) g = M;
  if (g < 1) g = 1;
  const int64_t per = (M + g - 1) / g;
  return LbPlan{(M + per - 1) / per, per};
}

template <typename T, typename Wt, typename S>
static int run_lb(const void* dyv, const void* xv, const void* mv, const void* rv, const void* wv, void* dxv, void* dwv, void* dbv,
                  int64_t M, int64_t N, void* ws, hipStream_t st) {
  const T *dy = static_cast<const T*>(dyv), *x = static_cast<const T*>(xv);
  const S *mean = static_cast<const S*>(mv), *rstd = static_cast<const S*>(rv);
  const Wt* w = static_cast<const Wt*>(wv);
  S* sums = static_cast<S*>(ws);
  S* partial = (dwv != nullptr || dbv != nullptr) ? sums + 2 * M : nullptr;
  const LbPlan p = lb_plan(M, N);
  if (dxv != nullptr)
    hipLaunchKernelGGL((lb_row_means_kernel<T, Wt, S>), dim3((unsigned)grid_for(M, 1, kNumCU * 32)), dim3(kLbBlock), 0, st, dy, x, mean, rstd, w, sums, M, N);
  hipLaunchKernelGGL((lb_columns_kernel<T, Wt, S>), dim3((unsigned)((N + kLbBlock - 1) / kLbBlock), (unsigned)p.groups), dim3(kLbBlock), 0, st, dy,
                     x, mean, rstd, w, sums, static_cast<T*>(dxv), partial, M, N, p.rows_per_group);
  if (partial)
    hipLaunchKernelGGL((lb_finish_kernel<Wt, S>), dim3((unsigned)((2 * N + 63) / 64)), dim3(kLbBlock), 0, st, partial,
                       static_cast<Wt*>(dwv), static_cast<Wt*>(dbv), N, (int)p.groups);
  return check_launch("mi355_layer_norm_backward");
}

}  // namespace mi355

using namespace mi355;

extern "C" int64_t mi355_layer_norm_backward_workspace_bytes(int64_t M, int64_t N, int dtype) {
  if (M <= 0 || N <= 0 || dtype_size(dtype) == 0) return 0;
  const int64_t acc = dtype == MI355_F64 ? 8 : 4;
  return (2 * M + lb_plan(M, N).groups * 2 * N) * acc;
}

extern "C" int mi355_layer_norm_backward(const void* dy, const void* x, int dtype, const void* mean, const void* rstd,
                                         const void* weight, int w_dtype, void* dx, void* dweight, void* dbias, int64_t M, int64_t N,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
  MI355_REQUIRE(M >= 0 && N >= 0, "mi355_layer_norm_backward: negative extent");
  MI355_REQUIRE(M > 0 || N == 0 || (dweight == nullptr && dbias == nullptr),
                "mi355_layer_norm_backward: no rows: the parameter gradients are zeros, which this call does not write");
  if (M == 0 || N == 0 || (dx == nullptr && dweight == nullptr && dbias == nullptr)) return MI355_OK;
  MI355_REQUIRE(dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr, "mi355_layer_norm_backward: NULL data pointer");
  MI355_REQUIRE(M < (int64_t(1) << 40) && N < (int64_t(1) << 28), "mi355_layer_norm_backward: extents too large (M=%lld N=%lld)",
                (long long)M, (long long)N);
  MI355_REQUIRE(workspace != nullptr && workspace_bytes >= mi355_layer_norm_backward_workspace_bytes(M, N, dtype) && aligned16(workspace),
                "mi355_layer_norm_backward: needs a 16-byte aligned workspace of %lld bytes",
                (long long)mi355_layer_norm_backward_workspace_bytes(M, N, dtype));
  hipStream_t st = static_cast<hipStream_t>(stream);
#define MI355_LB(DT, WDT, T_, W_, S_) \
  if (dtype == DT && w_dtype == WDT) return run_lb<T_, W_, S_>(dy, x, mean, rstd, weight, dx, dweight, dbias, M, N, workspace, st);
  MI355_LB(MI355_F32, MI355_F32, float, float, float)
  MI355_LB(MI355_F16, MI355_F16, f16_t, f16_t, float)
  MI355_LB(MI355_F16, MI355_F32, f16_t, float, float)
  MI355_LB(MI355_BF16, MI355_BF16, bf16_t, bf16_t, float)
  MI355_LB(MI355_BF16, MI355_F32, bf16_t, float, float)
  MI355_LB(MI355_F64, MI355_F64, double, double, double)
#undef MI355_LB
  return set_error(MI355_ERR_UNSUPPORTED, "mi355_layer_norm_backward: no kernel for rows of %s with parameters of %s", dtype_name(dtype),
                   dtype_name(w_dtype));
}
