// Layer norm, backward, over M dense rows of N: with xhat = (x - mean) rstd and g = dy w,
//   dx = rstd (g - mean_N(g) - xhat mean_N(g xhat)),   dw = sum_M dy xhat,   db = sum_M dy.
//
//   tile     rows of up to 16 K elements, one pass over x and dy: a row sits in the registers of 8 .. 1024 lanes, which
//            keep the same columns for every row they walk, so dw and db gather in registers too;
//   general  fp64 and longer rows, two passes over x and dy: a block per row leaves the row's two means, then every
//            thread walks one column down a group of rows, writing dx and carrying that column's dw and db;
//   finish   adds the partial dw and db of the blocks / row groups in a fixed order (no atomics: the same call gives
//            the same bits).
// Bound: HBM.  3 M N elements have to move; the tile kernel adds one fp32 partial of 2 N per block.
#include "../../include/mi355_train.h"
#include "rowtile.h"

namespace mi355 {

constexpr int kLbBlock = 256;
constexpr int kLbMaxGroups = 256;  // row groups that leave a partial dw / db each

// The tile kernel: blocks of 1024 threads, GL lanes per row, EL = NV x V elements per lane.  One block per CU (at most 256
// partials of dw / db, which the finish pass reads back from the last-level cache); sixteen waves of it, each with the
// next row's loads in flight while it reduces the current one, keep 64 KB per CU outstanding.  x and dy stay in the
// registers as loaded and are widened again after the two sums have met: 32 fp32 accumulators, two rows of raw vectors
// and the weights fit the 128 registers that sixteen waves leave.  Rows of more than one wave meet in LDS, one barrier
// per row (the slots alternate).
constexpr int kLbTile = 1024;
constexpr int kLbTileBlocks = kNumCU;

// V elements as loaded, in whole registers.
template <typename T, int V> struct LbRaw {
  static constexpr int R = sizeof(T) * V / 4;
  uint32_t r[R];
  __device__ __forceinline__ void set(const VecN<T, V>& v) {
    struct Regs { uint32_t r[R]; };
    const Regs t = __builtin_bit_cast(Regs, v);
#pragma unroll
    for (int i = 0; i < R; ++i) r[i] = t.r[i];
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, r[j]);
    else if constexpr (std::is_same<T, bf16_t>::value) return __builtin_bit_cast(float, j & 1 ? r[j >> 1] & 0xffff0000u : r[j >> 1] << 16);
    else return static_cast<float>(__builtin_bit_cast(T, (uint16_t)(r[j >> 1] >> (16 * (j & 1)))));
  }
  __device__ __forceinline__ void clear_unless(bool in) {
#pragma unroll
    for (int i = 0; i < R; ++i) r[i] = in ? r[i] : 0u;
  }
  __device__ __forceinline__ void clear_unless(bool in, int j) {  // element j alone
    if constexpr (sizeof(T) == 4) r[j] = in ? r[j] : 0u;
    else if (!in) r[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
  }
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int i = 0; i < R; ++i) asm volatile("" : "+v"(r[i]));
  }
};

template <typename T, typename Wt, int GL, int NV, bool VEC, bool AHEAD>
__global__ __launch_bounds__(kLbTile) void lb_tile_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         const Wt* __restrict__ w, T* __restrict__ dx, float* __restrict__ partial,
                                                         Wt* __restrict__ dw_out, Wt* __restrict__ db_out, int64_t M, int N) {
  constexpr int V = Vec<T>::N;
  constexpr int G = kLbTile / GL;                     // rows a block works on at a time
  constexpr int WPR = GL > kWave ? GL / kWave : 1;    // waves per row
  constexpr int WG = GL > kWave ? G : kLbTile / kWave;  // partial sums per column that meet in LDS at the end
  __shared__ float2 red[2][kLbTile / kWave];
  __shared__ __attribute__((aligned(16))) float meet[WG > 1 ? WG * (GL < kWave ? GL : kWave * WPR) * V : 1];
  const int t = threadIdx.x % GL, wave = threadIdx.x / kWave;
  // a row of whole waves: its number, and with it every row address, in scalar registers
  const int grp = GL >= kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / GL) : threadIdx.x / GL;
  auto col = [&](int k, int j) { return VEC ? (k * GL + t) * V + j : (k * V + j) * GL + t; };
  // Row data and weights as loaded.  `keep` hides them from the compiler between uses: it would otherwise carry the widened
  // fp32 values from one use to the next (and the weights' from row to row) and spill 60 - 150 registers.
  using Raw = LbRaw<T, V>;
  using WRaw = LbRaw<Wt, V>;
  WRaw gamma[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    VecN<Wt, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.v[j] = w && col(k, j) < N ? w[col(k, j)] : static_cast<Wt>(1.f);
    gamma[k].set(v);
  }
  struct Row {
    Raw x[NV], dy[NV];
    float mean, rstd;
  };
  // No branches: lanes past the row and rows past the last read the nearest element that is there; one_row puts zeros in
  // its place (with a branch per slab the compiler kept both sides of each in registers and spilled 100 of them).
  auto fetch = [&](int64_t row, Row& r) {
    const int64_t rc = row < M ? row : M - 1;
    r.mean = mean[rc];
    r.rstd = rstd[rc];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      VecN<T, V> xv, dv;
      if constexpr (VEC) {  // N % V == 0: a vector is inside the row or past it
        const int c = col(k, 0) < N ? col(k, 0) : N - V;
        xv = ld_nt<T, V>(x + rc * N + c);
        dv = ld_nt<T, V>(dy + rc * N + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = col(k, j) < N ? col(k, j) : N - 1;
          xv.v[j] = x[rc * N + c];
          dv.v[j] = dy[rc * N + c];
        }
      }
      r.x[k].set(xv);
      r.dy[k].set(dv);
    }
  };
  float dw[NV][V] = {}, db[NV][V] = {};
  const float inv_n = 1.f / (float)N;
  int parity = 0;
  auto one_row = [&](int64_t row, Row& r) {
    // Columns past the row and rows past the last become zeros: they add nothing to any sum.
    const bool live = row < M;
    if (!live) r.mean = r.rstd = 0.f;
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (VEC) {
        r.x[k].clear_unless(live && col(k, 0) < N);
        r.dy[k].clear_unless(live && col(k, 0) < N);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          r.x[k].clear_unless(live && col(k, j) < N, j);
          r.dy[k].clear_unless(live && col(k, j) < N, j);
        }
      }
      gamma[k].keep();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (2 * j == V) __builtin_amdgcn_sched_barrier(0);  // half a slab's temporaries at a time
        const float d = r.dy[k].get(j), xhat = (r.x[k].get(j) - r.mean) * r.rstd;
        const float g = d * gamma[k].get(j);
        s.x += g;
        s.y += g * xhat;
        dw[k][j] += d * xhat;
        db[k][j] += d;
      }
      r.x[k].keep();
      r.dy[k].keep();
      __builtin_amdgcn_sched_barrier(0);
    }
    if (dx == nullptr) return;
    if constexpr (GL < kWave) {
      s.x = sub_allreduce<GL>(s.x, SumOp());
      s.y = sub_allreduce<GL>(s.y, SumOp());
    } else {
      s.x = wave_allreduce(s.x, SumOp());
      s.y = wave_allreduce(s.y, SumOp());
    }
    if constexpr (WPR > 1) {
      if (threadIdx.x % kWave == 0) red[parity][wave] = s;
      __syncthreads();  // (the slots of the row before last are free: every wave has passed the last row's barrier)
      s = red[parity][wave / WPR * WPR + threadIdx.x % WPR];
      s.x = sub_allreduce<WPR>(s.x, SumOp());
      s.y = sub_allreduce<WPR>(s.y, SumOp());
      parity ^= 1;
    }
    if (!live) return;
    const float m1 = s.x * inv_n, m2 = s.y * inv_n;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      VecN<T, V> o;
      gamma[k].keep();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (2 * j == V) __builtin_amdgcn_sched_barrier(0);
        const float xhat = (r.x[k].get(j) - r.mean) * r.rstd;
        o.v[j] = static_cast<T>(r.rstd * (r.dy[k].get(j) * gamma[k].get(j) - m1 - xhat * m2));
        if constexpr (!VEC)
          if (col(k, j) < N) dx[row * N + col(k, j)] = o.v[j];
      }
      if constexpr (VEC)
        if (col(k, 0) < N) st_nt<T, V>(dx + row * N + col(k, 0), o);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t base = (int64_t)blockIdx.x * G;  // uniform over the block: every thread meets every barrier
  if constexpr (AHEAD) {
    Row a, b;
    fetch(base + grp, a);
    while (base < M) {  // two rows per trip, the two register sets trading places
      fetch(base + step + grp, b);
      one_row(base + grp, a);
      base += step;
      if (base >= M) break;
      fetch(base + step + grp, a);
      one_row(base + grp, b);
      base += step;
    }
  } else {
    for (; base < M; base += step) {
      Row a;
      fetch(base + grp, a);
      one_row(base + grp, a);
    }
  }
  if (partial == nullptr && dw_out == nullptr && db_out == nullptr) return;
  // This block's dw, then its db, V x GL columns at a time: the row groups' values meet in LDS (groups smaller than a wave
  // first by exchanges inside it) and leave as one partial, or as the result when this is the only block.
  constexpr int COLS = GL * V;
  auto leave = [&](float (&acc)[NV][V], float* part, Wt* out) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      auto put = [&](int c, float v) {
        if (c >= N) return;
        if (partial != nullptr) part[c] = v;
        else if (out != nullptr) out[c] = static_cast<Wt>(v);
      };
      if constexpr (WG == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) put(col(k, j), acc[k][j]);
      } else {
        __syncthreads();  // the buffer's last values have been read
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float v = acc[k][j];
#pragma unroll
          for (int d = GL; d < kWave; d *= 2) v += __shfl_xor(v, d, kWave);
          if (GL >= kWave || threadIdx.x % kWave < GL) meet[(GL >= kWave ? grp : wave) * COLS + (VEC ? t * V + j : j * GL + t)] = v;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < COLS; c += kLbTile) {
          float v = 0.f;
#pragma unroll
          for (int g = 0; g < WG; ++g) v += meet[g * COLS + c];
          put(k * COLS + c, v);
        }
      }
    }
  };
  float* part = partial + (int64_t)blockIdx.x * 2 * N;
  leave(dw, part, dw_out);
  leave(db, part + N, db_out);
}

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

// dw and db from `groups` partials of [dw | db]: 16 x 16 threads, 4 neighbouring columns and every 16th partial each.
template <typename Wt, typename S>
__global__ __launch_bounds__(kLbBlock) void lb_finish_kernel(const S* __restrict__ partial, Wt* __restrict__ dw, Wt* __restrict__ db,
                                                            int64_t N, int groups) {
  __shared__ S part[16][64];
  const int q = threadIdx.x / 16, l = threadIdx.x % 16;
  const int64_t c0 = (int64_t)blockIdx.x * 64 + 4 * l;  // of the 2N columns [dw | db]
  S s[4] = {};
  if (N % 2 == 0) {  // every group of four columns starts on a 16-byte boundary (of fp32) and is inside or outside as a whole
    if (c0 < 2 * N) {
#pragma unroll 8
      for (int g = q; g < groups; g += 16) {
        const VecN<S, 4> v = ld<S, 4>(partial + (int64_t)g * 2 * N + c0);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += v.v[j];
      }
    }
  } else {
#pragma unroll 4
    for (int g = q; g < groups; g += 16)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + j < 2 * N) s[j] += partial[(int64_t)g * 2 * N + c0 + j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[q][4 * l + j] = s[j];
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x >= 64 || c >= 2 * N) return;
  S sum = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += part[i][threadIdx.x];
  Wt* out = c < N ? dw : db;
  if (out) out[c < N ? c : c - N] = static_cast<Wt>(sum);
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

// Lanes per row and slabs per lane of the tile kernel; lanes == 0: the general path.  Two-byte rows take at most two slabs
// of 8 elements per lane, fp32 rows two of 4, or four without the row ahead beyond 8 K elements.
struct LbTile {
  int lanes, slabs;
};
template <typename T> static LbTile lb_tile(int64_t N) {
  constexpr int V = 16 / sizeof(T);
  if (sizeof(T) == 8) return LbTile{0, 0};
  for (int lanes = 8; lanes <= kLbTile; lanes *= 2) {
    if (N <= (int64_t)lanes * V) return LbTile{lanes, 1};
    if (lanes >= kWave && N <= (int64_t)lanes * V * 2) return LbTile{lanes, 2};
  }
  if (sizeof(T) == 4 && N <= (int64_t)kLbTile * V * 4) return LbTile{kLbTile, 4};
  return LbTile{0, 0};
}
static int64_t lb_tile_blocks(int64_t M, const LbTile& p) {
  const int64_t rows = kLbTile / p.lanes;  // per block and trip
  const int64_t need = (M + rows - 1) / rows;
  return need < kLbTileBlocks ? need : kLbTileBlocks;
}

template <typename T, typename Wt>
static bool run_lb_tile(const T* dy, const T* x, const float* mean, const float* rstd, const Wt* w, T* dx, Wt* dw, Wt* db, int64_t M,
                        int64_t N, float* ws, hipStream_t st) {
  const LbTile p = lb_tile<T>(N);
  if (p.lanes == 0) return false;
  const int64_t blocks = lb_tile_blocks(M, p);
  const bool params = dw != nullptr || db != nullptr;
  float* partial = params && blocks > 1 ? ws : nullptr;
  const bool vec = N % Vec<T>::N == 0 && aligned16(dy) && aligned16(x) && aligned16(dx);
  auto go = [&](auto gl, auto nv) {
    constexpr int GL = decltype(gl)::value, NV = decltype(nv)::value;
    if (vec) hipLaunchKernelGGL((lb_tile_kernel<T, Wt, GL, NV, true, (NV <= 2)>), dim3((unsigned)blocks), dim3(kLbTile), 0, st, dy, x, mean, rstd, w, dx, partial, dw, db, M, (int)N);
    else hipLaunchKernelGGL((lb_tile_kernel<T, Wt, GL, NV, false, false>), dim3((unsigned)blocks), dim3(kLbTile), 0, st, dy, x, mean, rstd, w, dx, partial, dw, db, M, (int)N);
  };
  using std::integral_constant;
#define MI355_LB_TILE(GL_, NV_) \
  if (p.lanes == GL_ && p.slabs == NV_) go(integral_constant<int, GL_>(), integral_constant<int, NV_>());
  MI355_LB_TILE(8, 1) MI355_LB_TILE(16, 1) MI355_LB_TILE(32, 1)
  MI355_LB_TILE(64, 1) MI355_LB_TILE(128, 1) MI355_LB_TILE(256, 1) MI355_LB_TILE(512, 1) MI355_LB_TILE(1024, 1)
  MI355_LB_TILE(64, 2) MI355_LB_TILE(128, 2) MI355_LB_TILE(256, 2) MI355_LB_TILE(512, 2) MI355_LB_TILE(1024, 2)
  if constexpr (sizeof(T) == 4) MI355_LB_TILE(1024, 4)
#undef MI355_LB_TILE
  if (partial)
    hipLaunchKernelGGL((lb_finish_kernel<Wt, float>), dim3((unsigned)((2 * N + 63) / 64)), dim3(kLbBlock), 0, st, partial, dw, db, N, (int)blocks);
  return true;
}

template <typename T, typename Wt, typename S>
static int run_lb(const void* dyv, const void* xv, const void* mv, const void* rv, const void* wv, void* dxv, void* dwv, void* dbv,
                  int64_t M, int64_t N, void* ws, hipStream_t st) {
  const T *dy = static_cast<const T*>(dyv), *x = static_cast<const T*>(xv);
  const S *mean = static_cast<const S*>(mv), *rstd = static_cast<const S*>(rv);
  const Wt* w = static_cast<const Wt*>(wv);
  if constexpr (!std::is_same<T, double>::value) {
    if (run_lb_tile<T, Wt>(dy, x, mean, rstd, w, static_cast<T*>(dxv), static_cast<Wt*>(dwv), static_cast<Wt*>(dbv), M, N, static_cast<float*>(ws), st))
      return check_launch("mi355_layer_norm_backward");
  }
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
  const LbTile p = dtype == MI355_F32 ? lb_tile<float>(N) : dtype == MI355_F64 ? lb_tile<double>(N) : lb_tile<bf16_t>(N);
  if (p.lanes != 0) return lb_tile_blocks(M, p) * 2 * N * 4;
  return (2 * M + lb_plan(M, N).groups * 2 * N) * (dtype == MI355_F64 ? 8 : 4);
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
