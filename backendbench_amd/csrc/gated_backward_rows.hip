// The gated projection, backward, for few rows: dW = dpre^T x is a sum of M outer products and dx = dpre W a sum of 2F weighted
// rows, so both are bound by the weight's way in and its gradient's way out (2 F K elements each), and one pass does both:
// a weight row is loaded for dx while the same row of dW is computed and stored.  Nothing is copied or transposed and any
// strides and alignment are taken.  One row and 16, us (TB/s): 2 * 11008 x 4096 bf16 80 (4.5) and 104 (3.5), fp32 153 (4.7)
// and 171 (4.2).  From eight rows on the vector units bound it, below that what two waves per SIMD have in flight.
#include "gated.h"

namespace mi355 {

constexpr int kGbrWaves = 4;     // per workgroup, each with its own work
// Features of a step: their gate and up rows are all requested before the first is used (in 64 bits fewer fit the registers).
constexpr int gbr_features(int size) { return size == 8 ? 4 : 8; }

// The value another lane holds, as a scalar.
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ float lane_value(float v, int lane) { return __builtin_bit_cast(float, lane_value(__builtin_bit_cast(uint32_t, v), lane)); }
__device__ __forceinline__ double lane_value(double v, int lane) {
  int2 p = __builtin_bit_cast(int2, v);
  p.x = __builtin_amdgcn_readlane(p.x, lane);
  p.y = __builtin_amdgcn_readlane(p.y, lane);
  return __builtin_bit_cast(double, p);
}

// V elements as loaded, in whole registers (the compiler keeps every element of a 16-bit array in one of its own).
template <typename T, int V> struct Words {
  static constexpr int R = sizeof(T) * V / 4;
  uint32_t r[R];
  __device__ __forceinline__ void load(const T* p) {  // at any element's address
    const auto v = *reinterpret_cast<const typename AnyPart<sizeof(T) * V, sizeof(T)>::type*>(p);
#pragma unroll
    for (int i = 0; i < R; ++i) r[i] = v[i];
  }
  __device__ __forceinline__ typename OpMath<T>::type get(int j) const {
    if constexpr (sizeof(T) == 8) return __builtin_bit_cast(double, (uint64_t)r[2 * j] | (uint64_t)r[2 * j + 1] << 32);
    else return __builtin_bit_cast(float, r[j]);
  }
};

// 16-bit types: (element j of a, element j of b) in one register, and c + a.lo b.lo + a.hi b.hi with the products and the sum
// in fp32 (subnormal factors count; 2 2^-24 of the terms, measured).
template <typename T, int V> __device__ __forceinline__ uint32_t both(const Words<T, V>& a, const Words<T, V>& b, int j) {
  return __builtin_amdgcn_perm(b.r[j >> 1], a.r[j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
}
typedef __bf16 gbr_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 gbr_f16x2 __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(gbr_bf16x2, a), __builtin_bit_cast(gbr_bf16x2, b), c, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(gbr_f16x2, a), __builtin_bit_cast(gbr_f16x2, b), c, false);
}
template <typename T> __device__ __forceinline__ uint32_t bits16(float v) { return __builtin_bit_cast(uint16_t, static_cast<T>(v)); }

// A wave has a strip of 64 V columns and the features [c0, c1) of its group, N at a time.  Lane m N + i (then the next register's
// lanes) computes dpre of row m, feature i of the step, which the whole wave then takes from there as a scalar.
// x of the strip, MT rows, and its dx sums stay in registers.  partial [group][ld]: the sums [M][K]; one group: dx itself.
template <typename T, int MT, int V, bool DX, bool DW>
__global__ __launch_bounds__(64 * kGbrWaves, 2) void gated_backward_rows_kernel(GatedBackwardArgs g, typename OpMath<T>::type* __restrict__ partial,
                                                                               int64_t ld, int strips, int64_t per_group, int64_t items) {
  using A = typename OpMath<T>::type;
  constexpr int N = gbr_features(sizeof(T)), R = (MT * N + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t item = (int64_t)blockIdx.x * kGbrWaves + wave;
  if (item >= items) return;
  const int64_t group = item / strips, own = (item % strips) * (kWave * V) + lane * V;
  // A lane whose columns would stick out of the row moves back to end with it and computes what its neighbour does.
  const int64_t col = own + V <= g.K ? own : g.K - V;
  const bool stores = own < g.K;
  const T *X = static_cast<const T*>(g.x), *W = static_cast<const T*>(g.w), *P = static_cast<const T*>(g.pre), *H = static_cast<const T*>(g.dh);
  constexpr bool HALF = sizeof(T) == 2;
  Words<T, V> x[DW ? MT : 1] = {};  // (rows past M: zeros)
  uint32_t x2[DW && HALF ? MT / 2 : 1][V];  // rows 2 m and 2 m + 1, column by column
  if constexpr (DW) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < g.M) x[m].load(X + m * g.x_rs + col);
  }
  if constexpr (DW && HALF) {
#pragma unroll
    for (int m = 0; m < MT; m += 2)
#pragma unroll
      for (int j = 0; j < V; ++j) x2[m / 2][j] = both(x[m], x[m + 1], j);
  }
  A dx[DX ? MT : 1][V] = {};
  const int64_t c0 = group * per_group, c1 = c0 + per_group < g.F ? c0 + per_group : g.F;
  for (int64_t f0 = c0; f0 < c1; f0 += N) {
    Words<T, V> w[DX ? 2 * N : 1];
    A gate[R], up[R], dh[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t m = (r * kWave + lane) / N, f = f0 + lane % N;
      const int64_t mc = m < g.M ? m : g.M - 1, fc = f < c1 ? f : c1 - 1;
      gate[r] = static_cast<A>(P[mc * 2 * g.F + fc]);
      up[r] = static_cast<A>(P[mc * 2 * g.F + g.F + fc]);
      dh[r] = static_cast<A>(H[mc * g.F + fc]);
    }
    if constexpr (DX) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t f = f0 + i < c1 ? f0 + i : c1 - 1;
        w[2 * i].load(W + f * g.w_rs + col);
        w[2 * i + 1].load(W + (g.F + f) * g.w_rs + col);
      }
    }
    // dpre.  In 16 bits the pair (gate's, up's) rounded to the type, as the matrix instructions of more rows have to take it: one
    // definition whatever the number of rows (in f16 with its range: infinite beyond 65504), and two terms to an operation, a third
    // of the operations.
    A dgate[R], dup[R];
    uint32_t d2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if ((r * kWave + lane) / N >= g.M) gate[r] = up[r] = dh[r] = A(0);  // rows past M add nothing (0 * inf)
      auto gradients = [&](auto ACT_) __attribute__((always_inline)) {
        const A q = gate_q<decltype(ACT_)::value, GateMath<T>>(gate[r]);
        dgate[r] = dh[r] * up[r] * gate_grad<decltype(ACT_)::value, GateMath<T>>(gate[r], q);
        dup[r] = dh[r] * (gate[r] * q);
      };
      if (g.act == MI355_SILU) gradients(std::integral_constant<int, MI355_SILU>{});
      else if (g.act == MI355_GELU) gradients(std::integral_constant<int, MI355_GELU>{});
      else gradients(std::integral_constant<int, MI355_GELU_TANH>{});
      if constexpr (HALF) d2[r] = bits16<T>(dgate[r]) | bits16<T>(dup[r]) << 16;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (f0 + i >= c1) break;
      __builtin_amdgcn_sched_barrier(0);  // not two features at once: their temporaries would be spilled
      A og[V] = {}, ou[V] = {};
      if constexpr (HALF) {
        uint32_t w2[DX ? V : 1];
        if constexpr (DX) {
#pragma unroll
          for (int j = 0; j < V; ++j) w2[j] = both(w[2 * i], w[2 * i + 1], j);
        }
#pragma unroll
        for (int m = 0; m < MT; m += 2) {
          const uint32_t a = lane_value(d2[m * N / kWave], m * N % kWave + i), b = lane_value(d2[(m + 1) * N / kWave], (m + 1) * N % kWave + i);
          const uint32_t gates = (a & 0xffffu) | b << 16, ups = a >> 16 | (b & 0xffff0000u);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if constexpr (DX) {
              dx[m][j] = dot2<T>(w2[j], a, dx[m][j]);
              dx[m + 1][j] = dot2<T>(w2[j], b, dx[m + 1][j]);
            }
            if constexpr (DW) {
              og[j] = dot2<T>(x2[m / 2][j], gates, og[j]);
              ou[j] = dot2<T>(x2[m / 2][j], ups, ou[j]);
            }
          }
        }
      } else {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const A a = lane_value(dgate[m * N / kWave], m * N % kWave + i), b = lane_value(dup[m * N / kWave], m * N % kWave + i);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if constexpr (DX) dx[m][j] += a * w[2 * i].get(j) + b * w[2 * i + 1].get(j);
            if constexpr (DW) {
              og[j] += a * x[m].get(j);
              ou[j] += b * x[m].get(j);
            }
          }
        }
      }
      if (DW && stores) {
        VecN<T, V> vg, vu;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          vg.v[j] = static_cast<T>(og[j]);
          vu.v[j] = static_cast<T>(ou[j]);
        }
        T* out = static_cast<T*>(g.dw) + (f0 + i) * g.K + col;
        store_any(out, vg);
        store_any(out + g.F * g.K, vu);
      }
    }
  }
  if (DX && stores) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= g.M) break;
      if (partial != nullptr) {
        A* p = partial + group * ld + m * g.K + col;
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = dx[m][j];
      } else {
        VecN<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = static_cast<T>(dx[m][j]);
        store_any(static_cast<T*>(g.dx) + m * g.K + col, o);
      }
    }
  }
}

// dx [n] = the groups' sums, in a fixed order: 32 neighbouring elements per block, 8 lanes of 4 by 32 threads that take
// every 32nd group; they meet by exchanges inside a wave and in LDS.
template <typename T, typename A>
__global__ __launch_bounds__(256) void gated_backward_join_kernel(const A* __restrict__ partial, T* __restrict__ dx, int64_t n, int64_t ld, int groups) {
  __shared__ A part[4][32];
  const int q = threadIdx.x / 8, l = threadIdx.x % 8;
  const int64_t e0 = (int64_t)blockIdx.x * 32 + 4 * l;
  A s[4] = {};
  if (e0 < ld) {
#pragma unroll 4
    for (int g = q; g < groups; g += 32) {
      const VecN<A, 4> v = *reinterpret_cast<const VecN<A, 4>*>(partial + (int64_t)g * ld + e0);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += v.v[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int d = 8; d < kWave; d *= 2) s[j] += __shfl_xor(s[j], d, kWave);
    if (threadIdx.x % kWave < 8) part[threadIdx.x / kWave][4 * l + j] = s[j];
  }
  __syncthreads();
  const int64_t e = (int64_t)blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x >= 32 || e >= n) return;
  dx[e] = static_cast<T>((part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]));
}

struct GbrPlan {
  int v, strips;
  int64_t per_group, groups, ld;  // features of a group, a multiple of a step; elements of a partial dx
};
// Columns per lane: 16 bytes, 8 in two-byte types with more than eight rows (x and the sums of 16 take twice the registers).
// Two waves per SIMD: more groups add partial sums, M K of them each (eight rows, 2 * 11008 x 4096 bf16: 8, 12 and 16 waves
// per CU take 89, 91 and 98 us; 2 * 5001 x 5001 fp32 99, 108 and 111).
static GbrPlan gbr_plan(int64_t M, int64_t F, int64_t K, int dtype) {
  GbrPlan p;
  const int size = dtype_size(dtype);
  p.v = size == 2 && M > 8 ? 4 : 16 / size;
  p.strips = (int)((K + kWave * p.v - 1) / (kWave * p.v));
  const int64_t step = gbr_features(size), steps = (F + step - 1) / step, want = 8 * kNumCU / p.strips;
  const int64_t groups = want < 1 ? 1 : want < steps ? want : steps;
  p.per_group = (steps + groups - 1) / groups * step;
  p.groups = (F + p.per_group - 1) / p.per_group;
  p.ld = (M * K + 3) / 4 * 4;
  return p;
}

// Against the products (dpre kernel, copies, two products), us: 16 rows bf16 104 / 115 at 2 * 11008 x 4096, 40 / 40 at
// 2 * 5504 x 2048, 77 / 127 at 2 * 5001 x 5001, 11 / 19 at 2 * 290 x 342; fp32 171 / 267, 59 / 88, 114 / 333 and 13 / 20.
bool gated_backward_rows_takes(int64_t M, int64_t K) { return M <= 16 && K >= 8; }  // (K: a lane's columns are there)

int64_t gated_backward_rows_workspace(int64_t M, int64_t F, int64_t K, int dtype) {
  const GbrPlan p = gbr_plan(M, F, K, dtype);
  return (p.groups * p.ld * (dtype == MI355_F64 ? 8 : 4) + 255) / 256 * 256;
}

template <typename T> static int run_gated_backward_rows(const GatedBackwardArgs& a, void* workspace, hipStream_t st) {
  using A = typename OpMath<T>::type;
  const GbrPlan p = gbr_plan(a.M, a.F, a.K, a.dtype);
  const int64_t items = p.groups * p.strips;
  A* partial = a.dx != nullptr && p.groups > 1 ? static_cast<A*>(workspace) : nullptr;
  auto launch = [&](auto mt, auto v, auto dx, auto dw) {
    hipLaunchKernelGGL((gated_backward_rows_kernel<T, decltype(mt)::value, decltype(v)::value, decltype(dx)::value, decltype(dw)::value>),
                       dim3((unsigned)((items + kGbrWaves - 1) / kGbrWaves)), dim3(64 * kGbrWaves), 0, st, a, partial, p.ld, p.strips,
                       p.per_group, items);
  };
  auto go = [&](auto mt, auto v) {
    using std::false_type;
    using std::true_type;
    if (a.dx != nullptr && a.dw != nullptr) launch(mt, v, true_type(), true_type());
    else if (a.dx != nullptr) launch(mt, v, true_type(), false_type());
    else launch(mt, v, false_type(), true_type());
  };
  constexpr int V = 16 / sizeof(T);
  if constexpr (sizeof(T) == 2) {
    if (a.M <= 4) {
      go(std::integral_constant<int, 4>(), std::integral_constant<int, V>());
    } else if (a.M <= 8) go(std::integral_constant<int, 8>(), std::integral_constant<int, V>());
    else go(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
  } else if (a.M <= 8) go(std::integral_constant<int, 8>(), std::integral_constant<int, V>());
  else go(std::integral_constant<int, 16>(), std::integral_constant<int, V>());
  if (partial != nullptr)
    hipLaunchKernelGGL((gated_backward_join_kernel<T, A>), dim3((unsigned)((p.ld + 31) / 32)), dim3(256), 0, st, partial, static_cast<T*>(a.dx),
                       a.M * a.K, p.ld, (int)p.groups);
  return check_launch("mi355_gated_linear_backward");
}

int launch_gated_backward_rows(const GatedBackwardArgs& a, void* workspace, hipStream_t st) {
  switch (a.dtype) {
    case MI355_F32: return run_gated_backward_rows<float>(a, workspace, st);
    case MI355_F64: return run_gated_backward_rows<double>(a, workspace, st);
    case MI355_F16: return run_gated_backward_rows<f16_t>(a, workspace, st);
    default: return run_gated_backward_rows<bf16_t>(a, workspace, st);
  }
}

}  // namespace mi355
