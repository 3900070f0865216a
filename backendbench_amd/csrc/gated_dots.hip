// The gated projection for a handful of rows on the vector units: any float type, any strides and alignment.  The weight is
// read once and its stream is the bound (2 F K elements); with so few rows no matrix instruction is needed to keep up, and
// a wave can read 1 KB of one row at a time, at any address, where a fragment of a matrix instruction takes 64 bytes of
// each of 16 rows.  Measured, us (TB/s of the weight): one row, 2 * 5001 x 5001 bf16 22 (4.6; 55
// through copies in aligned rows), 2 * 11008 x 4096 fp32 58 (6.2; 145 as a product and an activation kernel), bf16 31 (5.9;
// 30 through LDS).
#include "gated.h"

namespace mi355 {

constexpr int kGdWaves = 4;  // per workgroup

// A wave has two features, their gate and up rows: of 64 V elements of K at a time, lane l takes the V from l V on, with
// the next step's loads in flight while it computes.  MT rows of x (fewer tokens: the last again, not stored).  WK waves share a pair of
// features, taking turns along K; a lane's sums are added over the wave, then over the WK waves, in a fixed order.
template <typename T, int MT, int WK>
__global__ __launch_bounds__(64 * kGdWaves) void gated_dots_kernel(GatedArgs g) {
  using A = typename OpMath<T>::type;
  constexpr int V = 16 / sizeof(T), STEP = kWave * V, PAIRS = kGdWaves / WK;
  using Any = typename AnyVec<sizeof(T)>::type;
  __shared__ A meet[kGdWaves][4][MT];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t f0 = ((int64_t)blockIdx.x * PAIRS + wave / WK) * 2;
  const T* w[4];  // rows gate, up of feature f0, gate, up of f0 + 1 (past the last feature: the last one's, not stored)
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t f = f0 + r / 2 < g.F ? f0 + r / 2 : g.F - 1;
    w[r] = static_cast<const T*>(g.w) + ((r & 1) ? g.F + f : f) * g.w_rs;
  }
  const T* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = static_cast<const T*>(g.x) + (m < g.M ? m : g.M - 1) * g.x_rs;
  A acc[4][MT] = {};
  struct Step {
    VecN<T, V> w[4], x[MT];
  };
  auto fetch = [&](int64_t k, Step& s) __attribute__((always_inline)) {
    const int64_t c = k + lane * V;
#pragma unroll
    for (int r = 0; r < 4; ++r) s.w[r] = __builtin_bit_cast(VecN<T, V>, __builtin_nontemporal_load(reinterpret_cast<const Any*>(w[r] + c)));
#pragma unroll
    for (int m = 0; m < MT; ++m) s.x[m] = __builtin_bit_cast(VecN<T, V>, *reinterpret_cast<const Any*>(x[m] + c));
  };
  auto multiply = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r][m] = __builtin_fma(static_cast<A>(s.w[r].v[j]), static_cast<A>(s.x[m].v[j]), acc[r][m]);
  };
  const int64_t whole = g.K / STEP * STEP;  // whole steps
  constexpr int64_t ROUND = (int64_t)STEP * WK;
  int64_t k = (int64_t)(wave % WK) * STEP;
  if (k < whole) {
    Step a, b;
    fetch(k, a);
    while (true) {  // two steps per trip, the two register sets trading places
      const int64_t kb = k + ROUND;
      if (kb < whole) fetch(kb, b);
      multiply(a);
      if (kb >= whole) {
        k = kb;
        break;
      }
      k = kb + ROUND;
      if (k < whole) fetch(k, a);
      multiply(b);
      if (k >= whole) break;
    }
  }
  if (k == whole && whole < g.K) {  // what is left of K, zeros behind its end in both operands (0 * inf): the wave whose turn it is
    Step s;
    const int64_t c = k + lane * V;
    if (g.K >= V) {
      u32x4 we[4], xe[MT];
#pragma unroll
      for (int r = 0; r < 4; ++r) we[r] = load_within(w[r], c, g.K);
#pragma unroll
      for (int m = 0; m < MT; ++m) xe[m] = load_within(x[m], c, g.K);
#pragma unroll
      for (int r = 0; r < 4; ++r) s.w[r] = __builtin_bit_cast(VecN<T, V>, placed<T>(we[r], c, g.K));
#pragma unroll
      for (int m = 0; m < MT; ++m) s.x[m] = __builtin_bit_cast(VecN<T, V>, placed<T>(xe[m], c, g.K));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) s.w[r] = load_short(w[r], c, g.K);
#pragma unroll
      for (int m = 0; m < MT; ++m) s.x[m] = load_short(x[m], c, g.K);
    }
    multiply(s);
  }
  // The 4 MT sums over the lanes: halves of the wave trade halves of the list until a lane holds one of them (4 MT - 1
  // exchanges instead of 6 * 4 MT), then what is left of the lanes is added up.
  constexpr int R = 4 * MT;
  A* v = &acc[0][0];
#pragma unroll
  for (int n = R / 2; n > 0; n /= 2) {
    const int d = kWave / 2 * n / (R / 2);
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const A keep = upper ? v[i + n] : v[i], send = upper ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor(send, d, kWave);
    }
  }
#pragma unroll
  for (int d = kWave / R / 2; d > 0; d /= 2) v[0] += __shfl_xor(v[0], d, kWave);
  if (lane % (kWave / R) == 0) (&meet[wave][0][0])[lane / (kWave / R)] = v[0];
  __syncthreads();
  // One feature of one token per thread.
  const int t = threadIdx.x;
  if (t >= PAIRS * 2 * MT) return;
  const int pair = t / (2 * MT), i = t / MT % 2, m = t % MT;
  const int64_t f = ((int64_t)blockIdx.x * PAIRS + pair) * 2 + i;
  if (f >= g.F || m >= g.M) return;
  A gv = meet[pair * WK][2 * i][m], uv = meet[pair * WK][2 * i + 1][m];
#pragma unroll
  for (int q = 1; q < WK; ++q) {
    gv += meet[pair * WK + q][2 * i][m];
    uv += meet[pair * WK + q][2 * i + 1][m];
  }
  A q = A(0);
  if (g.act == MI355_SILU) q = gate_q<MI355_SILU, GateMath<T>>(gv);
  else if (g.act == MI355_GELU) q = gate_q<MI355_GELU, GateMath<T>>(gv);
  else q = gate_q<MI355_GELU_TANH, GateMath<T>>(gv);
  static_cast<T*>(g.h)[m * g.F + f] = static_cast<T>(gv * q * uv);
  if (g.pre != nullptr) {
    T* pre = static_cast<T*>(g.pre) + 2 * m * g.F + f;
    pre[0] = static_cast<T>(gv);
    pre[g.F] = static_cast<T>(uv);
  }
}

template <typename T> static int run_gated_dots(const GatedArgs& a, hipStream_t st) {
  const int64_t pairs = (a.F + 1) / 2;
  auto launch = [&](auto mt, auto wk) {
    constexpr int MT = decltype(mt)::value, WK = decltype(wk)::value, PAIRS = kGdWaves / WK;
    hipLaunchKernelGGL((gated_dots_kernel<T, MT, WK>), dim3((unsigned)((pairs + PAIRS - 1) / PAIRS)), dim3(64 * kGdWaves), 0, st, a);
    return check_launch("mi355_gated_linear");
  };
  auto go = [&](auto mt) {
    using std::integral_constant;
    // Four waves to a pair of features from three steps of K on, one where K is over before the four are busy.  One wave against
    // four, us, one row: 2 * 11008 x 4096 bf16 33.5 / 30.6, fp32 64 / 61; 2 * 5001 x 5001 bf16 25 / 23.6, fp32 42 / 36.5;
    // 2 * 4096 x 1024 bf16 5.9 / 5.8; 2 * 20000 x 64 bf16 9 / 15; four rows: 2 * 1376 x 8192 bf16 23 / 18, 2 * 4096 x 1024 8.6 / 10.
    return a.K > 2 * kWave * (16 / (int64_t)sizeof(T)) ? launch(mt, integral_constant<int, kGdWaves>()) : launch(mt, integral_constant<int, 1>());
  };
  if (a.M == 1) return go(std::integral_constant<int, 1>());
  if (a.M == 2) return go(std::integral_constant<int, 2>());
  if constexpr (sizeof(T) > 2) {
    if (a.M <= 4) return go(std::integral_constant<int, 4>());
  }
  if constexpr (sizeof(T) > 4) {
    if (a.M <= 8) return go(std::integral_constant<int, 8>());
  }
  return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_linear: no vector kernel for %lld rows of %s", (long long)a.M, dtype_name(a.dtype));
}

// More rows make the vector units the bound.  Against the matrix instructions, us: 2 * 5001 x 5001 bf16 1, 2 and 3 rows 22 / 30,
// 28 / 39 and 38 / 32; 2 * 11008 x 4096 fp32 2, 4 and 8 rows 58 / 80, 71 / 76 and 108 / 75, 2 * 1376 x 8192 18 / 35, 21 / 33 and
// 32 / 33.  (fp64 has no other fused form.)  Fewer than 2^32 threads.
bool gated_dots_takes(const GatedArgs& a) {
  const int size = dtype_size(a.dtype);
  return size >= 2 && a.M <= size && a.F < (1 << 27) && a.K > 0;
}

int launch_gated_dots(const GatedArgs& a, hipStream_t st) {
  switch (a.dtype) {
    case MI355_F32: return run_gated_dots<float>(a, st);
    case MI355_F64: return run_gated_dots<double>(a, st);
    case MI355_F16: return run_gated_dots<f16_t>(a, st);
    case MI355_BF16: return run_gated_dots<bf16_t>(a, st);
    default: return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_linear: unsupported dtype %s", dtype_name(a.dtype));
  }
}

}  // namespace mi355
