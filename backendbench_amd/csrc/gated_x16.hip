// The gated projection h = act(x Wg^T) * (x Wu^T) in one kernel on the 256x256 tile of gemm_x16.h: 256 rows by 128
// features, gate and up products side by side in the accumulators, activation and product in the epilogue; bf16 / f16,
// K % 128 == 0, K >= 256.  What it saves against a product and an activation kernel is the 2F-wide result's way out and
// back (fp32: 16 bytes of traffic per feature).
#include "gated.h"
#include "gemm_x16.h"

namespace mi355 {

// Epilogue of a wave: 128 rows by 64 features, gate in acc[i][0 .. 3], up in acc[i][4 .. 7]; through a slab of the idle
// ring (128-byte rows, 16-byte slot s of row r at s ^ ((r / 2) % 8)) and out in whole 128-byte rows.
struct GatedStore {
  void* h;    // [M][F]
  void* pre;  // [M][2F] or null: gate and up, rounded, for the backward pass
  int act, vec;  // vec: rows of h and pre start on 16-byte boundaries

  template <typename T>
  __device__ __forceinline__ void store(const GemmArgs& g, f32x4 (&acc)[8][8], unsigned char* lds, int wave, int lane, int m0, int f0) const {
    const int lr = lane & 15, lg = lane >> 4;
    unsigned char* slab = lds + wave * (128 * 128);
    // Several paths read the accumulators: pinned here, behind the caller's wait states, so that no copy is made earlier.
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("" : "+a"(acc[i][j]));
    auto rows_out = [&](auto value, T* D, int64_t ld) __attribute__((always_inline)) {
      unsigned char* wr = slab + lr * 128 + (lg & 1) * 8;
      const int sx = (lr >> 1) & 7;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          VecN4<T> r;
#pragma unroll
          for (int e = 0; e < 4; ++e) r.v[e] = static_cast<T>(value(i, p, e));
          *reinterpret_cast<VecN4<T>*>(wr + i * (16 * 128) + (((p * 2 + (lg >> 1)) ^ sx) << 4)) = r;
        }
      // same wave wrote and reads: LDS operations of a wave complete in order
      if (vec) {
        const int s = lane & 7, r0 = lane >> 3;
        T* dst = D + (int64_t)(m0 + r0) * ld + f0 + s * 8;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const int row = r0 + 8 * t;
          const u32x4 v = *reinterpret_cast<const u32x4*>(slab + row * 128 + ((s ^ ((row >> 1) & 7)) << 4));
          if (m0 + row < g.M && f0 + s * 8 < g.N) *reinterpret_cast<u32x4*>(dst + (int64_t)(8 * t) * ld) = v;
        }
      } else {
        const int rows = g.M - m0 < 128 ? g.M - m0 : 128, cols = g.N - f0 < 64 ? g.N - f0 : 64;
        store_slab_rows_shifted<T, 128>(slab, D, ld, m0, rows, f0, cols, lane);
      }
    };
    if (pre != nullptr) {
      T* P = static_cast<T*>(pre);
      rows_out([&](int i, int p, int e) __attribute__((always_inline)) { return acc[i][p][e]; }, P, 2 * (int64_t)g.N);
      rows_out([&](int i, int p, int e) __attribute__((always_inline)) { return acc[i][4 + p][e]; }, P + g.N, 2 * (int64_t)g.N);
    }
    auto hidden = [&](auto ACT_) __attribute__((always_inline)) {
      rows_out([&](int i, int p, int e) __attribute__((always_inline)) {
        const float gv = acc[i][p][e];
        return gv * gate_q<decltype(ACT_)::value, GateHalf>(gv) * acc[i][4 + p][e];
      }, static_cast<T*>(h), g.N);
    };
    if (act == MI355_SILU) hidden(std::integral_constant<int, MI355_SILU>{});
    else if (act == MI355_GELU) hidden(std::integral_constant<int, MI355_GELU>{});
    else hidden(std::integral_constant<int, MI355_GELU_TANH>{});
  }
};

template <typename T>
__global__ __launch_bounds__(256) void gated_x16_kernel(GemmArgs g, GatedStore out) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  int tm, tn;
  tile_coords(g, tm, tn);
  x16_tile<T, false, 4, false, false, GatedStore>(g, lds, __builtin_amdgcn_readfirstlane(tm * 256), __builtin_amdgcn_readfirstlane(tn * 128), X16Split{}, &out);
}

template <typename T>
static int run_gated_x16(const GatedArgs& a, hipStream_t st) {
  GemmArgs g{};
  g.a = a.x;
  g.b = a.w;
  g.lda = a.x_rs;
  g.ldb = a.w_rs;
  g.M = (int32_t)a.M;
  g.N = (int32_t)a.F;
  g.K = (int32_t)a.K;
  g.alpha = 1.f;
  g.tiles_m = (int32_t)((a.M + 255) / 256);
  g.tiles_n = (int32_t)((a.F + 127) / 128);
  const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n;
  GatedStore out{a.h, a.pre, a.act, a.F % 8 == 0 && aligned16(a.h) && aligned16(a.pre)};
  const auto kern = gated_x16_kernel<T>;
  static std::atomic<uint64_t> devices{0};
  const int rc = allow_lds(reinterpret_cast<const void*>(kern), kX16Lds, devices, "mi355_gated_linear");
  if (rc != MI355_OK) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(256), kX16Lds, st, g, out);
  return check_launch("mi355_gated_linear");
}

bool gated_x16_takes(const GatedArgs& a) {
  // 32-bit byte offsets over up to 256 rows of either operand; fewer than 2^32 threads
  return a.K % 128 == 0 && a.K >= 256 && a.x_rs < (1 << 22) && a.w_rs < (1 << 22) &&
         ((a.M + 255) / 256) * ((a.F + 127) / 128) < (int64_t(1) << 24);
}

int launch_gated_x16(const GatedArgs& a, hipStream_t st) {
  return a.dtype == MI355_BF16 ? run_gated_x16<bf16_t>(a, st) : run_gated_x16<f16_t>(a, st);
}

}  // namespace mi355
