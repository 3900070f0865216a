// mm / addmm on v_mfma_f32_16x16x32: the kernels around x16_tile (gemm_x16.h), one workgroup per tile, persistent, split
// along K, and with two tile widths.
#include "gemm_x16.h"

namespace mi355 {

template <typename T, bool B_NN>
__global__ __launch_bounds__(256) void gemm_mfma_x16_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  if ((int)blockIdx.x >= g.tiles_m * g.tiles_n) return warm_operands<T, false, B_NN>(g, 0, g.K);
  int tm, tn;
  tile_coords(g, tm, tn);
  x16_tile<T, B_NN, 4>(g, lds, __builtin_amdgcn_readfirstlane(tm * BM), __builtin_amdgcn_readfirstlane(tn * BN));
}

// Fewer tiles than half the CUs and a long K: sk_splits workgroups per tile, each with its share of K.
// Blocks [r * sk_tiles8, (r + 1) * sk_tiles8) have one role: r < sk_splits - 1 the producers r + 1, the
// last group the summing workgroups (blocks are dispatched in order: a summing workgroup only ever waits
// for workgroups in front of it).  Block t of a group works on tile t; sk_tiles8 is a multiple of 8, so the
// workgroups of one tile share an XCD and its L2 (blocks go to the XCDs round robin), and blocks past the
// tile count have nothing to do.  K is shared out in units of 128, the summing workgroup gets the largest
// share (x16_split_summing_units): what it does with the planes only starts when the last producer has stored
// its plane, 3 us after its K loop, so the summing workgroup's own K loop should end about then.
template <typename T, bool B_NN>
__global__ __launch_bounds__(256) void gemm_mfma_x16_splitk_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int S = g.sk_splits, tiles = g.tiles_m * g.tiles_n;
  const int grp = __builtin_amdgcn_readfirstlane((int)blockIdx.x / g.sk_tiles8);
  const int t = __builtin_amdgcn_readfirstlane((int)blockIdx.x % g.sk_tiles8);
  if (t >= tiles) return;
  const int role = grp == S - 1 ? 0 : grp + 1;
  int tm, tn;
  tile_coords(g.tiles_m, g.tiles_n, t, tm, tn);
  const int units = g.K / kX16SplitUnit;
  const int cu = x16_split_summing_units(units, S);
  const int pu = units - cu, pbase = pu / (S - 1), prem = pu % (S - 1);
  int k0 = 0, ku = cu;
  if (role > 0) {
    const int q = role - 1;
    k0 = cu + q * pbase + (q < prem ? q : prem);
    ku = pbase + (q < prem ? 1 : 0);
  }
  GemmArgs gs = g;
  const T* A = static_cast<const T*>(g.a);
  const T* B = static_cast<const T*>(g.b);
  gs.a = A + (int64_t)k0 * kX16SplitUnit;
  gs.b = B_NN ? B + (int64_t)k0 * kX16SplitUnit * g.ldb : B + (int64_t)k0 * kX16SplitUnit;
  gs.K = ku * kX16SplitUnit;
  X16Split sk;
  const int64_t first = (int64_t)t * (S - 1) + (role > 0 ? role - 1 : 0);  // plane / flag index
  sk.planes = reinterpret_cast<f32x4*>(g.ws) + first * 16384;
  sk.flags = g.sk_flags + first;
  sk.epoch = g.sk_epoch;
  sk.spin_limit = g.sk_spin_limit;
  sk.role = role;
  sk.nprod = S - 1;
  x16_tile<T, B_NN, 4, false, true>(gs, lds, __builtin_amdgcn_readfirstlane(tm * BM), __builtin_amdgcn_readfirstlane(tn * BN), sk);
}

// Two tile widths in one launch: blocks [0, tiles_m * tiles_n) are 256 x 256 tiles of the columns
// [0, 256 tiles_n); the blocks behind them are 256 x 192 tiles of the columns from there on (tiles_m *
// tail_n of them).  Workgroups are dispatched in block order, so the narrow tiles form the last round.
template <typename T, bool B_NN>
__global__ __launch_bounds__(256) void gemm_mfma_x16_mixed_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int wide = g.tiles_m * g.tiles_n;
  int tm, tn;
  if ((int)blockIdx.x < wide) {
    tile_coords(g.tiles_m, g.tiles_n, blockIdx.x, tm, tn);
    x16_tile<T, B_NN, 4>(g, lds, __builtin_amdgcn_readfirstlane(tm * BM), __builtin_amdgcn_readfirstlane(tn * BN));
  } else {
    tile_coords(g.tiles_m, g.tail_n, blockIdx.x - wide, tm, tn);
    x16_tile<T, B_NN, 3>(g, lds, __builtin_amdgcn_readfirstlane(tm * BM), __builtin_amdgcn_readfirstlane(g.tiles_n * BN + tn * 192));
  }
}

// One workgroup per CU walks the tiles (x16_tile<..., PERSIST>): gridDim.x workgroups, tiles_m * tiles_n tiles.
template <typename T, bool B_NN>
__global__ __launch_bounds__(256) void gemm_mfma_x16_persistent_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  x16_tile<T, B_NN, 4, true>(g, lds, 0, 0);
}

const void* gemm_x16_persistent_kernel(bool is_bf16, bool b_nn) {
  if (is_bf16) return b_nn ? (const void*)gemm_mfma_x16_persistent_kernel<bf16_t, true> : (const void*)gemm_mfma_x16_persistent_kernel<bf16_t, false>;
  return b_nn ? (const void*)gemm_mfma_x16_persistent_kernel<f16_t, true> : (const void*)gemm_mfma_x16_persistent_kernel<f16_t, false>;
}

const void* gemm_x16_kernel(bool is_bf16, bool b_nn) {
  if (is_bf16) return b_nn ? (const void*)gemm_mfma_x16_kernel<bf16_t, true> : (const void*)gemm_mfma_x16_kernel<bf16_t, false>;
  return b_nn ? (const void*)gemm_mfma_x16_kernel<f16_t, true> : (const void*)gemm_mfma_x16_kernel<f16_t, false>;
}

const void* gemm_x16_splitk_kernel(bool is_bf16, bool b_nn) {
  if (is_bf16) return b_nn ? (const void*)gemm_mfma_x16_splitk_kernel<bf16_t, true> : (const void*)gemm_mfma_x16_splitk_kernel<bf16_t, false>;
  return b_nn ? (const void*)gemm_mfma_x16_splitk_kernel<f16_t, true> : (const void*)gemm_mfma_x16_splitk_kernel<f16_t, false>;
}

const void* gemm_x16_mixed_kernel(bool is_bf16, bool b_nn) {
  if (is_bf16) return b_nn ? (const void*)gemm_mfma_x16_mixed_kernel<bf16_t, true> : (const void*)gemm_mfma_x16_mixed_kernel<bf16_t, false>;
  return b_nn ? (const void*)gemm_mfma_x16_mixed_kernel<f16_t, true> : (const void*)gemm_mfma_x16_mixed_kernel<f16_t, false>;
}

}  // namespace mi355

extern "C" int mi355_gemm_status(void) {
  unsigned int word = 0, word2 = 0;
  hipError_t e = hipMemcpyFromSymbol(&word, HIP_SYMBOL(mi355::x16_gave_up_word), sizeof(word));
  if (e != hipSuccess) return mi355::set_error(MI355_ERR_LAUNCH, "mi355_gemm_status: reading the status word failed: %s", hipGetErrorString(e));
  if (word != 0) {
    const unsigned int zero = 0;
    e = hipMemcpyToSymbol(HIP_SYMBOL(mi355::x16_gave_up_word), &zero, sizeof(zero));
    if (e != hipSuccess) return mi355::set_error(MI355_ERR_LAUNCH, "mi355_gemm_status: clearing the status word failed: %s", hipGetErrorString(e));
  }
  const int e2 = mi355::read_insplit_status(&word2);  // the 128x128- and 64x64-tile kernels' word (gemm.hip)
  if (e2 != 0) return mi355::set_error(MI355_ERR_LAUNCH, "mi355_gemm_status: reading the status word failed: %s", hipGetErrorString((hipError_t)e2));
  if (word == 0 && word2 == 0) return MI355_OK;
  return mi355::set_error(MI355_ERR_LAUNCH,
                          "mi355_gemm: a split-K launch gave up waiting for a partial product (its output tile holds NaNs)");
}
