// Dropout from a counter-based generator, fused with the residual add; the mask is a function of (seed, offset,
// element index) and is never stored: the backward pass computes it again.
//
// Generator: Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011).  One
// counter gives 128 bits, used as eight 16-bit draws: an element is dropped when its draw is below t = round(p 2^16) (halves to even).
#include "../../include/mi355_train.h"
#include "elementwise.h"

namespace mi355 {

constexpr int kDropDraws = 8;  // elements per counter

// The 128 bits of counter `ctr` (its upper 64 bits are zero) under key `key`.
__device__ __forceinline__ u32x4 philox4x32_10(uint64_t ctr, uint64_t key) {
  u32x4 c = {(uint32_t)ctr, (uint32_t)(ctr >> 32), 0u, 0u};
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c[0] * 0xD2511F53u, p1 = (uint64_t)c[2] * 0xCD9E8D57u;
    c = u32x4{(uint32_t)(p1 >> 32) ^ c[1] ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c[3] ^ k1, (uint32_t)p0};
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// One counter's eight elements per thread and step.  VEC: all operands on 16-byte boundaries.
template <typename T, bool RES, bool VEC>
__global__ __launch_bounds__(256) void dropout_add_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                         const uint64_t* __restrict__ rng, uint64_t seed, uint64_t offset,
                                                         uint32_t threshold, typename OpMath<T>::type scale,
                                                         T* __restrict__ out, int64_t n) {
  using A = typename OpMath<T>::type;
  if (rng != nullptr) {
    seed = rng[0];
    offset = rng[1];
  }
  const int64_t groups = (n + kDropDraws - 1) / kDropDraws;
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
    const u32x4 bits = philox4x32_10(offset + (uint64_t)g, seed);
    const int64_t i0 = g * kDropDraws;
    auto apply = [&](int j, T xv, T rv) {
      const uint32_t draw = (bits[j >> 1] >> (16 * (j & 1))) & 0xffffu;
      A r = draw >= threshold ? static_cast<A>(xv) * scale : A(0);
      if constexpr (RES) r += static_cast<A>(rv);
      return static_cast<T>(r);
    };
    if (VEC && i0 + kDropDraws <= n) {
      const VecN<T, kDropDraws> xv = ld_nt<T, kDropDraws>(x + i0);
      VecN<T, kDropDraws> rv{}, o;
      if constexpr (RES) rv = ld_nt<T, kDropDraws>(res + i0);
#pragma unroll
      for (int j = 0; j < kDropDraws; ++j) o.v[j] = apply(j, xv.v[j], rv.v[j]);
      st_nt<T, kDropDraws>(out + i0, o);
    } else {
#pragma unroll
      for (int j = 0; j < kDropDraws; ++j)
        if (i0 + j < n) out[i0 + j] = apply(j, x[i0 + j], RES ? res[i0 + j] : T(0));
    }
  }
}

template <typename T>
static int run_dropout(const void* xv, const void* rv, uint32_t t, const void* rng, int64_t seed, int64_t offset, void* ov,
                       int64_t n, hipStream_t st) {
  using A = typename OpMath<T>::type;
  const T* x = static_cast<const T*>(xv);
  const T* res = static_cast<const T*>(rv);
  T* out = static_cast<T*>(ov);
  const A scale = t < 65536u ? static_cast<A>(65536.0 / (65536.0 - t)) : A(0);
  const bool vec = aligned16(x) && aligned16(out) && aligned16(res);
  const unsigned grid = (unsigned)grid_for((n + kDropDraws - 1) / kDropDraws, 256, 1 << 22);
  auto go = [&](auto has_res, auto v) {
    constexpr bool RES = decltype(has_res)::value, VEC = decltype(v)::value;
    hipLaunchKernelGGL((dropout_add_kernel<T, RES, VEC>), dim3(grid), dim3(256), 0, st, x, res, static_cast<const uint64_t*>(rng),
                       (uint64_t)seed, (uint64_t)offset, t, scale, out, n);
  };
  using std::true_type;
  using std::false_type;
  if (res != nullptr) vec ? go(true_type(), true_type()) : go(true_type(), false_type());
  else vec ? go(false_type(), true_type()) : go(false_type(), false_type());
  return check_launch("mi355_dropout_add");
}

}  // namespace mi355

using namespace mi355;

extern "C" int mi355_dropout_add(const void* x, const void* residual, int dtype, double p, const void* rng, int64_t seed,
                                 int64_t offset, void* out, int64_t n, void* stream) {
  MI355_REQUIRE(n >= 0, "mi355_dropout_add: negative extent");
  MI355_REQUIRE(p >= 0.0 && p <= 1.0, "mi355_dropout_add: p = %g is not in [0, 1]", p);
  if (n == 0) return MI355_OK;
  MI355_REQUIRE(x != nullptr && out != nullptr, "mi355_dropout_add: NULL data pointer");
  MI355_REQUIRE(reinterpret_cast<uintptr_t>(rng) % 8 == 0, "mi355_dropout_add: rng is not 8-byte aligned");
  const uint32_t t = (uint32_t)nearbyint(p * 65536.0);  // halves to the even neighbour
  MI355_DISPATCH_FLOAT(dtype, "mi355_dropout_add", return run_dropout<T>(x, residual, t, rng, seed, offset, out, n, static_cast<hipStream_t>(stream)));
}
