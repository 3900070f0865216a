// The gated projection for few rows (decoding: 1 .. 64 tokens), bf16 / f16: the weight is read once and its stream is the
// bound (4 F K bytes); v_mfma_f32_16x16x32 with the weight rows as the first operand, the waves of a workgroup share K and
// add their accumulators in LDS at the end.  Two forms: through LDS for aligned rows, straight into registers for the rest.
#include <string.h>

#include "gated.h"
#include "gemm_shared.h"

namespace mi355 {

typedef uint32_t gr_any __attribute__((ext_vector_type(4), aligned(2)));  // 8 elements at any element's address

template <typename T> struct GrMfma;
template <> struct GrMfma<bf16_t> {
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct GrMfma<f16_t> {
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// Element e of gv / uv: gate and up of feature f + e for token m.
template <typename T> __device__ __forceinline__ void store_rows(const GatedArgs& g, int64_t m, int64_t f, const f32x4& gv, const f32x4& uv) {
  if (m >= g.M) return;
  float hv[4];
  auto hidden = [&](auto ACT_) {
#pragma unroll
    for (int e = 0; e < 4; ++e) hv[e] = gv[e] * gate_q<decltype(ACT_)::value, GateHalf>(gv[e]) * uv[e];
  };
  if (g.act == MI355_SILU) hidden(std::integral_constant<int, MI355_SILU>{});
  else if (g.act == MI355_GELU) hidden(std::integral_constant<int, MI355_GELU>{});
  else hidden(std::integral_constant<int, MI355_GELU_TANH>{});
  T* h = static_cast<T*>(g.h) + m * g.F;
  T* pre = static_cast<T*>(g.pre) + 2 * m * g.F;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (f + e < g.F) {
      h[f + e] = static_cast<T>(hv[e]);
      if (g.pre != nullptr) {
        pre[f + e] = static_cast<T>(gv[e]);
        pre[g.F + f + e] = static_cast<T>(uv[e]);
      }
    }
}

// Aligned rows: the weight goes through LDS.  An MFMA fragment takes 64 bytes of each of 16 rows per load instruction; the
// memory system delivers such requests at 4.6 - 5.0 TB/s whatever their order, and pieces of 1 KB of one row, 2 KB of a row
// per workgroup at a time, at 6.3 - 6.5 (a [22016, 4096] weight read by nothing but loads).  So the rows are requested in
// 1 KB pieces straight into LDS (global_load_lds), two buffers of kRlChunk elements of each row, and the fragments are read
// from there: 16-byte unit c of row r sits at c ^ (r % 16), so that the 16 rows of a fragment read fall into 16 distinct
// columns of the 256-byte bank window.  Eight waves share a buffer, each takes its eighth of the chunk's k for all RB x 8
// features (8 gate rows and the 8 up rows of the same features make one 16-row operand) and MB x 16 tokens; x comes
// straight from L2 in fragments, one chunk ahead.
constexpr int kRlChunk = 1024, kRlWaves = 8;
constexpr int kRlRowBytes = kRlChunk * 2;

template <typename T, int MB, int RB>
__global__ __launch_bounds__(64 * kRlWaves, RB == 1 ? 4 : 2) void gated_rows_lds_kernel(GatedArgs g) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // two buffers; at the end the waves' accumulators
  constexpr int BUF = RB * 16 * kRlRowBytes;
  constexpr int FILLS = RB * 4;  // 1 KB requests of a wave per buffer: RB x 32 in all
  constexpr int P = kRlChunk / kRlWaves / 32;  // 32-k pieces of a wave per chunk
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * (8 * RB);
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  // Row r (0 .. 16 RB - 1) of the workgroup: feature f0 + 8 (r / 16) + r % 8, its gate row when r % 16 < 8, else its up row;
  // features past the last are computed on the last one's rows and not stored.
  auto row_of = [&](int r) {
    int64_t f = f0 + 8 * (r >> 4) + (r & 7);
    f = f < g.F ? f : g.F - 1;
    return static_cast<const T*>(g.w) + ((r & 8) ? g.F + f : f) * g.w_rs;
  };
  const T* xrow[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t m = mb * 16 + lr;
    xrow[mb] = static_cast<const T*>(g.x) + (m < g.M ? m : g.M - 1) * g.x_rs;
  }
  const int chunks = (int)(g.K / kRlChunk);
  // Rows are usually a power of two apart, so the memory channel of a piece is a matter of its k: workgroups that share an
  // L2 (every eighth) start at different chunks.
  const int turn = chunks > 0 ? (int)(blockIdx.x / kNumXCD % chunks) : 0;
  auto k_of = [&](int i) { return (int64_t)(i + turn < chunks ? i + turn : i + turn - chunks) * kRlChunk; };
  auto fill = [&](int i, int buf) {
    const int64_t k = k_of(i);
#pragma unroll
    for (int q = 0; q < FILLS; ++q) {
      const int piece = wave * FILLS + q, r = piece >> 1, half = piece & 1;
      lds_dma16s(lds_base + (uint32_t)(buf * BUF + piece * 1024), (uint32_t)((lane ^ (r & 15)) * 16), row_of(r) + k + half * 512);
    }
  };
  auto fetch_x = [&](int i, u32x4 (&x)[MB][P]) {
    const int64_t k = k_of(i) + wave * (32 * P) + 8 * lg;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int p = 0; p < P; ++p) x[mb][p] = *reinterpret_cast<const u32x4*>(xrow[mb] + k + 32 * p);
  };
  f32x4 acc[RB][MB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[rb][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int buf, const u32x4 (&x)[MB][P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = wave * (4 * P) + 4 * p + lg;  // 16-byte unit of the row
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(lds + buf * BUF + (rb * 16 + lr) * kRlRowBytes + (c >> 6) * 1024 + (((c & 63) ^ lr) << 4));
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[rb][mb] = GrMfma<T>::run(w, x[mb][p], acc[rb][mb]);
      }
    }
  };
  if (chunks > 0) {
    u32x4 xa[MB][P], xb[MB][P];
    fetch_x(0, xa);
    fill(0, 0);
    // One chunk: the next one's x and weight pieces are requested, then this one's pieces waited for (all but the last FILLS
    // requests are back: the wait covers x too) and met by every wave.  The barrier behind the multiplication frees the
    // buffer.
    auto chunk = [&](int i, const u32x4 (&x)[MB][P], u32x4 (&xn)[MB][P]) {
      if (i + 1 < chunks) {
        fetch_x(i + 1, xn);
        asm volatile("" ::: "memory");
        fill(i + 1, (i + 1) & 1);
        if constexpr (FILLS == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __syncthreads();
      multiply(i & 1, x);
      __syncthreads();
    };
    for (int i = 0; i < chunks; i += 2) {
      chunk(i, xa, xb);
      if (i + 1 < chunks) chunk(i + 1, xb, xa);
    }
  }
  // What is left of K, under a chunk: 32-k pieces, four per wave at most, all requested before the first is used; rows end
  // on a 16-byte unit, units behind the end are zeros in both operands (0 * inf).
  const int64_t k0 = (int64_t)chunks * kRlChunk;
  if (k0 < g.K) {
    const T* wrow[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) wrow[rb] = row_of(rb * 16 + lr);
    u32x4 w[P][RB], x[P][MB];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t k = k0 + 32 * (wave + kRlWaves * p) + 8 * lg;
      const bool in = k < g.K;
      const int64_t kc = in ? k : 0;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) w[p][rb] = *reinterpret_cast<const u32x4*>(wrow[rb] + kc);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) x[p][mb] = *reinterpret_cast<const u32x4*>(xrow[mb] + kc);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (k0 + 32 * (wave + kRlWaves * p) >= g.K) break;  // (uniform over the wave)
      const bool in = k0 + 32 * (wave + kRlWaves * p) + 8 * lg < g.K;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) w[p][rb][e] = in ? w[p][rb][e] : 0u;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) x[p][mb][e] = in ? x[p][mb][e] : 0u;
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[rb][mb] = GrMfma<T>::run(w[p][rb], x[p][mb], acc[rb][mb]);
    }
  }
  // The waves' parts meet in LDS (the buffers are free: every chunk ends in a barrier) and are added in a fixed order.
  f32x4* meet = reinterpret_cast<f32x4*>(lds);  // [wave][block][lane]
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) meet[(wave * (RB * MB) + rb * MB + mb) * kWave + lane] = acc[rb][mb];
  __syncthreads();
  for (int i = wave; i < RB * MB; i += kRlWaves) {
    if (lane >= 32) continue;  // lanes 0 .. 31 hold gate rows, lane + 32 the up rows of the same features
    f32x4 gv = meet[i * kWave + lane], uv = meet[i * kWave + lane + 32];
#pragma unroll
    for (int q = 1; q < kRlWaves; ++q) {
      gv += meet[(q * (RB * MB) + i) * kWave + lane];
      uv += meet[(q * (RB * MB) + i) * kWave + lane + 32];
    }
    store_rows<T>(g, (i % MB) * 16 + lr, f0 + (i / MB) * 8 + 4 * lg, gv, uv);
  }
}

// Rows at any address: fragments straight from global memory, a workgroup owns FB x 16 features, gate and up, and its W waves
// take turns along K, 32 S elements at a time, each with its next step's loads in flight while it computes.
// Operand fragment of a 32-k piece: lane l holds row l % 16, k = 8 (l / 16) .. + 7 of it.  With the weight as the first
// operand, element e of an accumulator in lane l is feature 4 (l / 16) + e of token l % 16.
template <typename T, int MB, int FB, int W, int S>
__global__ __launch_bounds__(64 * W) void gated_rows_kernel(GatedArgs g) {
  __shared__ f32x4 meet[W][MB * FB * 2][kWave];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * (16 * FB);
  const T* wrow[FB][2];
  const T* xrow[MB];
#pragma unroll
  for (int fb = 0; fb < FB; ++fb) {
    int64_t f = f0 + fb * 16 + lr;
    f = f < g.F ? f : g.F - 1;  // features past the last are computed on its row and not stored
    wrow[fb][0] = static_cast<const T*>(g.w) + f * g.w_rs;
    wrow[fb][1] = static_cast<const T*>(g.w) + (g.F + f) * g.w_rs;
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t m = mb * 16 + lr;
    xrow[mb] = static_cast<const T*>(g.x) + (m < g.M ? m : g.M - 1) * g.x_rs;
  }
  struct Step {
    u32x4 w[FB][2][S], x[MB][S];
  };
  auto fetch = [&](int64_t k, Step& s) {
#pragma unroll
    for (int p = 0; p < S; ++p) {
      const int64_t c = k + 32 * p + 8 * lg;
#pragma unroll
      for (int fb = 0; fb < FB; ++fb)
#pragma unroll
        for (int u = 0; u < 2; ++u) s.w[fb][u][p] = __builtin_nontemporal_load(reinterpret_cast<const gr_any*>(wrow[fb][u] + c));
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) s.x[mb][p] = *reinterpret_cast<const gr_any*>(xrow[mb] + c);
    }
  };
  f32x4 acc[FB][2][MB];
#pragma unroll
  for (int fb = 0; fb < FB; ++fb)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) acc[fb][u][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int p = 0; p < S; ++p)
#pragma unroll
      for (int fb = 0; fb < FB; ++fb)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) acc[fb][u][mb] = GrMfma<T>::run(s.w[fb][u][p], s.x[mb][p], acc[fb][u][mb]);
  };
  constexpr int64_t KS = 32 * S, ROUND = KS * W;
  const int64_t whole = g.K / KS * KS;  // whole steps
  int64_t k = wave * KS;
  if (k < whole) {
    Step a, b;
    fetch(k, a);
    while (true) {  // two steps per trip, the two register sets trading places
      const int64_t kb = k + ROUND;
      if (kb < whole) fetch(kb, b);
      multiply(a);
      if (kb >= whole) break;
      k = kb + ROUND;
      if (k < whole) fetch(k, a);
      multiply(b);
      if (k >= whole) break;
    }
  }
  // What is left of K, 32 elements per wave: eight elements of a row at a time when they are there, else one by one, zeros
  // behind the end (in both operands: 0 * inf).
  for (int64_t k1 = whole + 32 * wave; k1 < g.K; k1 += 32 * W) {
    const int64_t c = k1 + 8 * lg;
    auto piece = [&](const T* row) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (c + 8 <= g.K) {
        v = *reinterpret_cast<const gr_any*>(row + c);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < g.K) v[j >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, row[c + j]) << (16 * (j & 1));
      }
      return v;
    };
    u32x4 xv[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) xv[mb] = piece(xrow[mb]);
#pragma unroll
    for (int fb = 0; fb < FB; ++fb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 wv = piece(wrow[fb][u]);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[fb][u][mb] = GrMfma<T>::run(wv, xv[mb], acc[fb][u][mb]);
      }
  }
#pragma unroll
  for (int fb = 0; fb < FB; ++fb)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) meet[wave][(mb * FB + fb) * 2 + u][lane] = acc[fb][u][mb];
  __syncthreads();
  // Block (token block, feature block) i goes to wave i % W, which adds the waves' parts in a fixed order.
  for (int i = wave; i < MB * FB; i += W) {
    f32x4 gv = meet[0][2 * i][lane], uv = meet[0][2 * i + 1][lane];
#pragma unroll
    for (int q = 1; q < W; ++q) {
      gv += meet[q][2 * i][lane];
      uv += meet[q][2 * i + 1][lane];
    }
    store_rows<T>(g, (i / FB) * 16 + lr, f0 + (i % FB) * 16 + 4 * lg, gv, uv);
  }
}

template <typename T> static int run_gated_rows(const GatedArgs& a, hipStream_t st) {
  using std::integral_constant;
  using One = integral_constant<int, 1>;
  using Two = integral_constant<int, 2>;
  using Four = integral_constant<int, 4>;
  using Eight = integral_constant<int, 8>;
  auto lds = [&](auto mb, auto rb) {
    constexpr int MB = decltype(mb)::value, RB = decltype(rb)::value;
    const auto kern = gated_rows_lds_kernel<T, MB, RB>;
    constexpr int bytes = 2 * RB * 16 * kRlRowBytes;
    static_assert(bytes >= kRlWaves * RB * MB * kWave * 16, "the accumulators meet in the buffers");
    static std::atomic<uint64_t> devices{0};
    const int rc = allow_lds(reinterpret_cast<const void*>(kern), bytes, devices, "mi355_gated_linear");
    if (rc != MI355_OK) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)((a.F + 8 * RB - 1) / (8 * RB))), dim3(64 * kRlWaves), bytes, st, a);
    return check_launch("mi355_gated_linear");
  };
  auto direct = [&](auto mb, auto w, auto s) {
    constexpr int MB = decltype(mb)::value, W = decltype(w)::value, S = decltype(s)::value;
    hipLaunchKernelGGL((gated_rows_kernel<T, MB, 1, W, S>), dim3((unsigned)((a.F + 15) / 16)), dim3(64 * W), 0, st, a);
    return check_launch("mi355_gated_linear");
  };
  if (strcmp(knobs().gated_form, "direct") != 0 && a.x_rs % 8 == 0 && a.w_rs % 8 == 0 && a.K % 8 == 0 && aligned16(a.x) && aligned16(a.w)) {
    if (a.M <= 16) return lds(One(), One());
    if (a.M <= 32) return lds(Two(), Two());
    return lds(Four(), Two());
  }
  if (a.M <= 16) return direct(One(), Eight(), Four());
  if (a.M <= 32) return direct(Two(), Eight(), Two());
  return direct(Four(), Eight(), Two());
}

int launch_gated_rows(const GatedArgs& a, hipStream_t st) {
  return a.dtype == MI355_BF16 ? run_gated_rows<bf16_t>(a, st) : run_gated_rows<f16_t>(a, st);
}

}  // namespace mi355
