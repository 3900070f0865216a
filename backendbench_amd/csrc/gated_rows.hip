// The gated projection for few rows (decoding: 1 .. 64 tokens), bf16 / f16, and up to 32 in fp32: the weight is read once and
// its stream is the bound (2 F K elements); 16x16 matrix instructions with the weight rows as the first operand, the waves of a
// workgroup share K and add their accumulators in LDS at the end.
#include "gated.h"
#include "gemm_shared.h"

namespace mi355 {

// Behind the last matrix instruction on `v`, in front of its first other reader: 16 wait states, more than the 16x16x32
// instruction needs.  Not left to the compiler: in the LDS kernel's branch for K under a chunk it put none between the last
// v_mfma and the ds_write of its result, and the write took the registers' old contents (the generated code shows it, and
// [3, 1000] x 2 * 24 f16 came out wrong).
__device__ __forceinline__ void settle(f32x4& v) { asm volatile("s_nop 15" : "+v"(v)); }

// c + a b over 64 bytes of each of 16 rows: lane (r, g) = (lane % 16, lane / 16) holds bytes 16 g .. 16 g + 15 of row r of either.
template <typename T> struct GrMfma;
template <> struct GrMfma<float> {  // element j of every lane: the k of 4 g + j, the same in both operands
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    const f32x4 av = __builtin_bit_cast(f32x4, a), bv = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(av[j], bv[j], c, 0, 0, 0);
    return c;
  }
};
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
    for (int e = 0; e < 4; ++e) hv[e] = gv[e] * gate_q<decltype(ACT_)::value, GateMath<T>>(gv[e]) * uv[e];
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

// Weight and x go through LDS.  An MFMA fragment takes 64 bytes of each of 16 rows per load instruction; the
// memory system delivers such requests at 4.6 - 5.0 TB/s whatever their order, and 1 KB pieces of one row at 6.4 (a [22016,
// 4096] weight read by nothing but loads: 36 - 39 us against 28).  So both operands are requested in whole pieces straight
// into LDS (global_load_lds, 64 units of 16 bytes), a ring of NB buffers of KC elements of each row deep, and the fragments
// are read from there: unit c of row r sits at c ^ (r % 16), so that the 16 rows of a fragment read fall into 16 distinct
// columns of the 256-byte bank window.  Everything that is in flight is a request of one kind, counted by hand: a load into
// registers between them would have to be waited for together with all older requests.
// A block is RB x 8 features: their gate rows and the up rows of the same features, 8 + 8, make one 16-row operand; eight
// waves share it, each takes an eighth of a buffer's k.  RX rows of x are staged (fewer tokens than RX: the last one again).
constexpr int kRlWaves = 8;

// A request with the streaming hint (a weight is read once per call) or without.
template <bool STREAM> __device__ __forceinline__ void rl_fill(uint32_t lds_byte_offset, uint32_t lane_byte_offset, const void* base) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_byte_offset), "v"(lane_byte_offset), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_byte_offset), "v"(lane_byte_offset), "s"(base) : "memory");
}
template <int N> __device__ __forceinline__ void rl_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// KB: bytes of a row in a buffer.
template <int RX, int RB, int KB> struct RowsShape {
  static constexpr int MB = (RX + 15) / 16;            // token blocks
  static constexpr int ROWS = 16 * RB;                 // weight rows of a block
  static constexpr int UNITS = KB / 16;                // 16-byte units of a row
  static constexpr int RPI = 64 / UNITS;               // rows per request
  static constexpr int WFILLS = ROWS / RPI / kRlWaves;                               // requests of a wave per buffer: weight,
  static constexpr int XFILLS = RX / RPI >= kRlWaves ? RX / RPI / kRlWaves : 1;      // x (fewer than waves: some twice)
  static constexpr int FILLS = WFILLS + XFILLS;
  static constexpr int P = KB / kRlWaves / 64;         // 64-byte pieces of a wave per buffer
  static constexpr int BUF = (ROWS + RX) * KB;
  static constexpr int MEET = kRlWaves * RB * MB * kWave * 16;
};

// ANY: rows at any address and any K, which the requests into LDS do not take.  The pieces come through registers, NB sets of
// them in flight ahead, and are written to one of two buffers when their turn comes; the last chunk ends in zeros.  8, 32 and
// 64 rows: 2 * 5001 x 5001 37, 43 and 62 us (57, 59 and 76 through copies in aligned rows), 2 * 8430 x 8126 67, 82 and 119
// (144, 150 and 187), 2 * 4544 x 351 5.7, 6.6 and 11.7 (15.5, 17 and 16).  Chunks of 512 instead of 256 elements, two sets
// ahead: 45 us for the first.  fp32 (always this way): 16 and 32 rows of 2 * 11008 x 4096 76 and 94 us (a product and an
// activation kernel 141), of 2 * 2649 x 951 9 and 11 (28), of 2 * 1376 x 8192 34 and 45 (38 and 39).
template <typename T, int RX, int RB, int KB, int NB, int WAVES_PER_SIMD, bool ANY>
__global__ __launch_bounds__(64 * kRlWaves, WAVES_PER_SIMD) void gated_rows_lds_kernel(GatedArgs g) {
  using S = RowsShape<RX, RB, KB>;
  constexpr int V = 16 / sizeof(T), KC = KB / sizeof(T);  // elements of a unit, of a row in a buffer
  constexpr int MB = S::MB, P = S::P, UNITS = S::UNITS, RPI = S::RPI;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // the ring; at the end the waves' accumulators
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lr = lane & 15, lg = lane >> 4;
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const int64_t f0 = (int64_t)blockIdx.x * (8 * RB);
  // Row r of the block: feature f0 + 8 (r / 16) + r % 8, its gate row when r % 16 < 8, else its up row; features past the last
  // are computed on the last one's rows and not stored.
  auto row_of = [&](int r) {
    int64_t f = f0 + 8 * (r >> 4) + (r & 7);
    f = f < g.F ? f : g.F - 1;
    return ((r & 8) ? g.F + f : f) * g.w_rs;
  };
  const T* W = static_cast<const T*>(g.w);
  const T* X = static_cast<const T*>(g.x);
  const int chunks = (int)(ANY ? (g.K + KC - 1) / KC : g.K / KC);
  // Rows are usually a power of two apart, so the memory channel of a piece is a matter of its k: workgroups that share an
  // L2 (every eighth) start at different chunks.
  const int turn = chunks > 0 ? (int)(blockIdx.x / kNumXCD % chunks) : 0;
  // A request covers RPI rows; lane l fetches unit (l % UNITS) ^ (r % 16) of row r = first + l / UNITS, which lands at l.
  auto fill = [&](int c) {
    const int64_t k = (int64_t)(c + turn < chunks ? c + turn : c + turn - chunks) * KC;
    const uint32_t buf = lds_base + (uint32_t)(c % NB) * S::BUF;
#pragma unroll
    for (int q = 0; q < S::WFILLS; ++q) {
      const int first = (wave * S::WFILLS + q) * RPI;
      const int64_t row0 = row_of(first);
      uint32_t off = (uint32_t)(((lane % UNITS) ^ ((first + lane / UNITS) & 15)) * 16);
      if constexpr (RPI > 1) off += lane / UNITS ? (uint32_t)((row_of(first + 1) - row0) * 2) : 0u;  // (rows 2 i, 2 i + 1: neighbours)
      rl_fill<true>(buf + first * KB, off, W + row0 + k);
    }
#pragma unroll
    for (int q = 0; q < S::XFILLS; ++q) {
      const int first = (wave * S::XFILLS + q) * RPI % RX;
      const int64_t m0 = first < g.M ? first : g.M - 1, m1 = first + 1 < g.M ? first + 1 : g.M - 1;
      uint32_t off = (uint32_t)(((lane % UNITS) ^ ((first + lane / UNITS) & 15)) * 16);
      if constexpr (RPI > 1) off += lane / UNITS ? (uint32_t)((m1 - m0) * g.x_rs * 2) : 0u;
      rl_fill<false>(buf + (S::ROWS + first) * KB, off, X + m0 * g.x_rs + k);
    }
  };
  f32x4 acc[RB][MB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[rb][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int slot) {
    const unsigned char* buf = lds + slot * S::BUF;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int u = wave * (4 * P) + 4 * p + lg;  // this lane's unit of a row
      u32x4 x[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const int r = (mb * 16 + lr) % RX;  // (tokens past RX repeat: never stored)
        x[mb] = *reinterpret_cast<const u32x4*>(buf + (S::ROWS + r) * KB + ((u ^ (r & 15)) << 4));
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(buf + (rb * 16 + lr) * KB + ((u ^ lr) << 4));
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[rb][mb] = GrMfma<T>::run(w, x[mb], acc[rb][mb]);
      }
    }
  };
  if constexpr (ANY) {
    // Thread t has units t, t + 512, ... of a chunk's rows, the weight's and then x's.
    constexpr int THREADS = 64 * kRlWaves, WN = S::ROWS * UNITS / THREADS, XN = (RX * UNITS + THREADS - 1) / THREADS;
    const T* from[WN + XN];  // this thread's places in the first chunk
    uint32_t to[WN + XN];
#pragma unroll
    for (int q = 0; q < WN + XN; ++q) {
      const int i = (q < WN ? q : q - WN) * THREADS + (int)threadIdx.x, r = i / UNITS % (q < WN ? S::ROWS : RX), u = i % UNITS;
      from[q] = q < WN ? W + row_of(r) : X + (r < g.M ? r : g.M - 1) * g.x_rs;
      to[q] = (uint32_t)((q < WN ? r : S::ROWS + r) * KB + ((u ^ (r & 15)) << 4));
    }
    u32x4 piece[NB][WN + XN];
    const int unit = (int)threadIdx.x % UNITS * V;
    auto fetch = [&](int c, u32x4 (&p)[WN + XN]) __attribute__((always_inline)) {
      if (c >= chunks) return;
      const int64_t k = (int64_t)c * KC + unit, at = k + V <= g.K ? k : g.K - V;
#pragma unroll
      for (int q = 0; q < WN + XN; ++q) {
        const auto* a = reinterpret_cast<const typename AnyVec<sizeof(T)>::type*>(from[q] + at);
        p[q] = q < WN ? __builtin_nontemporal_load(a) : *a;
      }
    };
#pragma unroll
    for (int c = 0; c < NB; ++c) fetch(c, piece[c]);
    for (int c0 = 0; c0 < chunks; c0 += NB) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int c = c0 + n;
        if (c >= chunks) break;
        unsigned char* buf = lds + (c & 1) * S::BUF;
#pragma unroll
        for (int q = 0; q < WN + XN; ++q) {
          if (c + 1 == chunks) piece[n][q] = placed<T>(piece[n][q], (int64_t)c * KC + unit, g.K);  // zeros in both operands (0 * inf)
          *reinterpret_cast<u32x4*>(buf + to[q]) = piece[n][q];
        }
        // The barrier: chunk c is there for every wave, and every wave has multiplied chunk c - 1, whose buffer is next.
        __syncthreads();
        fetch(c + NB, piece[n]);
        multiply(c & 1);
      }
    }
  } else {
    // NB - 1 buffers ahead.  Chunk c: its requests are back when only those of the NB - 2 chunks behind it are out; the barrier
    // that follows says so for every wave, and that all have multiplied chunk c - 1, whose buffer is then refilled.
#pragma unroll
    for (int c = 0; c < NB - 1; ++c)
      if (c < chunks) fill(c);
    for (int c = 0; c < chunks; ++c) {
      if (c + NB - 1 <= chunks) rl_wait<(NB - 2) * S::FILLS>();
      else rl_wait<0>();  // (the last chunks: fewer are out)
      __syncthreads();
      if (c + NB - 1 < chunks) fill(c + NB - 1);
      multiply(c % NB);
    }
    // What is left of K, under a chunk: 32-k pieces, all requested before the first is used; rows end on a 16-byte unit, units
    // behind the end are zeros in both operands (0 * inf).
    const int64_t k0 = (int64_t)chunks * KC;
    if (k0 < g.K) {
      u32x4 w[P][RB], x[P][MB];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t k = k0 + 32 * (wave + kRlWaves * p) + 8 * lg;
        const int64_t kc = k < g.K ? k : 0;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) w[p][rb] = *reinterpret_cast<const u32x4*>(W + row_of(rb * 16 + lr) + kc);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const int64_t m = mb * 16 + lr;
          x[p][mb] = *reinterpret_cast<const u32x4*>(X + (m < g.M ? m : g.M - 1) * g.x_rs + kc);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int p = 0; p < P; ++p) {
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
  }
  // The waves' parts meet in LDS and are added in a fixed order.
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) settle(acc[rb][mb]);
  __syncthreads();  // every wave has read the last chunk
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

// Rows on 16-byte boundaries, of whole 16-byte units, and neighbours within a request's 32-bit byte offset.
bool gated_rows_aligned(const GatedArgs& a) {
  return a.x_rs % 8 == 0 && a.w_rs % 8 == 0 && a.K % 8 == 0 && aligned16(a.x) && aligned16(a.w) && a.x_rs < (1 << 30) && a.w_rs < (1 << 30);
}

template <typename T> static int run_gated_rows(const GatedArgs& a, hipStream_t st) {
  using std::integral_constant;
  using One = integral_constant<int, 1>;
  using Two = integral_constant<int, 2>;
  using Four = integral_constant<int, 4>;
  auto lds = [&](auto rx, auto rb, auto kb, auto nb, auto waves, auto any) {
    constexpr int RX = decltype(rx)::value, RB = decltype(rb)::value, KB = decltype(kb)::value, NB = decltype(nb)::value;
    constexpr bool ANY = decltype(any)::value;
    using S = RowsShape<RX, RB, KB>;
    const auto kern = gated_rows_lds_kernel<T, RX, RB, KB, NB, decltype(waves)::value, ANY>;
    constexpr int ring = (ANY ? 2 : NB) * S::BUF, bytes = ring > S::MEET ? ring : S::MEET;
    static std::atomic<uint64_t> devices{0};
    const int rc = allow_lds(reinterpret_cast<const void*>(kern), bytes, devices, "mi355_gated_linear");
    if (rc != MI355_OK) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)((a.F + 8 * RB - 1) / (8 * RB))), dim3(64 * kRlWaves), bytes, st, a);
    return check_launch("mi355_gated_linear");
  };
  using Whole = integral_constant<int, 1024>;  // a request's
  using Half = integral_constant<int, 512>;
  // Blocks of 8 features (x read twice as often) where those of 16 would leave half of the CUs without one: 2 * 1376 x 8192, 16
  // and 32 tokens, 17.3 -> 12.4 and 21.0 -> 16.3 us; 2 * 2752 x 4096 11.6 and 13.2 in blocks of 16, 14.3 and 17.8 in blocks of 8.
  const bool few = a.F <= 8 * kNumCU;
  if (sizeof(T) == 4 || !gated_rows_aligned(a)) {
    using Yes = std::true_type;
    if (a.M <= 16 && few) return lds(integral_constant<int, 16>(), One(), Half(), integral_constant<int, 6>(), Two(), Yes());
    if (a.M <= 16) return lds(integral_constant<int, 16>(), Two(), Half(), Four(), Two(), Yes());
    if (a.M <= 32 && few) return lds(integral_constant<int, 32>(), One(), Half(), Four(), Two(), Yes());
    if (a.M <= 32) return lds(integral_constant<int, 32>(), Two(), Half(), integral_constant<int, 3>(), Two(), Yes());
    if constexpr (sizeof(T) == 2) return lds(integral_constant<int, 64>(), Two(), Half(), integral_constant<int, 3>(), Two(), Yes());
  }
  if constexpr (sizeof(T) == 2) {
    if (a.M <= 4) return lds(Four(), One(), Whole(), Four(), Four(), std::false_type());
    if (a.M <= 16 && few) return lds(integral_constant<int, 16>(), One(), Whole(), integral_constant<int, 5>(), Two(), std::false_type());
    if (a.M <= 16) return lds(integral_constant<int, 16>(), Two(), Whole(), integral_constant<int, 3>(), Two(), std::false_type());
    if (a.M <= 32 && few) return lds(integral_constant<int, 32>(), One(), Half(), integral_constant<int, 6>(), Two(), std::false_type());
    if (a.M <= 32) return lds(integral_constant<int, 32>(), Two(), Half(), integral_constant<int, 5>(), Two(), std::false_type());
    return lds(integral_constant<int, 64>(), Two(), Half(), integral_constant<int, 3>(), Two(), std::false_type());
  }
  return set_error(MI355_ERR_UNSUPPORTED, "mi355_gated_linear: %lld rows are not few", (long long)a.M);
}

// fp32 up to 32 rows: 33 of them take 183 us at 2 * 11008 x 4096 (142 as a product), where 32 take 94.
bool gated_rows_takes(const GatedArgs& a) { return a.M <= (a.dtype == MI355_F32 ? 32 : 64) && a.F < (1 << 25) && a.K >= 8 && a.K < (1 << 30); }

int launch_gated_rows(const GatedArgs& a, hipStream_t st) {
  if (a.dtype == MI355_F32) return run_gated_rows<float>(a, st);
  return a.dtype == MI355_BF16 ? run_gated_rows<bf16_t>(a, st) : run_gated_rows<f16_t>(a, st);
}

}  // namespace mi355
