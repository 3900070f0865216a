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
// registers as loaded and are widened again after the two sums have met.  Sixteen waves leave 128 registers: a slab takes 40 - 89 of
// them, two slabs of 32 fp32 accumulators, two rows of raw vectors and 16-bit weights 120 - 128 (one to four spilled to scratch
// memory where N is no multiple of V).  fp32 weights beside 16-bit rows are too many: 6 registers spilled on 128 - 512 lanes, 16 on
// 64, 8 - 22 where N is no multiple of V, 0 and 2 on 1024; the four slabs of fp32 rows spill 7 or 8.  The kernel alone, [10738,
// 5056] bf16: 69 us with bf16 weights, 75 with fp32 ones, and 88 for 5053 columns, whose rows start off the vectors.
// Rows of more than one wave meet in LDS, one barrier per row (the slots alternate).
constexpr int kLbTile = 1024;
// Columns of one gradient in a partial: padded so that every partial starts on a 16-byte boundary.
__host__ __device__ constexpr int64_t lb_ld(int64_t N) { return (N + 3) / 4 * 4; }
constexpr int kLbTileBlocks = kNumCU;

// 16 bytes at an address that is only a multiple of an element's size.
typedef uint32_t lb_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t lb_any4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> using LbAny = std::conditional_t<sizeof(T) == 2, lb_any2, lb_any4>;

// V elements as loaded, in whole registers.
template <typename T, int V> struct LbRaw {
  static constexpr int R = sizeof(T) * V >= 4 ? sizeof(T) * V / 4 : 1;
  uint32_t r[R];
  // 16-byte (fp32 weights beside two-byte rows: 32-byte) vectors at any element's address.
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) * V >= 16) {
#pragma unroll
      for (int i = 0; i < R; i += 4) {
        const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const LbAny<T>*>(p + i * 4 / (int)sizeof(T)));
        r[i] = v[0]; r[i + 1] = v[1]; r[i + 2] = v[2]; r[i + 3] = v[3];
      }
    } else if constexpr (sizeof(T) == 4) {
      r[0] = __builtin_bit_cast(uint32_t, *p);
    } else {
      r[0] = __builtin_bit_cast(uint16_t, *p);
    }
  }
  __device__ __forceinline__ void fill(float v) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if constexpr (sizeof(T) == 4) r[i] = __builtin_bit_cast(uint32_t, v);
      else r[i] = (uint32_t)__builtin_bit_cast(uint16_t, static_cast<T>(v)) * 0x10001u;
    }
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
  __device__ __forceinline__ void clear_below(int first) {  // elements 0 .. first - 1
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (sizeof(T) == 4) r[j] = j < first ? 0u : r[j];
      else if (j < first) r[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
    }
  }
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int i = 0; i < R; ++i) asm volatile("" : "+v"(r[i]));
  }
};

// TAIL: N is no multiple of V.  The lane whose vector would stick out of the row moves it back to end with the row; the
// `skip` elements it then shares with its neighbour are the neighbour's.
template <typename T, typename Wt, int V, int GL, int NV, bool TAIL>
__global__ __launch_bounds__(kLbTile) void lb_tile_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         const Wt* __restrict__ w, T* __restrict__ dx, float* __restrict__ partial,
                                                         Wt* __restrict__ dw_out, Wt* __restrict__ db_out, int64_t M, int N) {
  constexpr int G = kLbTile / GL;                       // rows a block works on at a time
  constexpr int WPR = GL > kWave ? GL / kWave : 1;      // waves per row
  constexpr int WG = GL > kWave ? G : kLbTile / kWave;  // partial sums per column that meet in LDS at the end
  constexpr int COLS = NV * GL * V;
  static_assert(NV * V <= 16, "32 accumulators per lane");
  extern __shared__ __attribute__((aligned(16))) float lb_meet[];  // [dw, db][WG][COLS] when WG > 1
  __shared__ float2 red[2][kLbTile / kWave];
  const int t = threadIdx.x % GL, wave = threadIdx.x / kWave;
  // a row of whole waves: its number, and with it every row address, in scalar registers
  const int grp = GL >= kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / GL) : threadIdx.x / GL;
  // Row data and weights stay as loaded.  `keep` hides them from the compiler between uses: it would otherwise carry the
  // widened fp32 values from one use to the next (and the weights' from row to row) and spill 60 - 150 registers.
  struct Row {
    LbRaw<T, V> x[NV], dy[NV];
    float mean, rstd;
  };
  // First column of slab k's vector, its byte offset in a row (unsigned: one register beside a row address in scalars), and how
  // many of its elements are not this lane's.
  int first[NV], skip[NV];
  uint32_t at[NV];
  bool in[NV];
  LbRaw<Wt, V> gamma[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * GL + t) * V;
    in[k] = c < N;
    first[k] = c + V <= N ? c : N - V;
    at[k] = (uint32_t)first[k] * (uint32_t)sizeof(T);
    skip[k] = TAIL && in[k] ? c - first[k] : 0;
  }
  // No branches: lanes past the row and rows past the last read what is nearest; one_row puts zeros in its place (with a
  // branch per slab the compiler kept both sides of each in registers and spilled 100 of them).
  auto fetch = [&](int64_t row, Row& r) {
    const int64_t rc = row < M ? row : M - 1;
    r.mean = mean[rc];
    r.rstd = rstd[rc];
    const char *xr = reinterpret_cast<const char*>(x + rc * N), *dr = reinterpret_cast<const char*>(dy + rc * N);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      asm volatile("" : "+v"(at[k]));  // (else the loop carries a 64-bit pointer per slab and operand, and spills them)
      r.x[k].load(reinterpret_cast<const T*>(xr + at[k]));
      r.dy[k].load(reinterpret_cast<const T*>(dr + at[k]));
    }
  };
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t base = (int64_t)blockIdx.x * G;  // uniform over the block: every thread meets every barrier
  Row a;
  fetch(base + grp, a);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (w) gamma[k].load(w + first[k]);
    else gamma[k].fill(1.f);
  }
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
      r.x[k].clear_unless(live && in[k]);
      r.dy[k].clear_unless(live && in[k]);
      if constexpr (TAIL) r.x[k].keep();
      LbRaw<T, V> d = r.dy[k];
      if constexpr (TAIL) d.clear_below(skip[k]);
      gamma[k].keep();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (V > 4 && 2 * j == V) __builtin_amdgcn_sched_barrier(0);  // half a slab's temporaries at a time
        float xhat = (r.x[k].get(j) - r.mean) * r.rstd;
        if constexpr (TAIL) xhat = j < skip[k] ? 0.f : xhat;  // (0 * inf)
        const float g = d.get(j) * gamma[k].get(j);
        s.x += g;
        s.y += g * xhat;
        dw[k][j] += d.get(j) * xhat;
        db[k][j] += d.get(j);
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
      struct alignas(sizeof(T) * V) { T v[V]; } o;
      gamma[k].keep();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (V > 4 && 2 * j == V) __builtin_amdgcn_sched_barrier(0);
        const float xhat = (r.x[k].get(j) - r.mean) * r.rstd;
        o.v[j] = static_cast<T>(r.rstd * (r.dy[k].get(j) * gamma[k].get(j) - m1 - xhat * m2));
      }
      asm volatile("" : "+v"(at[k]));
      T* out = reinterpret_cast<T*>(reinterpret_cast<char*>(dx + row * N) + at[k]);
      if constexpr (V == 1) {
        if (in[k]) *out = o.v[0];
      } else if (in[k] && (!TAIL || skip[k] == 0)) {
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, o), reinterpret_cast<LbAny<T>*>(out));
      } else if (TAIL && in[k]) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j >= skip[k]) out[j] = o.v[j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The weights of columns that are not this lane's become zeros, like their dy (0 * inf).
  auto own_weights = [&]() {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      gamma[k].clear_unless(in[k]);
      if constexpr (TAIL) gamma[k].clear_below(skip[k]);
    }
  };
  if constexpr (NV <= 2) {
    Row b;
    fetch(base + step + grp, b);
    own_weights();
    while (base < M) {  // two rows per trip, the two register sets trading places
      one_row(base + grp, a);
      base += step;
      if (base >= M) break;
      fetch(base + step + grp, a);
      one_row(base + grp, b);
      base += step;
      if (base >= M) break;
      fetch(base + step + grp, b);
    }
  } else {  // no room for a second row
    own_weights();
    while (base < M) {
      one_row(base + grp, a);
      base += step;
      fetch(base + grp, a);
    }
  }
  if (partial == nullptr && dw_out == nullptr && db_out == nullptr) return;
  // This block's dw and db: the row groups' values meet in LDS (groups smaller than a wave first by exchanges inside it) and
  // leave as one partial [dw | db], each padded to lb_ld(N) columns, or as the result when this is the only block.
  const int64_t ld_n = lb_ld(N);
  float* part = partial + (int64_t)blockIdx.x * 2 * ld_n;
  if constexpr (WG == 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = first[k] + j;
        if (!in[k] || (TAIL && j < skip[k])) continue;
        if (partial != nullptr) {
          part[c] = dw[k][j];
          part[ld_n + c] = db[k][j];
        } else {
          if (dw_out != nullptr) dw_out[c] = static_cast<Wt>(dw[k][j]);
          if (db_out != nullptr) db_out[c] = static_cast<Wt>(db[k][j]);
        }
      }
  } else {
    auto park = [&](float (&acc)[NV][V], int which) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
          for (int d = GL; d < kWave; d *= 2) acc[k][j] += __shfl_xor(acc[k][j], d, kWave);
        if (!in[k] || (GL < kWave && threadIdx.x % kWave >= GL)) continue;
        float* dst = lb_meet + (which * WG + (GL >= kWave ? grp : wave)) * COLS + first[k];
        if constexpr (TAIL || V == 1) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j >= skip[k]) dst[j] = acc[k][j];
        } else {
#pragma unroll
          for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(dst + j) = float4{acc[k][j], acc[k][j + 1], acc[k][j + 2], acc[k][j + 3]};
        }
      }
    };
    park(dw, 0);
    park(db, 1);
    __syncthreads();
    const int quads = (int)ld_n / 4;
    for (int q = threadIdx.x; q < 2 * quads; q += kLbTile) {
      const int which = q >= quads, c = 4 * (which ? q - quads : q);
      float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < WG; ++g) {
        const float4 o = *reinterpret_cast<const float4*>(lb_meet + (which * WG + g) * COLS + c);
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      if (partial != nullptr) {  // (columns past N are padding: never read back)
        *reinterpret_cast<float4*>(part + which * ld_n + c) = v;
      } else {
        Wt* out = which ? db_out : dw_out;
        const float e[4] = {v.x, v.y, v.z, v.w};
        if (out != nullptr)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < N) out[c + j] = static_cast<Wt>(e[j]);
      }
    }
  }
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

// One column per thread, blockIdx.y = row group; partial[group][0 / 1][lb_ld(N)] = the group's dw / db.
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
    partial[(int64_t)blockIdx.y * 2 * lb_ld(N) + c] = dw;
    partial[((int64_t)blockIdx.y * 2 + 1) * lb_ld(N) + c] = db;
  }
}

// dw and db from `groups` partials of [dw | db]: 32 columns per block, 8 lanes of 4 neighbouring columns by 32 threads that
// take every 32nd partial; they meet by exchanges inside a wave (8 of them) and in LDS.
template <typename Wt, typename S>
__global__ __launch_bounds__(kLbBlock) void lb_finish_kernel(const S* __restrict__ partial, Wt* __restrict__ dw, Wt* __restrict__ db,
                                                            int64_t N, int groups) {
  __shared__ S part[kLbBlock / kWave][32];
  const int q = threadIdx.x / 8, l = threadIdx.x % 8;
  const int64_t ld_n = lb_ld(N), c0 = (int64_t)blockIdx.x * 32 + 4 * l;  // of the 2 ld_n columns [dw | db]
  S s[4] = {};
  if (c0 < 2 * ld_n) {
#pragma unroll 8
    for (int g = q; g < groups; g += 32) {
      const VecN<S, 4> v = ld<S, 4>(partial + (int64_t)g * 2 * ld_n + c0);
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
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const int64_t col = c < ld_n ? c : c - ld_n;
  if (threadIdx.x >= 32 || c >= 2 * ld_n || col >= N) return;
  const S sum = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
  Wt* out = c < ld_n ? dw : db;
  if (out) out[col] = static_cast<Wt>(sum);
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

// Lanes per row and slabs per lane of the tile kernel; lanes == 0: the general path.  A slab is one 16-byte vector per lane
// (single elements for rows shorter than that); two-byte rows take at most two, fp32 rows four.  More than a wave of lanes
// always hold two slabs: half as many lanes hold what one slab would.
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
// One block where four trips of it do: the finish pass is another launch (3 us), a trip about one.
static int64_t lb_tile_blocks(int64_t M, const LbTile& p) {
  const int64_t rows = kLbTile / p.lanes;  // per block and trip
  const int64_t need = (M + rows - 1) / rows;
  return need <= 4 ? 1 : need < kLbTileBlocks ? need : kLbTileBlocks;
}

template <typename T, typename Wt, int V, int GL, int NV, bool TAIL>
static int launch_lb_tile(int64_t blocks, const T* dy, const T* x, const float* mean, const float* rstd, const Wt* w, T* dx, float* partial,
                          Wt* dw, Wt* db, int64_t M, int64_t N, hipStream_t st) {
  constexpr int WG = GL > kWave ? kLbTile / GL : kLbTile / kWave;
  constexpr int bytes = WG > 1 ? 2 * WG * NV * GL * V * (int)sizeof(float) : 0;
  const auto kern = lb_tile_kernel<T, Wt, V, GL, NV, TAIL>;
  if (bytes > 48 * 1024) {
    static std::atomic<uint64_t> devices{0};
    const int rc = allow_lds(reinterpret_cast<const void*>(kern), bytes, devices, "mi355_layer_norm_backward");
    if (rc != MI355_OK) return rc;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kLbTile), bytes, st, dy, x, mean, rstd, w, dx, partial, dw, db, M, (int)N);
  return check_launch("mi355_layer_norm_backward");
}

template <typename T, typename Wt>
static int run_lb_tile(const LbTile& p, const T* dy, const T* x, const float* mean, const float* rstd, const Wt* w, T* dx, Wt* dw, Wt* db,
                       int64_t M, int64_t N, float* ws, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int64_t blocks = lb_tile_blocks(M, p);
  float* partial = (dw != nullptr || db != nullptr) && blocks > 1 ? ws : nullptr;
  int rc = MI355_ERR_UNSUPPORTED;
#define MI355_LB_TILE(GL_, NV_)                                                                                              \
  if (p.lanes == GL_ && p.slabs == NV_)                                                                                       \
    rc = N % V == 0 ? launch_lb_tile<T, Wt, V, GL_, NV_, false>(blocks, dy, x, mean, rstd, w, dx, partial, dw, db, M, N, st)  \
                    : launch_lb_tile<T, Wt, V, GL_, NV_, true>(blocks, dy, x, mean, rstd, w, dx, partial, dw, db, M, N, st);
  if (N < V) {
    rc = launch_lb_tile<T, Wt, 1, 8, 1, false>(blocks, dy, x, mean, rstd, w, dx, partial, dw, db, M, N, st);
  } else {
    MI355_LB_TILE(8, 1) MI355_LB_TILE(16, 1) MI355_LB_TILE(32, 1) MI355_LB_TILE(64, 1)
    MI355_LB_TILE(64, 2) MI355_LB_TILE(128, 2) MI355_LB_TILE(256, 2) MI355_LB_TILE(512, 2) MI355_LB_TILE(1024, 2)
    if constexpr (sizeof(T) == 4) MI355_LB_TILE(1024, 4)
  }
#undef MI355_LB_TILE
  if (rc == MI355_ERR_UNSUPPORTED) return set_error(rc, "mi355_layer_norm_backward: no kernel form of %d lanes and %d slabs", p.lanes, p.slabs);
  if (rc != MI355_OK || partial == nullptr) return rc;
  hipLaunchKernelGGL((lb_finish_kernel<Wt, float>), dim3((unsigned)((2 * lb_ld(N) + 31) / 32)), dim3(kLbBlock), 0, st, partial, dw, db, N, (int)blocks);
  return check_launch("mi355_layer_norm_backward");
}

template <typename T, typename Wt, typename S>
static int run_lb(const void* dyv, const void* xv, const void* mv, const void* rv, const void* wv, void* dxv, void* dwv, void* dbv,
                  int64_t M, int64_t N, void* ws, hipStream_t st) {
  const T *dy = static_cast<const T*>(dyv), *x = static_cast<const T*>(xv);
  const S *mean = static_cast<const S*>(mv), *rstd = static_cast<const S*>(rv);
  const Wt* w = static_cast<const Wt*>(wv);
  if constexpr (!std::is_same<T, double>::value) {
    const LbTile tile = lb_tile<T>(N);
    if (tile.lanes != 0)
      return run_lb_tile<T, Wt>(tile, dy, x, mean, rstd, w, static_cast<T*>(dxv), static_cast<Wt*>(dwv), static_cast<Wt*>(dbv), M, N,
                                static_cast<float*>(ws), st);
  }
  S* partial = (dwv != nullptr || dbv != nullptr) ? static_cast<S*>(ws) : nullptr;
  S* sums = static_cast<S*>(ws) + lb_plan(M, N).groups * 2 * lb_ld(N);  // behind the partials
  const LbPlan p = lb_plan(M, N);
  if (dxv != nullptr)
    hipLaunchKernelGGL((lb_row_means_kernel<T, Wt, S>), dim3((unsigned)grid_for(M, 1, kNumCU * 32)), dim3(kLbBlock), 0, st, dy, x, mean, rstd, w, sums, M, N);
  hipLaunchKernelGGL((lb_columns_kernel<T, Wt, S>), dim3((unsigned)((N + kLbBlock - 1) / kLbBlock), (unsigned)p.groups), dim3(kLbBlock), 0, st, dy,
                     x, mean, rstd, w, sums, static_cast<T*>(dxv), partial, M, N, p.rows_per_group);
  if (partial)
    hipLaunchKernelGGL((lb_finish_kernel<Wt, S>), dim3((unsigned)((2 * lb_ld(N) + 31) / 32)), dim3(kLbBlock), 0, st, partial,
                       static_cast<Wt*>(dwv), static_cast<Wt*>(dbv), N, (int)p.groups);
  return check_launch("mi355_layer_norm_backward");
}

}  // namespace mi355

using namespace mi355;

extern "C" int64_t mi355_layer_norm_backward_workspace_bytes(int64_t M, int64_t N, int dtype) {
  if (M <= 0 || N <= 0 || dtype_size(dtype) == 0) return 0;
  const LbTile p = dtype == MI355_F32 ? lb_tile<float>(N) : dtype == MI355_F64 ? lb_tile<double>(N) : lb_tile<bf16_t>(N);
  if (p.lanes != 0) return lb_tile_blocks(M, p) > 1 ? lb_tile_blocks(M, p) * 2 * lb_ld(N) * 4 : 0;
  return (2 * M + lb_plan(M, N).groups * 2 * lb_ld(N)) * (dtype == MI355_F64 ? 8 : 4);
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
  const int64_t need = mi355_layer_norm_backward_workspace_bytes(M, N, dtype);
  MI355_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && aligned16(workspace)),
                "mi355_layer_norm_backward: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
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
