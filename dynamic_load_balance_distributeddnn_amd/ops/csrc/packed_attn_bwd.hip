// Causal attention over packed sequences, backward (gfx950).
//
// With P_ij the forward's weights, recomputed from its row statistics:
//
//   delta_i = sum_d dO_id O_id            (= sum_j P_ij dO_i.v_j)
//   dS_ij   = P_ij (dO_i.v_j - delta_i)
//   dQ_i = scale sum_j dS_ij k_j          dV_j = sum_i P_ij dO_i
//   dK_j = scale sum_i dS_ij q_i          dtable[b] = sum of dS_ij, ij in b
//
// Two kernels, each the owner of what it writes: one holds 128 query rows
// and streams keys (dQ, delta), then one holds 128 keys and streams the
// queries of every head that shares them (dK, dV, the table's sums).
// The scores are computed in both, 7 products for 5; in return there are
// no atomics and no fp32 gradient buffer, and results do not depend on
// the order in which workgroups run.
//
// delta from the stored output carries the output's roundings to bf16
// (weights, result).  The first kernel sums dS over each row as it goes;
// the sum is 0 but for that error, so adding it to delta makes delta exact
// to fp32 for the second kernel: dK and the table's gradient lose nothing
// to it.  dQ itself is under way by then.  What the error costs it falls
// with the number of keys that a row's average spreads over, so the first
// 128 rows of a sequence, which can have few, take delta from a sweep over
// their one or two key tiles beforehand.
//
// Measured, both kernels and their joins: one sequence of 8192, 32 heads of
// 128 over 8, 1880 us (730 TFLOP/s by the formula's 5 products, 1020 by
// the 7 performed); seven of 8192 in all, 16 heads over 4, 290 us; eight
// of 512, 92 us; 20 of 35, 2 heads of 100, 26 us.  With a bias and its
// gradient: five of 4096 in all, 16 heads of 64, 112 us; one of 4001, 12
// heads, 180; one of 8192, 16 heads of 128 over 2, 1324.  Bound by the
// matrix units where sequences are long, else by the longest workgroup:
// the key kernel holds 128 keys for all heads of a group, so it is cut
// finer than the others.
#include "packed_attn.h"

// ---- The table's gradient: sums of dS along its diagonals, then of the
// diagonals of a bucket, all in a fixed order.  The last bucket, which has
// no end, a lane sums by itself (`far`).  A row's dS sum to 0, but minus the
// sum of the other buckets would leave their rounding where no pair has the
// last one or its weights are 0.  What that costs, backward and forward: five
// of 4096 in all, 16 heads of 64, 142 -> 144 us; one of 8192, 16 heads of 128
// over 2, 1511 -> 1598, of which the heads' order (see the kernel) is 35.
#define PA_DISTANCES 512  // with that many sums a wave
#define PA_FARHEADS 32    // of a group that LDS keeps the far bias of

// Lane l gets the value of lane (l + N) & 31 of its half.
template <int N>
__device__ inline float pa_rotate(float v) {
  return N == 0 ? v
                : __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(
                                                __builtin_bit_cast(int, v),
                                                0xc000 | (N << 5)));
}

// Diagonals of one 32 x 32 block of dS (queries x keys, the result layout;
// masked pairs 0): register r of half h, query i = c + 4 h, rotated by c
// leaves in lane x the distance 4 h - x, or 32 more where it wrapped.
__device__ PA_INLINE void pa_diagonals(const f32x16& ds, float& a, float& b,
                                       int x) {
  a = b = 0.f;
#define PA_DIAGONAL(R)                                   \
  {                                                      \
    constexpr int c = 8 * (R >> 2) + (R & 3);            \
    const float v = pa_rotate<c>(ds[R]);                 \
    if (x + c < 32) a += v; else b += v;                 \
  }
  PA_DIAGONAL(0) PA_DIAGONAL(1) PA_DIAGONAL(2) PA_DIAGONAL(3)
  PA_DIAGONAL(4) PA_DIAGONAL(5) PA_DIAGONAL(6) PA_DIAGONAL(7)
  PA_DIAGONAL(8) PA_DIAGONAL(9) PA_DIAGONAL(10) PA_DIAGONAL(11)
  PA_DIAGONAL(12) PA_DIAGONAL(13) PA_DIAGONAL(14) PA_DIAGONAL(15)
#undef PA_DIAGONAL
}

// Adds them to the wave's sums by distance; `n0` is the distance of query
// 0 and key 0 of the block.  The halves one after the other: no two lanes
// of an addition meet.
__device__ PA_INLINE void pa_add_diagonals(const f32x16& ds, int n0,
                                           int far_from, float* sums,
                                           float& far, int lane) {
  const int n = n0 + 4 * (lane >> 5) - (lane & 31);
  float a, b;
  pa_diagonals(ds, a, b, lane & 31);
  if (n >= far_from) far += a;
  if (n + 32 >= far_from) far += b;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if ((lane >> 5) == h) {
      if (n >= 0 && n < far_from)
        __hip_atomic_fetch_add(sums + n, a, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
      if (n + 32 >= 0 && n + 32 < far_from)
        __hip_atomic_fetch_add(sums + n + 32, b, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
}

// The same where there are too many distances for LDS: neighbouring
// diagonals of one bucket are added up lane by lane first.
__device__ PA_INLINE void pa_add_buckets(const f32x16& ds, int n0,
                                         const int* starts, int buckets,
                                         float* sums, int lane) {
  float part[2];
  pa_diagonals(ds, part[0], part[1], lane & 31);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // in the order of their distances: half by half, lanes downwards
    const int n = n0 + 4 * (lane >> 5) - (lane & 31) + 32 * i;
    const int z = 31 - (lane & 31);
    float v = part[i];
    const int b = n < 0 ? -1 : pa_bucket(starts, buckets, n);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const float pv = __shfl_down(v, off, 64);
      const int pb = __shfl_down(b, off, 64);
      if (z >= off && pb == b) v += pv;
    }
    const int nb = __shfl_up(b, 1, 64);
    const bool last = b >= 0 && (z == 31 || nb != b);
    // a bucket can end in both halves
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (last && (lane >> 5) == h)
        __hip_atomic_fetch_add(sums + b, v, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
  }
}

// A query row's end: N x 32 elements of its gradient from 32 * t0 on, with
// the first its delta.
template <int W, int N>
__device__ PA_INLINE void pa_bwd_q_end(const PaBwd& p, long first, int row,
                                       int len, int h,
                                       const f32x16 (&acc)[N], int t0,
                                       float delta) {
  if (row >= len) return;
  const int half = (threadIdx.x & 63) >> 5;
  if (half == 0 && t0 == 0) p.delta[(long)h * p.T + first + row] = delta;
  __bf16* ob = static_cast<__bf16*>(p.dq) + ((first + row) * p.H + h) * p.D;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bf16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = (__bf16)(acc[t][4 * g + e] * p.scale);
      pa_store4<W>(ob, (t0 + t) * 32 + 8 * g + 4 * half, p.D, v);
    }
}

// Three waves a SIMD where 168 registers do without spilling in the loop:
// with a bias, heads of 64, 145 -> 142 us (five of 4096 in all); without
// one 112 -> 117 us, so two there.  128 columns want 256 registers.
template <int DP, int W, bool BIAS, typename BiasArg>
__global__ void __launch_bounds__(PA_BLOCK, DP == 64 && BIAS ? 3 : 2)
pa_bwd_q_kernel(const PaBwd p, const BiasArg bias) {
  const int KS = DP / 16, DT = DP / 32;
  const int TILE = PA_STEP * DP;
  __shared__ __attribute__((aligned(1024))) __bf16 s_tiles[4][TILE];
  __bf16 (*s_k)[TILE] = s_tiles, (*s_v)[TILE] = s_tiles + 2;
  __shared__ float s_win[BIAS ? 2 : 1][BIAS ? 192 : 1];
  __shared__ float s_tab[BIAS ? PA_MAXBUCKETS : 1];
  __shared__ int s_start[BIAS ? PA_MAXBUCKETS : 1];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int h = pa_head(blockIdx.x % p.H, p.H);
  const PaChunk it = p.work_q.chunks[blockIdx.x / p.H];
  const int r0 = it.tile * PA_ROWS;
  const int w0 = r0 + wave * 32;
  const int row = w0 + col;
  const int len = it.len;
  const int whole = r0 / PA_STEP;  // tiles that all rows see whole
  PaStage<DP, W> ks(pa_at(p.k, it.first, h / p.G), p.k.row, len, p.D);
  PaStage<DP, W> vs(pa_at(p.v, it.first, h / p.G), p.v.row, len, p.D);
  if (p.D < DP) {
    pa_clear<DP>(s_k[0], 2 * PA_STEP);
    pa_clear<DP>(s_v[0], 2 * PA_STEP);
    __syncthreads();
  }
  // the first tile is under way before anything else is waited for
  ks.start(it.begin * PA_STEP, s_k[it.begin & 1]);
  vs.start(it.begin * PA_STEP, s_v[it.begin & 1]);

  float far_bias = 0.f;
  int far_from = 0;
  if constexpr (BIAS) {
    for (int b = threadIdx.x; b < bias.buckets; b += PA_BLOCK) {
      s_tab[b] = pa_bias(pa_table(bias, b, p.H, h), bias.is_bf16);
      s_start[b] = bias.starts[b];
    }
    __syncthreads();
    far_bias = s_tab[bias.buckets - 1];
    far_from = s_start[bias.buckets - 1];
  }
  auto window = [&](int k0) PA_INLINE {
    float x = 0.f;
    if constexpr (BIAS) {
      const int n = r0 - k0 - (PA_STEP - 1) + (int)threadIdx.x;
      if (n >= 0) x = s_tab[pa_bucket(s_start, bias.buckets, n)];
    }
    return x;
  };
  auto near = [&](int k0) PA_INLINE {
    return r0 - k0 - (PA_STEP - 1) < far_from || !pa_moderate(far_bias);
  };

  // a sequence's first rows, never in chunks: see above
  const bool sweep = it.tile == 0;
  float rest = 0.f;  // this half's sum of the row's dS

  bf16x8 qf[KS], gf[KS];
  float delta = 0.f, stat_m = 0.f, stat_l = INFINITY;
  {
    const long rr = (long)it.first + min(row, len - 1);
    const __bf16* qb = pa_at(p.q, rr, h);
    const __bf16* gb = pa_at(p.go, rr, h);
    const __bf16* ob = static_cast<const __bf16*>(p.o) +
                       (rr * p.H + h) * p.D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + half * 8;
      qf[s] = pa_load8<W>(qb, d, p.D);
      gf[s] = pa_load8<W>(gb, d, p.D);
      if (!sweep) {
        const bf16x8 of = pa_load8<W>(ob, d, p.D);
#pragma unroll
        for (int j = 0; j < 8; ++j) delta += (float)gf[s][j] * (float)of[j];
      }
    }
    delta = pa_half_sum(delta);
    const long at = (long)h * p.T + rr;
    if (row < len) {
      if constexpr (BIAS) {
        stat_m = p.stats[2 * at];
        stat_l = p.stats[2 * at + 1];
      } else {
        stat_l = p.stats[at];
      }
    }
  }
  // scores are exponents of 2, as in the forward
  const float mul = p.scale * PA_LOG2E;

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = pa_zero16();

  float win = 0.f;
  auto start = [&](int k0, int buf) PA_INLINE {
    ks.start(k0, s_k[buf]);
    vs.start(k0, s_v[buf]);
    if (BIAS && near(k0)) win = window(k0);
  };
  auto arrive = [&](int k0, int buf) PA_INLINE {
    if (BIAS && near(k0) && threadIdx.x < 192) s_win[buf][threadIdx.x] = win;
    ks.arrive(k0, s_k[buf]);
    vs.arrive(k0, s_v[buf]);
    __syncthreads();
  };
  const PaFrags<DP> lanes(s_tiles, lane);
  PaFrags<DP> frags = lanes;  // of the current buffer
  // weights times (dO.v - delta) of 32 keys of a tile
  auto gradient = [&](int k0, int j, int buf) PA_INLINE {
    const unsigned at = j * 32 * DP * 2;
    f32x16 s = pa_zero16(), dp = pa_zero16();
#pragma unroll
    for (int x = 0; x < KS; ++x)
      s = pa_mfma(frags.rows(at, x), qf[x], s);
#pragma unroll
    for (int x = 0; x < KS; ++x)
      dp = pa_mfma(frags.rows(at + 4 * TILE, x), gf[x], dp);
    float a = mul, off = -stat_l;
    if constexpr (BIAS) {
      if (near(k0)) {
        const float* w =
            s_win[buf] + wave * 32 + col + PA_STEP - 1;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = fmaf(s[r], mul,
                      w[-(j * 32 + 8 * (r >> 2) + 4 * half + (r & 3))]) -
                 stat_m;
        a = 1.f;
      } else {
        off = (far_bias - stat_m) - stat_l;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a, off)) * (dp[r] - delta);
    return s;
  };
  auto product = [&](bf16x8 w, int x) PA_INLINE {
#pragma unroll
    for (int d = 0; d < DT; ++d)
      acc[d] = pa_mfma(frags.cols(x * 16 * DP * 2, d), w, acc[d]);
  };

  // t < 0: the sweep's; its tiles stay in their two buffers.
  auto any_tile = [&](int t) PA_INLINE {
    const int tile = t < 0 ? t + it.end : t;
    const int k0 = tile * PA_STEP, buf = tile & 1;
    const bool more = t + 1 < (sweep ? 0 : it.end);
    if (more) start(k0 + PA_STEP, buf ^ 1);
    const bool works = k0 <= w0 + 31;
    bf16x8 w[4];
    frags = lanes.fresh(buf * TILE * 2);
    if (works) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f32x16 s = gradient(k0, j, buf);
        const int lim = row - k0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (j * 32 + 8 * (r >> 2) + (r & 3) > lim) s[r] = 0.f;
          rest += s[r];
        }
        w[2 * j] = pa_operand(s, 0);
        w[2 * j + 1] = pa_operand(s, 1);
      }
    }
    if (t >= 0) {
      if (__syncthreads_or(pa_tile_nonfinite<DP, PA_STEP>(s_k[buf]))) {
        pa_poison<DP, PA_STEP, true>(s_k[buf], acc, row - k0, lane);
        __syncthreads();
        pa_cleanse<DP, PA_STEP>(s_k[buf]);
        __syncthreads();
      }
      if (works) {
#pragma unroll
        for (int x = 0; x < 4; ++x) product(w[x], x);
      }
    }
    if (more) arrive(k0 + PA_STEP, buf ^ 1);
  };
  auto whole_tile = [&](int t) PA_INLINE {
    const int k0 = t * PA_STEP, buf = t & 1;
    const bool more = t + 1 < it.end;
    if (more) start(k0 + PA_STEP, buf ^ 1);
    frags = lanes.fresh(buf * TILE * 2);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x16 s = gradient(k0, j, buf);
#pragma unroll
      for (int r = 0; r < 16; ++r) rest += s[r];
      product(pa_operand(s, 0), 2 * j);
      product(pa_operand(s, 1), 2 * j + 1);
    }
    if (more) arrive(k0 + PA_STEP, buf ^ 1);
  };

  int t = sweep ? -it.end : it.begin;
  if (BIAS && near(it.begin * PA_STEP)) win = window(it.begin * PA_STEP);
  arrive(it.begin * PA_STEP, it.begin & 1);
  if (!sweep)  // then there are none
    for (; t < min(whole, it.end); ++t) whole_tile(t);
  for (; t < it.end; ++t) {
    if (t == 0 && sweep) {  // with delta 0 the sum of dS was delta
      delta = pa_half_sum(rest);
      rest = 0.f;
    }
    any_tile(t);
  }

  rest = pa_half_sum(rest);
  if (it.slot >= 0) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *pa_sums(p.work_q, it.slot, p.H, h, DT * 4, t * 4 + g) =
            f32x4{acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2],
                  acc[t][4 * g + 3]};
    if (half == 0) {
      float* to = pa_rows(p.work_q, it.slot, p.H, h, wave * 32 + col);
      to[0] = delta;
      to[1] = rest;
    }
    return;
  }
  pa_bwd_q_end<W, DT>(p, it.first, row, len, h, acc, 0, delta + rest);
}

// The sum of a tile's chunks: 32 elements of its rows, accumulators
// 4 t .. 4 t + 3 of n.  Four chunks' loads together in flight, added in
// their order.
__device__ PA_INLINE f32x16 pa_joined(const PaWork& w, const PaJoin& j,
                                      int heads, int h, int n, int t) {
  f32x16 acc = pa_zero16();
  for (int i0 = 0; i0 < j.n; i0 += 4) {
    f32x4 x[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        x[i][g] = *pa_sums(w, j.slot + min(i0 + i, j.n - 1), heads, h, n,
                           t * 4 + g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i0 + i >= j.n) break;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] += x[i][r >> 2][r & 3];
    }
  }
  return acc;
}

// Tiles in several chunks; blockIdx.y: 32 elements of the rows.
template <int DP, int W>
__global__ void __launch_bounds__(PA_BLOCK)
pa_bwd_q_join_kernel(const PaBwd p) {
  const int h = blockIdx.x % p.H;
  const PaJoin j = p.work_q.joins[blockIdx.x / p.H];
  const int in = (threadIdx.x >> 6) * 32 + (threadIdx.x & 31);
  float delta = pa_rows(p.work_q, j.slot, p.H, h, in)[0];
  for (int i = 0; i < j.n; ++i)
    delta += pa_rows(p.work_q, j.slot + i, p.H, h, in)[1];
  const f32x16 acc[1] = {
      pa_joined(p.work_q, j, p.H, h, DP / 8, blockIdx.y)};
  pa_bwd_q_end<W, 1>(p, j.first, j.tile * PA_ROWS + in, j.len, h, acc,
                     blockIdx.y, delta);
}

// N x 32 elements of a key row's gradient from 32 * t0 on.
template <int W, int N>
__device__ PA_INLINE void pa_bwd_kv_end(const PaBwd& p, void* out, long row,
                                        int hk, const f32x16 (&acc)[N],
                                        int t0, float scale) {
  const int half = (threadIdx.x & 63) >> 5;
  __bf16* to = static_cast<__bf16*>(out) + (row * (p.H / p.G) + hk) * p.D;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bf16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (__bf16)(acc[t][4 * g + e] * scale);
      pa_store4<W>(to, (t0 + t) * 32 + 8 * g + 4 * half, p.D, v);
    }
}

// Rows of a streamed tile: LDS holds two tiles of queries and two of
// gradients next to 128 values, for two workgroups a CU.  Heads of 64 with
// 32 rows: 198 us for 177 (one of 4001, 12 heads, a bias).
template <int DP>
struct PaKeys {
  static const int ROWS = DP == 64 ? 64 : 32;
};

// Three waves a SIMD where 168 registers do; with a bias they spill (five
// of 4096 in all, 16 heads of 64: 119 -> 159 us), so two there.
template <int DP, int W, bool BIAS, typename BiasArg>
__global__ void __launch_bounds__(PA_BLOCK, DP == 64 && !BIAS ? 3 : 2)
pa_bwd_kv_kernel(const PaBwd p, const BiasArg bias) {
  const int KS = DP / 16, DT = DP / 32;
  const int ROWS = PaKeys<DP>::ROWS;  // of a streamed tile
  const int TILE = ROWS * DP;
  __shared__ __attribute__((aligned(1024)))
  __bf16 s_tiles[4 + PA_ROWS / ROWS][TILE];
  __bf16 (*s_q)[TILE] = s_tiles, (*s_g)[TILE] = s_tiles + 2;
  __bf16* s_v = s_tiles[4];
  __shared__ __attribute__((aligned(16))) float s_l[2][ROWS];
  __shared__ __attribute__((aligned(16))) float s_delta[2][ROWS];
  __shared__ __attribute__((aligned(16))) float s_m[2][BIAS ? ROWS : 4];
  __shared__ float s_win[BIAS ? 2 : 1][BIAS ? 192 : 1];
  __shared__ int s_start[BIAS ? PA_MAXBUCKETS : 1];
  // far bias of each head of the group, buckets by distance
  __shared__ float s_far[BIAS ? PA_FARHEADS : 1];
  __shared__ unsigned char s_bucket[BIAS ? PA_DISTANCES : 1];
  // sums of each wave by distance, or by bucket where far_from is larger
  __shared__ float s_sums[BIAS ? 4 : 1][BIAS ? PA_DISTANCES : 1];
  __shared__ float s_far_sum[BIAS ? 4 : 1];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int kvh = p.H / p.G;
  const int hk = pa_head(blockIdx.x % kvh, kvh);
  const long chunk = blockIdx.x / kvh;
  const PaChunk it = p.work_kv.chunks[chunk];
  const int c0 = it.tile * PA_ROWS;  // first key of the workgroup
  const int w0 = c0 + wave * 32;
  const int key = w0 + col;
  const int len = it.len;
  // query tiles from the first that sees a key, for each head
  const int nt = (len - c0 + ROWS - 1) / ROWS;

  float far_bias = 0.f, next_far = 0.f;  // of this and the next step
  int far_from = 0;
  if constexpr (BIAS) far_from = bias.starts[bias.buckets - 1];

  // The order of the steps: first the tiles that need neither a mask nor
  // the table's sums, from the sequence's end backwards and every head of
  // a tile in turn, so that the workgroups of a sequence read the same
  // queries at the same time, from L2; then the others, head by head (with
  // the table's sums all of them).
  int other = min(PA_ROWS / ROWS, nt);  // tiles of the second part
  if (BIAS && p.part) other = nt;
  const int h0 = hk * p.G, bulk = (nt - other) * p.G;
  // tile and head of a step
  auto tile_of = [&](int s) PA_INLINE {
    return s < bulk ? nt - 1 - s / p.G : other - 1 - (s - bulk) % other;
  };
  auto head_of = [&](int s) PA_INLINE {
    return s < bulk ? s % p.G : (s - bulk) / other;
  };
  int step = it.begin, t = tile_of(step), g = head_of(step);

  // all that the first step needs is under way before any is waited for
  if (p.D < DP) {
    pa_clear<DP>(s_q[0], 2 * ROWS);
    pa_clear<DP>(s_g[0], 2 * ROWS);
    pa_clear<DP>(s_v, PA_ROWS);
    __syncthreads();
  }
  PaStage<DP, W, ROWS> qs(pa_at(p.q, it.first, h0 + g), p.q.row, len, p.D);
  PaStage<DP, W, ROWS> gs(pa_at(p.go, it.first, h0 + g), p.go.row, len, p.D);
  PaStage<DP, W, ROWS> vs(pa_at(p.v, it.first, hk), p.v.row, len, p.D);
  for (int r = 0; r < PA_ROWS && c0 + r < len; r += ROWS)
    vs.start(c0 + r, s_v + r * DP);
  qs.start(c0 + t * ROWS, s_q[step & 1]);
  gs.start(c0 + t * ROWS, s_g[step & 1]);

  if constexpr (BIAS) {
    for (int b = threadIdx.x; b < bias.buckets; b += PA_BLOCK)
      s_start[b] = bias.starts[b];
    for (int i = threadIdx.x; i < 4 * PA_DISTANCES; i += PA_BLOCK)
      s_sums[0][i] = 0.f;
    for (int x = threadIdx.x; x < min(p.G, PA_FARHEADS); x += PA_BLOCK)
      s_far[x] = pa_bias(pa_table(bias, bias.buckets - 1, p.H, hk * p.G + x),
                         bias.is_bf16);
    __syncthreads();
    for (int n = threadIdx.x; n < PA_DISTANCES; n += PA_BLOCK)
      s_bucket[n] = pa_bucket(s_start, bias.buckets, n);
    __syncthreads();
  }
  // Nothing that a step asks memory for is looked at before the step ends:
  // a wait for it would be a wait for the tiles asked for before.
  auto near = [&](int q0, float far) PA_INLINE {
    return q0 - c0 - (PA_ROWS - 1) < far_from || !pa_moderate(far);
  };
  auto window = [&](int q0, int h) PA_INLINE {
    unsigned x = 0;
    if constexpr (BIAS) {
      const int n = max(q0 - c0 - (PA_ROWS - 1) + (int)threadIdx.x, 0);
      const int b = n >= far_from      ? bias.buckets - 1
                    : n < PA_DISTANCES ? s_bucket[n]
                                       : pa_bucket(s_start, bias.buckets, n);
      x = pa_table(bias, b, p.H, h);
    }
    return x;
  };

  bf16x8 kf[KS];
  {
    const __bf16* kb = pa_at(p.k, (long)it.first + min(key, len - 1), hk);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      kf[s] = pa_load8<W>(kb, s * 16 + half * 8, p.D);
  }
  // scores are exponents of 2, as in the forward
  const float mul = p.scale * PA_LOG2E;

  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[t] = dv[t] = pa_zero16();

  unsigned win = 0;
  float st_l = 0.f, st_d = 0.f, st_m = 0.f;
  // what goes with a tile: its rows' statistics, its window
  auto start_rows = [&](int q0, int h) PA_INLINE {
    if constexpr (BIAS) {
      const int g = h - hk * p.G;
      next_far = g < PA_FARHEADS
                     ? s_far[g]
                     : pa_bias(pa_table(bias, bias.buckets - 1, p.H, h),
                               bias.is_bf16);
      if (near(q0, next_far)) win = window(q0, h);
    }
    const int r = min(q0 + (int)(threadIdx.x & (ROWS - 1)), len - 1);
    const long at = (long)h * p.T + it.first + r;
    if constexpr (BIAS) {
      st_m = p.stats[2 * at];
      st_l = p.stats[2 * at + 1];
    } else {
      st_l = p.stats[at];
    }
    st_d = p.delta[at];
  };
  auto start = [&](int q0, int h, int buf) PA_INLINE {
    qs.base = pa_at(p.q, it.first, h);
    gs.base = pa_at(p.go, it.first, h);
    qs.start(q0, s_q[buf]);
    gs.start(q0, s_g[buf]);
    start_rows(q0, h);
  };
  auto arrive = [&](int q0, int buf) PA_INLINE {
    qs.arrive(q0, s_q[buf]);
    gs.arrive(q0, s_g[buf]);
    const bool each = BIAS && near(q0, next_far);
    // a tile of one bias: all in one
    if (BIAS && !each) st_l -= next_far - st_m;
    // rows behind the sequence: weights of exp2(-inf)
    if (q0 + (int)threadIdx.x >= len) st_l = INFINITY;
    if (threadIdx.x < ROWS) {
      s_l[buf][threadIdx.x] = st_l;
      s_delta[buf][threadIdx.x] = st_d;
      if (BIAS) s_m[buf][threadIdx.x] = st_m;
    }
    if constexpr (BIAS) {
      if (each && threadIdx.x < 192)
        s_win[buf][threadIdx.x] = pa_bias(win, bias.is_bf16);
    }
    far_bias = next_far;
    __syncthreads();
  };

  const PaFrags<DP> lanes(s_tiles, lane);
  PaFrags<DP> frags = lanes;  // of the current buffer
  // s: the weights, dp: their gradient, of queries 32 j .. of a tile
  auto gradient = [&](f32x16& s, f32x16& dp, int q0, int j,
                      int buf) PA_INLINE {
    const unsigned from = j * 32 * DP * 2;
    const PaFrags<DP> vfrags = lanes.fresh(wave * (32 * DP * 2));
    s = dp = pa_zero16();
#pragma unroll
    for (int x = 0; x < KS; ++x)
      s = pa_mfma(frags.rows(from, x), kf[x], s);
#pragma unroll
    for (int x = 0; x < KS; ++x)
      dp = pa_mfma(frags.rows(from + 2 * TILE * 2, x),
                   vfrags.rows(4 * TILE * 2, x), dp);
    bool each = false;
    if constexpr (BIAS) each = near(q0, far_bias);
    const float a = each ? 1.f : mul;
    if (each) {
      const float* w = s_win[BIAS ? buf : 0] + PA_ROWS - 1 - wave * 32 - col;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * j + 8 * g + 4 * half;
        const f32x4 mv = *reinterpret_cast<const f32x4*>(
            &s_m[buf][BIAS ? at : 0]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[4 * g + e] = fmaf(s[4 * g + e], mul, w[at + e]) - mv[e];
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int at = 32 * j + 8 * g + 4 * half;
      const f32x4 lv = *reinterpret_cast<const f32x4*>(&s_l[buf][at]);
      const f32x4 ev = *reinterpret_cast<const f32x4*>(&s_delta[buf][at]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * g + e;
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a, -lv[e]));
        dp[r] = s[r] * (dp[r] - ev[e]);
      }
    }
  };
  float far_sum = 0.f;  // this lane's part of the last bucket
  auto table_sums = [&](const f32x16& dp, int q0) PA_INLINE {
    if constexpr (BIAS) {
      if (!p.part) return;
      const int n0 = q0 - w0;  // distance of diagonal 0
      f32x16 mine = dp;
      if (key >= len) mine = pa_zero16();
      // rows behind the sequence have weights of 0, but repeat a row that
      // may hold no numbers
      if (q0 + 31 >= len)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (q0 + 8 * (r >> 2) + 4 * half + (r & 3) >= len) mine[r] = 0.f;
      if (n0 - 31 >= far_from) {
        float sum[4] = {};
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r & 3] += mine[r];
        far_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      } else if (far_from <= PA_DISTANCES) {
        pa_add_diagonals(mine, n0, far_from, s_sums[wave], far_sum, lane);
      } else {
        pa_add_buckets(mine, n0, s_start, bias.buckets, s_sums[wave], lane);
      }
    }
  };
  // with 16 of its queries, 16 x ..
  auto product = [&](bf16x8 pw, bf16x8 sw, int x) PA_INLINE {
#pragma unroll
    for (int d = 0; d < DT; ++d)
      dv[d] = pa_mfma(
          frags.cols((2 * ROWS + x * 16) * DP * 2, d), pw, dv[d]);
#pragma unroll
    for (int d = 0; d < DT; ++d)
      dk[d] = pa_mfma(frags.cols(x * 16 * DP * 2, d), sw, dk[d]);
  };

  // Step `step`: query tile q0 of a head; q1 and h1 are the next step's.
  auto any_tile = [&](int step, int q0, int q1, int h1) PA_INLINE {
    const int buf = step & 1;
    const bool more = step + 1 < it.end;
    if (more) start(q1, h1, buf ^ 1);
    frags = lanes.fresh(buf * TILE * 2);
    bf16x8 pw[ROWS / 16], sw[ROWS / 16];
#pragma unroll
    for (int j = 0; j < ROWS / 32; ++j) {
      if (q0 + 32 * j + 31 < w0) continue;
      f32x16 s, dp;
      gradient(s, dp, q0, j, buf);
      const int lim = key - q0 - 32 * j - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) < lim) s[r] = dp[r] = 0.f;
      table_sums(dp, q0 + 32 * j);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        pw[2 * j + x] = pa_operand(s, x);
        sw[2 * j + x] = pa_operand(dp, x);
      }
    }
    if (__syncthreads_or(pa_tile_nonfinite<DP, ROWS>(s_q[buf]) ||
                         pa_tile_nonfinite<DP, ROWS>(s_g[buf]))) {
      pa_poison<DP, ROWS, false>(s_g[buf], dv, key - q0, lane);
      pa_poison<DP, ROWS, false>(s_q[buf], dk, key - q0, lane);
      __syncthreads();
      pa_cleanse<DP, ROWS>(s_g[buf]);
      pa_cleanse<DP, ROWS>(s_q[buf]);
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < ROWS / 16; ++x)
      if (q0 + 32 * (x >> 1) + 31 >= w0) product(pw[x], sw[x], x);
    if (more) arrive(q1, buf ^ 1);
  };
  auto whole_tile = [&](int step, int q0, int q1, int h1) PA_INLINE {
    const int buf = step & 1;
    const bool more = step + 1 < it.end;
    if (more) start(q1, h1, buf ^ 1);
    frags = lanes.fresh(buf * TILE * 2);
#pragma unroll
    for (int j = 0; j < ROWS / 32; ++j) {
      f32x16 s, dp;
      gradient(s, dp, q0, j, buf);
      table_sums(dp, q0 + 32 * j);
      product(pa_operand(s, 0), pa_operand(dp, 0), 2 * j);
      product(pa_operand(s, 1), pa_operand(dp, 1), 2 * j + 1);
    }
    if (more) arrive(q1, buf ^ 1);
  };

  start_rows(c0 + t * ROWS, h0 + g);
  for (int r = 0; r < PA_ROWS && c0 + r < len; r += ROWS)
    vs.arrive(c0 + r, s_v + r * DP);
  arrive(c0 + t * ROWS, step & 1);
  auto go = [&](auto tile) PA_INLINE {
    const int q0 = c0 + t * ROWS;
    const bool last = step + 1 < bulk ? g + 1 == p.G : t == 0;
    if (step + 1 < bulk) {
      t -= last;
      g = last ? 0 : g + 1;
    } else if (step + 1 == bulk) {
      t = other - 1;
      g = 0;
    } else {
      g += last;
      t = last ? other - 1 : t - 1;
    }
    tile(step++, q0, c0 + t * ROWS, h0 + g);
  };
  while (step < min(bulk, it.end)) go(whole_tile);
  const int g_first = g;
  while (step < it.end) {
    const int head = g;
    const int stop = min(bulk + (head + 1) * other, it.end);
    while (t >= PA_ROWS / ROWS && step < stop) go(whole_tile);
    while (step < stop) go(any_tile);
    if constexpr (BIAS) {
      if (p.part) {
        far_sum = wave_reduce_sum(far_sum);
        if (lane == 0) s_far_sum[wave] = far_sum;
        far_sum = 0.f;
        __syncthreads();
        float* out = p.part + (chunk * p.H + h0 + head) * bias.buckets;
        const bool by_distance = far_from <= PA_DISTANCES;
        // eight threads a bucket
        for (int b = threadIdx.x >> 3; b < bias.buckets; b += PA_BLOCK / 8) {
          const int from = by_distance ? s_start[b] : b;
          const int to = !by_distance              ? b + 1
                         : b + 1 < bias.buckets ? s_start[b + 1]
                                                : from;
          float v = 0.f;
          for (int n = from + (threadIdx.x & 7); n < to; n += 8)
            v += (s_sums[0][n] + s_sums[1][n]) +
                 (s_sums[2][n] + s_sums[3][n]);
          v += __shfl_xor(v, 1, 64);
          v += __shfl_xor(v, 2, 64);
          v += __shfl_xor(v, 4, 64);
          if (b == bias.buckets - 1)
            v += (s_far_sum[0] + s_far_sum[1]) +
                 (s_far_sum[2] + s_far_sum[3]);
          if ((threadIdx.x & 7) == 0) out[b] = v;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 4 * PA_DISTANCES; i += PA_BLOCK)
          s_sums[0][i] = 0.f;
        __syncthreads();
      }
    }
  }
  if constexpr (BIAS) {
    if (p.part) {  // heads that only other chunks have sums for
      const int g_end = (it.end - 1) / other;
      for (int x = 0; x < p.G; ++x)
        if (x < g_first || x > g_end)
          for (int b = threadIdx.x; b < bias.buckets; b += PA_BLOCK)
            p.part[(chunk * p.H + h0 + x) * bias.buckets + b] = 0.f;
    }
  }

  if (it.slot >= 0) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        *pa_sums(p.work_kv, it.slot, kvh, hk, DT * 8, t * 8 + g) =
            f32x4{dk[t][4 * g], dk[t][4 * g + 1], dk[t][4 * g + 2],
                  dk[t][4 * g + 3]};
        *pa_sums(p.work_kv, it.slot, kvh, hk, DT * 8, t * 8 + 4 + g) =
            f32x4{dv[t][4 * g], dv[t][4 * g + 1], dv[t][4 * g + 2],
                  dv[t][4 * g + 3]};
      }
    return;
  }
  if (key < len) {
    const long at = (long)it.first + key;
    pa_bwd_kv_end<W, DT>(p, p.dk, at, hk, dk, 0, p.scale);
    pa_bwd_kv_end<W, DT>(p, p.dv, at, hk, dv, 0, 1.f);
  }
}

// Tiles in several chunks; blockIdx.y: 32 elements of dK's rows or dV's.
template <int DP, int W>
__global__ void __launch_bounds__(PA_BLOCK)
pa_bwd_kv_join_kernel(const PaBwd p) {
  const int kvh = p.H / p.G, hk = blockIdx.x % kvh;
  const PaJoin j = p.work_kv.joins[blockIdx.x / kvh];
  const int key = j.tile * PA_ROWS + (threadIdx.x >> 6) * 32 +
                  (threadIdx.x & 31);
  const f32x16 acc[1] = {
      pa_joined(p.work_kv, j, kvh, hk, DP / 4, blockIdx.y)};
  const bool v = blockIdx.y & 1;
  if (key < j.len)
    pa_bwd_kv_end<W, 1>(p, v ? p.dv : p.dk, (long)j.first + key, hk, acc,
                        blockIdx.y >> 1, v ? 1.f : p.scale);
}

// dtable[b, h] from the chunks' partial sums; a workgroup a head, a lane a
// bucket, the chunks by turns to the waves, every sum in a fixed order.  42
// chunks of 16 heads: 2 us less than a wave a bucket and a lane a chunk.
#define PA_TABLE_WAVES 16
__global__ void __launch_bounds__(PA_TABLE_WAVES * 64)
pa_table_grad_kernel(const float* __restrict__ part, void* out, int is_bf16,
                     long chunks, int H, int buckets) {
  __shared__ float s_part[PA_TABLE_WAVES][64];
  const int h = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b0 = 0; b0 < buckets; b0 += 64) {
    const int b = min(b0 + lane, buckets - 1);
    float v[4] = {};
    for (long i = wave; i < chunks; i += 4 * PA_TABLE_WAVES)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long at = i + u * PA_TABLE_WAVES;
        const float x = part[(min(at, chunks - 1) * H + h) * buckets + b];
        v[u] += at < chunks ? x : 0.f;
      }
    s_part[wave][lane] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (wave == 0 && b0 + lane < buckets) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < PA_TABLE_WAVES; ++w) x += s_part[w][lane];
      const long at = (long)b * H + h;
      if (is_bf16)
        static_cast<__bf16*>(out)[at] = (__bf16)x;
      else
        static_cast<float*>(out)[at] = x;
    }
    __syncthreads();
  }
}

template <int DP, int W>
static void pa_bwd_q_go(const PaBwd& p, const PaBias* bias,
                        hipStream_t stream) {
  const dim3 block(PA_BLOCK), grid((unsigned)p.work_q.n_chunks * p.H);
  const dim3 joins((unsigned)p.work_q.n_joins * p.H, DP / 32);
  if (bias)
    hipLaunchKernelGGL((pa_bwd_q_kernel<DP, W, true, PaBias>), grid, block, 0,
                       stream, p, *bias);
  else
    hipLaunchKernelGGL((pa_bwd_q_kernel<DP, W, false, PaNoBias>), grid, block,
                       0, stream, p, PaNoBias{});
  if (joins.x)
    hipLaunchKernelGGL((pa_bwd_q_join_kernel<DP, W>), joins, block, 0, stream,
                       p);
}

template <int DP, int W>
static void pa_bwd_kv_go(const PaBwd& p, const PaBias* bias,
                         hipStream_t stream) {
  const unsigned kvh = p.H / p.G;
  const dim3 block(PA_BLOCK), grid(p.work_kv.n_chunks * kvh);
  const dim3 joins(p.work_kv.n_joins * kvh, DP / 16);
  if (bias)
    hipLaunchKernelGGL((pa_bwd_kv_kernel<DP, W, true, PaBias>), grid, block,
                       0, stream, p, *bias);
  else
    hipLaunchKernelGGL((pa_bwd_kv_kernel<DP, W, false, PaNoBias>), grid,
                       block, 0, stream, p, PaNoBias{});
  if (joins.x)
    hipLaunchKernelGGL((pa_bwd_kv_join_kernel<DP, W>), joins, block, 0,
                       stream, p);
}

#define PA_BWD_GO(GO)                                   \
  {                                                     \
    auto go = [&](auto go64, auto go128) {              \
      (p->D <= 64 ? go64 : go128)(*p, bias, stream);    \
    };                                                  \
    if (width == 16) go(GO<64, 16>, GO<128, 16>);       \
    else if (width == 4) go(GO<64, 4>, GO<128, 4>);     \
    else go(GO<64, 2>, GO<128, 2>);                     \
  }

// The two halves, so that the host can go on with the second's results
// while the first runs.  Queries: dq and delta.  width: as in the forward.
extern "C" void dlb_packed_attn_bwd_q(const PaBwd* p, const PaBias* bias,
                                      int width, hipStream_t stream) {
  PA_BWD_GO(pa_bwd_q_go)
}

// Keys, behind the queries: dk, dv and the table's gradient.
extern "C" void dlb_packed_attn_bwd_kv(const PaBwd* p, const PaBias* bias,
                                       int width, void* dtable,
                                       int dtable_bf16, hipStream_t stream) {
  PA_BWD_GO(pa_bwd_kv_go)
  if (bias && dtable)
    hipLaunchKernelGGL(pa_table_grad_kernel, dim3(p->H),
                       dim3(PA_TABLE_WAVES * 64), 0, stream, p->part, dtable,
                       dtable_bf16, (long)p->work_kv.n_chunks, p->H,
                       bias->buckets);
}
