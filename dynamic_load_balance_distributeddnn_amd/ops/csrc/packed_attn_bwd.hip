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
#include "packed_attn.h"

// Sums of the table's gradient over one 32 x 32 block of dS (queries x
// keys, the result layout; masked pairs 0): lane l first collects the
// diagonals l & 31 and (l & 31) - 32, then neighbouring diagonals of one
// bucket are added up lane by lane, in a fixed order.  `n0` is the
// distance of diagonal 0.  The last bucket is left out: a row's dS sum to
// 0, so it is minus the sum of the others.
__device__ inline void pa_bias_sums(const f32x16& ds, int n0,
                                    const int* starts, int buckets,
                                    float* hist, int lane) {
  const int x = lane & 31, half = lane >> 5;
  float hi = 0.f, lo = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = 8 * (r >> 2) + 4 * half + (r & 3);
    const float v = __shfl(ds[r], ((i - x) & 31) + 32 * half, 64);
    if (x <= i) hi += v; else lo += v;
  }
  hi = pa_half_sum(hi);
  lo = pa_half_sum(lo);
  float v = half ? lo : hi;
  const int z = lane ^ 32;  // diagonals in the order of their distance
  const int n = n0 - 32 + z;
  const int b = n < 0 ? -1 : pa_bucket(starts, buckets, n);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int src = ((z - off) & 63) ^ 32;
    const float pv = __shfl(v, src, 64);
    const int pb = __shfl(b, src, 64);
    if (z >= off && pb == b) v += pv;
  }
  const int nb = __shfl(b, ((z + 1) & 63) ^ 32, 64);
  if (b >= 0 && b < buckets - 1 && (z == 63 || nb != b)) hist[b] += v;
}

template <int DP, bool VEC, bool BIAS, typename BiasArg>
__global__ void __launch_bounds__(PA_BLOCK, 2)
pa_bwd_q_kernel(const PaBwd p, const BiasArg bias) {
  const int KS = DP / 16, DT = DP / 32;
  __shared__ __attribute__((aligned(16))) __bf16 s_k[2][PA_STEP * DP];
  __shared__ __attribute__((aligned(16))) __bf16 s_v[2][PA_STEP * DP];
  __shared__ float s_win[BIAS ? 2 : 1][BIAS ? 192 : 1];
  __shared__ float s_tab[BIAS ? PA_MAXBUCKETS : 1];
  __shared__ int s_start[BIAS ? PA_MAXBUCKETS : 1];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, half = lane >> 5;
  const int h = pa_head(blockIdx.x % p.H, p.H);
  const PaItem it = p.items[blockIdx.x / p.H];
  const int r0 = it.tile * PA_ROWS;
  const int w0 = r0 + wave * 32;
  const int row = w0 + col;
  const int len = it.len;
  const int tiles = (min(r0 + PA_ROWS, len) + PA_STEP - 1) / PA_STEP;
  const __bf16* kb = pa_at(p.k, it.first, h / p.G);
  const __bf16* vb = pa_at(p.v, it.first, h / p.G);

  float far_bias = 0.f;
  int far_from = 0;
  if constexpr (BIAS) {
    for (int b = threadIdx.x; b < bias.buckets; b += PA_BLOCK) {
      s_tab[b] = pa_table(bias, b, p.H, h);
      s_start[b] = bias.starts[b];
    }
    __syncthreads();
    far_bias = s_tab[bias.buckets - 1];
    far_from = s_start[bias.buckets - 1];
  }
  auto window = [&](int k0) {
    float x = 0.f;
    if constexpr (BIAS) {
      const int n = r0 - k0 - (PA_STEP - 1) + (int)threadIdx.x;
      if (n >= 0) x = s_tab[pa_bucket(s_start, bias.buckets, n)];
    }
    return x;
  };
  auto near = [&](int k0) { return r0 - k0 - (PA_STEP - 1) < far_from; };

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
      const int dd = VEC ? min(d, p.D - 8) : min(d, p.D - 1);
      qf[s] = pa_load8<VEC>(qb + dd, p.D - d);
      gf[s] = pa_load8<VEC>(gb + dd, p.D - d);
      if (!sweep) {
        const bf16x8 of = pa_load8<VEC>(ob + dd, p.D - d);
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
  const float to2 = BIAS ? PA_LOG2E : p.scale * PA_LOG2E;

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = pa_zero16();

  PaStage<DP, VEC> ks, vs;
  float win = 0.f;
  ks.load(kb, p.k.row, 0, len, p.D);
  vs.load(vb, p.v.row, 0, len, p.D);
  const int buf0 = sweep ? -tiles & 1 : 0;
  ks.store(s_k[buf0]);
  vs.store(s_v[buf0]);
  if constexpr (BIAS) {
    if (threadIdx.x < 192) s_win[buf0][threadIdx.x] = window(0);
  }
  bool bad = __syncthreads_or(PA_STEP > r0 && ks.nonfinite());

  for (int t = sweep ? -tiles : 0; t < tiles; ++t) {
    if (t == 0 && sweep) {  // with delta 0 the sum of dS was delta
      delta = pa_half_sum(rest);
      rest = 0.f;
    }
    const int k0 = (t < 0 ? t + tiles : t) * PA_STEP, buf = t & 1;
    const bool more = t + 1 < tiles;
    const int k1 = t == -1 ? 0 : k0 + PA_STEP;  // of the next tile
    if (more) {
      ks.load(kb, p.k.row, k1, len, p.D);
      vs.load(vb, p.v.row, k1, len, p.D);
      if (BIAS && near(k1)) win = window(k1);
    }
    const bool works = k0 <= w0 + 31;
    bf16x8 w[4];
    if (works) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f32x16 s = pa_zero16(), dp = pa_zero16();
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          s = pa_mfma(pa_row_frag<DP>(s_k[buf], j * 32 + col, 2 * x + half),
                      qf[x], s);
          dp = pa_mfma(pa_row_frag<DP>(s_v[buf], j * 32 + col, 2 * x + half),
                       gf[x], dp);
        }
        if constexpr (BIAS) {
          if (near(k0)) {
            const float* win_at = s_win[buf] + wave * 32 + col + PA_STEP - 1;
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[r] = fmaf(s[r], p.scale,
                          win_at[-(j * 32 + 8 * (r >> 2) + 4 * half +
                                   (r & 3))]);
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[r] = fmaf(s[r], p.scale, far_bias);
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = BIAS ? fmaf(s[r] - stat_m, to2, -stat_l)
                               : fmaf(s[r], to2, -stat_l);
          s[r] = __builtin_amdgcn_exp2f(e) * (dp[r] - delta);
        }
        if (k0 + PA_STEP - 1 > w0) {
          const int lim = row - k0 - 4 * half;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j * 32 + 8 * (r >> 2) + (r & 3) > lim) s[r] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) rest += s[r];
        w[2 * j] = pa_operand(s, 0);
        w[2 * j + 1] = pa_operand(s, 1);
      }
    }
    if (bad && t >= 0) {
      __syncthreads();
      pa_poison<DP, true>(s_k[buf], acc, row - k0, lane);
      __syncthreads();
      pa_cleanse<DP>(s_k[buf]);
      __syncthreads();
    }
    if (works && t >= 0) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          acc[d] = pa_mfma(pa_col_frag<DP>(s_k[buf], x * 16, d * 32, lane),
                           w[x], acc[d]);
    }
    if (more) {
      ks.store(s_k[buf ^ 1]);
      vs.store(s_v[buf ^ 1]);
      if (BIAS && near(k1) && threadIdx.x < 192)
        s_win[buf ^ 1][threadIdx.x] = win;
      if (k1 + PA_STEP > r0)
        bad = __syncthreads_or(ks.nonfinite());
      else
        __syncthreads();
    }
  }

  delta += pa_half_sum(rest);
  if (row < len) {
    if (half == 0) p.delta[(long)h * p.T + it.first + row] = delta;
    __bf16* ob = static_cast<__bf16*>(p.dq) +
                 (((long)it.first + row) * p.H + h) * p.D;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = t * 32 + 8 * g + 4 * half;
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = (__bf16)(acc[t][4 * g + e] * p.scale);
        if (VEC) {
          if (d < p.D) *reinterpret_cast<bf16x4*>(ob + d) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < p.D) ob[d + e] = v[e];
        }
      }
  }
}

template <int DP, bool VEC, bool BIAS, typename BiasArg>
__global__ void __launch_bounds__(PA_BLOCK, 1)
pa_bwd_kv_kernel(const PaBwd p, const BiasArg bias) {
  const int KS = DP / 16, DT = DP / 32;
  __shared__ __attribute__((aligned(16))) __bf16 s_q[2][PA_STEP * DP];
  __shared__ __attribute__((aligned(16))) __bf16 s_g[2][PA_STEP * DP];
  __shared__ __attribute__((aligned(16))) float s_l[2][PA_STEP];
  __shared__ __attribute__((aligned(16))) float s_delta[2][PA_STEP];
  __shared__ __attribute__((aligned(16))) float s_m[2][BIAS ? PA_STEP : 4];
  __shared__ float s_win[BIAS ? 2 : 1][BIAS ? 192 : 1];
  __shared__ int s_start[BIAS ? PA_MAXBUCKETS : 1];
  __shared__ float s_hist[BIAS ? 4 : 1][BIAS ? PA_MAXBUCKETS : 1];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, half = lane >> 5;
  const int kvh = p.H / p.G;
  const int hk = pa_head(blockIdx.x % kvh, kvh);
  const long item = blockIdx.x / kvh;
  const PaItem it = p.items[item];
  const int c0 = it.tile * PA_ROWS;  // first key of the block
  const int w0 = c0 + wave * 32;
  const int key = w0 + col;
  const int len = it.len;
  const int t0 = c0 / PA_STEP;       // first query tile that sees one
  const int nt = (len + PA_STEP - 1) / PA_STEP - t0;
  const int steps = nt * p.G;

  float far_bias = 0.f;
  int far_from = 0;
  if constexpr (BIAS) {
    for (int b = threadIdx.x; b < bias.buckets; b += PA_BLOCK) {
      s_start[b] = bias.starts[b];
      for (int w = 0; w < 4; ++w) s_hist[w][b] = 0.f;
    }
    far_from = bias.starts[bias.buckets - 1];
  }
  auto near = [&](int q0) { return q0 - c0 - (PA_ROWS - 1) < far_from; };
  auto window = [&](int q0, int h) {
    float x = 0.f;
    if constexpr (BIAS) {
      const int n = q0 - c0 - (PA_ROWS - 1) + (int)threadIdx.x;
      if (n >= 0)
        x = pa_table(bias, pa_bucket(s_start, bias.buckets, n), p.H, h);
    }
    return x;
  };

  bf16x8 kf[KS], vf[KS];
  {
    const long rr = (long)it.first + min(key, len - 1);
    const __bf16* kb = pa_at(p.k, rr, hk);
    const __bf16* vb = pa_at(p.v, rr, hk);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + half * 8;
      const int dd = VEC ? min(d, p.D - 8) : min(d, p.D - 1);
      kf[s] = pa_load8<VEC>(kb + dd, p.D - d);
      vf[s] = pa_load8<VEC>(vb + dd, p.D - d);
    }
  }
  const float to2 = BIAS ? PA_LOG2E : p.scale * PA_LOG2E;

  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[t] = dv[t] = pa_zero16();

  PaStage<DP, VEC> qs, gs;
  float win = 0.f, st_l = 0.f, st_d = 0.f, st_m = 0.f;
  auto fetch = [&](int step) {
    const int h = hk * p.G + step / nt;
    const int q0 = (t0 + step % nt) * PA_STEP;
    qs.load(pa_at(p.q, it.first, h), p.q.row, q0, len, p.D);
    gs.load(pa_at(p.go, it.first, h), p.go.row, q0, len, p.D);
    if (threadIdx.x < PA_STEP) {
      // rows behind the sequence: weights of exp2(-inf)
      st_l = INFINITY;
      st_d = st_m = 0.f;
      const int r = q0 + (int)threadIdx.x;
      if (r < len) {
        const long at = (long)h * p.T + it.first + r;
        if constexpr (BIAS) {
          st_m = p.stats[2 * at];
          st_l = p.stats[2 * at + 1];
        } else {
          st_l = p.stats[at];
        }
        st_d = p.delta[at];
      }
    }
    if (BIAS) {
      if (near(q0)) win = window(q0, h);
      else win = 0.f;
    }
  };
  auto put = [&](int buf) {
    qs.store(s_q[buf]);
    gs.store(s_g[buf]);
    if (threadIdx.x < PA_STEP) {
      s_l[buf][threadIdx.x] = st_l;
      s_delta[buf][threadIdx.x] = st_d;
      if (BIAS) s_m[buf][threadIdx.x] = st_m;
    }
    if (BIAS && threadIdx.x < 192) s_win[buf][threadIdx.x] = win;
  };
  auto diagonal = [&](int step) {
    return (t0 + step % nt) * PA_STEP < c0 + PA_ROWS;
  };

  if (BIAS) __syncthreads();
  fetch(0);
  put(0);
  bool bad = __syncthreads_or(qs.nonfinite() || gs.nonfinite());
  int head_now = -1;

  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1;
    const int q0 = (t0 + step % nt) * PA_STEP;
    const bool more = step + 1 < steps;
    if (more) fetch(step + 1);
    if constexpr (BIAS) {
      const int h = hk * p.G + step / nt;
      if (h != head_now) {
        head_now = h;
        far_bias = pa_table(bias, bias.buckets - 1, p.H, h);
      }
    }
    const bool works = q0 + PA_STEP - 1 >= w0;
    bf16x8 pw[4], sw[4];
    if (works) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f32x16 s = pa_zero16(), dp = pa_zero16();
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          s = pa_mfma(pa_row_frag<DP>(s_q[buf], j * 32 + col, 2 * x + half),
                      kf[x], s);
          dp = pa_mfma(pa_row_frag<DP>(s_g[buf], j * 32 + col, 2 * x + half),
                       vf[x], dp);
        }
        if constexpr (BIAS) {
          if (near(q0)) {
            const float* win_at = s_win[buf] + PA_ROWS - 1 - wave * 32 - col;
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[r] = fmaf(s[r], p.scale,
                          win_at[j * 32 + 8 * (r >> 2) + 4 * half + (r & 3)]);
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[r] = fmaf(s[r], p.scale, far_bias);
          }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at = j * 32 + 8 * g + 4 * half;
          const f32x4 lv = *reinterpret_cast<const f32x4*>(&s_l[buf][at]);
          const f32x4 ev = *reinterpret_cast<const f32x4*>(&s_delta[buf][at]);
          f32x4 mv = {0.f, 0.f, 0.f, 0.f};
          if constexpr (BIAS)
            mv = *reinterpret_cast<const f32x4*>(&s_m[buf][at]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            s[r] = __builtin_amdgcn_exp2f(
                BIAS ? fmaf(s[r] - mv[e], to2, -lv[e])
                     : fmaf(s[r], to2, -lv[e]));
            dp[r] = s[r] * (dp[r] - ev[e]);
          }
        }
        if (q0 < w0 + 31) {
          const int lim = key - q0 - 4 * half;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j * 32 + 8 * (r >> 2) + (r & 3) < lim) s[r] = dp[r] = 0.f;
        }
        if constexpr (BIAS) {
          const int n0 = q0 + j * 32 - w0;  // of diagonal 0
          if (p.part && n0 - 31 < far_from) {
            f32x16 mine = dp;
            if (key >= len) mine = pa_zero16();
            pa_bias_sums(mine, n0, s_start, bias.buckets, s_hist[wave],
                         lane);
          }
        }
        pw[2 * j] = pa_operand(s, 0);
        pw[2 * j + 1] = pa_operand(s, 1);
        sw[2 * j] = pa_operand(dp, 0);
        sw[2 * j + 1] = pa_operand(dp, 1);
      }
    }
    if (bad) {
      __syncthreads();
      pa_poison<DP, false>(s_g[buf], dv, key - q0, lane);
      pa_poison<DP, false>(s_q[buf], dk, key - q0, lane);
      __syncthreads();
      pa_cleanse<DP>(s_g[buf]);
      pa_cleanse<DP>(s_q[buf]);
      __syncthreads();
    }
    if (works) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          dv[d] = pa_mfma(pa_col_frag<DP>(s_g[buf], x * 16, d * 32, lane),
                          pw[x], dv[d]);
          dk[d] = pa_mfma(pa_col_frag<DP>(s_q[buf], x * 16, d * 32, lane),
                          sw[x], dk[d]);
        }
    }
    if constexpr (BIAS) {
      if (p.part && (step + 1) % nt == 0) {  // a head is done
        __syncthreads();
        float* out = p.part +
                     (item * p.H + hk * p.G + step / nt) * bias.buckets;
        for (int b = threadIdx.x; b < bias.buckets; b += PA_BLOCK) {
          out[b] = (s_hist[0][b] + s_hist[1][b]) +
                   (s_hist[2][b] + s_hist[3][b]);
          for (int w = 0; w < 4; ++w) s_hist[w][b] = 0.f;
        }
      }
    }
    if (more) {
      put(buf ^ 1);
      if (diagonal(step + 1))
        bad = __syncthreads_or(qs.nonfinite() || gs.nonfinite());
      else {
        bad = false;
        __syncthreads();
      }
    }
  }

  if (key >= len) return;
  const long at = (((long)it.first + key) * kvh + hk) * p.D;
  __bf16* okb = static_cast<__bf16*>(p.dk) + at;
  __bf16* ovb = static_cast<__bf16*>(p.dv) + at;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = t * 32 + 8 * g + 4 * half;
      bf16x4 a, b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = (__bf16)(dk[t][4 * g + e] * p.scale);
        b[e] = (__bf16)dv[t][4 * g + e];
      }
      if (VEC) {
        if (d < p.D) {
          *reinterpret_cast<bf16x4*>(okb + d) = a;
          *reinterpret_cast<bf16x4*>(ovb + d) = b;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < p.D) {
            okb[d + e] = a[e];
            ovb[d + e] = b[e];
          }
      }
    }
}

// dtable[b, h] from the items' partial sums; a workgroup a head, a wave a
// bucket at a time, every sum in a fixed order.
__global__ void __launch_bounds__(PA_BLOCK)
pa_table_grad_kernel(const float* __restrict__ part, void* out, int is_bf16,
                     long items, int H, int buckets) {
  __shared__ float s_sum[PA_MAXBUCKETS];
  const int h = blockIdx.x, lane = threadIdx.x & 63;
  for (int b = threadIdx.x >> 6; b < buckets - 1; b += PA_BLOCK / 64) {
    float v = 0.f;
    for (long i = lane; i < items; i += 64)
      v += part[(i * H + h) * buckets + b];
    v = wave_reduce_sum(v);
    if (lane == 0) s_sum[b] = v;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = 0.f;
    for (int b = 0; b < buckets - 1; ++b) all += s_sum[b];
    s_sum[buckets - 1] = -all;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += PA_BLOCK) {
    const long at = (long)b * H + h;
    if (is_bf16)
      static_cast<__bf16*>(out)[at] = (__bf16)s_sum[b];
    else
      static_cast<float*>(out)[at] = s_sum[b];
  }
}

template <int DP, bool VEC>
static void pa_bwd_go(const PaBwd& p, const PaBwd& pk, const PaBias* bias,
                      unsigned grid, unsigned grid_kv, hipStream_t stream) {
  if (bias) {
    hipLaunchKernelGGL((pa_bwd_q_kernel<DP, VEC, true, PaBias>), dim3(grid),
                       dim3(PA_BLOCK), 0, stream, p, *bias);
    hipLaunchKernelGGL((pa_bwd_kv_kernel<DP, VEC, true, PaBias>),
                       dim3(grid_kv), dim3(PA_BLOCK), 0, stream, pk, *bias);
  } else {
    hipLaunchKernelGGL((pa_bwd_q_kernel<DP, VEC, false, PaNoBias>),
                       dim3(grid), dim3(PA_BLOCK), 0, stream, p, PaNoBias{});
    hipLaunchKernelGGL((pa_bwd_kv_kernel<DP, VEC, false, PaNoBias>),
                       dim3(grid_kv), dim3(PA_BLOCK), 0, stream, pk,
                       PaNoBias{});
  }
}

// `items_kv`: the same tiles as keys, longest remainder first.
extern "C" void dlb_packed_attn_bwd(const PaBwd* p, const PaBias* bias,
                                    const PaItem* items_kv, long items,
                                    int vec, void* dtable, int dtable_bf16,
                                    hipStream_t stream) {
  PaBwd pk = *p;
  pk.items = items_kv;
  const unsigned grid = (unsigned)(items * p->H);
  const unsigned grid_kv = (unsigned)(items * (p->H / p->G));
  if (p->D <= 64)
    vec ? pa_bwd_go<64, true>(*p, pk, bias, grid, grid_kv, stream)
        : pa_bwd_go<64, false>(*p, pk, bias, grid, grid_kv, stream);
  else
    vec ? pa_bwd_go<128, true>(*p, pk, bias, grid, grid_kv, stream)
        : pa_bwd_go<128, false>(*p, pk, bias, grid, grid_kv, stream);
  if (bias && dtable)
    hipLaunchKernelGGL(pa_table_grad_kernel, dim3(p->H), dim3(PA_BLOCK), 0,
                       stream, p->part, dtable, dtable_bf16, items, p->H,
                       bias->buckets);
}
