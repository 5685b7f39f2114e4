// Causal attention over packed sequences, forward (gfx950).
//
//   S_ij = scale q_i.k_j (+ bias of head h at distance i - j),  j <= i
//   O_i  = sum_j exp(S_ij - m_i) v_j / sum_j exp(S_ij - m_i)
//
// One pass over the keys with a running maximum m and sum l per row; the
// [n, n] scores are never stored.  A workgroup owns 128 query rows of one
// head, 32 a wave, and streams 64-key tiles through LDS; S is computed
// transposed (keys x queries) so that a lane holds one query's scores and
// the softmax needs one lane exchange a tile.  Rows of a sequence are
// found through the packing's item list, longest first.
#include "packed_attn.h"

template <int DP, bool VEC, bool BIAS, typename BiasArg>
__global__ void __launch_bounds__(PA_BLOCK, 2)
pa_fwd_kernel(const PaFwd p, const BiasArg bias) {
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
  const int w0 = r0 + wave * 32;     // this wave's first row
  const int row = w0 + col;          // this lane's
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
  // bias of the distances a 128 x 64 tile spans, r0 - k0 - 63 upwards
  auto window = [&](int k0) {
    float x = 0.f;
    if constexpr (BIAS) {
      const int n = r0 - k0 - (PA_STEP - 1) + (int)threadIdx.x;
      if (n >= 0) x = s_tab[pa_bucket(s_start, bias.buckets, n)];
    }
    return x;
  };
  auto near = [&](int k0) { return r0 - k0 - (PA_STEP - 1) < far_from; };

  bf16x8 qf[KS];
  {
    const __bf16* qb = pa_at(p.q, (long)it.first + min(row, len - 1), h);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + half * 8;
      qf[s] = pa_load8<VEC>(qb + (VEC ? min(d, p.D - 8) : min(d, p.D - 1)),
                            p.D - d);
    }
  }

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = pa_zero16();
  float m = -INFINITY;   // running maximum: of q.k, with bias of S
  float l = 0.f;         // this half's part of the sum
  const float to2 = BIAS ? PA_LOG2E : p.scale * PA_LOG2E;

  PaStage<DP, VEC> ks, vs;
  float win = 0.f;
  ks.load(kb, p.k.row, 0, len, p.D);
  vs.load(vb, p.v.row, 0, len, p.D);
  ks.store(s_k[0]);
  vs.store(s_v[0]);
  if constexpr (BIAS) {
    if (threadIdx.x < 192) s_win[0][threadIdx.x] = window(0);
  }
  bool bad = __syncthreads_or(PA_STEP > r0 && vs.nonfinite());

  for (int t = 0; t < tiles; ++t) {
    const int k0 = t * PA_STEP, buf = t & 1;
    const bool more = t + 1 < tiles;
    if (more) {
      ks.load(kb, p.k.row, k0 + PA_STEP, len, p.D);
      vs.load(vb, p.v.row, k0 + PA_STEP, len, p.D);
      if (BIAS && near(k0 + PA_STEP)) win = window(k0 + PA_STEP);
    }
    if (bad) {
      pa_poison<DP, true>(s_v[buf], acc, row - k0, lane);
      __syncthreads();
      pa_cleanse<DP>(s_v[buf]);
      __syncthreads();
    }
    if (k0 <= w0 + 31) {
      f32x16 s[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j] = pa_zero16();
#pragma unroll
        for (int x = 0; x < KS; ++x)
          s[j] = pa_mfma(pa_row_frag<DP>(s_k[buf], j * 32 + col,
                                         2 * x + half), qf[x], s[j]);
      }
      if constexpr (BIAS) {
        if (near(k0)) {
          const float* w = s_win[buf] + wave * 32 + col + (PA_STEP - 1);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[j][r] = fmaf(s[j][r], p.scale,
                             w[-(j * 32 + 8 * (r >> 2) + 4 * half + (r & 3))]);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[j][r] = fmaf(s[j][r], p.scale, far_bias);
        }
      }
      if (k0 + PA_STEP - 1 > w0) {
        const int lim = row - k0 - 4 * half;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j * 32 + 8 * (r >> 2) + (r & 3) > lim) s[j][r] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[j][r]);
      top = fmaxf(m, pa_half_max(top));
      // The sum and the output are held relative to m; they are scaled
      // anew only when a maximum grew by more than 2^8, which fp32 and
      // the bf16 weights (their step is relative) carry without loss.
      if (__any((top - m) * to2 > 8.f || m == -INFINITY)) {
        const float now = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f((m - now) * to2);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        l *= f;
        m = top;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      const float off = ref * to2;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          // with a bias the scores may stand at the type's lowest value:
          // the difference is taken before the change of base
          const float e = BIAS ? (s[j][r] - ref) * to2
                               : fmaf(s[j][r], to2, -off);
          s[j][r] = __builtin_amdgcn_exp2f(e);
          l += s[j][r];
        }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const bf16x8 w = pa_operand(s[x >> 1], x & 1);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          acc[d] = pa_mfma(pa_col_frag<DP>(s_v[buf], x * 16, d * 32, lane), w,
                           acc[d]);
      }
    }
    if (more) {
      ks.store(s_k[buf ^ 1]);
      vs.store(s_v[buf ^ 1]);
      if (BIAS && near(k0 + PA_STEP) && threadIdx.x < 192)
        s_win[buf ^ 1][threadIdx.x] = win;
      if (k0 + 2 * PA_STEP > r0)
        bad = __syncthreads_or(vs.nonfinite());
      else
        __syncthreads();
    }
  }

  l = pa_half_sum(l);
  if (row >= len) return;
  // no weight anywhere (a bias of -inf on all a row sees): zeros, and
  // statistics under which the backward's weights are 0 too
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __bf16* ob = static_cast<__bf16*>(p.o) +
               (((long)it.first + row) * p.H + h) * p.D;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = t * 32 + 8 * g + 4 * half;
      bf16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (__bf16)(acc[t][4 * g + e] * inv);
      if (VEC) {
        if (d < p.D) *reinterpret_cast<bf16x4*>(ob + d) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < p.D) ob[d + e] = v[e];
      }
    }
  if (half == 0) {
    const long at = (long)h * p.T + it.first + row;
    const float lg = l == 0.f ? INFINITY : __builtin_amdgcn_logf(l);
    if constexpr (BIAS) {
      p.stats[2 * at] = m == -INFINITY ? 0.f : m;
      p.stats[2 * at + 1] = lg;
    } else {
      p.stats[at] = (m == -INFINITY ? 0.f : m * to2) + lg;
    }
  }
}

template <int DP, bool VEC>
static void pa_fwd_go(const PaFwd& p, const PaBias* bias, unsigned grid,
                      hipStream_t stream) {
  if (bias)
    hipLaunchKernelGGL((pa_fwd_kernel<DP, VEC, true, PaBias>), dim3(grid),
                       dim3(PA_BLOCK), 0, stream, p, *bias);
  else
    hipLaunchKernelGGL((pa_fwd_kernel<DP, VEC, false, PaNoBias>), dim3(grid),
                       dim3(PA_BLOCK), 0, stream, p, PaNoBias{});
}

// vec: head size, strides and addresses allow 16-byte loads.
extern "C" void dlb_packed_attn_fwd(const PaFwd* p, const PaBias* bias,
                                    long items, int vec, hipStream_t stream) {
  const unsigned grid = (unsigned)(items * p->H);
  if (p->D <= 64)
    vec ? pa_fwd_go<64, true>(*p, bias, grid, stream)
        : pa_fwd_go<64, false>(*p, bias, grid, stream);
  else
    vec ? pa_fwd_go<128, true>(*p, bias, grid, stream)
        : pa_fwd_go<128, false>(*p, bias, grid, stream);
}
