// Causal attention over packed sequences, forward (gfx950).
//
//   S_ij = scale q_i.k_j (+ bias of head h at distance i - j),  j <= i
//   O_i  = sum_j exp(S_ij - m_i) v_j / sum_j exp(S_ij - m_i)
//
// One pass over the keys with a running maximum m and sum l per row; the
// [n, n] scores are never stored.  A workgroup owns 128 query rows of one
// head, 32 a wave, and streams 64-key tiles through LDS; S is computed
// transposed (keys x queries) so that a lane holds one query's scores and
// the softmax needs one lane exchange a tile.  The packing's list says
// which rows and keys, most work first; a tile whose keys are shared out
// to several workgroups is put together by a second kernel.
//
// 32 rows a wave let one lane's registers hold a row's scores, 64 keys a
// step are two score tiles to overlap with their exponentials, and two
// buffers of keys and values of 128 leave room for two workgroups a CU.
// Measured: one sequence of 8192, 32 heads of 128 over 8, 498 to 535 us, 1030
// to 1100 TFLOP/s where a plain product of 8192 x 8192 x 8192 reaches 1190; seven
// of 8192 in all, 16 heads over 4, 78 us, 780 TFLOP/s; eight of 512, 21 us;
// 20 of 35, 2 heads of 100, 9 us.  Bound by the matrix units and the
// exponentials that share the issue with them where sequences are long
// (without the exponentials 3 to 10 % less, without the loads' addressing
// 15 % before that was cut to a scalar add a load), else by the longest
// workgroup and by the trips to memory at its start and end.
#include "packed_attn.h"

// A row's end: N x 32 elements of its output from 32 * t0 on, with the
// first its statistics.
template <int W, bool BIAS, int N>
__device__ PA_INLINE void pa_fwd_end(const PaFwd& p, long first, int row,
                                     int len, int h, const f32x16 (&acc)[N],
                                     int t0, float m, float l) {
  if (row >= len) return;
  const int half = (threadIdx.x & 63) >> 5;
  // no weight anywhere (a bias of -inf on all a row sees): zeros, and
  // statistics under which the backward's weights are 0 too
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __bf16* ob = static_cast<__bf16*>(p.o) + ((first + row) * p.H + h) * p.D;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bf16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (__bf16)(acc[t][4 * g + e] * inv);
      pa_store4<W>(ob, (t0 + t) * 32 + 8 * g + 4 * half, p.D, v);
    }
  if (half == 0 && t0 == 0) {
    const long at = (long)h * p.T + first + row;
    const float lg = l == 0.f ? INFINITY : __builtin_amdgcn_logf(l);
    const float top = m == -INFINITY ? 0.f : m;
    if constexpr (BIAS) {
      p.stats[2 * at] = top;
      p.stats[2 * at + 1] = lg;
    } else {
      p.stats[at] = top + lg;
    }
  }
}

template <int DP, int W, bool BIAS, typename BiasArg>
__global__ void __launch_bounds__(PA_BLOCK, 2)
pa_fwd_kernel(const PaFwd p, const BiasArg bias) {
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
  const PaChunk it = p.work.chunks[blockIdx.x / p.H];
  const int r0 = it.tile * PA_ROWS;
  const int w0 = r0 + wave * 32;     // this wave's first row
  const int row = w0 + col;          // this lane's
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
  // bias of the distances a 128 x 64 tile spans, r0 - k0 - 63 upwards
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

  bf16x8 qf[KS];
  {
    const __bf16* qb = pa_at(p.q, (long)it.first + min(row, len - 1), h);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[s] = pa_load8<W>(qb, s * 16 + half * 8, p.D);
  }

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = pa_zero16();
  // Scores are exponents of 2, a s + b: in tiles of one bias (or none) s is
  // q.k as the product leaves it, elsewhere the sum, with a = 1, b = 0.
  float m = -INFINITY;   // running maximum
  float l = 0.f;         // this half's part of the sum
  const float mul = p.scale * PA_LOG2E;
  float a = mul, b = far_bias;

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
  if (BIAS && near(it.begin * PA_STEP)) win = window(it.begin * PA_STEP);
  arrive(it.begin * PA_STEP, it.begin & 1);

  const PaFrags<DP> lanes(s_tiles, lane);
  PaFrags<DP> frags = lanes;  // of the current buffer
  auto scores = [&](f32x16 (&s)[2], int k0, int buf) PA_INLINE {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[j] = pa_zero16();
#pragma unroll
      for (int x = 0; x < KS; ++x)
        s[j] = pa_mfma(frags.rows(j * 32 * DP * 2, x),
                       qf[x], s[j]);
    }
    if constexpr (BIAS) {
      const bool each = near(k0);
      a = each ? 1.f : mul;
      b = each ? 0.f : far_bias;
      if (each) {
        const float* w = s_win[buf] + wave * 32 + col + (PA_STEP - 1);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[j][r] = fmaf(s[j][r], mul,
                           w[-(j * 32 + 8 * (r >> 2) + 4 * half + (r & 3))]);
      }
    }
  };
  auto maximum = [&](const f32x16 (&s)[2]) PA_INLINE {
    float top = s[0][0];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[j][r]);
    return fmaxf(m, fmaf(pa_half_max(top), a, b));
  };
  // scores to weights; returns their sum
  auto weights = [&](f32x16 (&s)[2], float ref) PA_INLINE {
    const float off = b - ref;
    float sum[4] = {};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[j][r] = __builtin_amdgcn_exp2f(fmaf(s[j][r], a, off));
        sum[r & 3] += s[j][r];
      }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  auto values = [&](const f32x16 (&s)[2]) PA_INLINE {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bf16x8 w = pa_operand(s[x >> 1], x & 1);
#pragma unroll
      for (int d = 0; d < DT; ++d)
        acc[d] = pa_mfma(
            frags.cols((2 * PA_STEP + x * 16) * DP * 2, d), w,
            acc[d]);
    }
  };

  // Any tile: with keys ahead of some row, and with a new maximum.
  auto any_tile = [&](int t) PA_INLINE {
    const int k0 = t * PA_STEP, buf = t & 1;
    const bool more = t + 1 < it.end;
    if (more) start(k0 + PA_STEP, buf ^ 1);
    if (t >= whole) {
      if (__syncthreads_or(pa_tile_nonfinite<DP, PA_STEP>(s_v[buf]))) {
        pa_poison<DP, PA_STEP, true>(s_v[buf], acc, row - k0, lane);
        __syncthreads();
        pa_cleanse<DP, PA_STEP>(s_v[buf]);
        __syncthreads();
      }
    }
    frags = lanes.fresh(buf * TILE * 2);
    if (k0 <= w0 + 31) {
      f32x16 s[2];
      scores(s, k0, buf);
      const int lim = row - k0 - 4 * half;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (j * 32 + 8 * (r >> 2) + (r & 3) > lim) s[j][r] = -INFINITY;
      const float top = maximum(s);
      const float ref = top == -INFINITY ? 0.f : top;
      // before the first weight there is nothing to scale but infinities that
      // were taken out of the values: 0 of those would be NaN
      const float f =
          m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= f;
      l *= f;
      m = top;
      l += weights(s, ref);
      values(s);
    }
    if (more) arrive(k0 + PA_STEP, buf ^ 1);
  };

  // A tile that all rows see whole, with the maximum as it is held: the
  // sum and the output are scaled anew only once the weights of a tile come
  // to more than 2^16, which fp32 and the bf16 weights (their step is
  // relative) carry without loss.  So no tile looks for its maximum (one of
  // 8192, 32 heads of 128 over 8: 544 -> 532 us).  False, with nothing
  // done, where they did; the wave then takes any_tile, which has as many
  // barriers, to its end: with keys that grow to six times along the
  // sequence 521 -> 555 us, and with a bias of -inf from 113 on, where most
  // rows have no weight in their first tile, 53 -> 73 (4001, 12 heads of 64).
  auto whole_tile = [&](int t) PA_INLINE {
    const int k0 = t * PA_STEP, buf = t & 1;
    const bool more = t + 1 < it.end;
    if (more) start(k0 + PA_STEP, buf ^ 1);
    frags = lanes.fresh(buf * TILE * 2);
    f32x16 s[2];
    scores(s, k0, buf);
    const float sum = weights(s, m);
    if (__any(sum > 65536.f)) return false;
    l += sum;
    values(s);
    if (more) arrive(k0 + PA_STEP, buf ^ 1);
    return true;
  };

  const int fast = min(whole, it.end);
  for (int t = it.begin; t < it.end;) {
    any_tile(t++);
    // a row without a weight so far has no maximum to hold
    if (t == it.begin + 1 && !__any(m == -INFINITY))
      while (t < fast && whole_tile(t)) ++t;
  }

  l = pa_half_sum(l);
  if (it.slot >= 0) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *pa_sums(p.work, it.slot, p.H, h, DT * 4, t * 4 + g) =
            f32x4{acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2],
                  acc[t][4 * g + 3]};
    if (half == 0) {
      float* to = pa_rows(p.work, it.slot, p.H, h, wave * 32 + col);
      to[0] = m;
      to[1] = l;
    }
    return;
  }
  pa_fwd_end<W, BIAS, DT>(p, it.first, row, len, h, acc, 0, m, l);
}

// Tiles in several chunks: with the largest maximum of a row,
// O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i; blockIdx.y: 32
// elements of the rows.
template <int DP, int W, bool BIAS>
__global__ void __launch_bounds__(PA_BLOCK)
pa_fwd_join_kernel(const PaFwd p) {
  const int DT = DP / 32;
  const int h = blockIdx.x % p.H, t = blockIdx.y;
  const PaJoin j = p.work.joins[blockIdx.x / p.H];
  const int in = (threadIdx.x >> 6) * 32 + (threadIdx.x & 31);
  float m = -INFINITY, l = 0.f;
  f32x16 acc[1] = {pa_zero16()};
  // four chunks at a time, their loads together in flight; the running
  // maximum as in the tiles
  for (int i0 = 0; i0 < j.n; i0 += 4) {
    f32x4 x[4][4];
    float mi[4], li[4], top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = j.slot + min(i0 + i, j.n - 1);
      const float* from = pa_rows(p.work, slot, p.H, h, in);
      const bool there = i0 + i < j.n;
      mi[i] = there ? from[0] : -INFINITY;
      li[i] = there ? from[1] : 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g)
        x[i][g] = *pa_sums(p.work, slot, p.H, h, DT * 4, t * 4 + g);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, mi[i]);
    const float ref = top == -INFINITY ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref);
    m = top;
    l *= f;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][r] *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i0 + i >= j.n) break;
      const float fi = __builtin_amdgcn_exp2f(mi[i] - ref);
      l += fi * li[i];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[0][r] = fmaf(fi, x[i][r >> 2][r & 3], acc[0][r]);
    }
  }
  pa_fwd_end<W, BIAS, 1>(p, j.first, j.tile * PA_ROWS + in, j.len, h, acc, t,
                         m, l);
}

template <int DP, int W>
static void pa_fwd_go(const PaFwd& p, const PaBias* bias,
                      hipStream_t stream) {
  const dim3 grid((unsigned)p.work.n_chunks * p.H), block(PA_BLOCK);
  const dim3 joins((unsigned)p.work.n_joins * p.H, DP / 32);
  if (bias) {
    hipLaunchKernelGGL((pa_fwd_kernel<DP, W, true, PaBias>), grid, block, 0,
                       stream, p, *bias);
    if (joins.x)
      hipLaunchKernelGGL((pa_fwd_join_kernel<DP, W, true>), joins, block, 0,
                         stream, p);
  } else {
    hipLaunchKernelGGL((pa_fwd_kernel<DP, W, false, PaNoBias>), grid, block,
                       0, stream, p, PaNoBias{});
    if (joins.x)
      hipLaunchKernelGGL((pa_fwd_join_kernel<DP, W, false>), joins, block, 0,
                         stream, p);
  }
}

// width: 16, 4 or 2 bytes, what the head size, strides and addresses of
// all tensors are multiples of.
extern "C" void dlb_packed_attn_fwd(const PaFwd* p, const PaBias* bias,
                                    int width, hipStream_t stream) {
  auto go = [&](auto go64, auto go128) {
    (p->D <= 64 ? go64 : go128)(*p, bias, stream);
  };
  if (width == 16) go(pa_fwd_go<64, 16>, pa_fwd_go<128, 16>);
  else if (width == 4) go(pa_fwd_go<64, 4>, pa_fwd_go<128, 4>);
  else go(pa_fwd_go<64, 2>, pa_fwd_go<128, 2>);
}
