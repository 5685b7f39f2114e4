// Learned relative position bias by buckets (gfx950).
//
//   out[h, i, j] = table[bucket(i + K - Q - j), h]      [H, Q, K]
//   dtable[b, h] = sum of dout[h, i, j] over the pairs of bucket b
//
// The queries are the last Q of the K positions.  bucket() is constant
// along a diagonal j - i and, being monotone in the distance, gives runs
// of neighbouring diagonals one bucket.  Both directions move H*Q*K
// elements once and are bound by memory, so both move them in vectors of
// 16 bytes, N elements.  Measured in bf16: 32 heads of 4096 x 4096 166 us
// forward (6.4 TB/s; a fill writes 6.85), 219 us backward alone (4.9 TB/s;
// a bare read of as much 6.2); 16 of 2048 x 2048 26 us (5.2 TB/s) and 38 us,
// of 2047 x 2047 forward 46: a row of 257 vectors takes a second strip of
// workgroups for the last; the smallest 4 and 6 us, of which a launch is
// most.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.h"
#include "longctx_args.h"

#define RB_BLOCK 256
#define RB_ROWS 64    // most rows of a workgroup

typedef __attribute__((ext_vector_type(4))) unsigned rb_vec;
typedef rb_vec __attribute__((aligned(4))) rb_words;  // on any word

__device__ inline int rb_bucket(const RbArgs& a, const int* starts, long far) {
  const int n0 = (int)min(max(far, -(1l << 30)), 1l << 30);
  if (n0 < 0 && !a.both) return 0;
  const int n = abs(n0), extra = n0 < 0 ? a.side : 0;
  // the first half of the buckets hold one distance each
  int lo = a.side / 2, hi = a.side - 1;
  if (n < lo) return n + extra;
  if (n >= starts[hi]) return hi + extra;
  while (hi - lo > 1) {  // starts[lo] <= n < starts[hi]
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= n) lo = mid; else hi = mid;
  }
  return lo + extra;
}

// Sum over a wave, in every lane.
__device__ inline float rb_wave_sum(float v) {
#define RB_STEP(CTRL, ROWS)                                              \
  v += __builtin_bit_cast(                                               \
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),  \
                                         CTRL, ROWS, 0xf, false));
  RB_STEP(0x111, 0xf) RB_STEP(0x112, 0xf)  // row_shr:1, 2, 4, 8
  RB_STEP(0x114, 0xf) RB_STEP(0x118, 0xf)
  RB_STEP(0x142, 0xa) RB_STEP(0x143, 0xc)  // row_bcast:15, 31
#undef RB_STEP
  return __builtin_bit_cast(
      float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// A workgroup writes `rows` rows of one head, 2^lanes vectors of each and
// RB_BLOCK >> lanes rows at a time.  It lays out the vectors of N values
// that start on each of its diagonals in LDS, one list for each remainder
// by N, so that a wave reads consecutive ones: one LDS read and one store a
// vector, and the stores are aligned, whatever K is (a row's vectors start
// at the columns that make them so).
// Where all its pairs are of one bucket (far behind or far ahead) there is
// nothing to lay out.  What a row has before its first and after its last
// whole vector is written element by element.
template <typename W>  // unsigned short or unsigned: the values' bits
__global__ void __launch_bounds__(RB_BLOCK)
rb_fwd_kernel(const W* __restrict__ table, W* __restrict__ out,
              const RbArgs a, const int rows, const int lanes) {
  const int N = 16 / sizeof(W);
  const int LIST = RB_BLOCK + RB_ROWS / N + 2;  // vectors of a shift
  const int SPAN = N * LIST;                    // diagonals
  __shared__ W s_diag[SPAN + N];
  typedef __attribute__((ext_vector_type(N))) W Vec;
  __shared__ Vec s_vec[N * LIST];
  __shared__ int s_start[RB_MAXBUCKETS];
  __shared__ W s_tab[RB_MAXBUCKETS];
  const int t = threadIdx.x;
  const long h = blockIdx.z;
  const long i0 = (long)blockIdx.y * rows;
  const int nrows = (int)min((long)rows, a.Q - i0);
  const int width = N << lanes;  // columns
  // columns of all rows' vectors: jlo .. jlo + width + N - 2
  const long jlo = (long)blockIdx.x * width - (N - 1);
  for (int b = t; b < a.side; b += RB_BLOCK) s_start[b] = a.starts[b];
  for (int b = t; b < a.buckets; b += RB_BLOCK)
    s_tab[b] = table[(long)b * a.H + h];
  __syncthreads();
  // diagonal x: j - i = jlo - (i0 + nrows - 1) + x
  const long top = i0 + nrows - 1 + a.K - a.Q - jlo;  // distance at x = 0
  const int span = width + N + nrows;
  const int b0 = rb_bucket(a, s_start, top);
  const bool plain = b0 == rb_bucket(a, s_start, top - (span - 1));
  Vec same = s_tab[b0];
  if (!plain) {
    for (int x = t; x < span; x += RB_BLOCK)
      s_diag[x] = s_tab[rb_bucket(a, s_start, top - x)];
    __syncthreads();
    for (int x = t; x + N <= span; x += RB_BLOCK) {
      Vec v;
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = s_diag[x + e];
      s_vec[(x % N) * LIST + x / N] = v;
    }
    __syncthreads();
  }

  const int u = t & ((1 << lanes) - 1);
  for (int r = t >> lanes; r < nrows; r += RB_BLOCK >> lanes) {
    const long row = (h * a.Q + i0 + r) * a.K;
    // the row's vectors start where row + j is a multiple of N
    const int phase = (int)((-row) & (N - 1));
    const long j0 = jlo + (N - 1) + (phase ? phase - N : 0) + (long)u * N;
    const int x0 = (int)(j0 - jlo) + nrows - 1 - r;
    Vec v = same;
    if (!plain) v = s_vec[(x0 % N) * LIST + x0 / N];
    if (j0 >= 0 && j0 + N <= a.K) {
      *reinterpret_cast<Vec*>(out + row + j0) = v;
    } else if (j0 + N > 0 && j0 < a.K) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j0 + e >= 0 && j0 + e < a.K) out[row + j0 + e] = v[e];
    }
  }
}

// Element e of a vector.
template <typename T>
__device__ inline float rb_element(rb_vec q, int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(q[e]);
  } else {
    const unsigned w = q[e >> 1];
    if constexpr (std::is_same<T, __hip_bfloat16>::value)
      return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    else
      return (float)__builtin_bit_cast(
          _Float16, (unsigned short)(e & 1 ? w >> 16 : w));
  }
}
__device__ inline void rb_put(__hip_bfloat16* p, float v) {
  *p = __float2bfloat16(v);
}
__device__ inline void rb_put(__half* p, float v) { *p = __float2half(v); }
__device__ inline void rb_put(float* p, float v) { *p = v; }

// The 16 bytes behind an address that is a multiple of 4 plus 2 * odd,
// from the words that hold them: `q` starts odd halves of a word early,
// `next` holds the half behind it.
__device__ inline rb_vec rb_shift(rb_vec q, unsigned next, int odd) {
  const int s = odd * 16;
  return rb_vec{__builtin_amdgcn_alignbit(q[1], q[0], s),
                __builtin_amdgcn_alignbit(q[2], q[1], s),
                __builtin_amdgcn_alignbit(q[3], q[2], s),
                __builtin_amdgcn_alignbit(next, q[3], s)};
}

// Elements d .. of a vector, zeros where it has none (d may be negative).
template <typename T>
__device__ inline rb_vec rb_move(rb_vec q, long d) {
  const int bits = 8 * sizeof(T), n = 16 / sizeof(T);
  unsigned __int128 x = __builtin_bit_cast(unsigned __int128, q);
  if (d < 0)
    x = d > -n ? x << (bits * (int)-d) : 0;
  else
    x = d < n ? x >> (bits * (int)d) : 0;
  return __builtin_bit_cast(rb_vec, x);
}

// A wave sums 64 * N diagonals over `rows` rows of one head, N neighbouring
// ones a lane, which stay in its registers while it walks down the rows.
// From one row to the next a lane's vector moves by K + 1 elements.
// Vectors on any word cost the cache no more than aligned ones, but between
// the words each lane would be an access of its own (64 instead of 16 for
// 1 KB): those are loaded half a word early and shifted, with the half that
// is missing from the next lane.  The four waves of a workgroup take
// neighbouring places of the head's (chunk of rows, 64 * N diagonals) and
// write their sums by bucket: part[workgroup of the head][h][bucket].
// K >= N.
template <typename T>
__global__ void __launch_bounds__(RB_BLOCK)
rb_bwd_kernel(const T* __restrict__ dout, float* __restrict__ part,
              const RbArgs a, const int rows, const int strips) {
  const int N = 16 / sizeof(T), SPAN = 64 * N;
  const bool HALVES = sizeof(T) == 2;
  __shared__ __attribute__((aligned(16))) float s_diag[4][SPAN];
  __shared__ float s_sum[4][RB_MAXBUCKETS];
  __shared__ int s_start[RB_MAXBUCKETS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long h = blockIdx.y;
  const long place = (long)blockIdx.x * 4 + wave;
  const long i0 = place / strips * rows;  // may be behind the last row
  const int nrows = (int)min(max(a.Q - i0, 0l), (long)rows);
  // j - i of this wave's diagonal 0
  const long d0 = place % strips * SPAN - (i0 + nrows - 1);
  for (int b = threadIdx.x; b < a.side; b += RB_BLOCK)
    s_start[b] = a.starts[b];
  for (int b = threadIdx.x; b < a.buckets; b += RB_BLOCK)
    s_sum[0][b] = s_sum[1][b] = s_sum[2][b] = s_sum[3][b] = 0.f;

  float sum[N] = {};
  // rows where the wave's columns reach into the matrix, eight at a time
  const long jw = d0 + i0;  // first column in row i0
  const int from = (int)min(max(-(jw + SPAN - 1), 0l), (long)nrows);
  const int last = (int)min(max(a.K - jw, 0l), (long)nrows);
  const T* row = dout + (h * a.Q + i0 + from) * a.K;
  for (int r0 = from; r0 < last; r0 += 8, row += 8 * a.K) {
    const long w = jw + r0;
    rb_vec q[8];
    unsigned end[8];
    if (w >= 1 && w + 7 + SPAN <= a.K && r0 + 8 <= last) {
      // the wave is inside in all of them
      int odd[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const T* at = row + r * a.K + w + r;  // of lane 0
        odd[r] = HALVES ? (int)(reinterpret_cast<__UINTPTR_TYPE__>(at) >> 1) &
                              1
                        : 0;
        q[r] = *reinterpret_cast<const rb_words*>(at - odd[r] + lane * N);
        if (HALVES)
          end[r] = *reinterpret_cast<const unsigned short*>(at + SPAN - 1);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (HALVES) {
          const unsigned next = __builtin_amdgcn_update_dpp(
              end[r], q[r][0], 0x130 /* wave_shl:1 */, 0xf, 0xf, false);
          q[r] = rb_shift(q[r], next, odd[r]);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += rb_element<T>(q[r], e);
      }
      continue;
    }
    // lanes may reach over a row's start or end: they load the row's first
    // or last vector and move it
    const long j = w + lane * N;
    int odd[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const T* at = row + min(r, last - 1 - r0) * a.K +
                    min(max(j + r, 0l), a.K - N);
      odd[r] = HALVES
                   ? (int)(reinterpret_cast<__UINTPTR_TYPE__>(at) >> 1) & 1
                   : 0;
      q[r] = *reinterpret_cast<const rb_words*>(at - odd[r]);
      if (HALVES)
        end[r] = *reinterpret_cast<const unsigned short*>(at + N - 1);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (HALVES) q[r] = rb_shift(q[r], end[r], odd[r]);
      q[r] = rb_move<T>(q[r], r0 + r < last
                                  ? j + r - min(max(j + r, 0l), a.K - N)
                                  : N);
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += rb_element<T>(q[r], e);
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s_diag[wave][lane * N + e] = sum[e];
  __syncthreads();

  // The diagonals of a bucket are neighbours: distance top - x.  A lane
  // takes a bucket; what is long for one lane (the far bucket of most
  // waves) the wave adds up together.
  const long top = a.K - a.Q - d0;
  if (from < last)
    for (int b0 = 0; b0 < a.buckets; b0 += 64) {
      const int b = b0 + lane;
      int first = 0, stop = 0;  // diagonals first .. stop - 1
      if (b < a.buckets) {
        const bool back = b >= a.side;  // keys ahead of the query
        const int s = back ? b - a.side : b;
        const long none = (long)1 << 60;
        // distances lo .. hi - 1; distance 0 is not ahead, and without
        // `both` what is ahead counts as distance 0
        const long lo = back ? max(s_start[s], 1)
                             : s == 0 && !a.both ? -none : s_start[s];
        const long hi = s + 1 < a.side ? s_start[s + 1] : none;
        const long xlo = back ? top + lo : top - hi + 1;
        const long xhi = back ? top + hi : top - lo + 1;
        first = (int)min(max(xlo, 0l), (long)SPAN);
        stop = (int)min(max(xhi, 0l), (long)SPAN);
      }
      const bool together = stop - first > 32;
      float v = 0.f;
      if (!together)
        for (int x = first; x < stop; ++x) v += s_diag[wave][x];
      for (unsigned long long m = __ballot(together); m; m &= m - 1) {
        const int l = __builtin_ctzll(m);
        const int x0 = __builtin_amdgcn_readlane(first, l);
        const int x1 = __builtin_amdgcn_readlane(stop, l);
        float w = 0.f;
        for (int x = x0 + lane; x < x1; x += 64) w += s_diag[wave][x];
        w = rb_wave_sum(w);
        if (lane == l) v = w;
      }
      if (b < a.buckets) s_sum[wave][b] = v;
    }
  __syncthreads();
  float* mine = part + ((long)blockIdx.x * a.H + h) * a.buckets;
  for (int b = threadIdx.x; b < a.buckets; b += RB_BLOCK)
    mine[b] = (s_sum[0][b] + s_sum[1][b]) + (s_sum[2][b] + s_sum[3][b]);
}

// Sums of part over its first index; a workgroup a (bucket, head).
template <typename T>
__global__ void __launch_bounds__(RB_BLOCK)
rb_reduce_kernel(const float* __restrict__ part, T* __restrict__ dtable,
                 const long blocks, const long n) {
  __shared__ float s_sum[RB_BLOCK / 64];
  const long h = blockIdx.x, b = blockIdx.y;
  const long at = h * gridDim.y + b;
  float v = 0.f;
  for (long i = threadIdx.x; i < blocks; i += RB_BLOCK) v += part[i * n + at];
  v = wave_reduce_sum(v);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    rb_put(dtable + b * gridDim.x + h,
           (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
}

static long rb_div(long a, long b) { return (a + b - 1) / b; }

// Rows of a workgroup: as many as leave 512 workgroups, within bounds.
// What a workgroup lays out costs as much as some 30 rows.
static int rb_rows(const RbArgs& a, long strips, int least, int most) {
  const long rows = a.H * strips * a.Q / 512;
  return (int)(rows < least ? least : rows > most ? most : rows);
}

// size: bytes of an element.  out is 16-byte aligned.
extern "C" void dlb_relbias_fwd(const void* table, void* out,
                                const RbArgs* a, int size,
                                hipStream_t stream) {
  const int n = 16 / size;
  // a row's vectors, one more where they do not start with the row
  const long vectors = rb_div(a->K, n) + (a->K % n != 0);
  int lanes = 0;
  while (lanes < 8 && (1l << lanes) < vectors) ++lanes;
  const long strips = rb_div(vectors, 1l << lanes);
  const int rows = rb_rows(*a, strips, RB_BLOCK >> lanes, RB_ROWS);
  const dim3 grid(strips, rb_div(a->Q, rows), a->H);
  if (size == 2)
    hipLaunchKernelGGL(rb_fwd_kernel<unsigned short>, grid, dim3(RB_BLOCK), 0,
                       stream, (const unsigned short*)table,
                       (unsigned short*)out, *a, rows, lanes);
  else
    hipLaunchKernelGGL(rb_fwd_kernel<unsigned>, grid, dim3(RB_BLOCK), 0,
                       stream, (const unsigned*)table, (unsigned*)out, *a,
                       rows, lanes);
}

// The backward's places: rows of a chunk, waves beside each other on its
// diagonals, workgroups of a head.  n: elements of a vector.
static void rb_bwd_shape(const RbArgs& a, int n, int* rows, long* strips,
                         long* blocks) {
  // About 12 waves a CU: 16 run at a time, and a last few alone would cost
  // as much as the first.  32 heads of 4096 x 4096 in bf16: 219 us (4.9
  // TB/s), with 64 rows a wave 270; 16 of 2047 x 2047: 38, with twice the
  // waves 55 where once took 45.
  const long span = 64 * n;
  const long all = (a.H * rb_div(a.K, span) * a.Q / (12 * 256) + 8) / 8 * 8;
  *rows = (int)(all > 512 ? 512 : all);
  *strips = rb_div(a.K + *rows - 1, span);
  *blocks = rb_div(*strips * rb_div(a.Q, *rows), 4);
}

// Workgroups of a head in the backward: rows of its partial sums.
extern "C" long dlb_relbias_bwd_blocks(const RbArgs* a, int size) {
  int rows;
  long strips, blocks;
  rb_bwd_shape(*a, 16 / size, &rows, &strips, &blocks);
  return blocks;
}

template <typename T>
static void rb_sum(const void* dout, float* part, const RbArgs& a, dim3 grid,
                   int rows, long strips, hipStream_t stream) {
  hipLaunchKernelGGL(rb_bwd_kernel<T>, grid, dim3(RB_BLOCK), 0, stream,
                     (const T*)dout, part, a, rows, (int)strips);
}
template <typename T>
static void rb_reduce(const float* part, void* dtable, const RbArgs& a,
                      long blocks, hipStream_t stream) {
  hipLaunchKernelGGL(rb_reduce_kernel<T>, dim3(a.H, a.buckets),
                     dim3(RB_BLOCK), 0, stream, part, (T*)dtable, blocks,
                     a.H * a.buckets);
}

// types: 0 bf16, 1 fp16, 2 fp32.  part: [blocks, H, buckets].  Rows have
// 16 bytes at least.
extern "C" void dlb_relbias_bwd(const void* dout, int type, float* part,
                                void* dtable, int table_type,
                                const RbArgs* a, hipStream_t stream) {
  int rows;
  long strips, blocks;
  rb_bwd_shape(*a, type == 2 ? 4 : 8, &rows, &strips, &blocks);
  const dim3 grid(blocks, a->H);
  if (type == 0)
    rb_sum<__hip_bfloat16>(dout, part, *a, grid, rows, strips, stream);
  else if (type == 1)
    rb_sum<__half>(dout, part, *a, grid, rows, strips, stream);
  else
    rb_sum<float>(dout, part, *a, grid, rows, strips, stream);
  if (table_type == 0)
    rb_reduce<__hip_bfloat16>(part, dtable, *a, blocks, stream);
  else if (table_type == 1)
    rb_reduce<__half>(part, dtable, *a, blocks, stream);
  else
    rb_reduce<float>(part, dtable, *a, blocks, stream);
}
