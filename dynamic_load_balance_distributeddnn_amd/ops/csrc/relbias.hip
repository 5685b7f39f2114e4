// Learned relative position bias by buckets (gfx950).
//
//   out[h, i, j] = table[bucket(i + K - Q - j), h]      [H, Q, K]
//   dtable[b, h] = sum of dout[h, i, j] over the pairs of bucket b
//
// The queries are the last Q of the K positions; bucket() is constant
// along a diagonal and, being monotone in the distance, takes a run of
// neighbouring diagonals to one bucket.  Both directions move H*Q*K
// elements once and are bound by memory: the forward spreads a short
// table of the tile's diagonals from LDS with 16-byte stores, the
// backward lets a thread keep the sums of its diagonals in registers
// while it walks down the rows.
#include <hip/hip_fp16.h>

#include "common.h"
#include "longctx_args.h"

#define RB_BLOCK 256
#define RB_ROWS 64    // most rows of a workgroup
#define RB_DIAGS 4    // diagonals of a thread in the backward

__device__ inline int rb_bucket(const RbArgs& a, const int* starts, long n) {
  int extra = 0;
  if (n < 0) {
    if (!a.both) return 0;
    n = -n;
    extra = a.side;
  }
  int lo = 0, hi = a.side;  // starts[lo] <= n < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= n) lo = mid; else hi = mid;
  }
  return lo + extra;
}

// Padded place of a diagonal in LDS: lanes that read eight neighbours each
// then start in different banks.
__device__ inline int rb_at(int x) { return x + (x >> 3); }

// A workgroup writes `rows` rows x 256 vectors of one head.  A vector of
// 16 bytes starts where the ADDRESS is a multiple of 16, which is another
// column in each row where K is odd; what a row has before its first and
// after its last whole vector is written element by element.
template <typename W>  // unsigned short or unsigned: the values' bits
__global__ void __launch_bounds__(RB_BLOCK)
rb_fwd_kernel(const W* __restrict__ table, W* __restrict__ out,
              const RbArgs a, const int rows) {
  const int N = 16 / sizeof(W);
  const int SPAN = RB_BLOCK * N + RB_ROWS + 2 * N;
  __shared__ W s_diag[SPAN + SPAN / 8 + 1];
  __shared__ int s_start[RB_MAXBUCKETS];
  const int t = threadIdx.x;
  const long h = blockIdx.z;
  const long i0 = (long)blockIdx.y * rows;
  const int nrows = (int)min((long)rows, a.Q - i0);
  // columns of all rows' vectors: jlo .. jlo + RB_BLOCK * N + N - 2
  const long jlo = (long)blockIdx.x * RB_BLOCK * N - (N - 1);
  for (int b = t; b < a.side; b += RB_BLOCK) s_start[b] = a.starts[b];
  __syncthreads();
  // diagonal x: j - i = jlo - (i0 + nrows - 1) + x
  const long top = i0 + nrows - 1 + a.K - a.Q - jlo;  // distance at x = 0
  const int span = RB_BLOCK * N + N + nrows;
  for (int x = t; x < span; x += RB_BLOCK)
    s_diag[rb_at(x)] = table[(long)rb_bucket(a, s_start, top - x) * a.H + h];
  __syncthreads();

  for (int r = 0; r < nrows; ++r) {
    const long row = (h * a.Q + i0 + r) * a.K;
    // first column of lane 0: the vector starts of this row lie at
    // columns that bring row + j to a multiple of N
    const int phase = (int)((-row) & (N - 1));  // 0 .. N-1
    const long j0 = jlo + (N - 1) + (phase ? phase - N : 0) + (long)t * N;
    const int x0 = (int)(j0 - jlo) + nrows - 1 - r;
    W v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = s_diag[rb_at(x0 + e)];
    if (j0 >= 0 && j0 + N <= a.K) {
      *reinterpret_cast<uint4*>(out + row + j0) =
          *reinterpret_cast<const uint4*>(v);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j0 + e >= 0 && j0 + e < a.K) out[row + j0 + e] = v[e];
    }
  }
}

__device__ inline float rb_float(__hip_bfloat16 x) {
  return __bfloat162float(x);
}
__device__ inline float rb_float(__half x) { return __half2float(x); }
__device__ inline float rb_float(float x) { return x; }
__device__ inline void rb_put(__hip_bfloat16* p, float v) {
  *p = __float2bfloat16(v);
}
__device__ inline void rb_put(__half* p, float v) { *p = __float2half(v); }
__device__ inline void rb_put(float* p, float v) { *p = v; }

// A workgroup sums RB_BLOCK * RB_DIAGS diagonals over `rows` rows of one
// head, 64 neighbouring ones a wave and load, and writes the sums by
// bucket: part[workgroup of the head][h][bucket].
template <typename T>
__global__ void __launch_bounds__(RB_BLOCK)
rb_bwd_kernel(const T* __restrict__ dout, float* __restrict__ part,
              const RbArgs a, const int rows) {
  const int SPAN = RB_BLOCK * RB_DIAGS;
  __shared__ float s_diag[SPAN];
  __shared__ int s_start[RB_MAXBUCKETS];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long h = blockIdx.z;
  const long i0 = (long)blockIdx.y * rows;
  const int nrows = (int)min((long)rows, a.Q - i0);
  // j - i of this workgroup's diagonal 0
  const long d0 = (long)blockIdx.x * SPAN - (i0 + nrows - 1);
  for (int b = t; b < a.side; b += RB_BLOCK) s_start[b] = a.starts[b];

  float sum[RB_DIAGS] = {};
  const T* base = dout + (h * a.Q + i0) * a.K;
  long j = d0 + i0 + t;
#pragma unroll 4
  for (int r = 0; r < nrows; ++r) {
#pragma unroll
    for (int u = 0; u < RB_DIAGS; ++u) {
      const long jj = j + u * RB_BLOCK;
      const long at = min(max(jj, 0l), a.K - 1);
      const float v = rb_float(base[at]);
      sum[u] += jj == at ? v : 0.f;
    }
    base += a.K;
    ++j;
  }
#pragma unroll
  for (int u = 0; u < RB_DIAGS; ++u) s_diag[u * RB_BLOCK + t] = sum[u];
  __syncthreads();

  // the diagonals of a bucket are neighbours: distance top - x
  const long top = a.K - a.Q - d0;
  const long block = (long)blockIdx.y * gridDim.x + blockIdx.x;
  float* mine = part + (block * a.H + h) * a.buckets;
  for (int b = wave; b < a.buckets; b += RB_BLOCK / 64) {
    const bool back = b >= a.side;  // keys ahead of the query
    const int s = back ? b - a.side : b;
    // distances lo .. hi - 1 (infinite: LONG_MAX / 2)
    long lo = s_start[s];
    long hi = s + 1 < a.side ? s_start[s + 1] : (long)1 << 60;
    long xlo, xhi;  // diagonals xlo .. xhi - 1
    if (back) {
      if (lo == 0) lo = 1;  // distance 0 belongs to the other side
      xlo = top + lo;
      xhi = top + hi;
    } else {
      if (!a.both && s == 0) lo = -((long)1 << 60);  // keys ahead: 0
      xlo = top - hi + 1;
      xhi = top - lo + 1;
    }
    const int from = (int)min(max(xlo, 0l), (long)SPAN);
    const int to = (int)min(max(xhi, 0l), (long)SPAN);
    float v = 0.f;
    for (int x = from + lane; x < to; x += 64) v += s_diag[x];
    v = wave_reduce_sum(v);
    if (lane == 0) mine[b] = v;
  }
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

// Rows of a workgroup: as many as leave work for the whole chip.
static int rb_rows(const RbArgs& a, long strips) {
  long rows = a.H * strips * a.Q / 2048;
  return (int)(rows < 1 ? 1 : rows > RB_ROWS ? RB_ROWS : rows);
}
static long rb_div(long a, long b) { return (a + b - 1) / b; }

// size: bytes of an element.  out is 16-byte aligned.
extern "C" void dlb_relbias_fwd(const void* table, void* out,
                                const RbArgs* a, int size,
                                hipStream_t stream) {
  const int n = 16 / size;
  const long strips = rb_div(a->K + n - 1, (long)RB_BLOCK * n);
  const int rows = rb_rows(*a, strips);
  const dim3 grid(strips, rb_div(a->Q, rows), a->H);
  if (size == 2)
    hipLaunchKernelGGL(rb_fwd_kernel<unsigned short>, grid, dim3(RB_BLOCK), 0,
                       stream, (const unsigned short*)table,
                       (unsigned short*)out, *a, rows);
  else
    hipLaunchKernelGGL(rb_fwd_kernel<unsigned>, grid, dim3(RB_BLOCK), 0,
                       stream, (const unsigned*)table, (unsigned*)out, *a,
                       rows);
}

static void rb_bwd_shape(const RbArgs& a, int* rows, long* strips) {
  const long span = RB_BLOCK * RB_DIAGS;
  *rows = rb_rows(a, rb_div(a.K + RB_ROWS - 1, span));
  *strips = rb_div(a.K + *rows - 1, span);
}

// Workgroups of a head in the backward: rows of its partial sums.
extern "C" long dlb_relbias_bwd_blocks(const RbArgs* a) {
  int rows;
  long strips;
  rb_bwd_shape(*a, &rows, &strips);
  return strips * rb_div(a->Q, rows);
}

template <typename T>
static void rb_sum(const void* dout, float* part, const RbArgs& a, dim3 grid,
                   int rows, hipStream_t stream) {
  hipLaunchKernelGGL(rb_bwd_kernel<T>, grid, dim3(RB_BLOCK), 0, stream,
                     (const T*)dout, part, a, rows);
}
template <typename T>
static void rb_reduce(const float* part, void* dtable, const RbArgs& a,
                      long blocks, hipStream_t stream) {
  hipLaunchKernelGGL(rb_reduce_kernel<T>, dim3(a.H, a.buckets),
                     dim3(RB_BLOCK), 0, stream, part, (T*)dtable, blocks,
                     a.H * a.buckets);
}

// types: 0 bf16, 1 fp16, 2 fp32.  part: [blocks, H, buckets].
extern "C" void dlb_relbias_bwd(const void* dout, int type, float* part,
                                void* dtable, int table_type,
                                const RbArgs* a, hipStream_t stream) {
  int rows;
  long strips;
  rb_bwd_shape(*a, &rows, &strips);
  const long chunks = rb_div(a->Q, rows);
  const dim3 grid(strips, chunks, a->H);
  if (type == 0)
    rb_sum<__hip_bfloat16>(dout, part, *a, grid, rows, stream);
  else if (type == 1)
    rb_sum<__half>(dout, part, *a, grid, rows, stream);
  else
    rb_sum<float>(dout, part, *a, grid, rows, stream);
  if (table_type == 0)
    rb_reduce<__hip_bfloat16>(part, dtable, *a, strips * chunks, stream);
  else if (table_type == 1)
    rb_reduce<__half>(part, dtable, *a, strips * chunks, stream);
  else
    rb_reduce<float>(part, dtable, *a, strips * chunks, stream);
}
