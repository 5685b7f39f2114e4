// Pieces shared by the packed causal attention kernels (gfx950).
//
// All three kernels (forward, query gradient, key/value gradient) are
// built on v_mfma_f32_32x32x16_bf16 with the operands ordered so that a
// product's result is the next product's operand WITHOUT leaving the
// lane that holds it:
//
//   result    lane l holds column n = l & 31 and, with half = l >> 5,
//             rows m = 8*(r >> 2) + 4*half + (r & 3), r = 0..15;
//   operand   lane l holds row/column l & 31 and eight steps of the
//             summed index.  A sum does not care in which order its
//             index runs, so the eight steps of a 16-step slice are taken
//             as 8*(e >> 2) + 4*half + (e & 3), which is what the result
//             registers 8*s .. 8*s+7 hold, and the other operand is read
//             in the same order (four consecutive rows a transposing LDS
//             read, twice).
//
// So the weights go from the scores' registers to the value product by a
// conversion to bf16 alone: no LDS round trip, no lane exchange.
//
// LDS tiles are rows of DP elements in 16-byte chunks; chunk c of row r
// stands at c ^ pa_swz(r).  Row reads (32 rows, one chunk) and transposing
// reads (4 rows, 4 neighbouring chunks) both touch each bank once.
#pragma once

#include "common.h"
#include "longctx_args.h"

#define PA_BLOCK 256
#define PA_ROWS 128      // rows of a block's own tile: 4 waves of 32
#define PA_STEP 64       // rows of a streamed tile

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

#define PA_LOG2E 1.4426950408889634f

struct PaNoBias {};

template <int DP>
__device__ inline int pa_swz(int row) {
  if (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  return ((row & 2) << 1) | ((row >> 2) & 3);
}

__device__ inline f32x16 pa_zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

__device__ inline f32x16 pa_mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Lanes l and l ^ 32 hold the two halves of one row.
__device__ inline float pa_half_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                            __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float pa_half_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                            __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Result registers 8*s .. 8*s+7 as an operand; the one rounding of the
// weights (and of their gradient) to bf16, half a step of 2^-8 each.
__device__ inline bf16x8 pa_operand(const f32x16& c, int s) {
  union { bf16x2 h[4]; bf16x8 v; } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x2 f = {c[8 * s + 2 * i], c[8 * s + 2 * i + 1]};
    u.h[i] = __builtin_convertvector(f, bf16x2);
  }
  return u.v;
}

// Eight elements from global memory: `left` of them exist (<= 0: none).
// VEC: 16-byte aligned, and left is <= 0 or >= 8.  The address is clamped
// by the caller; elements that do not exist are 0.
template <bool VEC>
__device__ inline bf16x8 pa_load8(const __bf16* p, int left) {
  bf16x8 v;
  if (VEC) {
    v = *reinterpret_cast<const bf16x8*>(p);
    u32x4 z = {0u, 0u, 0u, 0u};
    return left > 0 ? v : __builtin_bit_cast(bf16x8, z);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int jj = j < left ? j : 0;
    v[j] = p[jj];
    v[j] = j < left ? v[j] : (__bf16)0.f;
  }
  return v;
}

// Whether any of eight values is an infinity or a NaN.
__device__ inline bool pa_nonfinite(bf16x8 v) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// Operand from the rows of an LDS tile: row `row`, chunk 2*ks + half.
template <int DP>
__device__ inline bf16x8 pa_row_frag(const __bf16* tile, int row, int chunk) {
  return *reinterpret_cast<const bf16x8*>(
      tile + row * DP + ((chunk ^ pa_swz<DP>(row)) << 3));
}

// Operand from the columns of an LDS tile: lane l gets column
// col0 + (l & 31) of the eight rows row0 + 8*(e >> 2) + 4*half + (e & 3).
#define PA_LDS __attribute__((address_space(3)))
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 pa_trvec;
template <int DP>
__device__ inline bf16x8 pa_col_frag(const __bf16* tile, int row0, int col0,
                                     int lane) {
  const int r = row0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
  const int c = (col0 >> 3) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int in = (lane & 1) * 4;
  auto p0 = (PA_LDS pa_trvec*)((PA_LDS __bf16*)tile + r * DP +
                               ((c ^ pa_swz<DP>(r)) << 3) + in);
  auto p1 = (PA_LDS pa_trvec*)((PA_LDS __bf16*)tile + (r + 8) * DP +
                               ((c ^ pa_swz<DP>(r + 8)) << 3) + in);
  union { struct { pa_trvec a, b; } t; bf16x8 v; } u;
  u.t.a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(p0);
  u.t.b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(p1);
  return u.v;
}

// A streamed [PA_STEP][DP] tile on its way through registers: the next
// tile's loads are in flight while this one's products run.
template <int DP, bool VEC>
struct PaStage {
  static const int CH = DP / 8;
  static const int N = PA_STEP * CH / PA_BLOCK;
  bf16x8 v[N];

  // Rows row0 .. of one sequence of `len` rows; `base` its first row's
  // head slice.  Rows behind the sequence come as zeros.
  __device__ inline void load(const __bf16* base, long stride, int row0,
                              int len, int D) {
    const __bf16* at = base + (long)row0 * stride;
    const int last = len - 1 - row0;  // >= 0: the tile has a row
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = threadIdx.x + u * PA_BLOCK;
      const int r = id / CH, d = (id % CH) * 8;
      const int rr = min(r, last);
      const int dd = VEC ? min(d, D - 8) : min(d, D - 1);
      v[u] = pa_load8<VEC>(at + (unsigned)(rr * (int)stride + dd),
                           r <= last ? D - d : 0);
    }
  }
  __device__ inline void store(__bf16* tile) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = threadIdx.x + u * PA_BLOCK;
      const int r = id / CH, c = id % CH;
      *reinterpret_cast<bf16x8*>(tile + r * DP +
                                 ((c ^ pa_swz<DP>(r)) << 3)) = v[u];
    }
  }
  __device__ inline bool nonfinite() const {
    bool bad = false;
#pragma unroll
    for (int u = 0; u < N; ++u) bad |= pa_nonfinite(v[u]);
    return bad;
  }
};

// A product sums over masked pairs too, with a weight of 0; an infinity
// or NaN there would come through as NaN.  A tile on the diagonal that
// holds one is taken apart: acc[column l & 31] += x for each such x of a
// row that the column may see, and the tile keeps zeros in their place.
// Columns see row i if i <= lim (DOWN) or i >= lim.
template <int DP, bool DOWN>
__device__ inline void pa_poison(const __bf16* tile, f32x16 (&acc)[DP / 32],
                                 int lim, int lane) {
  for (int i = 0; i < PA_STEP; ++i) {
    const bool sees = DOWN ? i <= lim : i >= lim;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = t * 4 + g;
        const bf16x4 x = *reinterpret_cast<const bf16x4*>(
            tile + i * DP + ((c ^ pa_swz<DP>(i)) << 3) + 4 * (lane >> 5));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = (float)x[e];
          if (sees && (__float_as_uint(f) & 0x7f800000u) == 0x7f800000u)
            acc[t][4 * g + e] += f;
        }
      }
  }
}
template <int DP>
__device__ inline void pa_cleanse(__bf16* tile) {
  for (int id = threadIdx.x; id < PA_STEP * DP / 2; id += PA_BLOCK) {
    unsigned* w = reinterpret_cast<unsigned*>(tile) + id;
    unsigned x = *w;
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
    if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu;
    *w = x;
  }
}

// ---- the bias of a block's head, in LDS
// Largest bucket whose least distance is <= n; starts[0] = 0.
__device__ inline int pa_bucket(const int* starts, int buckets, int n) {
  int lo = 0, hi = buckets;  // starts[lo] <= n < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= n) lo = mid; else hi = mid;
  }
  return lo;
}
__device__ inline float pa_table(const PaBias& b, int bucket, int heads,
                                 int h) {
  const long at = (long)bucket * heads + h;
  return b.is_bf16 ? (float)static_cast<const __bf16*>(b.table)[at]
                   : static_cast<const float*>(b.table)[at];
}

__device__ inline const __bf16* pa_at(const PaTensor& t, long row, int head) {
  return static_cast<const __bf16*>(t.p) + row * t.row + head * t.head;
}

// Workgroups go round the 8 XCDs in turn.  Where the heads divide, an XCD
// gets neighbouring heads, which share keys and values in its L2.
__device__ inline int pa_head(int c, int heads) {
  return (heads & 7) ? c : (c & 7) * (heads >> 3) + (c >> 3);
}
