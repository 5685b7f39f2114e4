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
#define PA_INLINE __attribute__((always_inline))
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

// How a launch moves its tensors: W bytes at a time, 16 where the head
// size, strides and addresses allow it, else 4, else 2.

// Elements d .. d+7 of a row of D in global memory; those that do not
// exist are 0.
template <int W>
__device__ inline bf16x8 pa_load8(const __bf16* row, int d, int D) {
  if constexpr (W == 16) {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(row + min(d, D - 8));
    const u32x4 z = {0u, 0u, 0u, 0u};
    return d < D ? v : __builtin_bit_cast(bf16x8, z);
  } else if constexpr (W == 4) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = d + 2 * j;
      const unsigned x =
          *reinterpret_cast<const unsigned*>(row + min(at, D - 2));
      v[j] = at < D ? x : 0u;
    }
    return __builtin_bit_cast(bf16x8, v);
  } else {
    bf16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __bf16 x = row[min(d + j, D - 1)];
      v[j] = d + j < D ? x : (__bf16)0.f;
    }
    return v;
  }
}

// Elements d .. d+3 of a dense row of D.
template <int W>
__device__ inline void pa_store4(__bf16* row, int d, int D, bf16x4 v) {
  if constexpr (W == 16) {
    if (d < D) *reinterpret_cast<bf16x4*>(row + d) = v;
  } else if constexpr (W == 4) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    if (d < D) *reinterpret_cast<unsigned*>(row + d) = w[0];
    if (d + 2 < D) *reinterpret_cast<unsigned*>(row + d + 2) = w[1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < D) row[d + e] = v[e];
  }
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

// Operands out of LDS tiles.  The swizzle is an exclusive or in bits that
// a lane's first address and the tiles' bases leave alone, so one address a
// lane serves all tiles: row operands differ by x << 5, column operands by
// t << 6, the eight rows further down by 32 and a constant.  fresh() keeps
// the compiler from holding all of them in registers.
#define PA_LDS __attribute__((address_space(3)))
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 pa_trvec;

template <int DP>
struct PaFrags {
  unsigned row;  // chunk `half` of row l & 31
  unsigned col;  // where lane l starts its transposing reads

  // tiles: 1024-byte aligned
  __device__ inline explicit PaFrags(const void* tiles, int lane) {
    const unsigned at = (unsigned)(__UINTPTR_TYPE__)(
        (PA_LDS const char*)(const char*)tiles);
    const int r = lane & 31, half = lane >> 5;
    row = at + r * (DP * 2) + ((half ^ pa_swz<DP>(r)) << 4);
    const int rc = 4 * half + ((lane & 15) >> 2);
    const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    col = at + rc * (DP * 2) + ((c ^ pa_swz<DP>(rc)) << 4) + (lane & 1) * 8;
  }
  // The same of tiles `off` bytes on (a multiple of 1024).
  __device__ PA_INLINE PaFrags fresh(unsigned off = 0) const {
    PaFrags f = *this;
    f.row += off;
    f.col += off;
    asm volatile("" : "+v"(f.row), "+v"(f.col));
    return f;
  }
  // Row l & 31 of the 32 that start `off` bytes into the tiles, elements
  // 16 x + 8 half + 0 .. 7.
  __device__ PA_INLINE bf16x8 rows(unsigned off, int x) const {
    return *(PA_LDS const bf16x8*)(__UINTPTR_TYPE__)((row ^ (x << 5)) + off);
  }
  // Column 32 t + (l & 31) of the 16 rows that start `off` bytes into the
  // tiles (a multiple of 16 rows), rows 8*(e >> 2) + 4*half + (e & 3).
  __device__ PA_INLINE bf16x8 cols(unsigned off, int t) const {
    union { struct { pa_trvec a, b; } t; bf16x8 v; } u;
    u.t.a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (PA_LDS pa_trvec*)(__UINTPTR_TYPE__)((col ^ (t << 6)) + off));
    u.t.b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (PA_LDS pa_trvec*)(__UINTPTR_TYPE__)((col ^ (t << 6 | 32)) + off +
                                             8 * DP * 2));
    return u.v;
  }
};

// W (16 or 4) bytes a lane from base + offset (bytes) to tile + W * lane;
// base and tile are the wave's.  Written out because the compiler would let
// every LDS read, of the other buffer too, wait for the load it knows of.
// Nobody but s_waitcnt vmcnt(0) and a barrier says that the data is there.
// The compiler counts no wait states here: the base is copied by a scalar
// instruction, as a load that reads it too soon after a vector instruction
// wrote it (a readlane) would not wait for it, and the copy is the state that
// M0 wants between its write and the load.
template <int W>
__device__ inline void pa_to_lds(const __bf16* base, unsigned offset,
                                 __bf16* tile) {
  const unsigned to = (unsigned)(__UINTPTR_TYPE__)(
      (__attribute__((address_space(3))) __bf16*)tile);
  const __bf16* from;
  if constexpr (W == 16)
    asm volatile(
        "s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\t"
        "global_load_lds_dwordx4 %2, %0"
        : "=&s"(from) : "s"(to), "v"(offset), "s"(base) : "m0");
  else
    asm volatile(
        "s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\t"
        "global_load_lds_dword %2, %0"
        : "=&s"(from) : "s"(to), "v"(offset), "s"(base) : "m0");
}

// Brings [ROWS][DP] tiles of one sequence's head slice into LDS, the
// next one while this one's products run: straight from memory, 64 lanes
// an instruction, the swizzle in the lane's choice of its source.  What is
// behind D is not loaded: the caller zeroes the buffers once.  Rows behind
// the sequence repeat its last row; their weights are 0.  W = 2 has no such
// load and moves its elements in arrive() instead.
//
// start() after the barrier that frees the buffer, arrive() before the one
// that hands it over; both are called by the whole workgroup.
template <int DP, int W, int ROWS = PA_STEP>
struct PaStage {
  static const int LANES = DP * 2 / W;          // of a row
  static const int N = ROWS * LANES / PA_BLOCK;
  static const int STEP = PA_BLOCK / LANES;     // rows of 256 lanes
  const __bf16* base;  // of the sequence's row 0
  int stride;  // below 2^24
  int len, D;
  unsigned from, col;  // a thread's first load: its row and column, bytes

  __device__ PA_INLINE PaStage(const __bf16* base, long stride, int len,
                               int D)
      : base(base), stride((int)stride), len(len), D(D) {
    const int r = threadIdx.x / LANES, in = threadIdx.x % LANES * (W / 2);
    from = (unsigned)(r * this->stride) * 2;
    col = ((((in >> 3) ^ pa_swz<DP>(r)) << 3) + (in & 7)) * 2;
  }
  // f(u, byte of the sequence from `row0` on) for each of the thread's
  // loads; WHOLE: the tile has all its rows, the byte counts from row
  // STEP u on.  The loads are STEP rows apart, and the swizzle of STEP u
  // rows on is another by one exclusive or: four of 2048, 16 heads of 100
  // over 4, 4 bytes a lane, forward 163 -> 108 us, backward 472 -> 362.
  template <bool WHOLE, typename F>
  __device__ PA_INLINE void each(int row0, F f) {
    const int last = len - 1 - row0;  // >= 0: the tile has a row
    int row = threadIdx.x / LANES;
    unsigned in = col;
    // made anew here, not held in registers for every u
    if (!WHOLE) asm volatile("" : "+v"(row));
    if (!WHOLE || W < 16) asm volatile("" : "+v"(in));
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const unsigned c = in ^ (unsigned)(pa_swz<DP>(u * STEP) << 4);
      if (c >= (unsigned)D * 2) continue;
      if (WHOLE)
        f(u, from + c);
      else
        f(u, (unsigned)(min(row + u * STEP, last) * stride) * 2 + c);
    }
  }
  __device__ PA_INLINE void start(int row0, __bf16* tile) {
    if constexpr (W > 2) {
      const __bf16* at = base + (long)row0 * stride;
      const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      __bf16* to = tile + wave * 64 * (W / 2);
      if (row0 + ROWS <= len)
        each<true>(row0, [&](int u, unsigned byte) PA_INLINE {
          pa_to_lds<W>(at + (long)(u * STEP) * stride, byte,
                       to + u * PA_BLOCK * (W / 2));
        });
      else
        each<false>(row0, [&](int u, unsigned byte) PA_INLINE {
          pa_to_lds<W>(at, byte, to + u * PA_BLOCK * (W / 2));
        });
    }
  }
  __device__ PA_INLINE void arrive(int row0, __bf16* tile) {
    if constexpr (W > 2) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
      const __bf16* at = base + (long)row0 * stride;
      each<false>(row0, [&](int u, unsigned byte) PA_INLINE {
        tile[u * PA_BLOCK + threadIdx.x] = at[byte / 2];
      });
    }
  }
};

// Zeroes `rows` rows.
template <int DP>
__device__ inline void pa_clear(__bf16* tile, int rows) {
  const u32x4 z = {0u, 0u, 0u, 0u};
  for (int i = threadIdx.x; i < rows * DP / 8; i += PA_BLOCK)
    reinterpret_cast<u32x4*>(tile)[i] = z;
}

// Whether a tile holds an infinity or NaN (this thread's share of it).
template <int DP, int ROWS>
__device__ inline bool pa_tile_nonfinite(const __bf16* tile) {
  bool bad = false;
#pragma unroll
  for (int u = 0; u < ROWS * DP / 8 / PA_BLOCK; ++u)
    bad |= pa_nonfinite(*reinterpret_cast<const bf16x8*>(
        tile + (threadIdx.x + u * PA_BLOCK) * 8));
  return bad;
}

// A product sums over masked pairs too, with a weight of 0; an infinity
// or NaN there would come through as NaN.  A tile on the diagonal that
// holds one is taken apart: acc[column l & 31] += x for each such x of a
// row that the column may see, and the tile keeps zeros in their place.
// Columns see row i if i <= lim (DOWN) or i >= lim.
template <int DP, int ROWS, bool DOWN>
__device__ inline void pa_poison(const __bf16* tile, f32x16 (&acc)[DP / 32],
                                 int lim, int lane) {
  for (int i = 0; i < ROWS; ++i) {
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
template <int DP, int ROWS>
__device__ inline void pa_cleanse(__bf16* tile) {
  for (int id = threadIdx.x; id < ROWS * DP / 2; id += PA_BLOCK) {
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
// A table's entry as it stands in memory.
__device__ inline unsigned pa_table(const PaBias& b, int bucket, int heads,
                                    int h) {
  const long at = (long)bucket * heads + h;
  if (b.is_bf16) return static_cast<const unsigned short*>(b.table)[at];
  return static_cast<const unsigned*>(b.table)[at];
}
// A bias in the base-2 exponents that scores are held in.  Finite ones
// beyond 1e37 (the types' lowest values, as masks) count as that: they
// still drown any score, and stay finite.
__device__ inline float pa_bias(unsigned entry, int is_bf16) {
  const float x = __uint_as_float(is_bf16 ? entry << 16 : entry);
  const bool finite = x > -INFINITY && x < INFINITY;
  const float y = x * PA_LOG2E;
  return finite ? fminf(fmaxf(y, -1e37f), 1e37f) : y;
}
// Whether a tile's one bias can be added outside of the scores' fma, to the
// maximum that is taken off them: that is the sum with a score, and what the
// sum's rounding drops of the score stays in the exponent.  Up to 2^14 that
// is 2^-11 at most, a tenth of the weights' own step in bf16; beyond 2^30 it
// could be the score itself, without a maximum taken off.  There each score
// is rounded with the bias before the maximum is, as in tiles of several
// biases: one of 4001, 12 heads of 64, forward 54 -> 67 us.
__device__ inline bool pa_moderate(float x) { return fabsf(x) <= 16384.f; }

__device__ inline const __bf16* pa_at(const PaTensor& t, long row, int head) {
  return static_cast<const __bf16*>(t.p) + row * t.row + head * t.head;
}

// Where a workgroup's accumulator `i` (of n, four values a thread) of a
// chunk goes: consecutive threads next to each other.
__device__ inline f32x4* pa_sums(const PaWork& w, int slot, int heads, int h,
                                 int n, int i) {
  return reinterpret_cast<f32x4*>(w.sums) +
         (((long)slot * heads + h) * n + i) * PA_BLOCK + threadIdx.x;
}
// And its statistics of row `r` of the tile.
__device__ inline float* pa_rows(const PaWork& w, int slot, int heads, int h,
                                 int r) {
  return w.rows + (((long)slot * heads + h) * PA_ROWS + r) * 2;
}

// Workgroups go round the 8 XCDs in turn.  Where the heads divide, an XCD
// gets neighbouring heads, which share keys and values in its L2.
__device__ inline int pa_head(int c, int heads) {
  return (heads & 7) ? c : (c & 7) * (heads >> 3) + (c >> 3);
}
