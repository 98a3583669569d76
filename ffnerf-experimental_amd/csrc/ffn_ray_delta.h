// ffn_ray_delta.h -- a matrix state a ray and head, written by the delta rule with decay, and its gradients: the kernels, which
// ffn_ray_delta_f32.hip, _f16.hip and _bf16.hip make for their types.
//
//   S_t = a_t S_{t-1} + k_t n_t^T,  n_t = b_t (v_t - a_t S_{t-1}^T k_t),  a_t = exp(decay_t),  o_t = scale S_t^T q_t
//
// In chunks of 16 rows, one matrix tile.  Inside a chunk, with D_ij = exp(decay_{j+1} + .. + decay_i) and e_i the same
// from the chunk's start, the rows' writes n solve a unit triangular system, and everything else is a matrix product:
//   A_ij = b_i D_ij k_i.k_j (j < i),  T = (I + A)^-1,  n = T R,  R_i = b_i (v_i - e_i S^T k_i)
//   P_ij = scale D_ij q_i.k_j (j <= i),  o_i = scale e_i S^T q_i + sum_j P_ij n_j,  S' = e_15 S + sum_j D_15,j k_j n_j^T
// Marched rays are short: a chunk of 16 wastes less of their last tile than a longer one, and its triangle is solved by
// substitution (sums of powers of A would cancel where neighbouring keys are alike, as they are along a ray).  Sums of
// decays are taken anew for every pair, so that neither a reset (decay = -infinity) nor a strong decay before a row costs
// the pairs after it their accuracy.
//
// A block is a ray and head; its wavefronts each hold 16 columns of S, whose columns do not touch each other, in product
// layout (lane c + 16 g: column c, rows 4 g + r of each 16), which is that of a product's second operand as well.  T and P
// belong to the rows alone: the wavefronts make those of a segment's chunks side by side and share them through LDS.
//
// Products: in float, by the K = 4 instruction.  Of bfloat16 inputs the rows are exact operands of the 16-bit instruction,
// and what they meet (S, n, dS: float) goes as three bfloat16 parts, which together are the float itself: three products
// at 16 times the rate (K = 32; 8 times at K = 16), to the same accuracy.  (A product whose second operand has K = 16 too
// stays in float where making its parts would cost the vector ALU more than the matrix cores save.)
//
// What bounds it, us a kernel in a trace (calls in a row, as the variants further down are compared, take up to a tenth less)
// with what memory alone would take of q, k, v, o and their gradients (4.63 TB/s): 8192 marched rays, 4 heads of 32 x 32, bf16,
// forward 137 (43), backward 365 (43): the vector ALU, 61 to 65 % busy, beside the waits of short rays' few chunks; 24 rays of
// up to 4096 rows, 8 heads of 64 x 64 on 4, bf16, 471 and 1350 + 61 (98 in all): what a block does for a chunk, the chain from
// state to state and all else between its barriers, 1.8 and 5.3 us for each of a ray's 256, at less than a wavefront a SIMD;
// 3001 rays, 3 heads of 24 x 40, fp32, with states, 111 and 291 (92): vector ALU and fp32 matrix cores a third each.  Not kept,
// us when each was tried: the next segment's v ahead in the forward 163 (149 without); the heads of a ray one after the other
// in a block 204 and 602 (139 and 352: the longest ray's chain is four times as long).  Not built: states kept every chunk
// (twice the marks).  Backward passes of 128 x 128, and of 128 x 16 in fp32, spill 31 to 154 registers (1024 marched rays, 2
// heads of 128 x 128, bf16, 408 us in a row).
#pragma once
#include <algorithm>
#include <type_traits>

#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int DL_C = 16;              // rows of a chunk
constexpr int DL_SEG = 2;             // chunks between two states that are kept for the backward pass
constexpr int DL_MARK = DL_C * DL_SEG;
constexpr int DL_LD = 20;             // LDS row of a 16 x 16 matrix
constexpr int DL_VEC = 64;            // a chunk's b, e, D_15 and (first of the last 16) e_15
constexpr float DL_RESET = -1e30f;    // stands for a decay of -infinity, which must not meet a zero in a product
constexpr int DL_BLOCKS = 4096;       // heads of rays, 16 a CU: more than run at once
constexpr int DL_FEW = 8;             // rows of a ray that are taken row by row at most
constexpr int DL_PICK = 509;          // blocks that look for rays of more, two a CU; a prime, as rays may be long in a pattern
constexpr int DL_CLEAR = 1024;        // rows that one block looks through for those of no ray

// ---------------------------------------------------------------------------
// products

__device__ __forceinline__ f32x4 mma4(float a, float b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(const b16x4& a, const b16x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma32(const b16x4& a0, const b16x4& a1, const b16x4& b0, const b16x4& b1, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7),
                                                 __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7), c, 0, 0, 0);
}
// A b for a 16 x 16 A, this lane's four values of its row c and columns 4 g + s, on a product
__device__ __forceinline__ f32x4 mul16(const f32x4& a, const f32x4& b, f32x4 to) {
#pragma unroll
  for (int s = 0; s < 4; ++s) to = mma4(a[s], b[s], to);
  return to;
}

// Four floats as three bfloat16 parts, by cutting 8 bits of the 24 each time, which together are the float itself.
struct Parts {
  b16x4 p[3];
};
__device__ __forceinline__ b16x4 upper_of(const f32x4& x) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x4 w = __builtin_bit_cast(u32x4, x);
  const u32x2 up = {__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
  return __builtin_bit_cast(b16x4, up);
}
__device__ __forceinline__ f32x4 rest_of(const f32x4& x) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  return x - __builtin_bit_cast(f32x4, __builtin_bit_cast(u32x4, x) & 0xFFFF0000u);
}
__device__ __forceinline__ Parts parts_of(const f32x4& x) {
  const f32x4 r = rest_of(x);
  return {{upper_of(x), upper_of(r), upper_of(rest_of(r))}};
}

// How a type's rows enter products.  Row: four neighbouring values of a row.  Full: a float operand.
template <typename T> struct Delta {
  static constexpr bool EXACT = false;
  typedef f32x4 Row;
  typedef f32x4 Full;
  static __device__ __forceinline__ Full full(const f32x4& x) { return x; }
  static __device__ __forceinline__ f32x4 value(const Row& x) { return x; }
  // on a product: 16 values of K from each operand's lane parts, then 32
  template <typename A, typename B> static __device__ __forceinline__ f32x4 mul(const A& a, const B& b, const f32x4& c) { return mul16(a, b, c); }
  template <typename A, typename B>
  static __device__ __forceinline__ f32x4 mul(const A& a0, const A& a1, const B& b0, const B& b1, const f32x4& c) {
    return mul16(a1, b1, mul16(a0, b0, c));
  }
};
template <> struct Delta<__bf16> {
  static constexpr bool EXACT = true;
  typedef b16x4 Row;
  typedef Parts Full;
  static __device__ __forceinline__ Full full(const f32x4& x) { return parts_of(x); }
  static __device__ __forceinline__ f32x4 value(const Row& x) { return __builtin_convertvector(x, f32x4); }
  static __device__ __forceinline__ f32x4 mul(const Row& a, const Row& b, const f32x4& c) { return mma16(a, b, c); }
  static __device__ __forceinline__ f32x4 mul(const Row& a, const Full& b, f32x4 c) {
#pragma unroll
    for (int i = 2; i >= 0; --i) c = mma16(a, b.p[i], c);
    return c;
  }
  static __device__ __forceinline__ f32x4 mul(const Full& a, const Row& b, f32x4 c) {
#pragma unroll
    for (int i = 2; i >= 0; --i) c = mma16(a.p[i], b, c);
    return c;
  }
  // of two floats: the six largest of nine products, the smallest first.  Those left out are some 2^-24 of a b, and 2^-20 at
  // most; with two of them more no result was nearer to 64 bits, and the backward's registers cost a wavefront a SIMD.
  static __device__ __forceinline__ f32x4 mul(const Full& a, const Full& b, f32x4 c) {
#pragma unroll
    for (int s = 2; s >= 0; --s) {
#pragma unroll
      for (int i = 0; i <= s; ++i) c = mma16(a.p[i], b.p[s - i], c);
    }
    return c;
  }
  static __device__ __forceinline__ f32x4 mul(const Row& a0, const Row& a1, const Row& b0, const Row& b1, const f32x4& c) {
    return mma32(a0, a1, b0, b1, c);
  }
  static __device__ __forceinline__ f32x4 mul(const Row& a0, const Row& a1, const Full& b0, const Full& b1, f32x4 c) {
#pragma unroll
    for (int i = 2; i >= 0; --i) c = mma32(a0, a1, b0.p[i], b1.p[i], c);
    return c;
  }
  static __device__ __forceinline__ f32x4 mul(const Full& a0, const Full& a1, const Row& b0, const Row& b1, f32x4 c) {
#pragma unroll
    for (int i = 2; i >= 0; --i) c = mma32(a0.p[i], a1.p[i], b0, b1, c);
    return c;
  }
  static __device__ __forceinline__ f32x4 mul(const Full& a0, const Full& a1, const Full& b0, const Full& b1, f32x4 c) {
#pragma unroll
    for (int s = 2; s >= 0; --s) {
#pragma unroll
      for (int i = 0; i <= s; ++i) c = mma32(a0.p[i], a1.p[i], b0.p[s - i], b1.p[s - i], c);
    }
    return c;
  }
};

// sum over the tiles of a and b, an even number
template <typename T, int N, typename A, typename B>
__device__ __forceinline__ f32x4 mul_tiles(const A (&a)[N], const B (&b)[N], f32x4 c) {
  if constexpr (Delta<T>::EXACT) {
#pragma unroll
    for (int t = 0; t < N; t += 2) c = Delta<T>::mul(a[t], a[t + 1], b[t], b[t + 1], c);
    return c;
  } else {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};  // two chains
#pragma unroll
    for (int t = 0; t < N; t += 2) {
      c = Delta<T>::mul(a[t], b[t], c);
      d = Delta<T>::mul(a[t + 1], b[t + 1], d);
    }
    return c + d;
  }
}

// ---------------------------------------------------------------------------
// rows and states

template <typename T> __device__ __forceinline__ f32x4 load4(const T* p) {
  typedef T tvec __attribute__((ext_vector_type(4)));
  return __builtin_convertvector(*reinterpret_cast<const tvec*>(p), f32x4);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const f32x4& x) {
  typedef T tvec __attribute__((ext_vector_type(4)));
  *reinterpret_cast<tvec*>(p) = __builtin_convertvector(x, tvec);
}
// A tile of 16 rows and 16 columns in LDS, LD values a row: an operand by rows (this lane's row c, columns 4 g + s) or, the
// transposed one, by columns (column c, rows 4 g + s).  Neither meets a bank twice.
template <typename T> struct Tile {
  static constexpr int LD = sizeof(T) == 4 ? 20 : Delta<T>::EXACT ? 16 : 24, SIZE = DL_C * LD;
};
// where a tile has the four values from column 4 u of row r: in 16 bits rows lie side by side, and the lower eight have their
// halves changed over, so that 32 lanes that take a row each and a four of it meet every bank once
template <typename T> __device__ __forceinline__ int four_at(int r, int u) {
  if constexpr (Delta<T>::EXACT) return r * 16 + 4 * (u ^ ((r >> 3) << 1));
  else return r * Tile<T>::LD + 4 * u;
}
// the same of a matrix of floats whose rows lie side by side
__device__ __forceinline__ int float4_at(int r, int u) { return r * 16 + 4 * (u ^ (r >> 2)); }
template <typename T> __device__ __forceinline__ typename Delta<T>::Row row_of(const T* tile, int c, int g) {
  const T* p = tile + four_at<T>(c, g);
  if constexpr (Delta<T>::EXACT) return *reinterpret_cast<const b16x4*>(p);
  else return load4(p);
}
template <typename T> __device__ __forceinline__ typename Delta<T>::Row col_of(const T* tile, int c, int g) {
  if constexpr (Delta<T>::EXACT) {
    typedef __attribute__((address_space(3))) s16x4* lds_quad;
    return __builtin_bit_cast(b16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(tile + four_at<T>(4 * g + (c >> 2), c & 3))));
  } else {
    f32x4 x;
#pragma unroll
    for (int s = 0; s < 4; ++s) x[s] = (float)tile[(4 * g + s) * Tile<T>::LD + c];
    return x;
  }
}

// x of another lane of this lane's 16, by one of the moves within them (0 where there is none)
template <int MOVE> __device__ __forceinline__ float moved(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), MOVE, 0xF, 0xF, true));
}
// sum over the 16 lanes of a group: within pairs, fours, halves, and of both
__device__ __forceinline__ f32x4 sum16(f32x4 x) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    x[r] += moved<0xB1>(x[r]);
    x[r] += moved<0x4E>(x[r]);
    x[r] += moved<0x141>(x[r]);
    x[r] += moved<0x140>(x[r]);
  }
  return x;
}
// sum over this lane and those after it in its 16
__device__ __forceinline__ float sum_after(float x) {
  x += moved<0x101>(x);
  x += moved<0x102>(x);
  x += moved<0x104>(x);
  x += moved<0x108>(x);
  return x;
}

// The rows of a ray in the order of the recurrence.
struct Chain {
  int64_t first;  // lowest row
  int count;
  bool back;
};
__device__ __forceinline__ Chain chain_of(const ffn_ray_delta& a, int64_t ray) {
  const int64_t n = a.rays.n, o = min((int64_t)a.rays.offsets[ray], n), c = min((int64_t)a.rays.counts[ray], n - o);
  return {o, (int)c, a.reverse != 0};
}
// where the state before place p (a multiple of DL_MARK above 0) is kept: places of one ray, and of rays that do not
// overlap, never share a slot
__device__ __forceinline__ int64_t mark_slot(const Chain& ch, int p) { return (uint32_t)(ch.first + p) / DL_MARK; }

// The rows of the chunk at place p0: `many` of them from row `low` on.  Place i's row is low + at(i); past the ray's end it
// is that of the last place, whose values are then dropped: under a branch each load would wait for the one before it.
struct Chunk {
  uint32_t low;
  int many;
  bool back;
  __device__ __forceinline__ Chunk(const Chain& ch, int p0)
      : low(0), many(min(DL_C, ch.count - p0)), back(ch.back) {
    low = (uint32_t)ch.first + (uint32_t)(back ? ch.count - p0 - many : p0);
  }
  // its first row in an array of rows `stride` < 2^24 bytes apart
  template <typename T> __device__ __forceinline__ T* in(T* p, int64_t stride) const {
    typedef typename std::conditional<std::is_const<T>::value, const char, char>::type byte;
    return reinterpret_cast<T*>(reinterpret_cast<byte*>(p) + (uint64_t)low * ((uint32_t)stride * (uint32_t)sizeof(T)));
  }
  __device__ __forceinline__ uint32_t at(int i) const {
    const int j = min(i, many - 1);
    return back ? many - 1 - j : j;
  }
};

// `at` < 16 rows and `col` elements on from p, rows `stride` < 2^24 bytes apart: a base of the wavefront and 32 bits of the lane
template <typename T> __device__ __forceinline__ T* row_ptr(T* p, uint32_t at, int64_t stride, uint32_t col) {
  typedef typename std::conditional<std::is_const<T>::value, const char, char>::type byte;
  const uint32_t off = __umul24(at, (uint32_t)(stride * (int64_t)sizeof(T))) + col * (uint32_t)sizeof(T);
  return reinterpret_cast<T*>(reinterpret_cast<byte*>(p) + off);
}
// the rows of places 4 g + r of a chunk
struct Rows4 {
  uint32_t at[4];
  __device__ __forceinline__ Rows4(const Chunk& ck, int g) {
#pragma unroll
    for (int r = 0; r < 4; ++r) at[r] = ck.at(4 * g + r);
  }
};

// column `col` of a chunk's rows 4 g + r, those that are there; p: the chunk's first row
template <typename T>
__device__ __forceinline__ void put_rows(T* p, const Chunk& ck, const Rows4& rows, int g, int stride, int col, const f32x4& x) {
  if (ck.many == DL_C) {
#pragma unroll
    for (int r = 0; r < 4; ++r) *row_ptr(p, rows.at[r], stride, col) = (T)x[r];
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * g + r < ck.many) *row_ptr(p, rows.at[r], stride, col) = (T)x[r];
  }
}

// this lane's part of a chunk's row c: four values of every 16 columns, as they lie in memory
template <typename T, int N> struct RawRow {
  typedef T tvec __attribute__((ext_vector_type(4)));
  tvec v[N];
  __device__ __forceinline__ void load(const T* base, int64_t stride, const Chunk& ck, int c, int g, int cols) {
    const uint32_t at = ck.at(c);
    if (cols == 16 * N) {
      const T* p = row_ptr(ck.in(base, stride), at, stride, 4 * g);
#pragma unroll
      for (int t = 0; t < N; ++t) v[t] = *reinterpret_cast<const tvec*>(p + 16 * t);
    } else {
#pragma unroll
      for (int t = 0; t < N; ++t)
        v[t] = *reinterpret_cast<const tvec*>(row_ptr(ck.in(base, stride), at, stride, 16 * t + 4 * g < cols ? 16 * t + 4 * g : 0));
    }
  }
  // 0 past the ray's end or the columns
  __device__ __forceinline__ void trim(const Chunk& ck, int c, int g, int cols) {
    if (ck.many == DL_C && cols == 16 * N) return;
#pragma unroll
    for (int t = 0; t < N; ++t) v[t] = c < ck.many && 16 * t + 4 * g < cols ? v[t] : tvec{};
  }
  __device__ __forceinline__ void operands(typename Delta<T>::Row (&to)[N]) const {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      if constexpr (Delta<T>::EXACT) to[t] = v[t];
      else to[t] = __builtin_convertvector(v[t], f32x4);
    }
  }
};
// column `col` of the chunk's rows 4 g + r
template <typename T> struct RawCol {
  T v[4];
  __device__ __forceinline__ void load(const T* base, int64_t stride, const Chunk& ck, const Rows4& rows, int col, int cols) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = *row_ptr(ck.in(base, stride), rows.at[r], stride, col < cols ? col : 0);
  }
  __device__ __forceinline__ f32x4 value(const Chunk& ck, int g, int col, int cols) const {
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = (float)v[r];
    if (ck.many < DL_C || cols % 16 || col >= cols) {  // (a wavefront may lie past the columns as a whole)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = 4 * g + r < ck.many && col < cols ? x[r] : 0.f;
    }
    return x;
  }
};
// the decays of the chunk's rows 4 g + r and the strength of its row c
template <typename T> struct RawGates {
  T d[4], b;
  __device__ __forceinline__ void load(const ffn_ray_delta& a, int h, const Chunk& ck, const Rows4& rows, int c) {
    const T *dp = ck.in((const T*)a.decay + h * a.decay_head, a.decay_row), *bp = ck.in((const T*)a.beta + h * a.beta_head, a.beta_row);
    b = *row_ptr(bp, ck.at(c), a.beta_row, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) d[r] = *row_ptr(dp, rows.at[r], a.decay_row, 0);
  }
  __device__ __forceinline__ f32x4 decay(const Chunk& ck, int g) const {
    f32x4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = 4 * g + r < ck.many ? (float)d[r] : 0.f;
      y[r] = x < DL_RESET ? DL_RESET : x;
    }
    return y;
  }
  __device__ __forceinline__ float beta(const Chunk& ck, int c) const { return c < ck.many ? (float)b : 0.f; }
};

// A state's 16 columns from `w16` on, in product layout, from or to [dk][dv].
template <int NT>
__device__ __forceinline__ void load_state(f32x4 (&S)[NT], const float* from, const ffn_ray_delta& a, int c, int g, int w16) {
#pragma unroll
  for (int t = 0; t < NT; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!from) return;
  const int v = min(w16 + c, a.val_dim - 1);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) S[t][r] = from[(int64_t)min(16 * t + 4 * g + r, a.key_dim - 1) * a.val_dim + v];
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (16 * t + 4 * g + r >= a.key_dim || w16 + c >= a.val_dim) S[t][r] = 0.f;
  }
}
template <int NT>
__device__ __forceinline__ void store_state(float* to, const f32x4 (&S)[NT], const ffn_ray_delta& a, int c, int g, int w16) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 16 * t + 4 * g + r, v = w16 + c;
      if (k < a.key_dim && v < a.val_dim) to[(int64_t)k * a.val_dim + v] = S[t][r];
    }
  }
}

// A state that is kept for the backward pass, as the wavefronts hold it: lane after lane, tile after tile.
template <int NT> __device__ __forceinline__ void load_mark(f32x4 (&S)[NT], const float* from, int w, int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t) S[t] = *reinterpret_cast<const f32x4*>(from + (w * NT + t) * 256 + 4 * lane);
}
template <int NT> __device__ __forceinline__ void store_mark(float* to, const f32x4 (&S)[NT], int w, int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(to + (w * NT + t) * 256 + 4 * lane) = S[t];
}

// exp(x): the product with log2(e) in two parts, so that the result is as accurate as the hardware's 2^x
__device__ __forceinline__ float exp_of(float x) {
  const float hi = x * 1.442695041f, lo = __builtin_fmaf(x, 1.442695041f, -hi);
  const float y = __builtin_amdgcn_exp2f(hi);
  return __builtin_fmaf(y, lo * 0.6931471806f, y);
}

// x[I] += a of lane I of this lane's 16, times x[J], for all I > J in a row of instructions.  The two waits are for the
// lanes' values of a, which a vector instruction may just have written.
#define DL_TAKE(I) "v_fmac_f32_dpp %" #I ", %16, %17 row_newbcast:" #I " row_mask:0xf bank_mask:0xf\n"
template <int J> __device__ __forceinline__ void take_off(float a, float (&x)[DL_C]) {
  const float y = x[J];
#define DL_X "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]), "+v"(x[8]), \
    "+v"(x[9]), "+v"(x[10]), "+v"(x[11]), "+v"(x[12]), "+v"(x[13]), "+v"(x[14]), "+v"(x[15])
#define DL_STEP(N, CODE) \
  if constexpr (J == N) asm("s_nop 1\n" CODE : DL_X : "v"(a), "v"(y));
  DL_STEP(14, DL_TAKE(15))
  DL_STEP(13, DL_TAKE(14) DL_TAKE(15))
  DL_STEP(12, DL_TAKE(13) DL_TAKE(14) DL_TAKE(15))
  DL_STEP(11, DL_TAKE(12) DL_TAKE(13) DL_TAKE(14) DL_TAKE(15))
#define DL_12 DL_TAKE(12) DL_TAKE(13) DL_TAKE(14) DL_TAKE(15)
  DL_STEP(10, DL_TAKE(11) DL_12)
  DL_STEP(9, DL_TAKE(10) DL_TAKE(11) DL_12)
  DL_STEP(8, DL_TAKE(9) DL_TAKE(10) DL_TAKE(11) DL_12)
#define DL_8 DL_TAKE(8) DL_TAKE(9) DL_TAKE(10) DL_TAKE(11) DL_12
  DL_STEP(7, DL_8)
  DL_STEP(6, DL_TAKE(7) DL_8)
  DL_STEP(5, DL_TAKE(6) DL_TAKE(7) DL_8)
  DL_STEP(4, DL_TAKE(5) DL_TAKE(6) DL_TAKE(7) DL_8)
#define DL_4 DL_TAKE(4) DL_TAKE(5) DL_TAKE(6) DL_TAKE(7) DL_8
  DL_STEP(3, DL_4)
  DL_STEP(2, DL_TAKE(3) DL_4)
  DL_STEP(1, DL_TAKE(2) DL_TAKE(3) DL_4)
  DL_STEP(0, DL_TAKE(1) DL_TAKE(2) DL_TAKE(3) DL_4)
#undef DL_TAKE
#undef DL_X
#undef DL_STEP
#undef DL_12
#undef DL_8
#undef DL_4
}
// Column c of X with (I + A) X = I: x[J] is done when the rows before it have been taken off.  a[j] = -A[c][j].  (By rows of
// X a NaN in a row of A would meet the zeros of the rows before it.)
template <int J> __device__ __forceinline__ void solve(const float (&a)[DL_C], float (&x)[DL_C]) {
  take_off<J>(a[J], x);
  if constexpr (J + 2 < DL_C) solve<J + 1>(a, x);
}

// What a chunk's rows do to each other, by one wavefront: T, P and (if Dm) D as [row i][column j], and the rows' vectors.
// decay: those of rows 4 g + r (at least DL_RESET), beta: that of row c.  Sums of decays are products with zeros and ones.
template <typename T, int NT>
__device__ __forceinline__ void prepare_chunk(const typename Delta<T>::Row (&kf)[NT], const typename Delta<T>::Row (&qf)[NT],
                                              const f32x4& decay, float beta, float scale, int c, int g, float* Tm, float* Pm,
                                              float* Dm, float* vec) {
  // row j = 4 g + r, column i = c: the sum of decays from j + 1 to i, k_j.k_i and k_j.q_i
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 sum = zero;
#pragma unroll
  for (int s = 0; s < 4; ++s) sum = mma4(4 * g + s > c ? 1.f : 0.f, 4 * g + s <= c ? decay[s] : 0.f, sum);
  const f32x4 kk = mul_tiles<T>(kf, kf, zero), kq = mul_tiles<T>(kf, qf, zero);
  f32x4 D, P, A;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = 4 * g + r;
    const float d = exp_of(sum[r]);
    D[r] = j <= c ? d : 0.f;
    P[r] = j <= c ? scale * d * kq[r] : 0.f;
    A[r] = j < c ? -beta * d * kk[r] : 0.f;
  }
  *reinterpret_cast<f32x4*>(Tm + c * DL_LD + 4 * g) = A;
  *reinterpret_cast<f32x4*>(Pm + c * DL_LD + 4 * g) = P;
  if (Dm) *reinterpret_cast<f32x4*>(Dm + float4_at(c, g)) = D;
  const float e = exp_of(decay[0] + sum[0]);  // in the first group, from the chunk's start to row c
  if (g == 0) {
    vec[c] = beta;
    vec[16 + c] = e;
    if (c == DL_C - 1) vec[48] = e;
  }
  if (c == DL_C - 1) *reinterpret_cast<f32x4*>(vec + 32 + 4 * g) = D;
  wave_sync();
  float a[DL_C], x[DL_C];
#pragma unroll
  for (int i = 0; i < DL_C; i += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(Tm + c * DL_LD + i);
#pragma unroll
    for (int r = 0; r < 4; ++r) a[i + r] = v[r], x[i + r] = i + r == c ? 1.f : 0.f;
  }
  solve<0>(a, x);
  wave_sync();
#pragma unroll
  for (int r = 0; r < 4; ++r) Tm[(4 * g + r) * DL_LD + c] = g == 0 ? x[r] : g == 1 ? x[4 + r] : g == 2 ? x[8 + r] : x[12 + r];
}

__device__ __forceinline__ bool finite4(const f32x4& x) {
  return fabsf(x[0]) <= 3.4e38f && fabsf(x[1]) <= 3.4e38f && fabsf(x[2]) <= 3.4e38f && fabsf(x[3]) <= 3.4e38f;
}
// A x for a lower triangular A where x holds infinities or NaN: they must not meet the zeros above the diagonal, so they
// are left out, and the rows from the first of them on are NaN.
__device__ __forceinline__ f32x4 mul16_sick(const f32x4& A, f32x4 x, const f32x4& to, int g) {
  int first = DL_C;
#pragma unroll
  for (int r = 3; r >= 0; --r) {
    if (!(fabsf(x[r]) <= 3.4e38f)) {
      first = 4 * g + r;
      x[r] = 0.f;
    }
  }
  first = min(first, __shfl_xor(first, 16));
  first = min(first, __shfl_xor(first, 32));
  f32x4 y = mul16(A, x, to);
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * g + r >= first) y[r] = __builtin_nanf("");
  return y;
}

// rows of no ray: 0 in `heads` x `cols` of each output
template <typename T>
__device__ __forceinline__ void clear_rows(const ffn_ray_delta& a, int64_t block, T* p, int64_t width) {
  for (int64_t i = block * DL_CLEAR + threadIdx.x; i < min((block + 1) * DL_CLEAR, (int64_t)a.rays.n); i += blockDim.x) {
    const uint32_t r = a.rays.ray_ids[i];
    if (r < a.rays.num_rays) {
      const int64_t o = a.rays.offsets[r];
      if (i >= o && i - o < (int64_t)a.rays.counts[r]) continue;
    }
    for (int64_t j = 0; j < width; ++j) p[i * width + j] = (T)0.f;
  }
}

// a / b of a block's number: both fit 32 bits in nearly every call
__device__ __forceinline__ int64_t quotient(int64_t a, int b) {
  return a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// wavefronts a SIMD that the forward's registers are held to, where no spill comes of it
template <typename T, int DK, int W> constexpr int DL_FWD_WAVES = Delta<T>::EXACT && DK == 32 && W <= 2 ? 5 : 1;

// PICK: of the rays alone that have more rows than `longer`.  A block then looks at 64 heads of rays at once, the number of
// blocks apart (long rays lie side by side), and takes the long ones one after the other.
template <typename T, int DK, int W, bool PICK>
__global__ __launch_bounds__(64 * W, (PICK ? 1 : DL_FWD_WAVES<T, DK, W>)) void k_delta_fwd(const ffn_ray_delta a, int longer) {
  constexpr int NT = DK / 16, TILE = Tile<T>::SIZE, CH = W < 4 ? W : 4;
  typedef Delta<T> Ops;
  typedef typename Ops::Row Row;
  __shared__ float Tm[CH][DL_C * DL_LD], Pm[CH][DL_C * DL_LD], vec[CH][DL_VEC];
  __shared__ __align__(16) T Kl[CH * NT * TILE], Ql[CH * NT * TILE];
  const int64_t teams = (int64_t)a.rays.num_rays * a.v_heads;
  int64_t block = block_number();
  const int lane = threadIdx.x & 63, w = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w16 = 16 * w;
  const int64_t base = block, apart = (int64_t)gridDim.x * gridDim.y;
  uint64_t found = 1;
  if constexpr (PICK) {
    const int64_t mine = base + lane * apart;
    found = __ballot(mine < teams && chain_of(a, quotient(min(mine, teams - 1), a.v_heads)).count > longer);
  }
  for (; found; found &= found - 1) {
    bool first = false;
    if constexpr (PICK) {
      block = base + __builtin_ctzll(found) * apart;
    } else {
      first = longer && block < teams;  // of two turns: the rays with more rows than `longer`
      if (longer && !first) block -= teams;
      if (block >= teams) {
        clear_rows(a, block - teams, (T*)a.o, (int64_t)a.v_heads * a.val_dim);
        return;
      }
    }
    const int64_t ray = quotient(block, a.v_heads);
    const int h = (int)(block - ray * a.v_heads), hk = h / (a.v_heads / a.heads);
    const Chain ch = chain_of(a, ray);
    if (!PICK && longer && (ch.count > longer) != first) return;
    int c = lane & 15, g = lane >> 4;
    const T* q = (const T*)a.q + hk * a.q_head;
    const T* k = (const T*)a.k + hk * a.k_head;
    const T* v = (const T*)a.v + h * a.v_head;
    const int64_t size = (int64_t)a.key_dim * a.val_dim;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    // the next segment's rows are on their way while a segment is worked on
    RawRow<T, NT> kr, qr;
    RawGates<T> gates;
    const auto fetch = [&](int p) {
      if (w < CH && p < ch.count) {
        const Chunk ck(ch, p);
        kr.load(k, a.k_row, ck, c, g, a.key_dim);
        qr.load(q, a.q_row, ck, c, g, a.key_dim);
        gates.load(a, h, ck, Rows4(ck, g), c);
      }
    };
    fetch(DL_C * w);
    f32x4 S[NT];
    load_state(S, a.h0 ? a.h0 + block * size : nullptr, a, c, g, w16);
#pragma unroll 1
    for (int p0 = 0; p0 < ch.count; p0 += CH * DL_C) {
      asm volatile("" : "+v"(c), "+v"(g));  // opaque: else all that goes by the lane alone is formed ahead, and held
      RawCol<T> vr[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (p0 + DL_C * i < ch.count) {
          const Chunk ck(ch, p0 + DL_C * i);
          vr[i].load(v, a.v_row, ck, Rows4(ck, g), w16 + c, a.val_dim);
        }
      if (w < CH && p0 + DL_C * w < ch.count) {
        const Chunk ck(ch, p0 + DL_C * w);
        kr.trim(ck, c, g, a.key_dim);
        qr.trim(ck, c, g, a.key_dim);
        Row kf[NT], qf[NT];
        kr.operands(kf);
        qr.operands(qf);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          typedef typename RawRow<T, NT>::tvec tvec;
          *reinterpret_cast<tvec*>(Kl + (w * NT + t) * TILE + four_at<T>(c, g)) = kr.v[t];
          *reinterpret_cast<tvec*>(Ql + (w * NT + t) * TILE + four_at<T>(c, g)) = qr.v[t];
        }
        prepare_chunk<T>(kf, qf, gates.decay(ck, g), gates.beta(ck, c), a.scale, c, g, Tm[w], Pm[w], (float*)nullptr, vec[w]);
        fetch(p0 + DL_C * (CH + w));
      }
      if constexpr (W > 1) __syncthreads();
      else wave_sync();
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int p = p0 + DL_C * i;
        if (p < ch.count) {
          const Chunk ck(ch, p);
          if (a.marks && p && p % DL_MARK == 0) store_mark(a.marks + (mark_slot(ch, p) * a.v_heads + h) * (NT * W * 256), S, w, lane);
          const T *Kc = Kl + i * NT * TILE, *Qc = Ql + i * NT * TILE;
          Row kf[NT], qf[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            kf[t] = row_of(Kc + t * TILE, c, g);
            qf[t] = row_of(Qc + t * TILE, c, g);
          }
          const f32x4 beta = *reinterpret_cast<const f32x4*>(&vec[i][4 * g]);
          const f32x4 e = *reinterpret_cast<const f32x4*>(&vec[i][16 + 4 * g]);
          const f32x4 left = *reinterpret_cast<const f32x4*>(&vec[i][32 + 4 * g]);
          const float all = vec[i][48];
          const f32x4 Tr = *reinterpret_cast<const f32x4*>(&Tm[i][c * DL_LD + 4 * g]);
          const f32x4 Pr = *reinterpret_cast<const f32x4*>(&Pm[i][c * DL_LD + 4 * g]);
          typename Ops::Full full[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) full[t] = Ops::full(S[t]);
          const f32x4 R = beta * (vr[i].value(ck, g, w16 + c, a.val_dim) - e * mul_tiles<T>(kf, full, zero));
          const f32x4 qs = a.scale * e * mul_tiles<T>(qf, full, zero);
          const f32x4 n = mul16(Tr, R, zero);
          f32x4 y = mul16(Pr, n, qs);
          const typename Ops::Full nl = Ops::full(left * n);
#pragma unroll
          for (int t = 0; t < NT; ++t) S[t] = Ops::mul(col_of(Kc + t * TILE, c, g), nl, all * S[t]);
          // a sick row leaves its columns of the state sick whatever the rows before it wrote, but not those rows' o
          if (__any(!finite4(n))) y = mul16_sick(Pr, mul16_sick(Tr, R, zero, g), qs, g);
          T* o = ck.in((T*)a.o + h * a.val_dim, a.v_heads * a.val_dim);
          if (w16 + c < a.val_dim) {
            put_rows(o, ck, Rows4(ck, g), g, a.v_heads * a.val_dim, w16 + c, y);
          }
        }
      }
      if constexpr (W > 1) __syncthreads();
      else wave_sync();
    }
    if (a.last) store_state(a.last + block * size, S, a, c, g, w16);
  }
}

// Few rows a ray (one more sample of each): the state goes through once, row by row on the vector ALU, and memory bounds
// it.  Rays of more than `most` rows are left to the chunks.  A wavefront takes 32 columns of a state: 8 lanes of four
// columns, 8 groups of rows dk = 8 i + group.
template <typename T, int DK>
__global__ __launch_bounds__(256, DK <= 32 ? 6 : DK <= 64 ? 5 : 3) void k_delta_step(const ffn_ray_delta a, int most) {
  constexpr int N = DK / 8;
  const int parts = (a.val_dim + 31) / 32;
  const int64_t teams = (int64_t)a.rays.num_rays * a.v_heads * parts, blocks = (teams + 3) / 4;
  if (block_number() >= blocks) {
    clear_rows(a, block_number() - blocks, (T*)a.o, (int64_t)a.v_heads * a.val_dim);
    return;
  }
  const int64_t team = block_number() * 4 + (threadIdx.x >> 6);
  if (team >= teams) return;
  const int64_t state = quotient(team, parts), ray = quotient(state, a.v_heads);
  const int h = (int)(state - ray * a.v_heads), hk = h / (a.v_heads / a.heads);
  const int lane = threadIdx.x & 63, rg = lane >> 3, col = (int)(team - state * parts) * 32 + 4 * (lane & 7);
  const bool in = col < a.val_dim;
  const Chain ch = chain_of(a, ray);
  if (ch.count > most) return;
  const int64_t at = state * a.key_dim * a.val_dim;
  f32x4 S[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int kd = 8 * i + rg;
    S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.h0 && in && kd < a.key_dim) S[i] = load4(a.h0 + at + (int64_t)kd * a.val_dim + col);
  }
  for (int p = 0; p < ch.count; ++p) {
    const int64_t row = ch.back ? ch.first + ch.count - 1 - p : ch.first + p;
    const T* q = (const T*)a.q + row * a.q_row + hk * a.q_head;
    const T* k = (const T*)a.k + row * a.k_row + hk * a.k_head;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (in) v = load4((const T*)a.v + row * a.v_row + h * a.v_head + col);
    const float decay = expf((float)((const T*)a.decay)[row * a.decay_row + h * a.decay_head]);
    const float beta = (float)((const T*)a.beta)[row * a.beta_row + h * a.beta_head];
    float kk[N], qq[N], qk = 0.f;
    f32x4 ks = {0.f, 0.f, 0.f, 0.f}, qs = ks;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int kd = 8 * i + rg;
      kk[i] = kd < a.key_dim ? (float)k[kd] : 0.f;
      qq[i] = kd < a.key_dim ? (float)q[kd] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      S[i] = decay * S[i];
      qk = __builtin_fmaf(qq[i], kk[i], qk);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] = __builtin_fmaf(kk[i], S[i][e], ks[e]);
        qs[e] = __builtin_fmaf(qq[i], S[i][e], qs[e]);
      }
    }
#pragma unroll
    for (int d = 8; d < 64; d *= 2) {
      qk += __shfl_xor(qk, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] += __shfl_xor(ks[e], d);
        qs[e] += __shfl_xor(qs[e], d);
      }
    }
    const f32x4 n = beta * (v - ks);
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][e] = __builtin_fmaf(kk[i], n[e], S[i][e]);
    }
    if (rg == 0 && in) store4((T*)a.o + (row * a.v_heads + h) * a.val_dim + col, a.scale * (qs + qk * n));
  }
  if (!a.last) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int kd = 8 * i + rg;
    if (in && kd < a.key_dim) store4(a.last + at + (int64_t)kd * a.val_dim + col, S[i]);
  }
}

// The backward pass.  Segments of two chunks from the ray's end, each from the state that the forward kept: its chunks'
// states and writes again, then the chunks back to front.  With dS the gradient of the state after a chunk:
//   dn = P^T do + D_15 K dS,  dR = T^T dn,  dv = b dR,  X = scale D (do n^T) (j <= i),  Y = -D (dR n^T) (j < i)
//   dq_i = scale e_i S do_i + sum_j X_ij k_j,  left_i = -e_i S dR_i + sum_j Y_ij k_j
//   right_j = D_15,j dS n_j + sum_i (X_ij q_i + b_i Y_ij k_i),  dk = b left + right,  db_i = k_i.left_i + v_i.dR_i
//   dS' = e_15 dS + sum_i (scale e_i q_i do_i^T - b_i e_i k_i dR_i^T)
// Every factor e or D a row i was multiplied with gives its sum of products to the decays up to i:
//   ddecay = sums, from each row to the chunk's end, of q.dq + b k.left - k.right, and at the end dS.S
// to the accuracy of those terms: where a decay is so strong that they cancel, not to its own.
// dn, dR, dv and dS go by columns, as S does; dq and dk are sums over the columns: S, dS, n and dR pass through LDS, and a
// wavefront takes 16 columns of dq and dk.

// Tiles of 16 x 16 floats in LDS, put down by columns as products leave them (column c, rows 4 g + r) and taken up by rows,
// as operands: floats, or three parts each.
template <typename T> struct Tiles {
  static constexpr int WORDS = Delta<T>::EXACT ? 3 * 128 : 256;  // of a tile
  float* p;
  __device__ __forceinline__ void set(int tile, int c, int g, const f32x4& x) const {
    if constexpr (Delta<T>::EXACT) {
      set(tile, c, g, parts_of(x));
    } else {
      // row 4 g + r is the (4 r + g)th, its fours of columns in an order that goes by r: neither side meets a bank twice
#pragma unroll
      for (int r = 0; r < 4; ++r) p[tile * WORDS + (4 * r + g) * 16 + 4 * ((c >> 2) ^ r) + (c & 3)] = x[r];
    }
  }
  __device__ __forceinline__ void set(int tile, int c, int g, const Parts& x) const {
    __bf16* q = (__bf16*)(p + tile * WORDS) + four_at<__bf16>(c, g);  // transposed, so that four rows lie side by side
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<b16x4*>(q + 256 * i) = x.p[i];
  }
  __device__ __forceinline__ typename Delta<T>::Full get(int tile, int c, int g) const {
    if constexpr (Delta<T>::EXACT) {
      const __bf16* q = (const __bf16*)(p + tile * WORDS);
      return {{col_of(q, c, g), col_of(q + 256, c, g), col_of(q + 512, c, g)}};
    } else {
      return *reinterpret_cast<const f32x4*>(p + tile * WORDS + (4 * (c & 3) + (c >> 2)) * 16 + 4 * (g ^ (c & 3)));
    }
  }
};
// A 16 x 16 matrix of floats, put down as this lane's row c, columns 4 g + s, and taken up by rows or by columns.
template <typename T> struct Square {
  static constexpr int WORDS = Tiles<T>::WORDS;
  float* p;
  __device__ __forceinline__ void set(int c, int g, const f32x4& x) const {
    if constexpr (Delta<T>::EXACT) {
      const Parts y = parts_of(x);
      __bf16* q = (__bf16*)p + four_at<__bf16>(c, g);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<b16x4*>(q + 256 * i) = y.p[i];
    } else {
      *reinterpret_cast<f32x4*>(p + float4_at(c, g)) = x;
    }
  }
  __device__ __forceinline__ typename Delta<T>::Full row(int c, int g) const {
    if constexpr (Delta<T>::EXACT) {
      const __bf16* q = (const __bf16*)p + four_at<__bf16>(c, g);
      return {{*reinterpret_cast<const b16x4*>(q), *reinterpret_cast<const b16x4*>(q + 256), *reinterpret_cast<const b16x4*>(q + 512)}};
    } else {
      return *reinterpret_cast<const f32x4*>(p + float4_at(c, g));
    }
  }
  __device__ __forceinline__ typename Delta<T>::Full col(int c, int g) const {
    if constexpr (Delta<T>::EXACT) {
      const __bf16* q = (const __bf16*)p;
      return {{col_of(q, c, g), col_of(q + 256, c, g), col_of(q + 512, c, g)}};
    } else {
      f32x4 x;
#pragma unroll
      for (int s = 0; s < 4; ++s) x[s] = p[(4 * g + s) * 16 + 4 * ((c >> 2) ^ g) + (c & 3)];
      return x;
    }
  }
};
// values of the type, as Tiles
template <typename T> struct RowTiles {
  T* p;
  __device__ __forceinline__ void set(int tile, int c, int g, const f32x4& x) const {
    if constexpr (Delta<T>::EXACT) {
      *reinterpret_cast<b16x4*>(p + tile * Tile<T>::SIZE + four_at<T>(c, g)) = __builtin_convertvector(x, b16x4);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) p[tile * Tile<T>::SIZE + (4 * g + r) * Tile<T>::LD + c] = (T)x[r];
    }
  }
  __device__ __forceinline__ typename Delta<T>::Row get(int tile, int c, int g) const {
    if constexpr (Delta<T>::EXACT) return col_of(p + tile * Tile<T>::SIZE, c, g);
    else return row_of(p + tile * Tile<T>::SIZE, c, g);
  }
};

// sum over the W tiles of the operands that a and b give for a tile
template <typename T, int W, typename A, typename B>
__device__ __forceinline__ f32x4 mul_cols(A a, B b, f32x4 c) {
#pragma unroll
  for (int u = 0; u + 1 < W; u += 2) c = Delta<T>::mul(a(u), a(u + 1), b(u), b(u + 1), c);
  // the last odd one in sums of its own: a product of K = 16 right behind one of K = 32 on the same sums gave wrong results
  if constexpr (W % 2) c = c + Delta<T>::mul(a(W - 1), b(W - 1), f32x4{0.f, 0.f, 0.f, 0.f});
  return c;
}

template <typename T, int DK, int W> struct DeltaLds {
  static constexpr int SQ = DL_C * DL_LD, NT = DK / 16;
  static constexpr int RL = W * Tiles<T>::WORDS, XYZ = 3 * Square<T>::WORDS;  // of dR, and of X, Y and Z after it
  static constexpr int WORDS = DL_SEG * (2 * SQ + 256 + DL_VEC) + (RL > XYZ ? RL : XYZ) + (1 + NT) * W * Tiles<T>::WORDS + W * 32;
  static constexpr int BYTES = WORDS * 4 + (2 * DL_SEG * NT + W) * Tile<T>::SIZE * (int)sizeof(T);
};

// Wavefronts a SIMD that the backward's registers are held to, where no spill comes of it.
template <typename T, int DK, int W> constexpr int DL_BWD_WAVES = Delta<T>::EXACT && DK == 32 && W == 2 ? 3 : 1;

// AHEAD: a segment's rows and state are asked for while the one after it is worked on, where its registers cost no wavefront a
// SIMD (24 rays of up to 4096 rows, 8 heads of 64 x 64, bf16: 1416 us, 1482 without; 8192 marched rays, 4 heads of 32 x 32,
// 426 with two wavefronts and 342 without with three; 2048 of 64 x 32 255 with one and 148 without with two), and there is
// more than one wavefront to prepare a segment's chunks.  Rows that are held as floats cost one, 128 columns leave none.
template <typename T, int DK, int W>
__global__ __launch_bounds__(64 * W, (DL_BWD_WAVES<T, DK, W>)) void k_delta_bwd(const ffn_ray_delta a, int longer) {
  typedef Delta<T> Ops;
  typedef typename Ops::Row Row;
  typedef DeltaLds<T, DK, W> L;
  constexpr bool AHEAD = Ops::EXACT && (DK == 32 ? W > 2 : DK == 64 && W == 4);
  constexpr int NT = DK / 16, TP = (NT + W - 1) / W, SQ = L::SQ, TILE = Tile<T>::SIZE;
  extern __shared__ __align__(16) float lds[];
  const int64_t teams = (int64_t)a.rays.num_rays * a.v_heads;
  int64_t block = block_number();
  const bool first = longer && block < teams;  // of two turns: the rays with more rows than `longer`
  if (longer && !first) block -= teams;
  const bool shared = a.heads != a.v_heads;
  if (block >= teams) {
    const int64_t width = (int64_t)a.v_heads * a.key_dim;
    if (shared) {
      clear_rows(a, block - teams, (float*)a.workspace, width);
      clear_rows(a, block - teams, (float*)a.workspace + a.rays.n * width, width);
    } else {
      clear_rows(a, block - teams, (T*)a.dq, width);
      clear_rows(a, block - teams, (T*)a.dk, width);
    }
    clear_rows(a, block - teams, (T*)a.dv, (int64_t)a.v_heads * a.val_dim);
    clear_rows(a, block - teams, (T*)a.ddecay, (int64_t)a.v_heads);
    clear_rows(a, block - teams, (T*)a.dbeta, (int64_t)a.v_heads);
    return;
  }
  const int64_t ray = quotient(block, a.v_heads);
  const int h = (int)(block - ray * a.v_heads), hk = h / (a.v_heads / a.heads);
  const Chain ch = chain_of(a, ray);
  if (longer && (ch.count > longer) != first) return;
  const int lane = threadIdx.x & 63, w = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w16 = 16 * w;
  int c = lane & 15, g = lane >> 4;
  float* Tm = lds;
  float* Pm = Tm + DL_SEG * SQ;
  float* Dm = Pm + DL_SEG * SQ;
  float* vecs = Dm + DL_SEG * 256;
  // n, dR; S and dS, tile t W + u: rows of tile t, columns of wavefront u
  const Tiles<T> Nl{vecs + DL_SEG * DL_VEC}, Sl{Nl.p + W * Tiles<T>::WORDS}, Rl{Sl.p + NT * W * Tiles<T>::WORDS};
  const Square<T> Xm{Rl.p}, Ym{Xm.p + Square<T>::WORDS}, Zm{Ym.p + Square<T>::WORDS};  // where dR was
  float* sums = Rl.p + (L::RL > L::XYZ ? L::RL : L::XYZ);
  T* Kl = (T*)(sums + W * 32);
  T* Ql = Kl + DL_SEG * NT * TILE;
  const RowTiles<T> Gl{Ql + DL_SEG * NT * TILE};  // do
  const T* q = (const T*)a.q + hk * a.q_head;
  const T* k = (const T*)a.k + hk * a.k_head;
  const T* v = (const T*)a.v + h * a.v_head;
  const T* dout = (const T*)a.dout + h * a.do_head;
  const int64_t size = (int64_t)a.key_dim * a.val_dim;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const auto sync = [] {
    if constexpr (W > 1) __syncthreads();
    else wave_sync();
  };
  f32x4 dS[NT];
  load_state(dS, a.dlast ? a.dlast + block * size : nullptr, a, c, g, w16);
  constexpr int MINE = (DL_SEG + W - 1) / W;  // chunks that a wavefront prepares
  RawRow<T, NT> kr[MINE], qr[MINE];
  RawGates<T> gates[MINE];
  RawCol<T> vn[DL_SEG], gn[DL_SEG];
  f32x4 Sn[NT];
  const auto fetch = [&](int p0) {
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int p = p0 + DL_C * (w + j * W);
      if (w + j * W < DL_SEG && p < ch.count) {
        const Chunk ck(ch, p);
        kr[j].load(k, a.k_row, ck, c, g, a.key_dim);
        qr[j].load(q, a.q_row, ck, c, g, a.key_dim);
        gates[j].load(a, h, ck, Rows4(ck, g), c);
      }
    }
#pragma unroll
    for (int i = 0; i < DL_SEG; ++i) {
      if (p0 + DL_C * i < ch.count) {
        const Chunk ck(ch, p0 + DL_C * i);
        const Rows4 rows(ck, g);
        vn[i].load(v, a.v_row, ck, rows, w16 + c, a.val_dim);
        gn[i].load(dout, a.do_row, ck, rows, w16 + c, a.val_dim);
      }
    }
    if (p0) load_mark(Sn, a.marks + (mark_slot(ch, p0) * a.v_heads + h) * (NT * W * 256), w, lane);
    else load_state(Sn, a.h0 ? a.h0 + block * size : nullptr, a, c, g, w16);
  };
  const int last = ch.count ? (ch.count - 1) / DL_MARK * DL_MARK : -1;
  if (AHEAD && last >= 0) fetch(last);
#pragma unroll 1
  for (int p0 = last; p0 >= 0; p0 -= DL_MARK) {
    asm volatile("" : "+v"(c), "+v"(g));
    if (!AHEAD) fetch(p0);
    RawCol<T> vr[DL_SEG], gr[DL_SEG];
    f32x4 S[DL_SEG][NT], n[DL_SEG];
#pragma unroll
    for (int i = 0; i < DL_SEG; ++i) vr[i] = vn[i], gr[i] = gn[i];
#pragma unroll
    for (int t = 0; t < NT; ++t) S[0][t] = Sn[t];
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int i = w + j * W, p = p0 + DL_C * i;
      if (i < DL_SEG && p < ch.count) {
        const Chunk ck(ch, p);
        kr[j].trim(ck, c, g, a.key_dim);
        qr[j].trim(ck, c, g, a.key_dim);
        Row kf[NT], qf[NT];
        kr[j].operands(kf);
        qr[j].operands(qf);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          typedef typename RawRow<T, NT>::tvec tvec;
          *reinterpret_cast<tvec*>(Kl + (i * NT + t) * TILE + four_at<T>(c, g)) = kr[j].v[t];
          *reinterpret_cast<tvec*>(Ql + (i * NT + t) * TILE + four_at<T>(c, g)) = qr[j].v[t];
        }
        prepare_chunk<T>(kf, qf, gates[j].decay(ck, g), gates[j].beta(ck, c), a.scale, c, g, Tm + i * SQ, Pm + i * SQ, Dm + i * 256,
                         vecs + i * DL_VEC);
      }
    }
    if (AHEAD && p0) fetch(p0 - DL_MARK);
    sync();
    // the states before the segment's chunks, and their writes n
#pragma unroll
    for (int i = 0; i < DL_SEG; ++i) {
      if (p0 + DL_C * i < ch.count) {
        const Chunk ck(ch, p0 + DL_C * i);
        const T* Kc = Kl + i * NT * TILE;
        const float* vec = vecs + i * DL_VEC;
        Row kf[NT];
        typename Ops::Full full[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          kf[t] = row_of(Kc + t * TILE, c, g);
          full[t] = Ops::full(S[i][t]);
        }
        const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + 4 * g), e = *reinterpret_cast<const f32x4*>(vec + 16 + 4 * g);
        const f32x4 R = beta * (vr[i].value(ck, g, w16 + c, a.val_dim) - e * mul_tiles<T>(kf, full, zero));
        n[i] = mul16(*reinterpret_cast<const f32x4*>(Tm + i * SQ + c * DL_LD + 4 * g), R, zero);
        if (i + 1 == DL_SEG || p0 + DL_C * (i + 1) >= ch.count) continue;
        const typename Ops::Full nl = Ops::full(*reinterpret_cast<const f32x4*>(vec + 32 + 4 * g) * n[i]);
#pragma unroll
        for (int t = 0; t < NT; ++t) S[i + 1 < DL_SEG ? i + 1 : i][t] = Ops::mul(col_of(Kc + t * TILE, c, g), nl, vec[48] * S[i][t]);
      }
    }
#pragma unroll
    for (int i = DL_SEG - 1; i >= 0; --i) {
      const int p = p0 + DL_C * i;
      if (p < ch.count) {
        asm volatile("" : "+v"(c), "+v"(g));
        const Chunk ck(ch, p);
        const T *Kc = Kl + i * NT * TILE, *Qc = Ql + i * NT * TILE;
        const float *vec = vecs + i * DL_VEC, *Tc = Tm + i * SQ, *Pc = Pm + i * SQ, *Dc = Dm + i * 256;
        const int vcol = w16 + c;
        const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + 4 * g), e = *reinterpret_cast<const f32x4*>(vec + 16 + 4 * g);
        const f32x4 left = *reinterpret_cast<const f32x4*>(vec + 32 + 4 * g);
        // by columns: dn, dR, dv
        const f32x4 go = gr[i].value(ck, g, vcol, a.val_dim), vv = vr[i].value(ck, g, vcol, a.val_dim);
        f32x4 dn, dR, col;
        typename Ops::Full full[NT];  // of dS
        {
          Row kf[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            kf[t] = row_of(Kc + t * TILE, c, g);
            full[t] = Ops::full(dS[t]);
          }
          dn = left * mul_tiles<T>(kf, full, zero);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) col[s] = Pc[(4 * g + s) * DL_LD + c];
        dn = mul16(col, go, dn);  // in float: the vector ALU, which would make the parts, is the busier one
#pragma unroll
        for (int s = 0; s < 4; ++s) col[s] = Tc[(4 * g + s) * DL_LD + c];
        dR = mul16(col, dn, zero);
        f32x4 to_beta = vv * dR, to_decay = zero;
        const Rows4 rows(ck, g);
        if (vcol < a.val_dim) {
          T* dv = ck.in((T*)a.dv + h * a.val_dim, a.v_heads * a.val_dim);
          put_rows(dv, ck, rows, g, a.v_heads * a.val_dim, vcol, beta * dR);
        }
        Nl.set(w, c, g, n[i]);
        Rl.set(w, c, g, dR);
        Gl.set(w, c, g, go);
        float inner = 0.f;  // dS . S at the chunk's end: what was there at its start ..
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int r = 0; r < 4; ++r) inner = __builtin_fmaf(dS[t][r], S[i][t][r], inner);
          Sl.set(t * W + w, c, g, S[i][t]);
        }
        inner *= vec[48];
        sync();
        const auto g_row = [&](int u) { return Gl.get(u, c, g); };
        const auto n_row = [&](int u) { return Nl.get(u, c, g); };
        const auto r_row = [&](int u) { return Rl.get(u, c, g); };
        // X and Y (the first and the second wavefront, where there are two); products with S
        f32x4 x = zero, y = zero;
        if (w == 0 || w == 1) {
          const f32x4 D = *reinterpret_cast<const f32x4*>(Dc + float4_at(c, g));
          if (w == 0) {
            x = mul_cols<T, W>(n_row, g_row, zero);  // rows j, column i
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = 4 * g + r <= c ? a.scale * D[r] * x[r] : 0.f;
          }
          if (w == 1 || W == 1) {
            y = mul_cols<T, W>(n_row, r_row, zero);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = 4 * g + r < c ? -D[r] * y[r] : 0.f;
          }
        }
        f32x4 sq[TP], lf[TP];
#pragma unroll
        for (int j = 0; j < TP; ++j) {
          const int t = w + j * W;
          if (t < NT) {
            const auto s_row = [&](int u) { return Sl.get(t * W + u, c, g); };
            sq[j] = mul_cols<T, W>(g_row, s_row, zero);
            lf[j] = mul_cols<T, W>(r_row, s_row, zero);
          }
        }
        sync();
        if (w == 0) Xm.set(c, g, x);
        if (w == 1 || W == 1) {
          Ym.set(c, g, y);
          Zm.set(c, g, vec[c] * y);
        }
        // dS out, and back to the chunk's start
        const typename Ops::Full fo = Ops::full(a.scale * e * go), fr = Ops::full(-(beta * e) * dR);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          Sl.set(t * W + w, c, g, full[t]);
          dS[t] = Ops::mul(col_of(Kc + t * TILE, c, g), fr, Ops::mul(col_of(Qc + t * TILE, c, g), fo, vec[48] * dS[t]));
        }
        sync();
        const typename Ops::Full xr = Xm.row(c, g), yr = Ym.row(c, g), xt = Xm.col(c, g), zt = Zm.col(c, g);
#pragma unroll
        for (int j = 0; j < TP; ++j) {
          const int t = w + j * W, kcol = 16 * t + c;
          if (t < NT) {
            const auto s_row = [&](int u) { return Sl.get(t * W + u, c, g); };
            const Row kt = col_of(Kc + t * TILE, c, g), qt = col_of(Qc + t * TILE, c, g);
            const f32x4 kv = Ops::value(kt), qv = Ops::value(qt);
            const f32x4 gq = Ops::mul(xr, kt, a.scale * e * sq[j]);
            const f32x4 gl = Ops::mul(yr, kt, -(e * lf[j]));
            const f32x4 end = left * mul_cols<T, W>(n_row, s_row, zero), right = Ops::mul(zt, kt, Ops::mul(xt, qt, end));
#pragma unroll
            for (int r = 0; r < 4; ++r) inner = __builtin_fmaf(kv[r], end[r], inner);  // .. and what the chunk wrote
            const f32x4 gk = beta * gl + right;
            to_beta += kv * gl;
            to_decay += qv * gq + beta * (kv * gl) - kv * right;
            if (kcol < a.key_dim) {
              if (shared) {
                const int stride = a.v_heads * a.key_dim;
                const int64_t other = (int64_t)a.rays.n * stride;
                float* part = ck.in((float*)a.workspace + h * a.key_dim, stride);
                put_rows(part, ck, rows, g, stride, kcol, gq);
                put_rows(part + other, ck, rows, g, stride, kcol, gk);
              } else {
                const int stride = a.heads * a.key_dim;
                T *dq = ck.in((T*)a.dq + h * a.key_dim, stride), *dk = ck.in((T*)a.dk + h * a.key_dim, stride);
                put_rows(dq, ck, rows, g, stride, kcol, gq);
                put_rows(dk, ck, rows, g, stride, kcol, gk);
              }
            }
          }
        }
        inner += __shfl_xor(inner, 16);
        inner += __shfl_xor(inner, 32);
        if (g == 3) to_decay[3] += inner;  // the chunk's last row
        to_beta = sum16(to_beta);
        to_decay = sum16(to_decay);
        if (c == 0) {
          *reinterpret_cast<f32x4*>(sums + w * 32 + 4 * g) = to_beta;
          *reinterpret_cast<f32x4*>(sums + w * 32 + 16 + 4 * g) = to_decay;
        }
        // a row that nothing passes through, a reset or the first one of a ray, has a decay's gradient of 0, and not what is
        // left of sums that cancel
        const float passed = c ? Dc[float4_at(c, (c - 1) >> 2) + ((c - 1) & 3)] : p || a.h0 ? vec[16] : 0.f;
        sync();
        if (w == 0 && g == 0) {
          float db = 0.f, dd = 0.f;
#pragma unroll
          for (int u = 0; u < W; ++u) {
            db += sums[u * 32 + c];
            dd += sums[u * 32 + 16 + c];
          }
          dd = sum_after(dd);
          if (passed == 0.f && fabsf(dd) <= 3.4e38f) dd = 0.f;
          if (c < ck.many) {
            const int64_t to = (int64_t)(ck.low + ck.at(c)) * a.v_heads + h;
            ((T*)a.ddecay)[to] = (T)dd;
            ((T*)a.dbeta)[to] = (T)db;
          }
        }
      }
    }
  }
  if (a.dh0) store_state(a.dh0 + block * size, dS, a, c, g, w16);
}

// dq and dk of key heads that value heads share, in a fixed order; four neighbouring columns a thread
template <typename T>
__global__ __launch_bounds__(256) void k_delta_join(const ffn_ray_delta a) {
  const uint32_t quads = (uint32_t)a.key_dim / 4, per = (uint32_t)(a.v_heads / a.heads);
  const int64_t all = (int64_t)a.rays.n * a.heads * quads, i = block_number() * 256 + threadIdx.x;
  if (i >= all) return;
  const int64_t head = quotient(i, (int)quads);  // of row and key head
  const int64_t at = (head * per * quads + (i - head * quads)) * 4, other = (int64_t)a.rays.n * a.v_heads * a.key_dim;
  f32x4 q = {0.f, 0.f, 0.f, 0.f}, k = q;
  for (uint32_t u = 0; u < per; ++u) {
    const float* from = (const float*)a.workspace + at + (int64_t)u * a.key_dim;
    q += load4(from);
    k += load4(from + other);
  }
  store4((T*)a.dq + 4 * i, q);
  store4((T*)a.dk + 4 * i, k);
}

// ---------------------------------------------------------------------------
// launches

// a state's rows and wavefronts of 16 columns, as the kernels hold it: those of 72 to 112 columns take the time of 128 (1024
// marched rays, 4 heads, bf16, us: 64 x 64 49 and 152, 64 x 80 127 and 343, 64 x 128 129 and 344); five to seven are not built
inline int delta_rows(int key_dim) { return key_dim <= 32 ? 32 : key_dim <= 64 ? 64 : 128; }
inline int delta_waves(int val_dim) { return val_dim <= 64 ? (val_dim + 15) / 16 : 8; }

inline int64_t delta_clear_blocks(const ffn_ray_delta& a) { return ((int64_t)a.rays.n + DL_CLEAR - 1) / DL_CLEAR; }

// Where rays are many, those of more than twice the mean and four chunks take their turn before the others: one that is
// begun last would be all that still runs (8192 marched rays, 4 heads of 32 x 32, bf16: forward 124 us, 130 in one turn,
// backward 341 and 360).
inline int delta_longer(const ffn_ray_delta& a) {
  if ((int64_t)a.rays.num_rays * a.v_heads < DL_BLOCKS) return 0;
  return (int)std::max<int64_t>(4 * DL_C, 2 * (int64_t)a.rays.n / a.rays.num_rays);
}

template <typename T, int DK, int W>
hipError_t start_delta(const ffn_ray_delta& a, bool back, bool few, hipStream_t st) {
  const int64_t teams = (int64_t)a.rays.num_rays * a.v_heads;
  if (few) {
    k_delta_step<T, DK><<<grid_of((teams * ((a.val_dim + 31) / 32) + 3) / 4 + delta_clear_blocks(a)), 256, 0, st>>>(a, DL_FEW);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.rays.n <= DL_FEW) return e;
    k_delta_fwd<T, DK, W, true><<<grid_of(std::max(std::min<int64_t>(teams, DL_PICK), (teams + 63) / 64)), 64 * W, 0, st>>>(a, DL_FEW);
    return hipGetLastError();
  }
  const int longer = delta_longer(a);
  const dim3 grid = grid_of(teams * (longer ? 2 : 1) + delta_clear_blocks(a));
  if (!back) {
    k_delta_fwd<T, DK, W, false><<<grid, 64 * W, 0, st>>>(a, longer);
    return hipGetLastError();
  }
  constexpr int bytes = DeltaLds<T, DK, W>::BYTES;
  static_assert(bytes <= 160 * 1024, "LDS");
  if (bytes > 64 * 1024) {  // has to be allowed, on the device that is current
    const hipError_t e = hipFuncSetAttribute((const void*)k_delta_bwd<T, DK, W>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
  }
  k_delta_bwd<T, DK, W><<<grid, 64 * W, bytes, st>>>(a, longer);
  return hipGetLastError();
}

template <typename T, int DK>
hipError_t delta_by_columns(const ffn_ray_delta& a, bool back, hipStream_t st) {
  // Row by row or in chunks: by the mean of rows a ray (2048 rays, 4 heads of 64 x 64, bf16, us: one row 55 and 83, three 64
  // and 82, six 94 and 87), and where row by row, by each ray's own: only the GPU knows it, and a second launch looks for
  // those of more than eight (3 us of these; one ray of 4096 rows and 2047 without any 488, 8900 row by row).
  const bool few = !back && !a.marks && a.rays.n <= 4ull * a.rays.num_rays;
  const int W = delta_waves(a.val_dim);
  const hipError_t e = W == 1   ? start_delta<T, DK, 1>(a, back, few, st)
                       : W == 2 ? start_delta<T, DK, 2>(a, back, few, st)
                       : W == 3 ? start_delta<T, DK, 3>(a, back, few, st)
                       : W == 4 ? start_delta<T, DK, 4>(a, back, few, st)
                                : start_delta<T, DK, 8>(a, back, few, st);
  if (!back || e != hipSuccess || a.heads == a.v_heads || !a.rays.n) return e;
  k_delta_join<T><<<grid_of(((int64_t)a.rays.n * a.heads * a.key_dim / 4 + 255) / 256), 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t delta_of_type(const ffn_ray_delta& a, bool back, hipStream_t st) {
  const int rows = delta_rows(a.key_dim);
  if (rows == 32) return delta_by_columns<T, 32>(a, back, st);
  if (rows == 64) return delta_by_columns<T, 64>(a, back, st);
  return delta_by_columns<T, 128>(a, back, st);
}

hipError_t delta_f32(const ffn_ray_delta& a, bool back, hipStream_t st);
hipError_t delta_f16(const ffn_ray_delta& a, bool back, hipStream_t st);
hipError_t delta_bf16(const ffn_ray_delta& a, bool back, hipStream_t st);

}  // namespace ffn
