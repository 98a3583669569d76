// ffn_ray_common.h -- pieces shared by the kernels that work along rays (attention, gated recurrence) and by the
// expert layers: element types, matrix fragments, and the rows of a packed ray set that see each other.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/ffnerf_hip.h"

namespace ffn {

// A launch counts an axis's threads in 32 bits, and one of more does a part of its work without an error.  So blocks go on
// along y after GRID_X of them (a multiple of the dies, 2^31 threads of 256 a block); those past the last one find no work.
constexpr int64_t GRID_X = 1 << 23;
inline dim3 grid_of(int64_t blocks) {
  return blocks <= GRID_X ? dim3((unsigned)blocks) : dim3((unsigned)GRID_X, (unsigned)((blocks + GRID_X - 1) / GRID_X));
}
__device__ __forceinline__ int64_t block_number() { return (int64_t)blockIdx.y * GRID_X + blockIdx.x; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8), aligned(16)));  // loaded as two 16-byte halves
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Between LDS writes of a wavefront and its own lanes' reads of them: the LDS takes a wavefront's accesses in order, so
// only the compiler has to be kept from moving them.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// one lane's eight K values of a 16x16x32 matrix operand, and its four values of the product
template <typename T> struct Mat;
template <> struct Mat<__bf16> {
  typedef b16x8 frag;
  typedef b16x4 quad;
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mat<_Float16> {
  typedef f16x8 frag;
  typedef f16x4 quad;
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
// float: the K = 4 instruction eight times.  Slot j of lane group g is K value 8 g + j of the 32 in both operands, so
// the same fragments serve all three types.
template <> struct Mat<float> {
  typedef f32x8 frag;
  typedef f32x4 quad;
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// LDS row of W values: 16 bytes of padding spread the 16 rows a fragment read touches over the banks
template <typename T, int W> constexpr int lds_row = W + 16 / (int)sizeof(T);

// K block ks (32 values) of LDS row `row` as this lane's fragment (rows of the operand = lanes & 15)
template <typename T, int W>
__device__ __forceinline__ typename Mat<T>::frag row_frag(const T* tile, int row, int ks, int lane) {
  return *reinterpret_cast<const typename Mat<T>::frag*>(tile + row * lds_row<T, W> + ks * 32 + (lane >> 4) * 8);
}

// Columns col0 .. col0 + 15 of LDS rows row0 .. row0 + 31 as an operand whose K runs over the rows.  Slots 0..3 of lane
// group g are rows 4 g .. 4 g + 3 and slots 4..7 the same ones 16 further on: where a product of two 16-row tiles
// leaves its values, so that a product's lanes hold the other operand without a move.  In 16 bits, the transposing
// LDS read: lane c of a 16-lane group gives the address of row c / 4, columns 4 (c % 4) .. + 3, and receives column c
// of the group's four rows.
template <typename T, int W>
__device__ __forceinline__ typename Mat<T>::frag col_frag(const T* tile, int row0, int col0, int lane) {
  constexpr int LD = lds_row<T, W>;
  const int g = lane >> 4, c = lane & 15;
  typename Mat<T>::frag f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = tile[(row0 + 16 * (j >> 2) + 4 * g + (j & 3)) * LD + col0 + c];
  } else {
    typedef __attribute__((address_space(3))) s16x4* lds_quad;
    const T* at = tile + (row0 + 4 * g + (c >> 2)) * LD + col0 + 4 * (c & 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(at + 16 * LD));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    f = __builtin_bit_cast(typename Mat<T>::frag, both);
  }
  return f;
}

// Two product tiles (rows 4 g + r and 16 + 4 g + r) as the K values of the next operand, in col_frag's order.  In 16 bits this
// rounds attention's weights, P and P (dP - D), to the type, while their sums stay in float: results end 1.4 times as far off
// as one rounding at the end would leave them (bf16 0.0024 of their size, not 0.0017).  Both halves of each weight would
// double the second products and add three vector instructions a pair to kernels that the vector ALU bounds.
template <typename T>
__device__ __forceinline__ typename Mat<T>::frag product_frag(const f32x4& lo, const f32x4& hi) {
  const f32x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_convertvector(both, typename Mat<T>::frag);
}

}  // namespace ffn
