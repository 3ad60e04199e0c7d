// Device helpers of the encoder kernels: 16-bit types, 32 x 32 x 16 MFMAs, LDS tiles.
//
// A 32 x 32 block's accumulator holds, in lane l and element e, column l % 32 and
// row 8 (e / 4) + 4 (l / 32) + e % 4.  The kernels hand operand rows to the matrix
// cores in the order tile_row() instead, so that a lane's elements 8 s .. 8 s + 7 are
// the consecutive rows 16 s + 8 (l / 32) + 0 .. 7: exactly what the B operand of a
// following product of depth 16 takes from that lane, and 16 contiguous bytes for
// a store.
//
// LDS tiles are lines of 128 bytes in 16-byte pieces; slot s of line r holds piece
// s ^ piece_swizzle(r).  Both ways of reading a tile are then free of bank
// conflicts: the same piece of 8 consecutive lines (rows as operand rows), and two
// neighbouring pieces of 4 consecutive lines (transposing reads, rows as depth).
#pragma once

#include "cvs_common.h"

namespace cvs {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef half8 V;
  static __device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<__bf16> {
  typedef bf16x8 V;
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

__device__ __forceinline__ constexpr int piece_swizzle(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }

// Row of a 32-row block that operand row m stands for.
__device__ __forceinline__ constexpr int tile_row(int m) {
  return 16 * (m >> 4) + 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3);
}
// Row of a block that element e of lane group g = lane / 32 holds, after tile_row.
__device__ __forceinline__ constexpr int elem_row(int e, int g) { return 16 * (e >> 3) + 8 * g + (e & 7); }

// Transposing read: lanes of a group of 16 address 8 bytes each; lane l gets, as
// element j, the (l % 4)-th 16-bit value at the address of lane 4 j + l / 4 (of its group).
__device__ __forceinline__ s16x4 read_tr(const void* lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds);
}

template <class T>
__device__ __forceinline__ typename Frag<T>::V join_tr(s16x4 lo, s16x4 hi) {
  const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(typename Frag<T>::V, v);
}

// Elements 8 s .. 8 s + 7 of an accumulator as the operand of the next product.
template <class T>
__device__ __forceinline__ typename Frag<T>::V pack8(const f32x16& v, int s) {
  typename Frag<T>::V r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)v[8 * s + j];
  return r;
}

__device__ __forceinline__ float swap_halves(float v) {  // lane l's value from lane l ^ 32
  return __shfl_xor(v, 32);
}

}  // namespace cvs
