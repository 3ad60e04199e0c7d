// Device helpers of the encoder kernels: 16-bit types, 32 x 32 x 16 MFMAs, LDS tiles.
//
// A 32 x 32 block's accumulator holds, in lane l and element e, column l % 32 and
// row 8 (e / 4) + 4 (l / 32) + e % 4.  The kernels hand operand rows to the matrix
// cores in the order tile_row() instead, so that a lane's elements 8 s .. 8 s + 7 are
// the consecutive rows 16 s + 8 (l / 32) + 0 .. 7: exactly what the B operand of a
// following product of depth 16 takes from that lane, and 16 contiguous bytes for
// a store.
//
// LDS tiles are lines of 128 bytes in 16-byte pieces, slot s of line r holding piece
// s ^ piece_swizzle(r).  LDS serves 256 bytes a cycle, from two neighbouring lines' slots.
// Both ways of reading a tile take each of the 16 once: the same piece of 16 consecutive
// rows (operand rows; 16 lanes a cycle), and four neighbouring pieces of 4 consecutive rows
// (transposing reads, rows as depth; 32 lanes of 8 bytes a cycle).
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

__device__ __forceinline__ constexpr int piece_swizzle(int r) { return (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }
// Rows of 256 bytes, two lines: of 16 pieces.
__device__ __forceinline__ constexpr int wide_swizzle(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
// Lines that hold two rows of 64 bytes.
__device__ __forceinline__ constexpr int pair_swizzle(int line) { return (line >> 1) & 3; }

// Byte offset of a row's 16-byte piece in a tile of rows of WIDTH 16-bit columns (32, 64 or 128).
template <int WIDTH>
__device__ __forceinline__ int row_offset(int row, int piece) {
  if constexpr (WIDTH == 32) {
    const int line = row >> 1;
    return line * 128 + ((((row & 1) * 4 + piece) ^ pair_swizzle(line)) << 4);
  } else if constexpr (WIDTH == 64) {
    return row * 128 + ((piece ^ piece_swizzle(row)) << 4);
  } else {
    return row * 256 + ((piece ^ wide_swizzle(row)) << 4);
  }
}

// A byte offset past the end of every buffer: loads there give zeros.
constexpr uint32_t kOutside = 0x80000000u;

typedef int i32x4s __attribute__((ext_vector_type(4)));

// 16 bytes a lane from base + voff into LDS at lds + 16 * lane; zeros where voff >= kOutside.
__device__ __forceinline__ void load_lds(uint32_t voff, const unsigned char* base, uint32_t lds) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  const i32x4s rsrc = {__builtin_amdgcn_readfirstlane((int)(uint32_t)b),
                       __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xffff), (int)kOutside, 0x00020000};
  const uint32_t m = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(m), "v"(voff), "s"(rsrc)
      : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

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

// Maximum and sum of lane l's value and lane l ^ 32's.
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Nothing moves across: LDS reads stay ahead of the products they are to wait under.  (Left
// to itself the compiler reads one operand, waits for it and multiplies, to save
// registers.)
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

}  // namespace cvs
