// LDS tiles of 64 or 32 rows of a head, and what the attention kernels share.
//
// Rows hold DP = 32, 64 or 128 columns (the head's width, zero-filled to DP).  Lines
// are 128 bytes: two rows of 32 columns, one of 64, half of one of 128.
#pragma once

#include "cvs_encoder.h"
#include "cvs_mfma.h"

namespace cvs {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <int DP>
__device__ __forceinline__ int tile_offset(int row, int piece) {  // bytes
  if constexpr (DP == 32) {
    const int line = row >> 1;
    return line * 128 + ((((row & 1) * 4 + piece) ^ (((line & 1) << 1) | ((line >> 1) & 1))) << 4);
  } else {
    return row * (2 * DP) + ((piece ^ piece_swizzle(row)) << 4);
  }
}

// Rows first .. first + ROWS - 1 of a head (zeros past `rows` and past the width `d`),
// in registers on their way to LDS.
template <int DP, int ROWS>
struct TileLoad {
  static constexpr int kPieces = ROWS * DP / 8;                        // 16-byte pieces of the tile
  static constexpr int N = (kPieces + kBlock - 1) / kBlock;
  u32x4 v[N];

  __device__ __forceinline__ void load(const unsigned char* base, int64_t stride_bytes, int first, int rows, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = threadIdx.x + i * kBlock;
      const int r = t / (DP / 8), p = t % (DP / 8);
      v[i] = u32x4{0, 0, 0, 0};
      if ((kPieces % kBlock == 0 || t < kPieces) && first + r < rows && p * 8 < d)
        v[i] = *reinterpret_cast<const u32x4*>(base + (first + r) * stride_bytes + p * 16);
    }
  }
  __device__ __forceinline__ void store(unsigned char* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = threadIdx.x + i * kBlock;
      if (kPieces % kBlock == 0 || t < kPieces)
        *reinterpret_cast<u32x4*>(lds + tile_offset<DP>(t / (DP / 8), t % (DP / 8))) = v[i];
    }
  }
};

// A operand: rows r0 .. r0 + 31 in tile_row order, columns 16 ks .. 16 ks + 15.
template <class T, int DP>
__device__ __forceinline__ typename Frag<T>::V row_frag(const unsigned char* lds, int r0, int ks) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const typename Frag<T>::V*>(lds + tile_offset<DP>(r0 + tile_row(lane & 31), 2 * ks + (lane >> 5)));
}

// A operand of the transposed tile: its rows are columns c0 .. c0 + 31 (in tile_row
// order), its depth rows r0 .. r0 + 15 of the tile.
template <class T, int DP>
__device__ __forceinline__ typename Frag<T>::V col_frag(const unsigned char* lds, int r0, int c0) {
  const int lane = threadIdx.x & 63, p = lane >> 4, s = lane & 15;
  const int c = ((s & 1) << 1) | ((s >> 1) & 1);
  const int col = c0 + 16 * (p & 1) + 4 * c;
  const int row = r0 + 8 * (p >> 1) + (s >> 2);
  const unsigned char* at = lds + (col & 4) * 2;
  return join_tr<T>(read_tr(at + tile_offset<DP>(row, col >> 3)), read_tr(at + tile_offset<DP>(row + 4, col >> 3)));
}

// B operand: column = row `row` of a head in memory (zeros when !in or past d), depth 16 ks + 8 (lane / 32) + 0 .. 7.
template <class T>
__device__ __forceinline__ typename Frag<T>::V global_frag(const unsigned char* row, int ks, int d, bool in) {
  const int lane = threadIdx.x & 63, c = 16 * ks + 8 * (lane >> 5);
  u32x4 v = {0, 0, 0, 0};
  if (in && c < d) v = *reinterpret_cast<const u32x4*>(row + 2 * c);
  return __builtin_bit_cast(typename Frag<T>::V, v);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// Columns 8 s' .. of a transposed accumulator (row = column of the head) to 16 bytes of the output row.
template <class T, int DP>
__device__ __forceinline__ void store_head_row(T* row, const f32x16* acc, float scale, int d) {
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = b * 32 + 16 * h + 8 * g;
      if (c < d) {
        typename Frag<T>::V v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (T)(acc[b][8 * h + j] * scale);
        *reinterpret_cast<typename Frag<T>::V*>(row + c) = v;
      }
    }
}

// The head's bias by relative position in LDS: tab[rel + max_distance].
__device__ __forceinline__ void load_diag(float* tab, const AttnArgs& a, int head) {
  const int n = 2 * a.max_distance + 1;
  for (int t = threadIdx.x; t < n; t += kBlock) tab[t] = a.diag[(int64_t)head * n + t];
}

__device__ __forceinline__ int key_count(const AttnArgs& a, int b) {
  return a.key_lengths == nullptr ? a.lk : min(max(a.key_lengths[b], 0), a.lk);
}
__device__ __forceinline__ int query_count(const AttnArgs& a, int b) {
  return a.query_lengths == nullptr ? a.lq : min(max(a.query_lengths[b], 0), a.lq);
}
__device__ __forceinline__ int query_offset(const AttnArgs& a, int b) {
  return a.query_start == nullptr ? a.lk - a.lq : min(max(a.query_start[b], -(1 << 29)), 1 << 29);
}

}  // namespace cvs
