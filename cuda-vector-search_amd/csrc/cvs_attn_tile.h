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

// Loads of tiles of ROWS rows of a head straight into LDS, by the four waves of a workgroup
// (WAVES = 1: by one, for itself): a lane's place in each 1 KiB load is the same in every
// tile.  Rows from `rows` on, rows before `low` and columns from `d` on become zeros: whatever lies
// there (0 times a NaN is one) is not read.
template <int DP, int ROWS, int WAVES = 4>
struct TileLoad {
  static constexpr int N = ROWS * DP * 2 / 1024 / WAVES;
  static_assert(N * WAVES * 1024 == ROWS * DP * 2, "whole loads");
  uint32_t at[N];
  int row[N];

  __device__ __forceinline__ TileLoad(int64_t stride_bytes, int d) {
    const int lane = threadIdx.x & 63, wave = WAVES > 1 ? threadIdx.x >> 6 : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int line = (wave + WAVES * i) * 8 + (lane >> 3), slot = lane & 7;
      int piece;
      if constexpr (DP == 32) {
        const int x = slot ^ pair_swizzle(line);
        row[i] = 2 * line + (x >> 2), piece = x & 3;
      } else if constexpr (DP == 64) {
        row[i] = line, piece = slot ^ piece_swizzle(line);
      } else {
        row[i] = line >> 1, piece = ((line & 1) * 8 + slot) ^ wide_swizzle(line >> 1);
      }
      at[i] = piece * 8 < d ? (uint32_t)(row[i] * (int)stride_bytes + piece * 16) : kOutside;
    }
  }
  // Rows first .. first + ROWS - 1 of the head at `base` (its row 0) to the tile at `lds`; 0 <= low <= rows.
  __device__ __forceinline__ void load(const unsigned char* base, int64_t stride_bytes, int first, int rows,
                                       const unsigned char* lds, int low = 0) const {
    const uint32_t to = lds_address(lds) + (WAVES > 1 ? threadIdx.x >> 6 : 0) * 1024;
#pragma unroll
    for (int i = 0; i < N; ++i)
      load_lds((unsigned)(first - low + row[i]) < (unsigned)(rows - low) ? at[i] : kOutside, base + first * stride_bytes, to + i * (WAVES * 1024));
  }
  // The same of rows low .. rows - 1 and of the first `head`.
  __device__ __forceinline__ void load_window(const unsigned char* base, int64_t stride_bytes, int first, int rows,
                                              const unsigned char* lds, int low, int head) const {
    const uint32_t to = lds_address(lds) + (WAVES > 1 ? threadIdx.x >> 6 : 0) * 1024;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = ((unsigned)(first - low + row[i]) < (unsigned)(rows - low)) | (first + row[i] < head);
      load_lds(in ? at[i] : kOutside, base + first * stride_bytes, to + i * (WAVES * 1024));
    }
  }
};

// What a window leaves of the keys for rows at positions p0 .. p1: the first `head` and low .. end - 1, in tiles of
// ROWS.  Tile u of these is the keys' tile u below `heads`, and u + gap from there.
template <int ROWS>
struct WindowTiles {
  int head, low, end, heads, gap, count;

  __device__ __forceinline__ WindowTiles() {}
  __device__ __forceinline__ WindowTiles(const AttnArgs& a, int nk, int p0, int p1) {
    const int last = a.causal ? min(nk, max(p1 + 1, 0)) : nk;
    head = p0 <= p1 ? min(a.sinks, last) : 0;
    low = min(max(p0 - a.before, 0), last);
    end = p0 <= p1 ? max(min(last, p1 + a.after + 1), low) : low;
    heads = (head + ROWS - 1) / ROWS;
    const int t0 = max(low / ROWS, heads), t1 = end > low ? (end + ROWS - 1) / ROWS : t0;
    gap = t0 - heads;
    count = heads + max(t1 - t0, 0);
  }
  __device__ __forceinline__ int tile(int u) const { return u < heads ? u : u + gap; }
};

// Whether rows at positions p0 .. p1 see a key of the `rows` ones from j0 on (were there that many).
__device__ __forceinline__ bool window_meets(const AttnArgs& a, int j0, int rows, int p0, int p1) {
  return (j0 < a.sinks || (j0 + rows > p0 - a.before && j0 <= p1 + a.after)) && (!a.causal || j0 <= p1);
}

// The keys that the row at position p sees, counted from `from` on: (unsigned)(key - low) <= span, or key < head.
struct WindowMask {
  int low, head;
  unsigned span;

  __device__ __forceinline__ WindowMask(const AttnArgs& a, int nk, int p, int from) {
    const int lo = p - a.before, hi = min(nk - 1, p + a.after);
    low = hi < lo ? 1 << 30 : lo - from;
    span = hi < lo ? 0 : hi - lo;
    head = min(nk, a.causal ? min(a.sinks, p + 1) : a.sinks) - from;
  }
  // Puts `out` in the places of a block (keys of 32 from `key` on, 8 (lane / 32) of them in `from`) that are not seen.
  __device__ __forceinline__ void apply(f32x16& x, int key, bool heads, float out) const {
    if (heads) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = key + elem_row(e, 0);
        x[e] = ((unsigned)(k - low) <= span) | (k < head) ? x[e] : out;  // (|: no branch an element)
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (unsigned)(key + elem_row(e, 0) - low) <= span ? x[e] : out;
    }
  }
};

// This wave's loads into LDS have landed and its LDS operations are done; then every wave's.
__device__ __forceinline__ void tile_barrier() {
  wait_vmcnt_lgkm0<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A operand: rows r0 .. r0 + 31 in tile_row order, columns 16 ks .. 16 ks + 15.
template <class T, int DP>
__device__ __forceinline__ typename Frag<T>::V row_frag(const unsigned char* lds, int r0, int ks) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const typename Frag<T>::V*>(lds + row_offset<DP>(r0 + tile_row(lane & 31), 2 * ks + (lane >> 5)));
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
  return join_tr<T>(read_tr(at + row_offset<DP>(row, col >> 3)), read_tr(at + row_offset<DP>(row + 4, col >> 3)));
}

// The same operands of a tile of 32 rows of 128 columns, from this lane's place in it (kept in one register, and the
// pieces' offsets, which the swizzle makes exclusive ors, taken from it anew: where all the offsets of a loop's
// operands do not fit the registers).
__device__ __forceinline__ uint32_t wide_row_place() {
  const int lane = threadIdx.x & 63, row = tile_row(lane & 31);
  return row * 256 + (((lane >> 5) ^ wide_swizzle(row)) << 4);
}
__device__ __forceinline__ uint32_t wide_col_place() {
  const int lane = threadIdx.x & 63, p = lane >> 4, s = lane & 15;
  const int c = ((s & 1) << 1) | ((s >> 1) & 1), row = 8 * (p >> 1) + (s >> 2);
  return row * 256 + (((2 * (p & 1) + (c >> 1)) ^ wide_swizzle(row)) << 4) + (c & 1) * 8;
}
template <class T>
__device__ __forceinline__ typename Frag<T>::V wide_row_frag(uint32_t at, int ks) {
  return *(const __attribute__((address_space(3))) typename Frag<T>::V*)(uintptr_t)(at ^ (ks << 5));
}
template <class T>
__device__ __forceinline__ typename Frag<T>::V wide_col_frag(uint32_t at, int r0, int c0) {
  typedef __attribute__((address_space(3))) s16x4* P;
  return join_tr<T>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)((at ^ (c0 << 1)) + r0 * 256)),
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)((at ^ (c0 << 1) ^ 16) + r0 * 256 + 1024)));
}

// B operand: column = row `row` of a head in memory (zeros when !in or past d), depth 16 ks + 8 (lane / 32) + 0 .. 7.
template <class T>
__device__ __forceinline__ typename Frag<T>::V global_frag(const unsigned char* row, int ks, int d, bool in) {
  const int lane = threadIdx.x & 63, c = 16 * ks + 8 * (lane >> 5);
  u32x4 v = {0, 0, 0, 0};
  if (in && c < d) v = *reinterpret_cast<const u32x4*>(row + 2 * c);
  return __builtin_bit_cast(typename Frag<T>::V, v);
}

__device__ __forceinline__ f32x16 splat16(float v) {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = v;
  return z;
}
__device__ __forceinline__ f32x16 zero16() { return splat16(0.f); }

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

// The same, unscaled, to fp32 partial sums.
template <int DP>
__device__ __forceinline__ void store_part_row(float* row, const f32x16* acc, int d) {
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = b * 32 + 16 * (q >> 1) + 8 * g + 4 * (q & 1);
      if (c < d) *reinterpret_cast<f32x4*>(row + c) = f32x4{acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
    }
}

// A head's learned bias by relative position, in LDS, in units of unscaled scores (so that it
// is what a block of scores starts from): tab[rel + reach], reach = far + kReach, far being
// the smallest distance of the last bucket.  A block of 32 queries and up to 64 keys that has
// a position nearer than far has none further than far + kReach; other blocks have one
// bias throughout.
constexpr int kReach = 96;

// Two dependent loads from memory, in steps that a kernel puts its other first loads between.
template <class T>
struct BiasLoad {
  static constexpr int N = (2 * (kMaxDistance + kReach) + kBlock) / kBlock;  // places a thread
  int u[N];
  float v[N];

  __device__ __forceinline__ void buckets(const AttnArgs& a) {
    const int reach = a.far + kReach;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int rel = min((int)threadIdx.x + n * kBlock, 2 * reach) - reach;
      u[n] = a.bucket_of[min(abs(rel), a.far)];
      if (rel > 0) u[n] = a.causal ? 0 : u[n] + a.one_way;
    }
  }
  __device__ __forceinline__ void values(const AttnArgs& a, int head) {
    const float unit = 1.f / a.scale;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = (float)((const T*)a.table)[u[n] * a.heads + head] * unit;
  }
  __device__ __forceinline__ void store(const AttnArgs& a, float* tab) const {
    const int reach = a.far + kReach;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int t = threadIdx.x + n * kBlock;
      if (t <= 2 * reach) tab[t] = v[n];
    }
  }
};

__device__ __forceinline__ int key_count(const AttnArgs& a, int b) {
  return a.key_lengths == nullptr ? a.lk : min(max(a.key_lengths[b], 0), a.lk);
}
__device__ __forceinline__ int query_count(const AttnArgs& a, int b) {
  return a.query_lengths == nullptr ? a.lq : min(max(a.query_lengths[b], 0), a.lq);
}
__device__ __forceinline__ int query_offset(const AttnArgs& a, int b) {
  return a.query_start == nullptr ? a.lk - a.lq : min(max(a.query_start[b], -(1 << 29)), 1 << 29);
}
// Whether no row sees more than a few keys.  Their gradients ds are then differences of few terms (of one key,
// zero), and delta is taken from those terms themselves, in a pass of its own.  (8 x 2048 rows, 12 heads of 64, windows
// of 64 keys: 99 us with it, 74 without, and dq wrong in its first digits where a row sees one key.)
__host__ __device__ inline bool window_narrow(const AttnArgs& a) { return a.windowed && a.before + a.after + a.sinks < 64; }

// The rows that see a key of a window: first .. end - 1.
__device__ __forceinline__ void window_rows(const AttnArgs& a, int nk, int nq, int off, int& first, int& end) {
  first = a.causal ? max(-off, 0) : a.sinks > 0 ? 0 : max(-off - a.after, 0);
  end = nk == 0 ? 0 : a.sinks > 0 ? nq : min(nq, nk + a.before - off);
  first = min(first, max(end, 0));
}
// The first row that sees a key, were there any, and the end of the keys that some row sees.
__device__ __forceinline__ int first_row(const AttnArgs& a, int off) { return a.causal ? max(-off, 0) : 0; }
__device__ __forceinline__ int seen_count(const AttnArgs& a, int nk, int nq, int off) {
  return a.causal ? min(nk, max(nq + off, 0)) : nk;
}

}  // namespace cvs
