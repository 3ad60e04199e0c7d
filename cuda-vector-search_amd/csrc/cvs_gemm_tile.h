// The matrix products' tile: operands through LDS, 32 x 32 x 16 MFMAs, epilogues.
//
//   out[i, j] = act(sum_r M(i, r) N(j, r) + bias[j]) + residual[i, j]
//
// Either operand may be stored with its reduction contiguous ([rows, k]) or strided
// ([k, rows]): y = x W^T reads x and W so, dx = dz W takes W strided, dW = dz^T x
// both.  Stages of 64 reduction steps come into LDS as lines of 128 bytes, straight
// from memory (buffer loads into LDS; a lane past the operand's edge gets an
// offset past the buffer's end, which reads as zero); strided operands are turned
// on the way out of LDS by transposing reads.
//
// Kinds of product beside that one:
//   gated      act(M N^T + bias) * (M N2^T + bias2): a tile's rows of N are half N's, half N2's of the same
//              columns, so that a wave holds both factors of an output and nothing but it is written;
//   two parts  sum over both of two reductions, M N^T + M' N2^T, M' at M + m_second, times *unit;
//   weights    both operands strided, times *unit, rows from m_first on to out2;
//   int8       8-bit whole numbers, two to a 16-bit unit of k and of the strides (a depth step's 16
//              bytes of a lane are 16 values, and a product takes as many cycles as one of 8 16-bit
//              values), 32-bit sums, times row_scale[i] col_scale[j].
#pragma once

#include <type_traits>

#include "cvs_encoder.h"
#include "cvs_mfma.h"

namespace cvs {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kDepth = 64;                    // reduction steps of a stage
// The normal distribution's Phi(z).  log2 Phi(-t), t >= 0, is nearly a parabola: a
// polynomial of degree 7 in t, fitted on [0, 7] for least error where t Phi(-t) is visible, gives
// Phi(-t) within 3.7e-6 of itself for t <= 3, 7e-5 for t <= 6, and below 1e-9, on its
// way to 0, from there.  (The error function of the math library costs some 40 instructions; a
// rational function times exp(-t^2 / 2) took 22 where this takes 15, and the epilogue of
// 16384 x 2048, k = 768 is bound by them.)
__device__ __forceinline__ float phi(float z) {
  const float t = fabsf(z);
  float r = -1.56350917e-06f;
  r = fmaf(r, t, 5.67471386e-05f);
  r = fmaf(r, t, -0.000897089475f);
  r = fmaf(r, t, 0.00839532736f);
  r = fmaf(r, t, -0.053766588f);
  r = fmaf(r, t, -0.458625503f);
  r = fmaf(r, t, -1.15119633f);
  r = __builtin_amdgcn_exp2f(fmaf(r, t, -1.f));
  return z < 0.f ? r : 1.f - r;
}

// tanh x = x (1 - x^2 / 3 + 2 x^4 / 15) near 0, where 1 - exp(-2 |x|) would lose digits.
__device__ __forceinline__ float tanh16(float x) {
  const float e = __builtin_amdgcn_exp2f(fabsf(x) * -2.8853900817779268f);
  const float t = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
  const float x2 = x * x;
  const float s = x * fmaf(x2, fmaf(x2, 0.13333333333333333f, -0.33333333333333333f), 1.f);
  return fabsf(x) < 0.0625f ? s : t;
}

// Eight neighbouring values through an activation, or times its slope (the same branch for a whole launch).
__device__ __forceinline__ void activate8(float* z, int act) {
  if (act == kActGelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] *= phi(z[e]);
  } else if (act == kActRelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = z[e] <= 0.f ? 0.f : z[e];  // (a NaN stays)
  } else if (act == kActTanh) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = tanh16(z[e]);
  }
}
__device__ __forceinline__ void times_slope8(float* dy, const float* z, int act) {
  if (act == kActGelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float g = __builtin_amdgcn_exp2f(z[e] * z[e] * -0.72134752044448170f);
      dy[e] *= fmaf(z[e] * 0.39894228040143268f, g, phi(z[e]));
    }
  } else if (act == kActRelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dy[e] = z[e] > 0.f ? dy[e] : 0.f;
  } else if (act == kActTanh) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // 1 - tanh^2 = 4 x / (1 + x)^2 with x = exp(-2 |z|), which keeps its digits far out
      const float x = __builtin_amdgcn_exp2f(fabsf(z[e]) * -2.8853900817779268f);
      const float r = __builtin_amdgcn_rcpf(1.f + x);
      dy[e] *= 4.f * x * r * r;
    }
  }
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  const auto v = *reinterpret_cast<const typename Frag<T>::V*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  typename Frag<T>::V v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)f[j];
  *reinterpret_cast<typename Frag<T>::V*>(p) = v;
}

// The epilogue of 8 neighbouring sums of row i, columns j .. j + 7, in place; pre receives them before the activation.
template <class T>
__device__ __forceinline__ void finish8(const GemmArgs& a, int i, int j, float* z, float* pre) {
  if (a.bias != nullptr) {
    float b[8];
    load8((const T*)a.bias + j, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += b[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) pre[e] = z[e];
  activate8(z, a.act);
  if (a.residual != nullptr) {
    float r[8];
    load8((const T*)a.residual + (int64_t)i * a.ld_res + j, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += r[e];
  }
}

// A 32 x 32 block of which lane l holds, of row l % 32, columns 8 g .. and 16 + 8 g .. (g = l / 32), packed
// for a store: 16 lanes exchange their pieces with the next 16 so that four lanes write 64 contiguous
// bytes of a row.
template <class T>
__device__ __forceinline__ void pack_block(const float* z0, const float* z1, u32x4& x, u32x4& y) {
  typename Frag<T>::V v0, v1;
#pragma unroll
  for (int e = 0; e < 8; ++e) v0[e] = (T)z0[e], v1[e] = (T)z1[e];
  x = __builtin_bit_cast(u32x4, v0), y = __builtin_bit_cast(u32x4, v1);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const auto s = __builtin_amdgcn_permlane16_swap(x[r], y[r], false, false);
    x[r] = s[0], y[r] = s[1];
  }
}
template <class T>
__device__ __forceinline__ void store_block(T* out, int64_t ld, int m, int n, int row0, int col0, const float* z0, const float* z1) {
  u32x4 x, y;
  pack_block<T>(z0, z1, x, y);
  const int lane = threadIdx.x & 63;
  const int row = row0 + (lane & 15), col = col0 + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);
  if (col < n) {
    T* to = out + (int64_t)row * ld + col;
    if (row < m) *reinterpret_cast<u32x4*>(to) = x;
    if (row + 16 < m) *reinterpret_cast<u32x4*>(to + 16 * ld) = y;
  }
}

// The same of rows of which those from `border` on are another matrix's.
template <class T>
__device__ __forceinline__ void store_block_of_two(T* out, T* out2, int border, int64_t ld, int m, int n, int row0, int col0,
                                                   const float* z0, const float* z1) {
  u32x4 x, y;
  pack_block<T>(z0, z1, x, y);
  const int lane = threadIdx.x & 63;
  const int row = row0 + (lane & 15), col = col0 + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);
  auto at = [&](int r) { return (r < border ? out + r * ld : out2 + (r - border) * ld) + col; };
  if (col < n) {
    if (row < m) *reinterpret_cast<u32x4*>(at(row)) = x;
    if (row + 16 < m) *reinterpret_cast<u32x4*>(at(row + 16)) = y;
  }
}

enum GemmKind : int { kPlain, kGated, kTwoParts, kWeights, kInt8 };

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

template <class T, int KIND>
struct Operand {
  typedef typename Frag<T>::V V;
  typedef f32x16 Sum;
  typedef typename std::conditional<KIND == kPlain, GemmArgs, GemmKindArgs>::type Args;
  static __device__ __forceinline__ Sum mfma(V a, V b, Sum c) { return Frag<T>::mfma(a, b, c); }
};
template <class T>
struct Operand<T, kInt8> {
  typedef i32x4 V;
  typedef i32x16 Sum;
  typedef GemmKindArgs Args;
  static __device__ __forceinline__ Sum mfma(V a, V b, Sum c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -kLog2e));
}

// Eight values through a gate's activation (the same branch for a whole launch).
__device__ __forceinline__ void gate8(float* z, int act) {
  if (act == kActSilu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] *= sigmoid(z[e]);
  } else if (act == kActSigmoid) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = sigmoid(z[e]);
  } else {
    activate8(z, act);
  }
}

// 8 neighbouring sums of both factors in place, with their biases (what pre receives); h: the output.
__device__ __forceinline__ void finish_gated8(int act, const float* bias, const float* bias2, float* gate, float* up, float* h) {
#pragma unroll
  for (int e = 0; e < 8; ++e) gate[e] += bias[e], up[e] += bias2[e], h[e] = gate[e];
  gate8(h, act);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] *= up[e];
}

// 8 neighbouring whole sums in units of both scales (one after the other: their product alone could leave fp32's
// range), with the bias, through the activation.
__device__ __forceinline__ void finish_int8(int act, float row, const float* col, const float* bias, float* z) {
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = fmaf(z[e] * col[e], row, bias[e]);
  activate8(z, act);
}

// 8 floats of LDS or memory, 16-byte aligned.
__device__ __forceinline__ void take8(const float* p, float* f) {
  const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = lo[e], f[4 + e] = hi[e];
}

// What a tile's epilogue takes of its rows and columns, in LDS: gated, both biases; int8, the columns' bias and
// scales, the rows' scales.  Loaded before the products, whose time hides it (block by block in the epilogue, each
// waited for, int8's 32768 x 4096, k = 1024 took 205 us instead of 177).
template <int KIND, int TM, int TN>
constexpr int gemm_vectors() { return KIND == kGated ? 2 * TN : KIND == kInt8 ? 2 * TN + TM : 4; }

// Workgroups of a product: tiles rounded up to a multiple of 8, times the parts of the reduction.
__host__ __device__ inline int gemm_grid(const GemmArgs& a, int tm, int tn) {
  return (((a.m + tm - 1) / tm) * ((a.n + tn - 1) / tn) + 7) / 8 * 8 * a.splits;
}

template <int WM, int WN, int BM, int BN, int RING>
constexpr int gemm_lds() { return RING * (WM * BM + WN * BN) * 32 * kDepth * 2; }

// Workgroup `id` of a product: WM x WN waves of BM x BN blocks of 32 x 32, RING stages in LDS (smem).
// (vectors: gemm_vectors floats of LDS of the gated and int8 kinds.)
template <class T, int WM, int WN, int BM, int BN, int RING, bool MS, bool NS, int KIND = kPlain>
__device__ __forceinline__ void gemm_tile(const typename Operand<T, KIND>::Args& a, int id, unsigned char* smem, float* vectors = nullptr) {
  static_assert((KIND != kGated || (BN % 2 == 0 && !MS && !NS)) && (KIND != kInt8 || (!MS && !NS)), "kinds' operands");
  constexpr int FN = KIND == kGated ? BN / 2 : BN;  // blocks of output columns of a wave
  constexpr int W = WM * WN, TM = WM * BM * 32, TN = WN * FN * 32, NROWS = WN * BN * 32;
  constexpr int MBYTES = TM * kDepth * 2, STAGE = (TM + NROWS) * kDepth * 2;
  constexpr int LM = MBYTES / 1024 / W, LN = (STAGE - MBYTES) / 1024 / W;  // 1 KiB loads a wave and stage
  static_assert(LM * 1024 * W == MBYTES && (LM + LN) * 1024 * W == STAGE, "whole loads");
  typedef Operand<T, KIND> Op;
  typedef typename Op::V V;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int l32 = lane & 31, g = lane >> 5;
  const int p16 = lane >> 4, s16 = lane & 15;

  // Tiles in an order that gives each XCD (consecutive workgroups go round the 8 of them)
  // neighbouring ones, in blocks of 4 tile rows, down the columns: the tiles under way
  // in an XCD share rows of both operands in its L2.
  constexpr int kRows = 4;
  const int tiles_n = (a.n + TN - 1) / TN, tiles_m = (a.m + TM - 1) / TM;
  const int tiles = tiles_n * tiles_m;
  const int per = (tiles + 7) / 8;
  const int split = id / (8 * per);
  const int tile = (id & 7) * per + (id - split * 8 * per) / 8;
  if (tile >= tiles) return;
  const int strip = tile / (kRows * tiles_n), in_strip = tile - strip * kRows * tiles_n;
  const int rows = min(kRows, tiles_m - strip * kRows);
  const int m0 = (strip * kRows + in_strip % rows) * TM, n0 = in_strip / rows * TN;

  // what the epilogue takes (a column, and a row, a thread): under way during the products, then to LDS
  static_assert(TN <= 64 * W && TM <= 64 * W, "a column and a row a thread");
  float of_col[2] = {0.f, 0.f}, of_row = 0.f;
  if constexpr (KIND == kGated || KIND == kInt8) {
    const int j = min(n0 + min(tid, TN - 1), a.n - 1);
    if (a.bias != nullptr) of_col[0] = (float)((const T*)a.bias)[j];
    if constexpr (KIND == kGated) {
      if (a.bias2 != nullptr) of_col[1] = (float)((const T*)a.bias2)[j];
    } else {
      of_col[1] = a.col_scale[j];
      of_row = a.row_scale[min(m0 + min(tid, TM - 1), a.m - 1)];
    }
  }

  float unit = 1.f;
  if constexpr (KIND == kTwoParts || KIND == kWeights)
    if (a.unit != nullptr) unit = *a.unit;

  const int part_stages = (a.k + kDepth - 1) / kDepth, stages = KIND == kTwoParts ? 2 * part_stages : part_stages;
  const int s_begin = (int)((int64_t)stages * split / a.splits);
  const int s_end = (int)((int64_t)stages * (split + 1) / a.splits);

  // This lane's place in each 1 KiB load: line and 16-byte piece of the tile.
  uint32_t vm[LM], vn[LN];
  int km[LM], kn[LN];  // reduction step of the load within a stage
  auto place = [&](int j, bool strided, int64_t ld, int first, int rows, uint32_t* voff, int* step) {
    const int line = (wave + W * j) * 8 + (lane >> 3);
    const int piece = (lane & 7) ^ piece_swizzle(line);
    if (strided) {
      const int col = line / kDepth * 64 + piece * 8;
      *step = line % kDepth;
      *voff = (uint32_t)(*step * ld * 2) + (uint32_t)(col * 2);
      if (first + col >= rows) *voff = kOutside;
    } else {
      *step = piece * 8;
      *voff = (uint32_t)(line * ld * 2) + (uint32_t)(piece * 16);
      if (first + line >= rows) *voff = kOutside;
    }
  };
#pragma unroll
  for (int j = 0; j < LM; ++j) place(j, MS, a.ldm, m0, a.m, &vm[j], &km[j]);
#pragma unroll
  for (int j = 0; j < LN; ++j) {
    if constexpr (KIND == kGated) {  // line 32 u + r: row r of wave column u / BN's block u % BN, of FN of N's, then of N2's
      const int line = (wave + W * j) * 8 + (lane >> 3), u = line >> 5;
      const int row = (u / BN * FN + u % BN % FN) * 32 + (line & 31);
      kn[j] = ((lane & 7) ^ piece_swizzle(line)) * 8;
      vn[j] = n0 + row < a.n ? (uint32_t)(row * a.ldn * 2) + (uint32_t)(kn[j] * 2) : kOutside;
    } else {
      place(j, NS, a.ldn, n0, a.n, &vn[j], &kn[j]);
    }
  }
  const unsigned char* mbase = (const unsigned char*)a.M + 2 * (MS ? (int64_t)m0 : m0 * a.ldm);
  const unsigned char* nbase = (const unsigned char*)a.N + 2 * (NS ? (int64_t)n0 : n0 * a.ldn);
  const int64_t mstep = 2 * (MS ? kDepth * a.ldm : (int64_t)kDepth), nstep = 2 * (NS ? kDepth * a.ldn : (int64_t)kDepth);
  const unsigned char* nbase2 = nullptr;  // gated: N2's tile, two parts: N of the second part
  if constexpr (KIND == kGated) {
    nbase2 = (const unsigned char*)a.N2 + 2 * n0 * a.ldn + s_begin * nstep;
  } else if constexpr (KIND == kTwoParts) {
    nbase2 = (const unsigned char*)a.N2 + 2 * (NS ? (int64_t)n0 : n0 * a.ldn);
  }
  const unsigned char* mbase2 = nullptr;  // two parts: M of the second part
  int first_stage = s_begin;              // of its part
  if constexpr (KIND == kTwoParts) {
    mbase2 = mbase + 2 * a.m_second;
    if (s_begin >= part_stages) mbase = mbase2, nbase = nbase2, first_stage -= part_stages;
  }
  mbase += first_stage * mstep;
  nbase += first_stage * nstep;
  const uint32_t lds0 = lds_address(smem);

  int load_s = s_begin, load_buf = 0;
  auto load_stage = [&]() {
    const uint32_t at = lds0 + (uint32_t)(load_buf * STAGE + wave * 1024);
    const int step = KIND == kTwoParts && load_s >= part_stages ? load_s - part_stages : load_s;
    const int left = a.k - step * kDepth;  // reduction steps from this stage on
#pragma unroll
    for (int j = 0; j < LM; ++j) load_lds(km[j] < left ? vm[j] : kOutside, mbase, at + j * (W * 1024));
#pragma unroll
    for (int j = 0; j < LN; ++j) {
      const unsigned char* base = nbase;
      if constexpr (KIND == kGated) base = (wave + W * j) / 4 % BN < FN ? nbase : nbase2;
      load_lds(kn[j] < left ? vn[j] : kOutside, base, at + MBYTES + j * (W * 1024));
    }
    mbase += mstep;
    nbase += nstep;
    ++load_s;
    if constexpr (KIND == kGated) nbase2 += nstep;
    if (KIND == kTwoParts && load_s == part_stages) mbase = mbase2, nbase = nbase2;
    load_buf = load_buf + 1 == RING ? 0 : load_buf + 1;
  };

  // Operand fragments of depth step ks (16 of the stage's 64), rows r0 .. r0 + 31 of the tile.
  auto frag = [&](const unsigned char* t, bool strided, int r0, int ks, bool reorder) -> V {
    if constexpr (KIND != kInt8) if (strided) {
      const int c = reorder ? ((s16 & 1) << 1) | ((s16 >> 1) & 1) : s16 & 3;
      const int col = r0 + 16 * (p16 & 1) + 4 * c;
      const int line = 16 * ks + 8 * (p16 >> 1) + (s16 >> 2);
      const unsigned char* panel = t + (col >> 6) * (kDepth * 128) + (col & 4) * 2;
      const int piece = (col & 63) >> 3;
      const s16x4 lo = read_tr(panel + line * 128 + ((piece ^ piece_swizzle(line)) << 4));
      const s16x4 hi = read_tr(panel + (line + 4) * 128 + ((piece ^ piece_swizzle(line + 4)) << 4));
      return join_tr<T>(lo, hi);
    }
    const int r = r0 + (reorder ? tile_row(l32) : l32);
    return *reinterpret_cast<const V*>(t + row_offset<kDepth>(r, 2 * ks + g));
  };

  typename Op::Sum acc[BM][BN];
#pragma unroll
  for (int i = 0; i < BM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  auto read = [&](int stage, int ks, V* fm, V* fn) {
    const unsigned char* tm = smem + stage * STAGE;
#pragma unroll
    for (int i = 0; i < BM; ++i) fm[i] = frag(tm, MS, (wm * BM + i) * 32, ks, false);
#pragma unroll
    for (int j = 0; j < BN; ++j) fn[j] = frag(tm + MBYTES, NS, (wn * BN + j) * 32, ks, true);
  };
  auto multiply = [&](const V* fm, const V* fn) {
#pragma unroll
    for (int i = 0; i < BM; ++i)
#pragma unroll
      for (int j = 0; j < BN; ++j) acc[i][j] = Op::mfma(fn[j], fm[i], acc[i][j]);
  };
  int buf = 0;
  if constexpr (W == 8) {
    // Two waves a SIMD, half a turn apart: while one reads the operands of two depth steps, the
    // other multiplies its own, and a barrier ends each such phase.  (Both at their own pace,
    // a barrier a stage: dW of 32768 x 2048, k = 2048 268 us instead of 248, dx of 32768 x 2048, k = 1024 123
    // instead of 118, 8192 x 8192, k = 2048 240 instead of 234; short reductions gain nothing,
    // 16384 x 2048, k = 768 52.5 instead of 54.)  The late waves are one phase behind; a stage's buffer is loaded
    // again from the phase on after the late waves' last read of it, and its loads have landed,
    // by each wave's own wait, before the barrier that the early waves' first read follows.
    static_assert(RING == 2, "two stages");
    const bool late = wave >= W / 2;
    auto phase_end = [&](bool landed) {
      keep_order();
      if (landed)
        wait_vmcnt_lgkm0<0>();
      else
        wait_vmcnt_lgkm0<63>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      keep_order();
    };
    if (s_begin < s_end) load_stage();
    if (s_begin + 1 < s_end) {
      load_stage();
      wait_vmcnt_lgkm0<LM + LN>();
    } else {
      wait_vmcnt_lgkm0<0>();
    }
    __builtin_amdgcn_s_barrier();
    if (late) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    for (int s = s_begin; s < s_end; ++s) {
      if (s > s_begin && load_s < s_end) load_stage();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        V fm[2][BM], fn[2][BN];
        read(buf, 2 * half, fm[0], fn[0]);
        read(buf, 2 * half + 1, fm[1], fn[1]);
        phase_end(half == 1 && late);
        multiply(fm[0], fn[0]);
        multiply(fm[1], fn[1]);
        phase_end(half == 1 && !late);
      }
      buf ^= 1;
    }
    if (!late) __builtin_amdgcn_s_barrier();
  } else {
#pragma unroll
    for (int s = 0; s < RING - 1; ++s)
      if (s_begin + s < s_end) load_stage();
    for (int s = s_begin; s < s_end; ++s) {
      // this stage's loads are in; those of the next RING - 2 may still be under way
      if (RING > 2 && s + 1 < s_end)
        wait_vmcnt_lgkm0<(RING - 2) * (LM + LN)>();
      else
        wait_vmcnt_lgkm0<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (load_s < s_end) load_stage();  // into the buffer that every wave has left
#pragma unroll
      for (int ks = 0; ks < kDepth / 16; ++ks) {
        V fm[BM], fn[BN];
        read(buf, ks, fm, fn);
        multiply(fm, fn);
      }
      buf = buf + 1 == RING ? 0 : buf + 1;
    }
  }

  if constexpr (KIND == kGated || KIND == kInt8) {
    if (a.splits == 1) {
      if (tid < TN) vectors[tid] = of_col[0], vectors[TN + tid] = of_col[1];
      if (KIND == kInt8 && tid < TM) vectors[2 * TN + tid] = of_row;
      __syncthreads();
    }
  }

  // Lane: a row of the output, two times 8 neighbouring columns of each block.
  if (KIND == kInt8 && a.splits == 1) {
    typename Frag<T>::V res[BM][FN][2];  // all of them under way together
    if (a.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < BM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            res[i][j][h] = *reinterpret_cast<const typename Frag<T>::V*>(
                (const T*)a.residual + (int64_t)min(m0 + (wm * BM + i) * 32 + l32, a.m - 1) * a.ld_res + min(n0 + (wn * FN + j) * 32 + 16 * h + 8 * g, a.n - 8));
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      float col[16], bias[16];
      const int at = (wn * FN + j) * 32 + 8 * g;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        take8(vectors + at + 16 * h, bias + 8 * h);
        take8(vectors + TN + at + 16 * h, col + 8 * h);
      }
#pragma unroll
      for (int i = 0; i < BM; ++i) {
        const float row = vectors[2 * TN + (wm * BM + i) * 32 + l32];
        float z[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = (float)acc[i][j][e];
        finish_int8(a.act, row, col, bias, z);
        finish_int8(a.act, row, col + 8, bias + 8, z + 8);
        if (a.residual != nullptr) {
#pragma unroll
          for (int e = 0; e < 16; ++e) z[e] += (float)res[i][j][e >> 3][e & 7];
        }
        store_block((T*)a.out, a.n, a.m, a.n, m0 + (wm * BM + i) * 32, n0 + (wn * FN + j) * 32, z, z + 8);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < BM; ++i) {
    const int row0 = m0 + (wm * BM + i) * 32, row = row0 + l32;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int col0 = n0 + (wn * FN + j) * 32, col = col0 + 8 * g;
      if (a.splits > 1) {
        constexpr int SUMS = KIND == kGated ? 2 : 1;
#pragma unroll
        for (int u = 0; u < SUMS; ++u) {
          float* p = a.partial + (((int64_t)split * a.m + row) * SUMS + u) * a.n + col;
          const auto& sum = acc[i][j + u * FN];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (row < a.m && col + 16 * h < a.n) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int e = 8 * h + 4 * q;
                if constexpr (KIND == kInt8)
                  *reinterpret_cast<i32x4*>(p + 16 * h + 4 * q) = i32x4{sum[e], sum[e + 1], sum[e + 2], sum[e + 3]};
                else
                  *reinterpret_cast<f32x4*>(p + 16 * h + 4 * q) = f32x4{sum[e], sum[e + 1], sum[e + 2], sum[e + 3]};
              }
            }
        }
      } else if constexpr (KIND == kGated) {
        float gate[16], up[16], h[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) gate[e] = acc[i][j][e], up[e] = acc[i][j + FN][e];
        float bias[16], bias2[16];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          take8(vectors + (wn * FN + j) * 32 + 8 * g + 16 * u, bias + 8 * u);
          take8(vectors + TN + (wn * FN + j) * 32 + 8 * g + 16 * u, bias2 + 8 * u);
        }
        finish_gated8(a.act, bias, bias2, gate, up, h);
        finish_gated8(a.act, bias + 8, bias2 + 8, gate + 8, up + 8, h + 8);
        if (a.pre != nullptr) {
          store_block((T*)a.pre, 2 * (int64_t)a.n, a.m, a.n, row0, col0, gate, gate + 8);
          store_block((T*)a.pre + a.n, 2 * (int64_t)a.n, a.m, a.n, row0, col0, up, up + 8);
        }
        store_block((T*)a.out, a.n, a.m, a.n, row0, col0, h, h + 8);
      } else if constexpr (KIND == kTwoParts || KIND == kWeights) {
        float z[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = acc[i][j][e] * unit;
        if constexpr (KIND == kWeights)
          store_block_of_two((T*)a.out, (T*)a.out2, a.m_first, a.n, a.m, a.n, row0, col0, z, z + 8);
        else
          store_block((T*)a.out, a.n, a.m, a.n, row0, col0, z, z + 8);
      } else {
        float z[16], pre[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = (float)acc[i][j][e];
        // rows and columns past the edge: those of the last ones again, not stored
        const int r = min(row, a.m - 1);
        finish8<T>(a, r, min(col, a.n - 8), z, pre);
        finish8<T>(a, r, min(col + 16, a.n - 8), z + 8, pre + 8);
        if (a.pre != nullptr) store_block((T*)a.pre, a.n, a.m, a.n, row0, col0, pre, pre + 8);
        store_block((T*)a.out, a.n, a.m, a.n, row0, col0, z, z + 8);
      }
    }
  }
}

}  // namespace

}  // namespace cvs
