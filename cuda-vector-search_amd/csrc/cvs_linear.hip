// Matrix product with bias, activation and residual in its epilogue, and the
// products of its backward pass, for 16-bit operands with fp32 sums.
//
//   out[i, j] = act(sum_r M(i, r) N(j, r) + bias[j]) + residual[i, j]
//
// Either operand may be stored with its reduction contiguous ([rows, k]) or strided
// ([k, rows]): y = x W^T reads x and W so, dx = dz W takes W strided, dW = dz^T x
// both.  Stages of 64 reduction steps come into LDS as lines of 128 bytes, straight
// from memory (buffer loads into LDS; a lane past the operand's edge gets an
// offset past the buffer's end, which reads as zero); strided operands are turned
// on the way out of LDS by transposing reads.
#include <algorithm>

#include "cvs_encoder.h"
#include "cvs_mfma.h"

namespace cvs {

namespace {

constexpr int kDepth = 64;                    // reduction steps of a stage
constexpr int64_t kLaunchThreads = (int64_t)1 << 32;
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

// Stores a 32 x 32 block of which lane l holds, of row l % 32, columns 8 g .. and 16 + 8 g ..
// (g = l / 32): 16 lanes exchange their pieces with the next 16 so that four lanes write
// 64 contiguous bytes of a row.
template <class T>
__device__ __forceinline__ void store_block(T* out, int64_t ld, int m, int n, int row0, int col0, const float* z0, const float* z1) {
  typename Frag<T>::V v0, v1;
#pragma unroll
  for (int e = 0; e < 8; ++e) v0[e] = (T)z0[e], v1[e] = (T)z1[e];
  u32x4 x = __builtin_bit_cast(u32x4, v0), y = __builtin_bit_cast(u32x4, v1);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const auto s = __builtin_amdgcn_permlane16_swap(x[r], y[r], false, false);
    x[r] = s[0], y[r] = s[1];
  }
  const int lane = threadIdx.x & 63;
  const int row = row0 + (lane & 15), col = col0 + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);
  if (col < n) {
    T* to = out + (int64_t)row * ld + col;
    if (row < m) *reinterpret_cast<u32x4*>(to) = x;
    if (row + 16 < m) *reinterpret_cast<u32x4*>(to + 16 * ld) = y;
  }
}

// Workgroups of a product: tiles rounded up to a multiple of 8, times the parts of the reduction.
__host__ __device__ inline int gemm_grid(const GemmArgs& a, int tm, int tn) {
  return (((a.m + tm - 1) / tm) * ((a.n + tn - 1) / tn) + 7) / 8 * 8 * a.splits;
}

template <int WM, int WN, int BM, int BN, int RING>
constexpr int gemm_lds() { return RING * (WM * BM + WN * BN) * 32 * kDepth * 2; }

// Workgroup `id` of a product: WM x WN waves of BM x BN blocks of 32 x 32, RING stages in LDS (smem).
template <class T, int WM, int WN, int BM, int BN, int RING, bool MS, bool NS>
__device__ __forceinline__ void gemm_tile(const GemmArgs& a, int id, unsigned char* smem) {
  constexpr int W = WM * WN, TM = WM * BM * 32, TN = WN * BN * 32;
  constexpr int MBYTES = TM * kDepth * 2, STAGE = (TM + TN) * kDepth * 2;
  constexpr int LM = MBYTES / 1024 / W, LN = (STAGE - MBYTES) / 1024 / W;  // 1 KiB loads a wave and stage
  static_assert(LM * 1024 * W == MBYTES && (LM + LN) * 1024 * W == STAGE, "whole loads");
  typedef typename Frag<T>::V V;

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

  const int stages = (a.k + kDepth - 1) / kDepth;
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
  for (int j = 0; j < LN; ++j) place(j, NS, a.ldn, n0, a.n, &vn[j], &kn[j]);
  const unsigned char* mbase = (const unsigned char*)a.M + 2 * (MS ? (int64_t)m0 : m0 * a.ldm);
  const unsigned char* nbase = (const unsigned char*)a.N + 2 * (NS ? (int64_t)n0 : n0 * a.ldn);
  const int64_t mstep = 2 * (MS ? kDepth * a.ldm : (int64_t)kDepth), nstep = 2 * (NS ? kDepth * a.ldn : (int64_t)kDepth);
  mbase += s_begin * mstep;
  nbase += s_begin * nstep;
  const uint32_t lds0 = lds_address(smem);

  int load_s = s_begin, load_buf = 0;
  auto load_stage = [&]() {
    const uint32_t at = lds0 + (uint32_t)(load_buf * STAGE + wave * 1024);
    const int left = a.k - load_s * kDepth;  // reduction steps from this stage on
#pragma unroll
    for (int j = 0; j < LM; ++j) load_lds(km[j] < left ? vm[j] : kOutside, mbase, at + j * (W * 1024));
#pragma unroll
    for (int j = 0; j < LN; ++j) load_lds(kn[j] < left ? vn[j] : kOutside, nbase, at + MBYTES + j * (W * 1024));
    mbase += mstep;
    nbase += nstep;
    ++load_s;
    load_buf = load_buf + 1 == RING ? 0 : load_buf + 1;
  };

  // Operand fragments of depth step ks (16 of the stage's 64), rows r0 .. r0 + 31 of the tile.
  auto frag = [&](const unsigned char* t, bool strided, int r0, int ks, bool reorder) -> V {
    if (strided) {
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

  f32x16 acc[BM][BN];
#pragma unroll
  for (int i = 0; i < BM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

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
      for (int j = 0; j < BN; ++j) acc[i][j] = Frag<T>::mfma(fn[j], fm[i], acc[i][j]);
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

  // Lane: a row of the output, two times 8 neighbouring columns of each block.
#pragma unroll
  for (int i = 0; i < BM; ++i) {
    const int row0 = m0 + (wm * BM + i) * 32, row = row0 + l32;
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      const int col0 = n0 + (wn * BN + j) * 32, col = col0 + 8 * g;
      if (a.splits > 1) {
        float* p = a.partial + ((int64_t)split * a.m + row) * a.n + col;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (row < a.m && col + 16 * h < a.n) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int e = 8 * h + 4 * q;
              *reinterpret_cast<f32x4*>(p + 16 * h + 4 * q) =
                  f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
            }
          }
      } else {
        float z[16], pre[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = acc[i][j][e];
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

template <class T, int WM, int WN, int BM, int BN, int RING, bool MS, bool NS>
__global__ __launch_bounds__(64 * WM * WN, (WM * BM + WN * BN) * RING <= 16 ? 2 : 1) void gemm_kernel(GemmArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[gemm_lds<WM, WN, BM, BN, RING>()];
  gemm_tile<T, WM, WN, BM, BN, RING, MS, NS>(a, blockIdx.x, smem);
}

// Two products that share an operand, dx (first) and dW, in one launch: neither fills the GPU
// where the rows are few.
template <class T, int WM, int WN, int BM, int BN, int RING>
__global__ __launch_bounds__(64 * WM * WN, (WM * BM + WN * BN) * RING <= 16 ? 2 : 1) void gemm_pair_kernel(GemmArgs a, GemmArgs b) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[gemm_lds<WM, WN, BM, BN, RING>()];
  const int first = gemm_grid(a, WM * BM * 32, WN * BN * 32);
  if ((int)blockIdx.x < first)
    gemm_tile<T, WM, WN, BM, BN, RING, false, true>(a, blockIdx.x, smem);
  else
    gemm_tile<T, WM, WN, BM, BN, RING, true, true>(b, blockIdx.x - first, smem);
}

// Adds the parts of a split reduction, in order, and finishes: 8 columns a thread.
template <class T>
__global__ __launch_bounds__(kBlock) void gemm_join_kernel(GemmArgs a) {
  const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int pieces = a.n / 8;
  const int64_t i = at / pieces;
  if (i >= a.m) return;
  const int j = (int)(at - i * pieces) * 8;
  const int64_t plane = (int64_t)a.m * a.n;
  const float* p = a.partial + i * a.n + j;
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = 0.f;
  for (int s = 0; s < a.splits; ++s, p += plane) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] += lo[e], z[4 + e] += hi[e];
  }
  float pre[8];
  finish8<T>(a, (int)i, j, z, pre);
  if (a.pre != nullptr) store8((T*)a.pre + i * a.n + j, pre);
  store8((T*)a.out + i * a.n + j, z);
}

template <class T>
hipError_t launch_join(const GemmArgs& a, hipStream_t s) {
  const int64_t threads = (int64_t)a.m * (a.n / 8);
  hipLaunchKernelGGL((gemm_join_kernel<T>), dim3((unsigned)((threads + kBlock - 1) / kBlock)), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

template <class T, int WM, int WN, int BM, int BN, int RING>
hipError_t launch_tiles(const GemmArgs& a, hipStream_t s) {
  const dim3 grid(gemm_grid(a, WM * BM * 32, WN * BN * 32)), block(64 * WM * WN);
  if (a.m_strided && a.n_strided)
    hipLaunchKernelGGL((gemm_kernel<T, WM, WN, BM, BN, RING, true, true>), grid, block, 0, s, a);
  else if (a.n_strided)
    hipLaunchKernelGGL((gemm_kernel<T, WM, WN, BM, BN, RING, false, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((gemm_kernel<T, WM, WN, BM, BN, RING, false, false>), grid, block, 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess && a.splits > 1 ? launch_join<T>(a, s) : e;
}

template <class T, int WM, int WN, int BM, int BN, int RING>
hipError_t launch_pair(const GemmArgs& a, const GemmArgs& b, hipStream_t s) {
  constexpr int TM = WM * BM * 32, TN = WN * BN * 32;
  hipLaunchKernelGGL((gemm_pair_kernel<T, WM, WN, BM, BN, RING>), dim3(gemm_grid(a, TM, TN) + gemm_grid(b, TM, TN)),
                     dim3(64 * WM * WN), 0, s, a, b);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.splits > 1) e = launch_join<T>(a, s);
  if (e == hipSuccess && b.splits > 1) e = launch_join<T>(b, s);
  return e;
}

template <class T>
hipError_t launch_typed(const GemmArgs& a, const GemmPlan& p, hipStream_t s) {
  if (p.tile == 256) return p.tile_n == 256 ? launch_tiles<T, 4, 2, 2, 4, 2>(a, s) : launch_tiles<T, 4, 2, 2, 3, 2>(a, s);
  if (p.tile == 128) return launch_tiles<T, 2, 2, 2, 2, 2>(a, s);
  return launch_tiles<T, 2, 2, 1, 1, 3>(a, s);
}

template <class T>
hipError_t launch_typed_pair(const GemmArgs& a, const GemmArgs& b, const GemmPlan& p, hipStream_t s) {
  if (p.tile == 128) return launch_pair<T, 2, 2, 2, 2, 2>(a, b, s);
  return launch_pair<T, 2, 2, 1, 1, 3>(a, b, s);
}

// Pieces of 8 columns of a workgroup of act_grad_kernel: few for few rows, which one part then
// has, so that it writes dbias itself.
__host__ __device__ inline int act_grad_width(int64_t m, int n) { return m <= 256 ? 16 : min(n / 8, kBlock); }

// dz = dy act'(pre) and its column sums, bound by memory.  A workgroup has up to 256
// pieces of 8 columns (blockIdx.x) and as many of its part's rows at a time as its threads
// cover; it adds its row lanes' sums in LDS and writes one partial row.
template <class T>
__global__ __launch_bounds__(kBlock) void act_grad_kernel(ActGradArgs a) {
  __shared__ float red[kBlock * 8];
  const int width = act_grad_width(a.m, a.n);
  const int pieces = min(a.n / 8 - (int)blockIdx.x * width, width), lanes = kBlock / pieces;
  const int p = threadIdx.x % pieces, rl = threadIdx.x / pieces;
  const int c = (blockIdx.x * width + p) * 8;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  const int64_t r0 = a.m * blockIdx.y / gridDim.y, r1 = a.m * (blockIdx.y + 1) / gridDim.y;
  if (rl < lanes) {
    const bool act = a.act != kActNone;
    constexpr int U = 4;  // rows under way
    for (int64_t r = r0 + rl; r < r1; r += U * lanes) {
      typename Frag<T>::V g[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = min(r + u * lanes, r1 - 1);
        g[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.dy + row * a.dy_stride + c);
        if (act) z[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.pre + row * a.n + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = r + u * lanes;
        if (row < r1) {
          float gf[8], zf[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) gf[e] = (float)g[u][e];
          if (act) {
#pragma unroll
            for (int e = 0; e < 8; ++e) zf[e] = (float)z[u][e];
            times_slope8(gf, zf, a.act);
            store8((T*)a.dz + row * a.n + c, gf);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += gf[e];
        }
      }
    }
  }
  if (a.dbias == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = sum[e];
  __syncthreads();
  const int64_t col0 = (int64_t)blockIdx.x * width * 8;
  for (int t = threadIdx.x; t < pieces * 8; t += kBlock) {
    float s = 0.f;
    for (int l = 0; l < lanes; ++l) s += red[l * pieces * 8 + t];
    if (gridDim.y == 1)
      ((T*)a.dbias)[col0 + t] = (T)s;
    else
      a.partial[(int64_t)blockIdx.y * a.n + col0 + t] = s;
  }
}

}  // namespace

// Tiles of 256 x 256 and 256 x 192 (8 waves, one workgroup a CU), 128 x 128 and 64 x 64 (4 waves,
// two and three workgroups a CU), and parts of the reduction where the tiles leave CUs idle: the
// choice of least estimated time.  A CU runs its workgroups in rounds; every XCD has an eighth of
// the tiles, rounded up, and all their parts (33 tiles in 7 parts are 35 workgroups on 32 CUs, two
// rounds: 100 us where 128 x 128 takes 60).  A stage of a round costs what was
// measured on long reductions (8192 x 8192, k = 2048: 1080, 850 and 480 TFLOP/s, that is 1.8 to
// 2.0, 1.2 and 0.9 us with 1, 2 and 3 workgroups; 256 x 192 has 1.7), a round 3 us more to fill
// and finish, and a split 3 us and its sums' way to memory and back.  At 16384 x 2048, k = 768
// that gives 256 x 256 (calls of the product alone, back to back: 54 us, with 128 x 128 58), at
// 16384 x 768, k = 2048 256 x 192 (its 256 tiles 48 us, 192 of 256 x 256 52), at 10007 x 768, k = 2048
// 128 x 128 (35, 256 x 256 47), at 2048 x 768, k = 16384 128 x 128 in 5 parts (61 with the join,
// 256 x 192 in parts 65).
//
// A launch has fewer than 2^32 threads: choices of more are passed over, and where that leaves none
// (splits 0), there is no plan.
GemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, int cus) {
  static constexpr struct { int m, n, wgs, threads; double stage; } kTiles[] = {
      {256, 256, 1, 512, 1.8}, {256, 192, 1, 512, 1.7}, {128, 128, 2, 256, 1.2}, {64, 64, 3, 256, 0.9}};
  const int64_t stages = (k + kDepth - 1) / kDepth;
  GemmPlan best = {};
  double least = 1e30;
  for (const auto& t : kTiles) {
    const int64_t tiles = ((m + t.m - 1) / t.m) * ((n + t.n - 1) / t.n);
    for (int64_t splits = 1; splits <= 16 && (splits == 1 || splits * 8 <= stages); ++splits) {
      const int64_t wgs = (tiles + 7) / 8 * 8 * splits, full = wgs / (t.wgs * (int64_t)cus);
      if (wgs * t.threads >= kLaunchThreads || (splits > 1 && m * (n / 8) + kBlock > kLaunchThreads)) break;
      // a last round of few workgroups has more of a CU for each, but not below a stage's latency
      const int64_t rest = (wgs - full * t.wgs * cus + cus - 1) / cus;
      const double per = full * t.stage + (rest > 0 ? std::max(rest * t.stage / t.wgs, 0.5) : 0.0);
      double us = (stages + splits - 1) / splits * per + 3.0 * (full + (rest > 0));
      if (splits > 1) us += 3.0 + 2.0 * splits * m * n * 4 / 4e6;
      if (us < least) {
        least = us;
        best.tile = t.m, best.tile_n = t.n, best.splits = (int)splits;
        best.ws_bytes = splits > 1 ? splits * m * n * 4 : 0;
      }
    }
  }
  return best;
}

hipError_t launch_gemm(const GemmArgs& a, const GemmPlan& p, hipStream_t s) {
  return a.type == kF16 ? launch_typed<_Float16>(a, p, s) : launch_typed<__bf16>(a, p, s);
}

hipError_t launch_gemm_pair(const GemmArgs& a, const GemmPlan& pa, const GemmArgs& b, const GemmPlan& pb, hipStream_t s) {
  const int64_t both = (int64_t)gemm_grid(a, pa.tile, pa.tile_n) + gemm_grid(b, pb.tile, pb.tile_n);
  if (pa.tile == pb.tile && pa.tile < 256 && both * 256 < kLaunchThreads)
    return a.type == kF16 ? launch_typed_pair<_Float16>(a, b, pa, s) : launch_typed_pair<__bf16>(a, b, pa, s);
  const hipError_t e = launch_gemm(a, pa, s);
  return e == hipSuccess ? launch_gemm(b, pb, s) : e;
}

int act_grad_parts(int64_t m, int64_t n, int cus) {
  const int64_t width = act_grad_width(m, (int)n);
  if (m <= 256) return 1;
  const int64_t blocks = (n / 8 + width - 1) / width, lanes = kBlock / width;
  return (int)std::max<int64_t>(1, std::min<int64_t>((m + lanes - 1) / lanes, 3 * cus / blocks));
}

hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t s) {
  const int width = act_grad_width(a.m, a.n);
  const dim3 grid((a.n / 8 + width - 1) / width, a.parts), block(kBlock);
  if (a.type == kF16)
    hipLaunchKernelGGL(act_grad_kernel<_Float16>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(act_grad_kernel<__bf16>, grid, block, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.dbias != nullptr && a.parts > 1)
    e = launch_column_sums(a.partial, a.parts, a.n, a.n, 0, a.type, a.dbias, nullptr, s);
  return e;
}

}  // namespace cvs
